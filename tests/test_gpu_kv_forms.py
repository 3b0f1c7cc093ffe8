"""Forms of the key/value cache's kernels that a call takes by its sizes alone: wide reads, blocks
written from registers and read twice, batches of single tokens beside a chunk; what lies
beside a call's arrays; calls on two streams at once."""
import numpy as np
import pytest
import torch

from kernels_amd import kq
from tests import _kv
from tests import test_gpu_kv as kv

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dim,heads,page,block", [(96, 2, 16, 16), (192, 1, 32, 16), (256, 2, 64, 64), (64, 1, 64, 64), (96, 1, 256, 256)])
@pytest.mark.parametrize("kind,dtype", [("i8", "f16"), ("e4m3", "bf16")])
def test_write_and_read(gpu, dim, heads, page, block, kind, dtype):
    kv.test_write_and_read(gpu, dim, heads, page, block, kind, dtype)


@pytest.mark.parametrize("out", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("dim,kind,heads,page,block", [(64, "e4m3", 1, 16, 16), (96, "i8", 2, 32, 32), (96, "e4m3", 3, 16, 16), (128, "i8", 2, 64, 64),
                                                       (128, "e4m3", 1, 16, 16), (192, "i8", 2, 16, 16), (192, "e4m3", 1, 128, 32), (256, "i8", 1, 64, 16), (256, "e4m3", 2, 16, 16)])
def test_wide_reads(gpu, dim, kind, heads, page, block, out):
    """Beyond 16384 workgroups of 16 tokens a wave, where heads of 64 are read by 64. Ragged lengths, whole sequences and parts of them, rows at negative
    positions, nothing at all."""
    rng = np.random.default_rng(dim)
    seqs = [(int(n), int(m)) for n, m in zip(rng.integers(0, 90, 520), rng.integers(0, 100, 520))]
    seqs[3], seqs[100], seqs[519] = (700, 700), (699, 530), (641, 641)
    b = kv.Batch(gpu, seqs, page, rng, pad=2)
    assert ((b.max_q - 1) // 16 + 2) * ((2 * heads + 3) // 4) * len(seqs) > 16384
    read_check(gpu, rng, b, dim, kind, heads, page, block, out)


def read_check(gpu, rng, b, dim, kind, heads, page, block, out):
    oracle = _kv.Cache(b.n_pages, heads, dim, page, block, kind)
    oracle.fill(rng)
    cache = kv.upload(oracle, gpu)
    got = {w: torch.full((b.rows, heads, dim), 7.0, dtype=kv.DTYPES[out], device=gpu) for w in "kv"}
    kq.kv_read(cache, b.c, got["k"], got["v"])
    torch.cuda.synchronize()
    top = torch.finfo(kv.DTYPES[out]).max
    for w in "kv":
        have = got[w].cpu()
        assert (have[b.starts[-1]:] == 7.0).all(), "rows behind the last sequence"
        for i, (n, m) in enumerate(b.seqs):
            rows = have[b.starts[i]:b.starts[i + 1]]
            want = torch.from_numpy(oracle.read(w, b.table[i], n, m)).clamp(-top, top).float().to(kv.DTYPES[out])
            there = torch.arange(m) >= m - n
            assert torch.equal(rows[there], want[there]) and (rows[~there] == 7.0).all(), (w, i)


@pytest.mark.parametrize("dim,kind,heads,page,block,out", [(64, "i8", 2, 16, 16, "f32"), (96, "i8", 2, 32, 32, "bf16"), (96, "e4m3", 1, 16, 16, "f16"),
                                                           (128, "e4m3", 2, 16, 16, "bf16"), (128, "i8", 1, 64, 64, "f16"), (192, "i8", 1, 16, 16, "bf16")])
def test_wider_reads(gpu, dim, kind, heads, page, block, out):
    """Beyond 65536 workgroups of 16 tokens, where heads of 96 and 128 and fp32 values of 64 are read by 64 too."""
    rng = np.random.default_rng(dim)
    seqs = [(int(n), int(m)) for n, m in zip(rng.integers(0, 70, 520), rng.integers(0, 80, 520))]
    seqs[7], seqs[200], seqs[519] = (2200, 2200), (2111, 700), (70, 70)
    b = kv.Batch(gpu, seqs, page, rng, pad=2)
    assert ((b.max_q - 1) // 16 + 2) * ((2 * heads + 3) // 4) * len(seqs) > 65536
    read_check(gpu, rng, b, dim, kind, heads, page, block, out)


class Guarded:
    """Tensors inside larger ones whose other bytes are to stay."""

    def __init__(self, gpu):
        self.gpu, self.all = gpu, []

    def tensor(self, dtype, shape, pad=4096):
        n = int(np.prod(shape)) * torch.empty((), dtype=dtype).element_size()
        whole = torch.full((n + 2 * pad,), 0xA5, dtype=torch.uint8, device=self.gpu)
        self.all.append((whole, pad, n))
        return whole[pad:pad + n].view(dtype).view(shape)

    def stayed(self):
        return all((w[:p] == 0xA5).all() and (w[p + n:] == 0xA5).all() for w, p, n in self.all)


@pytest.mark.parametrize("kind,max_q,heads,group", [("i8", 3, 2, 2), ("e4m3", 40, 1, 4), ("i8", 40, 2, 1)])
def test_arrays_that_lie_beside_others(gpu, kind, max_q, heads, group):
    """Lengths and rows beyond the host's bounds: cache, pages that no table names, rows and workspace's surroundings stay."""
    ints = dict(dtype=torch.int32, device=gpu)
    named = [1, 2, 4, 5, 7, 8, 10, 11]
    pages = torch.tensor(named, **ints).view(2, 4)
    other = [i for i in range(13) if i not in named]
    n = 2 * max_q
    for lens, starts in (([2**31 - 1, -5], [0, max_q, n]), ([60, 64], [-4, 2**31 - 1, n - 1]), ([64, 64], [n - 1, 2, 0]),
                         ([1000, 64], [0, 2**31 - 1, -2**31]), ([-2**31, 2**31 - 1], [-2**31, 0, 2**31 - 1])):
        g = Guarded(gpu)
        code = g.tensor(torch.int8, (13, heads, 16, 64)), g.tensor(torch.int8, (13, heads, 1, 64, 16))
        exps = [g.tensor(torch.uint8, (13, heads, 1)) for _ in "kv"]
        for t in (*code, *exps):
            t.fill_(90)
        cache = kq.KVCache(*(t.view(kv.CODE[kind]) for t in code), *exps)
        b = kq.KVBatch(pages, torch.tensor(lens, **ints), 64, q_start=torch.tensor(starts, **ints), max_q=max_q)
        q_heads = heads * group
        x = torch.randn((n, q_heads + 2 * heads, 64), device=gpu).half()
        out, lse = g.tensor(torch.float16, (n, q_heads, 64)), g.tensor(torch.float32, (n, q_heads))
        back = [g.tensor(torch.float32, (n, heads, 64)) for _ in "kv"]
        size = kq.kv_attn_workspace_size(cache, b, q_heads)
        ws = g.tensor(torch.uint8, (size,))
        print(f"{kind} {max_q} rows {lens} {starts}", flush=True)
        kq.kv_write(cache, b, x[:, q_heads:q_heads + heads], x[:, q_heads + heads:])
        kq.kv_attn(cache, b, x[:, :q_heads], out, ws, size, lse=lse)
        kq.kv_read(cache, b, *back)
        torch.cuda.synchronize()
        assert g.stayed()
        assert all((t[other] == 90).all() for t in (*code, *exps)), "pages of no table"


def mixed(gpu, rng, decode, chunk, heads, group, dim, window=0):
    """A step of single tokens beside one chunk: in one call, and in two: the tokens', the chunk's."""
    seqs = [(n, 1) for n in decode] + [chunk]
    b = kv.Batch(gpu, seqs, 16, rng, pad=1)
    oracle = _kv.Cache(b.n_pages, heads, dim)
    oracle.fill(rng)
    cache = kv.upload(oracle, gpu)
    q, q64 = kv.to(rng.normal(0, 1, (b.rows, heads * group, dim)), "f16", gpu)
    n = len(decode)
    starts, c = b.c.q_start, b.c
    parts = [kq.KVBatch(c.pages[:n], c.kv_len[:n], max(decode), q_start=starts[:n + 1], max_q=1),
             kq.KVBatch(c.pages[n:], c.kv_len[n:], chunk[0], q_start=starts[n:], max_q=chunk[1])]
    for batches in ([c], parts):
        out, lse = torch.full_like(q, 7.0), torch.full(q.shape[:2], 7.0, device=gpu)
        size = max(kq.kv_attn_workspace_size(cache, x, heads * group) for x in batches)
        ws = torch.empty(size, dtype=torch.uint8, device=gpu)
        for x in batches:
            kq.kv_attn(cache, x, q, out, ws, size, lse=lse, window=window)
        torch.cuda.synchronize()
        for i, (length, m) in enumerate(seqs):
            rows = slice(b.starts[i], b.starts[i + 1])
            want = _kv.attend(oracle, b.table[i], length, q64[rows], dim**-0.5, True, window)
            tol, tol_lse = _kv.attend_tolerance(*want, dim, *kv.EPS["f16"])
            assert (np.abs(out[rows].double().cpu().numpy() - want[0]) <= tol).all(), i
            assert (np.abs(lse[rows].double().cpu().numpy() - want[1]) <= tol_lse).all(), i
        assert (out[b.starts[-1]:] == 7.0).all() and (lse[b.starts[-1]:] == 7.0).all()


@pytest.mark.parametrize("decode,chunk,heads,group,dim,window", [
    ([700, 3, 64, 2000, 129], (300, 90), 2, 4, 64, 0), ([1500], (70, 70), 1, 8, 128, 0), ([40] * 70 + [2600], (200, 33), 1, 3, 64, 100)])
def test_single_tokens_beside_a_chunk(gpu, decode, chunk, heads, group, dim, window):
    mixed(gpu, np.random.default_rng(dim + len(decode)), decode, chunk, heads, group, dim, window)


def test_two_streams_at_once(gpu):
    """Two caches' calls on two streams, each with its own workspace, equal those made one after the other."""
    rng = np.random.default_rng(11)
    work = []
    for seqs, heads, group in (([(5000, 1), (300, 1)], 2, 4), ([(900, 80), (70, 70)], 1, 2)):
        b = kv.Batch(gpu, seqs, 16, rng)
        oracle = _kv.Cache(b.n_pages, heads, 64)
        oracle.fill(rng)
        cache = kv.upload(oracle, gpu)
        x = torch.randn((b.rows, heads * (group + 2), 64), device=gpu).half()
        size = kq.kv_attn_workspace_size(cache, b.c, heads * group)
        work.append((b, cache, x, heads, group, size, torch.empty(size, dtype=torch.uint8, device=gpu), torch.cuda.Stream()))
    got = []
    for at_once in (False, True):
        outs = []
        torch.cuda.synchronize()
        for _ in range(6):
            for b, cache, x, heads, group, size, ws, side in work:
                s = side if at_once else torch.cuda.current_stream()
                with torch.cuda.stream(s):
                    out = torch.zeros((b.rows, heads * group, 64), dtype=torch.float16, device=gpu)
                    kq.kv_write(cache, b.c, x[:, heads * group:-heads], x[:, -heads:])
                    kq.kv_attn(cache, b.c, x[:, :heads * group], out, ws, size)
                outs.append(out)
        torch.cuda.synchronize()
        got.append(outs)
    assert all(torch.equal(a, c) for a, c in zip(*got))
    assert all(torch.equal(a, c) for a, c in zip(got[0], got[0][2:]))


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0])
@pytest.mark.parametrize("dim,kind,dtype", [(64, "i8", "f16"), (128, "e4m3", "bf16"), (192, "i8", "bf16")])
def test_scales_of_many_rows(gpu, dim, kind, dtype, scale):
    kv.attn_case(gpu, [(100, 70), (65, 3), (0, 5), (300, 90)], 2, 2, dim, kind, dtype, scale=scale, sinks=scale < 0)


def test_query_range_of_many_rows(gpu):
    """Queries from the smallest to the largest of bf16, and rows of zeros, in the kernel for many rows."""
    def tiny(b, q_heads):
        return np.random.default_rng(1).normal(0, 1, (b.rows, q_heads, 64)) * 1e-36

    def huge(b, q_heads):
        x = np.random.default_rng(1).normal(0, 1, (b.rows, q_heads, 64)) * 1e36
        x[::5] = 0.0
        return x
    kv.attn_case(gpu, [(100, 40), (65, 33)], 2, 2, 64, dtype="bf16", scale=1e35, q=tiny)
    kv.attn_case(gpu, [(100, 40), (65, 33)], 2, 2, 64, "e4m3", dtype="bf16", scale=1e-37, q=huge)


@pytest.mark.parametrize("seqs,heads,group,dim", [([(70, 1), (0, 1), (33, 3)], 2, 4, 64), ([(1500, 1), (100, 1)], 1, 2, 96), ([(2600, 1)] + [(30, 1)] * 200, 1, 2, 64),
                                                  ([(64, 64), (90, 40)], 1, 3, 128), ([(2000, 70), (5, 5)], 1, 2, 256)])
def test_layouts_of_queries_and_outputs(gpu, seqs, heads, group, dim):
    """Heads of rows, rows with others' values between them, one row of queries for all: the same bits as rows of heads, and
    nothing beside them written."""
    rng = np.random.default_rng(dim)
    b = kv.Batch(gpu, seqs, 16, rng, pad=2)
    oracle = _kv.Cache(b.n_pages, heads, dim)
    oracle.fill(rng)
    cache = kv.upload(oracle, gpu)
    n, q_heads = b.rows, heads * group
    size = kq.kv_attn_workspace_size(cache, b.c, q_heads)
    ws = torch.empty(size, dtype=torch.uint8, device=gpu)

    def attend(q, out):
        kq.kv_attn(cache, b.c, q, out, ws, size)
        torch.cuda.synchronize()
        return out
    q = torch.randn((n, q_heads, dim), device=gpu).half()
    want = attend(q, torch.full_like(q, 7.0))
    by_head = torch.full((q_heads, n, dim), 7.0, dtype=torch.float16, device=gpu)
    assert torch.equal(attend(q.transpose(0, 1).contiguous().transpose(0, 1), by_head.transpose(0, 1)), want)
    wide = torch.full((n, 2 * q_heads + 1, dim + 8), 7.0, dtype=torch.float16, device=gpu)
    assert torch.equal(attend(q, wide[:, 1:2 * q_heads:2, :dim]), want)
    assert (wide[:, ::2] == 7.0).all() and (wide[:, :, dim:] == 7.0).all()
    one = q[:1].expand(n, q_heads, dim)
    assert torch.equal(attend(one, torch.full_like(q, 7.0)), attend(one.contiguous(), torch.full_like(q, 7.0)))
