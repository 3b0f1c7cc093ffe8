"""The 8-bit key/value cache and its attention on the GPU through the C ABI,
against the 64-bit oracle (tests/_kv.py): codes, exponents and values that were
read back exactly, attention within what the arithmetic allows."""
import numpy as np
import pytest
import torch

from kernels_amd import gen, kq
from tests import _kv
from tests._util import ATOL, RTOL, dev
from tests.test_gpu_graphs import replay_check

pytestmark = pytest.mark.gpu

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
CODE = {"i8": torch.int8, "e4m3": torch.float8_e4m3fn}
EPS = {"f16": (2.0**-10, 2.0**-25), "bf16": (2.0**-7, 2.0**-134)}  # eps, half the smallest step


def upload(cache, gpu):
    """The oracle's cache as the device holds it."""
    n, h, page, dim = cache.codes["v"].shape
    v = cache.codes["v"].reshape(n, h, page // 16, 16, dim).swapaxes(3, 4)
    k, v = (torch.from_numpy(np.ascontiguousarray(a).view(np.int8)).to(gpu).view(CODE[cache.kind]) for a in (cache.codes["k"], v))
    return kq.KVCache(k, v, *(torch.from_numpy(cache.exps[w].copy()).to(gpu) for w in "kv"))


def codes_of(c):
    """{k, v: uint8 codes in rows}, {k, v: exponents} of the device's cache."""
    k = c.k.view(torch.int8).cpu().numpy().view(np.uint8)
    v = c.v.view(torch.int8).cpu().numpy().view(np.uint8).swapaxes(3, 4)
    return {"k": k, "v": v.reshape(k.shape)}, {"k": c.k_exp.cpu().numpy(), "v": c.v_exp.cpu().numpy()}


def same_cache(device, oracle, what=""):
    codes, exps = codes_of(device)
    for w in "kv":
        assert np.array_equal(exps[w], oracle.exps[w]), f"{what}: {w} exponents"
        got, want = _kv.decode(codes[w], oracle.kind), _kv.decode(oracle.codes[w], oracle.kind)
        bad = np.argwhere((got != want) & ~(np.isnan(got) & np.isnan(want)))
        assert not len(bad), f"{what}: {w} code at {bad[0]}: {got[tuple(bad[0])]}, not {want[tuple(bad[0])]}; {len(bad)} in all"


class Batch:
    """Sequences (length, newest) on pages of their own, in any order; the table's other entries are no pages."""

    def __init__(self, gpu, seqs, page, rng, spare=2, q_start=True, pad=0, max_len=None, wide=0):
        self.seqs = seqs
        need = [-(-n // page) for n, _ in seqs]
        self.n_pages, wide = sum(need) + spare, max(max(need), 1) + wide
        order = rng.permutation(self.n_pages)
        self.table = np.full((len(seqs), wide), 2**30, np.int32)
        at = 0
        for i, k in enumerate(need):
            self.table[i, :k] = order[at:at + k]
            at += k
        self.max_q = max(max(m for _, m in seqs), 1)
        self.starts = np.concatenate([[0], np.cumsum([m for _, m in seqs])]).astype(np.int32)
        if not q_start:
            assert all(m == self.max_q for _, m in seqs)
        self.rows = int(self.starts[-1]) + pad
        self.max_len = max_len or max(max(n for n, _ in seqs), 1)
        self.c = kq.KVBatch(dev(self.table, gpu), torch.tensor([n for n, _ in seqs], dtype=torch.int32, device=gpu), self.max_len,
                            q_start=dev(self.starts, gpu) if q_start else None, max_q=self.max_q)


def to(x, dtype, gpu):
    """float64 -> tensor of the type on the GPU, and its values in 64 bits."""
    t = torch.from_numpy(x).to(DTYPES[dtype])
    return t.to(gpu), t.double().numpy()


def wild(rng, shape, dtype):
    """Values of many sizes, with zeros, infinities and NaN among them."""
    x = rng.normal(0, 1, shape) * np.exp(rng.normal(0, 1.5, shape[:-1] + (1,)))
    x[rng.random(shape) < 0.01] = 0.0
    flat = x.reshape(-1)
    n = len(flat)
    for v in (np.inf, -np.inf, np.nan, 6.0e4, -6.0e4, 127.0, 448.0, 2.0**-24, -0.0):
        flat[rng.integers(0, n, 2)] = v
    if dtype == "bf16":
        for v in (3.3e38, -3.3e38, 1e-38, 1e30, 1e-30):
            flat[rng.integers(0, n, 1)] = v
    return x


# lengths and newest tokens: nothing new, nothing at all, more rows than tokens,
# one token into each place of a block, tokens over several blocks and pages
SEQS = [(17, 1), (0, 0), (16, 1), (1, 1), (40, 0), (33, 2), (300, 1), (64, 64), (130, 77), (15, 15), (3, 5), (47, 16), (0, 2),
        (100, 100), (49, 18)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("dim,heads,page,block", [(64, 3, 16, 16), (128, 2, 64, 16), (96, 1, 32, 32), (192, 2, 64, 64),
                                                  (256, 1, 16, 16), (128, 1, 256, 128)])
def test_write_and_read(gpu, dim, heads, page, block, kind, dtype):
    rng = np.random.default_rng(dim + heads + page + block)
    b = Batch(gpu, SEQS, page, rng, pad=3)
    oracle = _kv.Cache(b.n_pages, heads, dim, page, block, kind)
    oracle.fill(rng)
    cache = upload(oracle, gpu)
    x = {w: to(wild(rng, (b.rows, heads, dim), dtype), dtype, gpu) for w in "kv"}
    kq.kv_write(cache, b.c, x["k"][0], x["v"][0])
    torch.cuda.synchronize()
    for w in "kv":
        for i, (n, m) in enumerate(SEQS):
            oracle.write(w, x[w][1][b.starts[i]:b.starts[i + 1]], b.table[i], n, m)
    same_cache(cache, oracle, "write")
    for out in ("f16", "bf16", "f32"):
        got = {w: torch.full((b.rows, heads, dim), 7.0, dtype=DTYPES[out], device=gpu) for w in "kv"}
        kq.kv_read(cache, b.c, got["k"], got["v"])
        torch.cuda.synchronize()
        top = torch.finfo(DTYPES[out]).max
        for w in "kv":
            for i, (n, m) in enumerate(SEQS):
                want = oracle.read(w, b.table[i], n, m)
                want = torch.from_numpy(want).clamp(-top, top).float().to(DTYPES[out])
                have = got[w][b.starts[i]:b.starts[i + 1]].cpu()
                there = torch.arange(m) >= m - n
                assert torch.equal(have[there], want[there]), (out, w, i)
                assert (have[~there] == 7.0).all(), (out, w, i)
            assert (got[w][b.starts[-1]:] == 7.0).all(), "rows behind the last sequence"


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
def test_appending_one_by_one(gpu, kind):
    """40 steps of single tokens whose sizes grow and fall: older codes are rounded anew where a
    block's exponent grows, and nothing else changes. Without q_start."""
    rng = np.random.default_rng(5)
    heads, dim, page, block, steps = 2, 64, 32, 32, 40
    start = [0, 13, 31]
    table = rng.permutation(12).reshape(3, 4).astype(np.int32)
    oracle = _kv.Cache(12, heads, dim, page, block, kind)
    oracle.fill(rng)
    cache = upload(oracle, gpu)
    pages, n = dev(table, gpu), torch.tensor(start, dtype=torch.int32, device=gpu)
    b = kq.KVBatch(pages, n, 100)
    for step in range(steps):
        n += 1
        k, v = (to(rng.normal(0, 1, (3, heads, dim)) * 2.0 ** rng.integers(-6, 7), "f16", gpu) for _ in "kv")
        kq.kv_write(cache, b, k[0], v[0])
        torch.cuda.synchronize()
        for i in range(3):
            for w, x in (("k", k), ("v", v)):
                oracle.write(w, x[1][i:i + 1], table[i], start[i] + step + 1, 1)
        same_cache(cache, oracle, f"step {step}")


def test_write_strides(gpu):
    """Slices of a fused projection's rows, other orders of heads and rows, and one row for all."""
    rng = np.random.default_rng(6)
    heads, dim, seqs = 2, 128, [(50, 20), (9, 9)]
    b = Batch(gpu, seqs, 16, rng)
    fused, v64 = to(rng.normal(0, 1, (b.rows, 7, dim)), "f16", gpu)
    by_head, h64 = to(rng.normal(0, 1, (heads, b.rows, dim)), "f16", gpu)
    one, o64 = to(rng.normal(0, 1, (1, 1, dim)), "f16", gpu)
    for k, k64 in ((fused[:, 3:5], v64[:, 3:5]), (by_head.transpose(0, 1), h64.swapaxes(0, 1)),
                   (one.expand(b.rows, heads, dim), np.broadcast_to(o64, (b.rows, heads, dim)))):
        oracle = _kv.Cache(b.n_pages, heads, dim)
        cache = upload(oracle, gpu)
        kq.kv_write(cache, b.c, k, fused[:, 5:7])
        torch.cuda.synchronize()
        for i, (n, m) in enumerate(seqs):
            rows = slice(b.starts[i], b.starts[i + 1])
            oracle.write("k", k64[rows], b.table[i], n, m)
            oracle.write("v", v64[rows, 5:7], b.table[i], n, m)
        same_cache(cache, oracle)
    # reading into slices leaves the rest as it was
    out = torch.full((b.rows, 5, dim), 7.0, device=gpu)
    kq.kv_read(cache, b.c, out[:, :2], out[:, 3:])
    torch.cuda.synchronize()
    want = torch.from_numpy(np.concatenate([oracle.read("v", b.table[i], n, m) for i, (n, m) in enumerate(seqs)]))
    assert torch.equal(out[:, 3:].cpu().double(), want) and (out[:, 2] == 7.0).all()


def attn_case(gpu, seqs, heads, group, dim, kind="i8", dtype="f16", page=16, block=16, causal=True, window=0, sinks=False,
              lse=True, q_start=True, pad=0, seed=0, nan=False, scale=None, max_len=None, spoil=None, q=None):
    """One call against the oracle. nan: e4m3 NaN codes wherever no sequence has a token."""
    rng = np.random.default_rng(seed + dim + group)
    b = Batch(gpu, seqs, page, rng, q_start=q_start, pad=pad, max_len=max_len)
    oracle = _kv.Cache(b.n_pages, heads, dim, page, block, kind)
    oracle.fill(rng)
    if nan:
        used = np.zeros((b.n_pages, page), bool)
        for i, (n, _) in enumerate(seqs):
            for t in range(n):
                used[b.table[i, t // page], t % page] = True
        for w in "kv":
            oracle.codes[w] = np.where(used[:, None, :, None], oracle.codes[w], 0x7F if kind == "e4m3" else 0x80).astype(np.uint8)
            blocks = used.reshape(b.n_pages, page // block, block).any(2)
            oracle.exps[w] = np.where(blocks[:, None], oracle.exps[w], 255).astype(np.uint8)
    if spoil is not None:
        spoil(b, gpu)
    cache = upload(oracle, gpu)
    q_heads = heads * group
    qt, q64 = to(rng.normal(0, 1, (b.rows, q_heads, dim)) * np.exp(rng.normal(0, 0.7, (b.rows, q_heads, 1))) if q is None else q(b, q_heads), dtype, gpu)
    s = rng.normal(0, 3, q_heads).astype(np.float32) if sinks is True else np.float32(sinks) if sinks else None
    out = torch.full((b.rows, q_heads, dim), 7.0, dtype=DTYPES[dtype], device=gpu)
    ls = torch.full((b.rows, q_heads), 7.0, device=gpu) if lse else None
    n = kq.kv_attn_workspace_size(cache, b.c, q_heads)
    ws = torch.full((n + 4096,), 0xA5, dtype=torch.uint8, device=gpu)
    args = dict(scale=scale, causal=causal, window=window, sinks=None if s is None else torch.from_numpy(s).to(gpu), lse=ls)
    print(f"attn {seqs} heads {heads} x {group} dim {dim} {kind} {dtype} page {page}/{block} window {window}", flush=True)
    kq.kv_attn(cache, b.c, qt, out, ws, n, **args)
    torch.cuda.synchronize()
    assert (ws[n:] == 0xA5).all(), "behind the workspace"
    first, first_lse = out.clone(), None if ls is None else ls.clone()
    eps, tiny = EPS[dtype]
    for i, (length, m) in enumerate(seqs):
        if not m:
            continue
        rows = slice(b.starts[i], b.starts[i + 1])
        want = _kv.attend(oracle, b.table[i], length, q64[rows], dim**-0.5 if scale is None else scale, causal, window, s)
        tol, tol_lse = _kv.attend_tolerance(*want, dim, eps, tiny)
        got = out[rows].double().cpu().numpy()
        off = np.abs(got - want[0])
        assert np.isfinite(got).all() and (off <= tol).all(), (i, float(np.nanmax(off / tol)), np.argwhere(~(off <= tol))[:3].tolist())
        if lse:
            have = ls[rows].double().cpu().numpy()
            none = np.isinf(want[1])
            assert np.array_equal(np.isinf(have), none) and np.array_equal(have[none], want[1][none])
            off = np.abs(have[~none] - want[1][~none])
            assert (off <= tol_lse[~none]).all(), (i, np.nanmax(off / tol_lse[~none]))
    assert (out[b.starts[-1]:] == 7.0).all() and (ls is None or (ls[b.starts[-1]:] == 7.0).all()), "rows behind the last sequence"
    kq.kv_attn(cache, b.c, qt, out, ws, n, **args)
    torch.cuda.synchronize()
    assert torch.equal(out, first) and (ls is None or torch.equal(ls, first_lse)), "a second run differs"


DECODE = [(1, 1), (0, 1), (15, 1), (16, 1), (17, 1), (63, 1), (64, 1), (65, 1), (255, 1), (256, 1), (257, 1), (700, 1)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 96, 128, 192, 256])
def test_decode(gpu, dim, kind, dtype):
    attn_case(gpu, DECODE, 2, 4, dim, kind, dtype, nan=True, pad=2)


@pytest.mark.parametrize("heads,group", [(1, 1), (3, 1), (8, 2), (1, 7), (2, 16), (1, 17), (1, 64), (5, 5)])
def test_decode_groups(gpu, heads, group):
    attn_case(gpu, [(90, 1), (33, 1), (0, 1)], heads, group, 64, q_start=False)


@pytest.mark.parametrize("page,block", [(16, 16), (32, 16), (64, 64), (128, 32), (256, 256), (1024, 16)])
@pytest.mark.parametrize("kind", ["i8", "e4m3"])
def test_decode_pages(gpu, page, block, kind):
    attn_case(gpu, [(1500, 1), (100, 1), (1, 1)], 2, 4, 128, kind, "bf16", page, block, sinks=True, nan=True)


@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 128, 600, 5000])
def test_window(gpu, window):
    attn_case(gpu, [(n, 1) for n in (1, 64, 127, 128, 129, 1000, 0)] + [(300, 9), (5, 9)], 2, 3, 64, window=window, sinks=window % 2 == 0, nan=True)


MANY = [(70, 70), (1, 1), (200, 33), (64, 64), (5, 9), (0, 3), (129, 2), (40, 0), (17, 16), (300, 111)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("dim,group", [(64, 8), (96, 3), (128, 4), (192, 1), (256, 2)])
def test_many_rows(gpu, dim, group, kind, dtype):
    attn_case(gpu, MANY, 2, group, dim, kind, dtype, pad=5, nan=kind == "i8", sinks=group == 8)


@pytest.mark.parametrize("few", [2, 3, 4, 5, 8])
@pytest.mark.parametrize("group", [1, 4, 8])
def test_few_rows(gpu, few, group):
    attn_case(gpu, [(100, few), (400, few), (few - 1, few)], 2, group, 128, "e4m3", q_start=False)


def test_not_causal(gpu):
    attn_case(gpu, MANY, 2, 4, 64, causal=False, sinks=True)
    attn_case(gpu, [(500, 1), (30, 4)], 2, 4, 128, "e4m3", "bf16", causal=False, lse=False)


def test_long_and_bounds_above(gpu):
    """A long sequence among short ones, and host bounds that are larger than any length."""
    attn_case(gpu, [(9001, 1), (30, 1)], 1, 8, 64, max_len=20000)
    attn_case(gpu, [(5000, 2), (3, 1)], 1, 2, 128, "e4m3", "bf16", max_len=100000, page=64, block=32)
    attn_case(gpu, [(4000, 70), (3, 1)], 1, 2, 64, max_len=50000, page=64, block=32)


def ragged(n, longest, seed, new=1):
    """n short sequences, empty ones among them, with a few long ones in between."""
    rng = np.random.default_rng(seed)
    lens = rng.integers(0, 40, n)
    lens[rng.integers(0, n, 4)] = rng.integers(longest // 2, longest, 4)
    lens[n // 3] = longest
    return [(int(x), int(m)) for x, m in zip(lens, rng.integers(0 if new > 1 else 1, new + 1, n))]


# the ways to share out few rows: parts of a row (up to 64 sequences, and more), equal shares (with fewer and more rows
# of work than workgroups; rows of several tiles; windows), a workgroup a row
@pytest.mark.parametrize("n,heads,group,longest,new,kw", [
    (40, 2, 4, 2700, 1, {}), (100, 1, 2, 2700, 1, {}), (70, 1, 16, 2500, 3, dict(kind="e4m3")),
    (300, 1, 2, 2700, 1, {}), (140, 4, 1, 2400, 1, dict(kind="e4m3", dtype="bf16")), (300, 1, 5, 2300, 5, {}),
    (150, 2, 9, 2300, 4, dict(dim=128)), (280, 1, 3, 2600, 2, dict(window=2200, sinks=True)), (1100, 1, 2, 2500, 1, {}),
    (30, 16, 1, 1500, 1, dict(dim=256)), (20, 8, 8, 2100, 8, dict(dim=192))])
def test_shares(gpu, n, heads, group, longest, new, kw):
    attn_case(gpu, ragged(n, longest, n), heads, group, **{"dim": 64, "nan": True, "pad": 1, **kw})


def test_more_page_ids_than_are_held(gpu):
    """Sequences longer than the page ids that a workgroup keeps at a time: few rows (a row each, for there are over 1024
    sequences) and many."""
    attn_case(gpu, [(1, 1)] * 600 + [(66100, 1)] + [(3, 1)] * 500, 1, 2, 64, max_len=70000)
    attn_case(gpu, [(17000, 70), (5, 5)], 1, 1, 64, "e4m3", "bf16")


@pytest.mark.parametrize("scale", [0.0, -0.3, 1.0])
def test_scales(gpu, scale):
    attn_case(gpu, [(100, 1), (65, 3)], 2, 2, 64, scale=scale)


@pytest.mark.parametrize("seqs,window", [([(0, 1), (1, 1), (70, 1), (2, 3)], 0), ([(1, 1), (5000, 1), (0, 1)], 0), ([(300, 1), (90, 40), (0, 20)], 7)])
def test_sinks_without_bounds(gpu, seqs, window):
    """A sink of -inf is none, also for a row that sees nothing; one of inf leaves nothing of the values."""
    attn_case(gpu, seqs, 2, 4, 128, window=window, sinks=[-np.inf, np.inf, 0.5, -np.inf, np.inf, -3e38, -np.inf, 3e38])


def test_query_range(gpu):
    """Queries from the smallest to the largest of bf16 (with a scale that keeps the scores moderate), and rows of zeros."""
    def tiny(b, q_heads):
        return np.random.default_rng(1).normal(0, 1, (b.rows, q_heads, 64)) * 1e-36

    def huge(b, q_heads):
        x = np.random.default_rng(1).normal(0, 1, (b.rows, q_heads, 64)) * 1e36
        x[0] = 0.0
        return x
    attn_case(gpu, [(100, 1), (65, 3)], 2, 2, 64, dtype="bf16", scale=1e35, q=tiny)
    attn_case(gpu, [(100, 1), (65, 3)], 2, 2, 64, dtype="bf16", scale=1e-37, q=huge)


def test_tiny_queries_on_huge_keys(gpu):
    """Queries of about 2^-110 and keys of about 2^110: their products are moderate, though neither factor nor the
    exponents' product is within float32's reach alone."""
    rng = np.random.default_rng(12)
    for n, m in ((70, 1), (200, 90)):
        b = Batch(gpu, [(n, m)], 16, rng)
        oracle = _kv.Cache(b.n_pages, 1, 64)
        oracle.fill(rng)
        oracle.exps["k"] = (oracle.exps["k"].astype(int) + 110).astype(np.uint8)
        q, q64 = to(rng.normal(0, 1, (m, 2, 64)) * 2.0**-110, "bf16", gpu)
        cache, out = upload(oracle, gpu), torch.zeros((m, 2, 64), dtype=torch.bfloat16, device=gpu)
        ws = torch.empty(kq.kv_attn_workspace_size(cache, b.c, 2), dtype=torch.uint8, device=gpu)
        kq.kv_attn(cache, b.c, q, out, ws, ws.numel())
        torch.cuda.synchronize()
        want = _kv.attend(oracle, b.table[0], n, q64, 64**-0.5)
        tol, _ = _kv.attend_tolerance(*want, 64, *EPS["bf16"])
        assert (np.abs(out.double().cpu().numpy() - want[0]) <= tol).all()


def test_single_row_of_any_stride(gpu):
    """One row and one head whose strides are no multiple of 8."""
    cache = kq.kv_cache(2, 1, 64, device=gpu)
    b = kq.KVBatch(torch.tensor([[1]], dtype=torch.int32, device=gpu), torch.tensor([1], dtype=torch.int32, device=gpu), 16)
    x = torch.randn(64, device=gpu).half()
    row = x.as_strided((1, 1, 64), (3, 5, 1))
    out = torch.zeros_like(x)
    kq.kv_write(cache, b, row, row)
    ws = torch.empty(kq.kv_attn_workspace_size(cache, b, 1), dtype=torch.uint8, device=gpu)
    kq.kv_attn(cache, b, row, out.as_strided((1, 1, 64), (1, 1, 1)), ws, ws.numel())
    back = torch.zeros((1, 1, 64), device=gpu)
    kq.kv_read(cache, b, back, torch.zeros_like(back))
    torch.cuda.synchronize()
    assert torch.equal(out.float(), back.view(-1).half().float())  # one token: its value


def test_scales_of_blocks_far_apart(gpu):
    """Values whose blocks differ by 2^60 in scale: the large ones have little probability."""
    rng = np.random.default_rng(3)
    b = Batch(gpu, [(64, 1)], 16, rng)
    oracle = _kv.Cache(b.n_pages, 1, 64)
    oracle.fill(rng)
    for j, e in enumerate((-30, 30, -10, 0)):
        oracle.exps["v"][b.table[0, j]] = 127 + e
    q, q64 = to(rng.normal(0, 1, (1, 2, 64)), "bf16", gpu)
    for t in range(16):  # the second block's keys point away from q
        oracle.codes["k"][b.table[0, 1], 0, t] = _kv.encode(-np.sign(q64[0, 0]) * 100.0, "i8")
    oracle.exps["k"][b.table[0, 1]] = 127 - 5
    cache, out = upload(oracle, gpu), torch.zeros((1, 2, 64), dtype=torch.bfloat16, device=gpu)
    ws = torch.empty(kq.kv_attn_workspace_size(cache, b.c, 2), dtype=torch.uint8, device=gpu)
    kq.kv_attn(cache, b.c, q, out, ws, ws.numel())
    torch.cuda.synchronize()
    want = _kv.attend(oracle, b.table[0], 64, q64, 64**-0.5)
    tol, _ = _kv.attend_tolerance(*want, 64, *EPS["bf16"])
    assert (np.abs(out.double().cpu().numpy() - want[0]) <= tol).all()


def test_nan_and_infinite_queries_stay_in_their_row(gpu):
    rng = np.random.default_rng(4)
    for kind, dtype in (("i8", "f16"), ("e4m3", "bf16")):
        b = Batch(gpu, [(100, 3), (80, 1)], 16, rng)
        oracle = _kv.Cache(b.n_pages, 1, 64, kind=kind)
        oracle.fill(rng)
        cache = upload(oracle, gpu)
        q = torch.randn((4, 4, 64), device=gpu).to(DTYPES[dtype])
        ws = torch.empty(kq.kv_attn_workspace_size(cache, b.c, 4), dtype=torch.uint8, device=gpu)
        clean, out = torch.zeros_like(q), torch.zeros_like(q)
        lse = torch.zeros((4, 4), device=gpu)
        kq.kv_attn(cache, b.c, q, clean, ws, ws.numel())
        q[1, 2, 5], q[3, 0, 0] = float("nan"), float("inf")
        kq.kv_attn(cache, b.c, q, out, ws, ws.numel(), lse=lse)
        torch.cuda.synchronize()
        bad = torch.zeros((4, 4), dtype=torch.bool, device=gpu)
        bad[1, 2] = bad[3, 0] = True
        assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], clean[~bad])
        assert torch.isnan(lse[bad]).all() and torch.isfinite(lse[~bad]).all()
        for sink in (-float("inf"), float("inf")):  # none; or one that takes all
            kq.kv_attn(cache, b.c, q, out, ws, ws.numel(), sinks=torch.full((4,), sink, device=gpu), lse=lse)
            torch.cuda.synchronize()
            assert torch.isnan(out[bad]).all() and torch.equal(out[~bad], clean[~bad] if sink < 0 else torch.zeros_like(clean[~bad]))
            assert torch.isnan(lse[bad]).all()


def test_pages_that_are_none(gpu):
    """Ids outside the pool: their tokens are neither attended to, nor read, nor written."""
    rng = np.random.default_rng(7)
    seqs = [(100, 30), (200, 1), (50, 50)]

    def spoil(b, gpu):
        b.table[0, 5], b.table[1, 0], b.table[1, 12], b.table[2, :] = -1, b.n_pages, 2**31 - 1, -7
        b.c.pages.copy_(dev(b.table, gpu))
    attn_case(gpu, seqs, 2, 4, 128, spoil=spoil)
    b = Batch(gpu, seqs, 16, rng)
    spoil(b, gpu)
    oracle = _kv.Cache(b.n_pages, 2, 64)
    oracle.fill(rng)
    cache = upload(oracle, gpu)
    x = {w: to(rng.normal(0, 1, (b.rows, 2, 64)), "f16", gpu) for w in "kv"}
    kq.kv_write(cache, b.c, x["k"][0], x["v"][0])
    out = {w: torch.full((b.rows, 2, 64), 7.0, device=gpu) for w in "kv"}
    kq.kv_read(cache, b.c, out["k"], out["v"])
    torch.cuda.synchronize()
    for w in "kv":
        for i, (n, m) in enumerate(seqs):
            rows = slice(b.starts[i], b.starts[i + 1])
            oracle.write(w, x[w][1][rows], b.table[i], n, m)
            assert np.array_equal(out[w][rows].double().cpu().numpy(), oracle.read(w, b.table[i], n, m))
    same_cache(cache, oracle)


def test_arrays_that_lie(gpu):
    """Lengths and rows beyond the host's bounds are cut to them: nothing outside the arrays is touched."""
    gpu_int = dict(dtype=torch.int32, device=gpu)
    pages = torch.arange(8, **gpu_int).view(2, 4)
    for lens, starts in (([2**31 - 1, -5], [0, 3, 6]), ([60, 64], [-4, 2**31 - 1, 5]), ([64, 64], [5, 2, 0]), ([1000, 64], [0, 2**31 - 1, -2**31])):
        b = kq.KVBatch(pages, torch.tensor(lens, **gpu_int), 64, q_start=torch.tensor(starts, **gpu_int), max_q=3)
        cache = kq.kv_cache(8, 2, 64, device=gpu)
        guard = torch.full((12, 4, 64), 7.0, dtype=torch.float16, device=gpu)
        x = torch.randn((6, 4, 64), device=gpu).half()
        ws = torch.empty(kq.kv_attn_workspace_size(cache, b, 4), dtype=torch.uint8, device=gpu)
        kq.kv_write(cache, b, x[:, :2], x[:, 2:])
        kq.kv_attn(cache, b, x, guard[3:9], ws, ws.numel())
        kq.kv_read(cache, b, guard[3:9, :2], guard[3:9, 2:])
        torch.cuda.synchronize()
        assert (guard[:3] == 7.0).all() and (guard[9:] == 7.0).all()


def test_other_stream_and_graph(gpu):
    """A step -- write, attend, read -- captured and replayed, eager work between the replays; two graphs on one workspace."""
    rng = np.random.default_rng(8)
    seqs = [(300, 2), (1000, 1), (17, 3), (40, 1)]
    b = Batch(gpu, seqs, 16, rng)
    oracle = _kv.Cache(b.n_pages, 2, 128)
    oracle.fill(rng)
    cache = upload(oracle, gpu)
    x = torch.randn((b.rows, 12, 128), device=gpu).half()
    out, lse = torch.zeros((b.rows, 8, 128), dtype=torch.float16, device=gpu), torch.zeros((b.rows, 8), device=gpu)
    back = [torch.zeros((b.rows, 2, 128), device=gpu) for _ in "kv"]
    ws = torch.empty(kq.kv_attn_workspace_size(cache, b.c, 8), dtype=torch.uint8, device=gpu)

    def step():
        kq.kv_write(cache, b.c, x[:, 8:10], x[:, 10:])
        kq.kv_attn(cache, b.c, x[:, :8], out, ws, ws.numel(), lse=lse)
        kq.kv_read(cache, b.c, *back)
    replay_check(step, [out, lse] + back)
    want = out.clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    out.fill_(0)
    side.wait_stream(torch.cuda.current_stream())
    kq.kv_attn(cache, b.c, x[:, :8], out, ws, ws.numel(), lse=lse, stream=side)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(out, want)
    # two graphs that share the workspace, with lengths that change between replays
    graphs, outs = [], []
    for w in (0, 32):
        o = torch.zeros_like(out)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            kq.kv_attn(cache, b.c, x[:, :8], o, ws, ws.numel(), window=w)
        graphs.append(g)
        outs.append(o)
    for take in (0, 1, 5):
        b.c.kv_len.sub_(take).clamp_(min=0)
        for g in graphs:
            g.replay()
        for o, w in zip(outs, (0, 32)):
            kq.kv_attn(cache, b.c, x[:, :8], out, ws, ws.numel(), window=w)
            torch.cuda.synchronize()
            assert torch.equal(o, out)


def test_python_checks(gpu):
    cache = kq.kv_cache(8, 2, 64, device=gpu)
    b = kq.KVBatch(torch.zeros((1, 4), dtype=torch.int32, device=gpu), torch.ones(1, dtype=torch.int32, device=gpu), 64)
    x = torch.zeros((1, 2, 64), dtype=torch.float16, device=gpu)
    q = torch.zeros((1, 4, 64), dtype=torch.float16, device=gpu)
    ws = torch.empty(kq.kv_attn_workspace_size(cache, b, 4), dtype=torch.uint8, device=gpu)
    for bad in ((x.cpu(), x), (x, x.float()), (x, x[:, :1]), (x[:, :, :32], x)):
        with pytest.raises(ValueError):
            kq.kv_write(cache, b, *bad)
    for kw in (dict(sinks=torch.zeros(4)), dict(sinks=torch.zeros(3, device=gpu)), dict(lse=torch.zeros((1, 3), device=gpu)), dict(window=-1)):
        with pytest.raises(ValueError):
            kq.kv_attn(cache, b, q, q.clone(), ws, ws.numel(), **kw)
    for f in (lambda: kq.kv_attn(cache, b, q, q.clone(), ws, 16), lambda: kq.kv_attn(cache, b, q.float(), q.float(), ws, ws.numel()),
              lambda: kq.kv_attn(cache, b, q, q.clone(), ws, ws.numel(), causal=False, window=4)):
        with pytest.raises(kq.KQError):
            f()


def test_most_sequences(gpu):
    """65535 sequences, of a token each: written, read back and attended to, which gives the value back."""
    n = 65535
    cache = kq.kv_cache(n, 1, 64, device=gpu)
    pages = torch.randperm(n, device=gpu).to(torch.int32).view(n, 1)
    b = kq.KVBatch(pages, torch.ones(n, dtype=torch.int32, device=gpu), 16)
    x = torch.randn((n, 3, 64), device=gpu).half()
    kq.kv_write(cache, b, x[:, 1:2], x[:, 2:])
    back = torch.zeros((n, 2, 64), device=gpu)
    kq.kv_read(cache, b, back[:, :1], back[:, 1:])
    ws = torch.empty(kq.kv_attn_workspace_size(cache, b, 1), dtype=torch.uint8, device=gpu)
    out = torch.zeros((n, 1, 64), dtype=torch.float16, device=gpu)
    kq.kv_attn(cache, b, x[:, :1], out, ws, ws.numel())
    torch.cuda.synchronize()
    assert torch.equal(out.float(), back[:, 1:])  # int8 times a power of two is fp16
    assert (back - x[:, 1:].float()).abs().max() <= 0.5 * 2.0**-4  # |x| < 8: steps of 2^-4 at most


@pytest.mark.parametrize("max_q", [1, 1 << 20, 100 << 20])
def test_longest_sequence(gpu, max_q):
    """The newest tokens of a sequence of nearly 2^31, all of whose pages are the same one: written and read back, whatever
    the bound on their number, with which blocks behind it would be counted past 2^31."""
    page, longest, new = 4096, 0x7FFEFFFF, 40
    cache = kq.kv_cache(3, 1, 64, page=page, block=16, device=gpu)
    table = torch.ones((1, -(-longest // page)), dtype=torch.int32, device=gpu)
    length, new = torch.tensor([longest], dtype=torch.int32, device=gpu), min(new, max_q)
    start = torch.tensor([0, new], dtype=torch.int32, device=gpu)
    b = kq.KVBatch(table, length, longest, q_start=start, max_q=max_q)
    x = torch.randn((new, 2, 64), device=gpu).half()
    before = [t.view(torch.int8).clone() for t in (cache.k, cache.v, cache.k_exp, cache.v_exp)]
    print(f"max_q {max_q}", flush=True)
    kq.kv_write(cache, b, x[:, :1], x[:, 1:])
    back = torch.zeros((new + 1, 2, 64), device=gpu)
    kq.kv_read(cache, b, back[:, :1], back[:, 1:])
    torch.cuda.synchronize()
    assert (back[:new] - x.float()).abs().max() <= 0.5 * 2.0**-4 and (back[new] == 0).all()  # |x| < 8
    last = (longest - 1) % page
    for t, old in zip((cache.k, cache.v, cache.k_exp, cache.v_exp), before):
        t = t.view(torch.int8)
        assert torch.equal(t[0], old[0]) and torch.equal(t[2], old[2])
    same = cache.k.view(torch.int8)[1, 0] == before[0][1, 0]
    assert same[:last - new + 1].all() and same[last + 1:].all()


def test_offsets_beyond_32_bits(gpu):
    """A cache of over 4 GiB of keys: the last pages' tokens."""
    heads, dim, page = 8, 128, 256
    n_pages = 2**32 // (heads * dim * page) + 8
    cache = kq.kv_cache(n_pages, heads, dim, page=page, block=64, device=gpu)
    ids = torch.tensor([[n_pages - 1, 3, n_pages - 5]], dtype=torch.int32, device=gpu)
    small = kq.kv_cache(3, heads, dim, page=page, block=64, device=gpu)
    n = 2 * page + 100
    length, start = torch.tensor([n], dtype=torch.int32, device=gpu), torch.tensor([0, n], dtype=torch.int32, device=gpu)
    x = torch.randn((n, 2 * heads, dim), device=gpu).half()
    q = torch.randn((1, 2 * heads, dim), device=gpu).half()
    got = []
    for c, pages in ((cache, ids), (small, torch.arange(3, dtype=torch.int32, device=gpu).view(1, 3))):
        kq.kv_write(c, kq.KVBatch(pages, length, n, q_start=start, max_q=n), x[:, :heads], x[:, heads:])
        b = kq.KVBatch(pages, length, n)
        ws = torch.empty(kq.kv_attn_workspace_size(c, b, 2 * heads), dtype=torch.uint8, device=gpu)
        out, back = torch.zeros_like(q), torch.zeros((n, 2 * heads, dim), device=gpu)
        kq.kv_attn(c, b, q, out, ws, ws.numel())
        kq.kv_read(c, kq.KVBatch(pages, length, n, q_start=start, max_q=n), back[:, :heads], back[:, heads:])
        torch.cuda.synchronize()
        got.append((out, back))
    assert torch.equal(got[0][0], got[1][0]) and torch.equal(got[0][1], got[1][1])
    assert got[0][1].abs().max() > 1


def test_decoder_layers_together(gpu):
    """Two layers of a small decoder as a server runs them: a prompt through int4 projections, cache and attention in
    two chunks, then six tokens one by one in a graph; every product, cache and attention against 64 bits."""
    rng = np.random.default_rng(9)
    hidden, heads, group, dim, layers = 512, 2, 4, 64, 2
    width = (heads * group + 2 * heads) * dim
    prompt, steps = 21, 6
    proj = [[gen.int4_problem(m, k, 64, seed=10 * i + j) for j, (m, k) in enumerate(((width, hidden), (hidden, heads * group * dim)))]
            for i in range(layers)]
    dense = [[gen_dense(p, m, k) for p, (m, k) in zip(ps, ((width, hidden), (hidden, heads * group * dim)))] for ps in proj]
    weights = [[(dev(p["W"], gpu), dev(p["SB"], gpu)) for p in ps] for ps in proj]
    total = prompt + steps
    tokens, _ = to(rng.normal(0, 1, (total, hidden)) * 0.2, "f16", gpu)
    caches = [kq.kv_cache(6, heads, dim, device=gpu) for _ in range(layers)]
    pages = torch.tensor([[4, 1, 5]], dtype=torch.int32, device=gpu)
    length = torch.zeros(1, dtype=torch.int32, device=gpu)

    def forward(x, batch, ws, seen):
        n = x.shape[0]
        for i in range(layers):
            qkv = torch.empty((n, width), dtype=torch.float16, device=gpu)
            kq.int4_gemv(*weights[i][0], x, qkv, kq.GemvParams(width, hidden), batch=n)
            qkv = qkv.mul_(0.05).view(n, -1, dim)
            out = torch.empty((n, heads * group, dim), dtype=torch.float16, device=gpu)
            kq.kv_write(caches[i], batch, qkv[:, heads * group:-heads], qkv[:, -heads:])
            kq.kv_attn(caches[i], batch, qkv[:, :heads * group], out, ws, ws.numel())
            y = torch.empty((n, hidden), dtype=torch.float16, device=gpu)
            kq.int4_gemv(*weights[i][1], out.view(n, -1), y, kq.GemvParams(hidden, heads * group * dim), batch=n)
            seen.append((x, qkv, out, y))
            x = x + y * 0.05
        return x
    calls = []  # (first token, tokens, what each layer computed)
    for a, n in ((0, 16), (16, 5)):
        length.fill_(a + n)
        b = kq.KVBatch(pages, length, 48, max_q=n)
        ws = torch.empty(kq.kv_attn_workspace_size(caches[0], b, heads * group), dtype=torch.uint8, device=gpu)
        seen = []
        forward(tokens[a:a + n], b, ws, seen)
        calls.append((a, n, [[t.clone() for t in s] for s in seen], [codes_of(c) for c in caches]))
    b = kq.KVBatch(pages, length, 48)
    ws = torch.empty(kq.kv_attn_workspace_size(caches[0], b, heads * group), dtype=torch.uint8, device=gpu)
    x, seen = torch.zeros((1, hidden), dtype=torch.float16, device=gpu), []
    scratch = [(c.k.clone(), c.v.clone(), c.k_exp.clone(), c.v_exp.clone()) for c in caches]
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        forward(x, b, ws, seen)
    for c, s in zip(caches, scratch):
        for t, u in zip((c.k, c.v, c.k_exp, c.v_exp), s):
            t.view(torch.uint8).copy_(u.view(torch.uint8))
    for i in range(steps):
        x.copy_(tokens[prompt + i])
        length.fill_(prompt + i + 1)
        g.replay()
        torch.cuda.synchronize()
        calls.append((prompt + i, 1, [[t.clone() for t in s] for s in seen], [codes_of(c) for c in caches]))
    oracles = [_kv.Cache(6, heads, dim) for _ in range(layers)]
    table = pages[0].cpu().numpy()
    for a, n, got, held in calls:
        for i in range(layers):
            x, qkv, out, y = (t.double().cpu().numpy() for t in got[i])
            for have, want in ((qkv.reshape(n, -1), x @ dense[i][0].T * 0.05), (y, out.reshape(n, -1) @ dense[i][1].T)):
                # the projections' own bar, and one more fp16 rounding
                assert (np.abs(have - want) <= ATOL + (RTOL + 2.0**-10) * np.abs(want)).all()
            oracles[i].write("k", qkv[:, heads * group:-heads], table, a + n, n)
            oracles[i].write("v", qkv[:, -heads:], table, a + n, n)
            for w in "kv":
                assert np.array_equal(held[i][1][w], oracles[i].exps[w])
                assert np.array_equal(_kv.decode(held[i][0][w], "i8"), _kv.decode(oracles[i].codes[w], "i8"))
            ref = _kv.attend(oracles[i], table, a + n, qkv[:, :heads * group], dim**-0.5)
            tol, _ = _kv.attend_tolerance(*ref, dim, *EPS["f16"])
            assert (np.abs(out - ref[0]) <= tol).all(), (a, i)


def gen_dense(p, m, k):
    """float64 [m][k] of an int4 problem with interleaved scales and biases."""
    W = np.asarray(p["W"]).view(np.uint32).reshape(m, k // 8)
    q = np.stack([W >> np.uint32(4 * j) & np.uint32(15) for j in range(8)], -1).reshape(m, k).astype(np.float64)
    sb = np.asarray(p["SB"]).view(np.float16).reshape(m, k // 64, 2).astype(np.float64)
    return q * np.repeat(sb[..., 0], 64, 1) + np.repeat(sb[..., 1], 64, 1)
