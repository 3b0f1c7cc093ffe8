"""The key/value cache's exponent bytes from 0 to 255, as a cache from elsewhere may
hold them: a code c of a block stands for c * 2^(byte - 127) whatever the byte,
against the 64-bit oracle (tests/_kv.py)."""
import numpy as np
import pytest
import torch

from kernels_amd import kq
from tests import _kv
from tests.test_gpu_kv import DTYPES, EPS, Batch, same_cache, to, upload

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("out", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("dim", [64, 96])
def test_read(gpu, dim, kind, out):
    """A block of every byte. The values are float32 numbers (the smallest 2^-136) or beyond its largest, which a
    type's largest then stands for: float64 -> float32 loses nothing, and one rounding is left."""
    rng = np.random.default_rng(dim)
    seqs = [(4096, 4096), (100, 30)]
    b = Batch(gpu, seqs, 16, rng)
    oracle = _kv.Cache(b.n_pages, 1, dim, kind=kind)
    oracle.fill(rng)
    for w in "kv":
        oracle.codes[w][..., ::7] = 0
        oracle.exps[w][b.table[0], 0, 0] = rng.permutation(256)
    cache = upload(oracle, gpu)
    got = {w: torch.full((b.rows, 1, dim), 7.0, dtype=DTYPES[out], device=gpu) for w in "kv"}
    kq.kv_read(cache, b.c, got["k"], got["v"])
    torch.cuda.synchronize()
    top = torch.finfo(DTYPES[out]).max
    for w in "kv":
        for i, (n, m) in enumerate(seqs):
            want = torch.from_numpy(oracle.read(w, b.table[i], n, m)).clamp(-top, top).float().to(DTYPES[out])
            have = got[w][b.starts[i]:b.starts[i + 1]].cpu()
            bad = (have != want).nonzero()
            first = tuple(bad[0].tolist()) if len(bad) else None
            assert first is None, (w, i, first, have[first].item(), want[first].item(), len(bad))


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("dim,block", [(64, 16), (128, 32)])
def test_write(gpu, dim, block, dtype, kind):
    """Tokens appended to blocks of any byte: the byte stays where it is the larger, and the new codes are x / 2^(byte - 127)."""
    rng = np.random.default_rng(dim)
    was = (0, 1, 10, 62, 63, 64, 127, 190, 246, 248, 252, 253, 254, 255)
    seqs = [(block + 9, 4)] * len(was)
    b = Batch(gpu, seqs, block, rng)
    oracle = _kv.Cache(b.n_pages, 1, dim, block, block, kind)
    oracle.fill(rng)
    for i, e in enumerate(was):
        for w in "kv":
            oracle.exps[w][b.table[i, 1]] = e
    cache = upload(oracle, gpu)
    size = 3.3e38 if dtype == "bf16" else 6e4
    x = {w: to(np.sign(rng.normal(0, 1, (b.rows, 1, dim))) * size * 2.0 ** -rng.integers(0, 9, (b.rows, 1, dim)), dtype, gpu) for w in "kv"}
    kq.kv_write(cache, b.c, x["k"][0], x["v"][0])
    torch.cuda.synchronize()
    for w in "kv":
        for i, (n, m) in enumerate(seqs):
            oracle.write(w, x[w][1][b.starts[i]:b.starts[i + 1]], b.table[i], n, m)
    same_cache(cache, oracle)


# few rows: a row of work each, in parts (joined by four waves or one), in equal shares; many rows: whole, in splits
FORMS = [([(70, 1), (1, 1), (0, 1), (33, 3)], 2, 4), ([(1500, 1), (100, 1), (0, 1)], 1, 2), ([(2300, 2), (700, 1)], 8, 16),
         ([(2600, 1)] + [(30, 1)] * 300, 1, 2), ([(64, 64), (90, 40), (0, 20), (200, 1)], 1, 3), ([(2000, 70), (5, 5)], 1, 2)]


def attend(gpu, seqs, heads, group, dim, kind, dtype, exps, sinks=False, window=0):
    """kq_kv_attn where exps(rng, shape) are V's bytes, against the oracle. Its tolerance's 96 for the exponents and
    the lift (in steps of 2^-24 times dim + 16) is 160 here: |byte - 127| <= 128, and |m| no more than that and the scores."""
    rng = np.random.default_rng(dim + group)
    b = Batch(gpu, seqs, 16, rng)
    oracle = _kv.Cache(b.n_pages, heads, dim, kind=kind)
    oracle.fill(rng)
    oracle.exps["v"] = exps(rng, oracle.exps["v"].shape).astype(np.uint8)
    cache = upload(oracle, gpu)
    q_heads = heads * group
    q, q64 = to(rng.normal(0, 1, (b.rows, q_heads, dim)), dtype, gpu)
    s = rng.normal(0, 3, q_heads).astype(np.float32) if sinks else None
    out, lse = torch.full((b.rows, q_heads, dim), 7.0, dtype=DTYPES[dtype], device=gpu), torch.full((b.rows, q_heads), 7.0, device=gpu)
    n = kq.kv_attn_workspace_size(cache, b.c, q_heads)
    ws = torch.empty(n, dtype=torch.uint8, device=gpu)
    kq.kv_attn(cache, b.c, q, out, ws, n, window=window, sinks=None if s is None else torch.from_numpy(s).to(gpu), lse=lse)
    torch.cuda.synchronize()
    eps, tiny = EPS[dtype]
    top = torch.finfo(DTYPES[dtype]).max
    for i, (length, m) in enumerate(seqs):
        rows = slice(b.starts[i], b.starts[i + 1])
        want = _kv.attend(oracle, b.table[i], length, q64[rows], dim**-0.5, True, window, s)
        tol, tol_lse = _kv.attend_tolerance(*want[:3], want[3] + 64.0, want[4], dim, eps, tiny)
        have, none = lse[rows].double().cpu().numpy(), np.isinf(want[1])
        assert np.array_equal(np.isinf(have), none) and np.array_equal(have[none], want[1][none]), (i, have[:2], want[1][:2])
        off = np.abs(have[~none] - want[1][~none])
        assert (off <= tol_lse[~none]).all(), (i, float(off.max()))
        got = out[rows].double().cpu().numpy()
        # off by its tolerance at most, or infinite where that reaches beyond the type's largest value
        over = np.isinf(got) & (np.sign(got) * want[0] + tol >= top)
        bad = np.argwhere(~((np.abs(got - want[0]) <= tol) | over))
        assert not len(bad), (i, bad[0].tolist(), got[tuple(bad[0])], want[0][tuple(bad[0])], tol[tuple(bad[0])], len(bad))


@pytest.mark.parametrize("seqs,heads,group", FORMS)
@pytest.mark.parametrize("byte", [0, 1, 10, 18, 62, 200, 244, 255])
def test_attention(gpu, byte, seqs, heads, group):
    attend(gpu, seqs, heads, group, 64, "e4m3" if byte % 2 else "i8", "bf16", lambda rng, shape: np.full(shape, byte), sinks=byte in (10, 200))


@pytest.mark.parametrize("dim,kind,dtype", [(64, "i8", "bf16"), (96, "e4m3", "bf16"), (128, "i8", "bf16"), (128, "e4m3", "f16"), (192, "i8", "f16"), (256, "e4m3", "bf16")])
@pytest.mark.parametrize("low", [0, 60, 155])
def test_attention_over_bytes_that_differ(gpu, low, dim, kind, dtype):
    """Bytes of a head that differ by up to 100, in any order, growing and falling."""
    for j, (seqs, heads, group) in enumerate(FORMS):
        if j % 2 == low // 60 % 2:
            orders = (lambda rng, shape: low + rng.integers(0, 101, shape), lambda rng, shape: low + np.arange(np.prod(shape)).reshape(shape) % 101)
            attend(gpu, seqs, heads, group, dim, kind, dtype, orders[j // 2 % 2], sinks=j == 1, window=37 if j == 4 else 0)


@pytest.mark.parametrize("seqs", [[(70, 1), (1, 1)], [(1500, 1)], [(80, 70)]])
@pytest.mark.parametrize("dtype,size,scale,byte", [("f16", 1.0, 2.0, 255), ("bf16", 1.0, 40.0, 255), ("bf16", 1e38, 0.1, 150)])
def test_keys_of_zero(gpu, dtype, size, scale, byte, seqs):
    """Zero codes are zeros, also where 2^(byte - 127) times the scale, or what a row of large queries goes by, is beyond
    float32's largest: every token has the same probability, 1 / n, and lse is log n."""
    rng = np.random.default_rng(byte)
    b = Batch(gpu, seqs, 16, rng)
    oracle = _kv.Cache(b.n_pages, 1, 64)
    oracle.fill(rng)
    oracle.codes["k"][:], oracle.exps["k"][:] = 0, byte
    cache = upload(oracle, gpu)
    q, q64 = to(np.clip(rng.normal(0, size, (b.rows, 2, 64)), -3e38, 3e38), dtype, gpu)  # finite
    out, lse = torch.full((b.rows, 2, 64), 7.0, dtype=DTYPES[dtype], device=gpu), torch.full((b.rows, 2), 7.0, device=gpu)
    ws = torch.empty(kq.kv_attn_workspace_size(cache, b.c, 2), dtype=torch.uint8, device=gpu)
    kq.kv_attn(cache, b.c, q, out, ws, ws.numel(), scale=scale, lse=lse)
    torch.cuda.synchronize()
    for i, (n, m) in enumerate(seqs):
        rows = slice(b.starts[i], b.starts[i + 1])
        want = _kv.attend(oracle, b.table[i], n, q64[rows], scale)
        tol, tol_lse = _kv.attend_tolerance(*want, 64, *EPS[dtype])
        assert (np.abs(out[rows].double().cpu().numpy() - want[0]) <= tol).all()
        assert (np.abs(lse[rows].double().cpu().numpy() - want[1]) <= tol_lse).all()
