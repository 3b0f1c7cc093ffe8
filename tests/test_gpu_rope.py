"""Rotary positions on the GPU through the C ABI, against 64 bits (tests/_rope.py): rows turned by
themselves, there and back, and on their way into the 8-bit cache."""
import numpy as np
import pytest
import torch

from kernels_amd import kq
from tests import _kv, _rope
from tests._util import dev
from tests.test_gpu_graphs import replay_check
from tests.test_gpu_kv import DTYPES, SEQS, Batch, same_cache, to, upload, wild

pytestmark = pytest.mark.gpu

EPS = {"f16": (2.0**-10, 2.0**-25), "bf16": (2.0**-7, 2.0**-134), "f32": (0.0, 0.0)}  # eps, half the smallest step


def freqs_of(rot, gpu, base=500000.0):
    f = np.array([base ** (-2.0 * i / rot) for i in range(rot // 2)], np.float32)
    return f, torch.from_numpy(f).to(gpu)


def check_turned(got, x64, pos, f, dtype, pairs, amplitude, inverse, what=""):
    want = _rope.turned(x64, pos, f, pairs, amplitude, inverse)
    far = float(np.abs(np.asarray(pos, np.float64)).max()) * float(np.abs(f).max()) if len(pos) else 0.0
    tol = _rope.tolerance(x64, want, 2 * len(f), pairs, amplitude, *EPS[dtype], far)
    off = np.abs(got.double().cpu().numpy() - want)
    assert (off <= tol).all(), (what, float(np.nanmax(off / tol)), np.argwhere(~(off <= tol))[:3].tolist())


def one(gpu, rows, heads, dim, rot, dtype, pairs=False, amplitude=1.0, inverse=False, far=5000, seed=0):
    rng = np.random.default_rng(seed + rows + heads + dim + rot)
    f, fd = freqs_of(rot, gpu)
    x, x64 = to(rng.normal(0, 1, (rows, heads, dim)), dtype, gpu)
    pos = rng.integers(-far, far + 1, rows).astype(np.int32)
    r = kq.Rope(fd, pairs, amplitude, inverse)
    out = torch.full_like(x, 7.0)
    print(f"rope {rows} x {heads} x {dim} rot {rot} {dtype} pairs {pairs}", flush=True)
    kq.rope(x, out, dev(pos, gpu), r)
    torch.cuda.synchronize()
    check_turned(out, x64, pos, f, dtype, pairs, amplitude, inverse)
    assert torch.equal(out[..., rot:], x[..., rot:]), "columns behind"
    kq.rope(x, x, dev(pos, gpu), r)
    torch.cuda.synchronize()
    assert torch.equal(x, out), "in place"


@pytest.mark.parametrize("pairs", [False, True])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,heads,dim,rot", [(1, 40, 128, 128), (5, 3, 128, 64), (7, 1, 64, 16), (3, 9, 96, 96), (2, 5, 80, 80),
                                                (4, 2, 256, 256), (3, 7, 192, 48), (1, 1, 8, 2), (5, 6, 96, 24), (3, 2, 128, 126),
                                                (2, 33, 512, 512), (3, 3, 512, 500), (300, 65, 64, 64)])
def test_rows(gpu, rows, heads, dim, rot, dtype, pairs):
    one(gpu, rows, heads, dim, rot, dtype, pairs)


def test_amplitude_and_inverse(gpu):
    for pairs in (False, True):
        one(gpu, 9, 4, 128, 96, "bf16", pairs, amplitude=1.1386)
        one(gpu, 9, 4, 128, 128, "f32", pairs, amplitude=-0.5, inverse=True)
        one(gpu, 3, 4, 64, 10, "f16", pairs, amplitude=0.0, inverse=True)


def test_far_positions(gpu):
    """The ends of int32: the fastest pair's angle is still exact to what 64 bits hold."""
    rng = np.random.default_rng(3)
    f, fd = freqs_of(64, gpu)
    pos = np.array([0, 1, -1, 131071, 2**20 + 1, 2**24 + 1, 2**31 - 1, -2**31, 16777215], np.int32)
    x, x64 = to(rng.normal(0, 1, (len(pos), 3, 64)), "f32", gpu)
    out = torch.empty_like(x)
    kq.rope(x, out, dev(pos, gpu), kq.Rope(fd))
    torch.cuda.synchronize()
    check_turned(out, x64, pos, f, "f32", False, 1.0, False)


def test_many_rows_and_strides(gpu):
    """So many rows that a wave takes all heads of one; slices of a fused projection, heads outermost, one row for all."""
    one(gpu, 6000, 36, 64, 64, "bf16")
    one(gpu, 17000, 3, 64, 62, "f16", pairs=True)
    rng = np.random.default_rng(4)
    f, fd = freqs_of(64, gpu)
    rows = 700
    pos = rng.integers(0, 9000, rows).astype(np.int32)
    fused, f64 = to(rng.normal(0, 1, (rows, 7, 64)), "bf16", gpu)
    by_head, h64 = to(rng.normal(0, 1, (5, rows, 64)), "bf16", gpu)
    single, s64 = to(rng.normal(0, 1, (1, 5, 64)), "bf16", gpu)
    for x, x64 in ((fused[:, 1:6], f64[:, 1:6]), (by_head.transpose(0, 1), h64.swapaxes(0, 1)),
                   (single.expand(rows, 5, 64), np.broadcast_to(s64, (rows, 5, 64)))):
        out = torch.full((rows, 9, 64), 7.0, dtype=x.dtype, device=gpu)
        kq.rope(x, out[:, 2:7], dev(pos, gpu), kq.Rope(fd))
        torch.cuda.synchronize()
        check_turned(out[:, 2:7], x64, pos, f, "bf16", False, 1.0, False)
        assert (out[:, :2] == 7.0).all() and (out[:, 7:] == 7.0).all(), "beside the rows"


@pytest.mark.parametrize("pairs", [False, True])
def test_gradient(gpu, pairs):
    """The inverse is the gradient: <dy, rope(x + e) - rope(x)> = <inverse(dy), e>, and differences of every input."""
    rng = np.random.default_rng(5)
    f, fd = freqs_of(16, gpu, 100.0)
    x, x64 = to(rng.normal(0, 1, (2, 2, 24)), "f32", gpu)
    dy, dy64 = to(rng.normal(0, 1, (2, 2, 24)), "f32", gpu)
    pos = np.array([3, 250], np.int32)
    dx = torch.empty_like(x)
    kq.rope(dy, dx, dev(pos, gpu), kq.Rope(fd, pairs, 1.25, inverse=True))
    torch.cuda.synchronize()
    got = dx.double().cpu().numpy()
    for i in np.ndindex(2, 2, 24):  # differences: rope is linear, so a step of 1 is exact but for rounding
        e = np.zeros_like(x64)
        e[i] = 1.0
        d = (dy64 * (_rope.turned(x64 + e, pos, f, pairs, 1.25) - _rope.turned(x64, pos, f, pairs, 1.25))).sum()
        assert abs(d - got[i]) <= 2.0**-23 * abs(d) + 1e-12, i
    check_turned(dx, dy64, pos, f, "f32", pairs, 1.25, True)


def test_freqs(gpu):
    """The device's copy of kq_rope_freqs turns rows as the host's formula does."""
    f, amplitude = kq.rope_freqs(64, 10000.0, "yarn", factor=8.0, original=4096.0)
    assert f.device.type == "cuda" and f.shape == (32,)
    rng = np.random.default_rng(6)
    x, x64 = to(rng.normal(0, 1, (3, 2, 64)), "f32", gpu)
    pos = np.array([1, 4096, 30000], np.int32)
    out = torch.empty_like(x)
    kq.rope(x, out, dev(pos, gpu), kq.Rope(f, amplitude=amplitude))
    torch.cuda.synchronize()
    check_turned(out, x64, pos, f.cpu().numpy(), "f32", False, amplitude, False)


def test_graph(gpu):
    rng = np.random.default_rng(7)
    f, fd = freqs_of(128, gpu)
    x, _ = to(rng.normal(0, 1, (5, 12, 128)), "f16", gpu)
    pos, out = dev(np.arange(5, dtype=np.int32), gpu), torch.empty_like(x)
    r = kq.Rope(fd)
    replay_check(lambda: kq.rope(x, out, pos, r), [out])


# ---- on the way into the cache

def write_both(gpu, b, oracle, rope, dtype, q_heads, pos, x, in_place=False):
    """kv_write_rope, and rope then kv_write on a copy of the cache: the same bits. Returns the cache and the turned queries."""
    one, two = upload(oracle, gpu), upload(oracle, gpu)
    heads = oracle.heads
    q, k, v = x[:, :q_heads], x[:, q_heads:q_heads + heads], x[:, q_heads + heads:]
    p = b.positions if pos is None else pos
    k2, q2 = torch.full(k.shape, 7.0, dtype=k.dtype, device=gpu), torch.full(q.shape, 7.0, dtype=q.dtype, device=gpu)
    kq.rope(k, k2, dev(p, gpu), rope)
    kq.rope(q, q2, dev(p, gpu), rope)
    kq.kv_write(two, b.c, k2, v)
    before = x.clone()
    out = q if in_place else torch.full(q.shape, 7.0, dtype=q.dtype, device=gpu)
    kq.kv_write_rope(one, b.c, rope, k, v, q=q, q_out=out, pos=None if pos is None else dev(pos, gpu))
    torch.cuda.synchronize()
    same = slice(q_heads if in_place else 0, None)
    assert torch.equal(x[:, same].nan_to_num(9.0), before[:, same].nan_to_num(9.0)), "inputs"
    for a, c in ((one.k, two.k), (one.v, two.v), (one.k_exp, two.k_exp), (one.v_exp, two.v_exp)):
        assert torch.equal(a.view(torch.uint8), c.view(torch.uint8)), "not what rope and kv_write leave"
    n = int(b.starts[-1])
    assert torch.equal(out[:n].nan_to_num(9.0), q2[:n].nan_to_num(9.0)), "queries"
    assert in_place or (out[n:] == 7.0).all(), "rows behind the last sequence"
    return one, k2


def positions(b, rng=None):
    """Of every row: its place in its sequence (rows of none: anything)."""
    p = np.full(b.rows, 77, np.int32)
    for i, (n, m) in enumerate(b.seqs):
        p[b.starts[i]:b.starts[i + 1]] = np.arange(n - m, n)
    return p


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("dim,heads,page,block,rot,pairs", [
    (64, 3, 16, 16, 64, False), (128, 2, 64, 16, 128, True), (128, 2, 16, 16, 128, False), (96, 1, 32, 32, 96, False),
    (96, 2, 16, 16, 48, True), (192, 2, 64, 64, 64, True), (256, 1, 16, 16, 256, False), (128, 1, 256, 128, 32, False),
    (192, 1, 16, 16, 176, False), (256, 3, 32, 32, 16, True)])
def test_write_rope(gpu, dim, heads, page, block, rot, pairs, kind, dtype):
    rng = np.random.default_rng(dim + heads + page + block + rot)
    b = Batch(gpu, SEQS, page, rng, pad=3)
    b.positions = positions(b)
    oracle = _kv.Cache(b.n_pages, heads, dim, page, block, kind)
    oracle.fill(rng)
    q_heads = 2 * heads + 1
    f, fd = freqs_of(rot, gpu)
    r = kq.Rope(fd, pairs, 1.0 if rot == dim else 0.9)
    x, _ = to(wild(rng, (b.rows, q_heads + 2 * heads, dim), dtype), dtype, gpu)
    cache, k2 = write_both(gpu, b, oracle, r, dtype, q_heads, None, x)
    k64, v64 = k2.double().cpu().numpy(), x[:, q_heads + heads:].double().cpu().numpy()
    for i, (n, m) in enumerate(SEQS):
        rows = slice(b.starts[i], b.starts[i + 1])
        oracle.write("k", k64[rows], b.table[i], n, m)
        oracle.write("v", v64[rows], b.table[i], n, m)
    same_cache(cache, oracle, "write_rope")
    # the keys that went in are the formula's, where it is finite
    x64 = x[:, q_heads:q_heads + heads].double().cpu().numpy()
    there = np.isfinite(x64).all(-1) & (np.abs(x64).max(-1) < 3e4)
    with np.errstate(invalid="ignore"):
        want = _rope.turned(np.where(there[..., None], x64, 0.0), b.positions, f, pairs, 1.0 if rot == dim else 0.9)
    tol = _rope.tolerance(np.where(there[..., None], x64, 0.0), want, rot, pairs, 1.0, *EPS[dtype], 400.0)
    assert (np.abs(k64 - want) <= tol)[there].all()


def test_write_rope_positions_and_in_place(gpu):
    """Positions of a tree, queries turned in place in the projection's rows; without q_start; a single token."""
    rng = np.random.default_rng(9)
    for seqs, q_start in (([(50, 20), (9, 9), (33, 1)], True), ([(40, 3), (3, 3), (17, 3)], False), ([(130, 1)], False)):
        b = Batch(gpu, seqs, 32, rng, q_start=q_start)
        oracle = _kv.Cache(b.n_pages, 2, 128, 32, 16)
        oracle.fill(rng)
        _, fd = freqs_of(64, gpu)
        pos = rng.integers(-5, 200000, b.rows).astype(np.int32)
        x, _ = to(rng.normal(0, 1, (b.rows, 9, 128)), "bf16", gpu)
        write_both(gpu, b, oracle, kq.Rope(fd), "bf16", 5, pos, x.clone())
        write_both(gpu, b, oracle, kq.Rope(fd, pairs=True), "bf16", 5, pos, x, in_place=True)


# more heads of queries than a wave takes of a row; blocks whose keys wait in LDS, and one that is too large for it
@pytest.mark.parametrize("dim,rot,q_heads,page,block", [(256, 256, 37, 16, 16), (128, 128, 70, 32, 32), (64, 64, 129, 64, 64), (64, 64, 3, 128, 128),
                                                        (96, 96, 43, 32, 16), (64, 48, 1, 32, 32)])
def test_write_rope_query_heads(gpu, dim, rot, q_heads, page, block):
    rng = np.random.default_rng(dim + rot + q_heads)
    b = Batch(gpu, [(150, 40), (9, 9), (33, 1), (7, 0), (70, 70)], page, rng, pad=2)
    oracle = _kv.Cache(b.n_pages, 1, dim, page, block)
    oracle.fill(rng)
    _, fd = freqs_of(rot, gpu)
    pos = rng.integers(-5, 200000, b.rows).astype(np.int32)
    x, _ = to(rng.normal(0, 1, (b.rows, q_heads + 2, dim)), "bf16", gpu)
    write_both(gpu, b, oracle, kq.Rope(fd), "bf16", q_heads, pos, x.clone())
    write_both(gpu, b, oracle, kq.Rope(fd, pairs=True), "bf16", q_heads, pos, x, in_place=True)


def test_write_rope_without_queries(gpu):
    rng = np.random.default_rng(10)
    b = Batch(gpu, [(50, 20), (9, 9)], 16, rng)
    b.positions = positions(b)
    oracle = _kv.Cache(b.n_pages, 2, 64)
    _, fd = freqs_of(64, gpu)
    x, _ = to(rng.normal(0, 1, (b.rows, 6, 64)), "f16", gpu)
    want, _ = write_both(gpu, b, oracle, kq.Rope(fd), "f16", 2, None, x)
    got = upload(oracle, gpu)
    kq.kv_write_rope(got, b.c, kq.Rope(fd), x[:, 2:4], x[:, 4:])
    torch.cuda.synchronize()
    assert torch.equal(got.k, want.k) and torch.equal(got.v, want.v) and torch.equal(got.k_exp, want.k_exp)


def test_write_rope_graph(gpu):
    """Captured, and replayed on tables and lengths that changed in between."""
    rng = np.random.default_rng(11)
    b = Batch(gpu, [(50, 4), (20, 4)], 16, rng, q_start=False, max_len=100, wide=4)
    _, fd = freqs_of(64, gpu)
    r = kq.Rope(fd)
    x, _ = to(rng.normal(0, 1, (b.rows, 4, 64)), "f16", gpu)
    cache = kq.kv_cache(b.n_pages, 1, 64)
    q_out = torch.empty((b.rows, 2, 64), dtype=torch.float16, device=gpu)
    outs = [torch.zeros((b.rows, 1, 64), dtype=torch.float16, device=gpu) for _ in "kv"]

    def step():
        kq.kv_write_rope(cache, b.c, r, x[:, 2:3], x[:, 3:], q=x[:, :2], q_out=q_out)
        kq.kv_read(cache, b.c, *outs)

    replay_check(step, [q_out, *outs])
