"""Trees of drafted tokens over the 8-bit cache on the GPU through the C ABI, against 64 bits
(tests/_spec.py): masks and positions exactly, attention within what the arithmetic allows."""
import numpy as np
import pytest
import torch

from kernels_amd import kq
from tests import _kv, _spec
from tests._util import dev
from tests.test_gpu_graphs import replay_check
from tests.test_gpu_kv import DTYPES, EPS, Batch, to, upload

pytestmark = pytest.mark.gpu


# ---- masks and positions

@pytest.mark.parametrize("window", [0, 1, 2, 5, 2000])
@pytest.mark.parametrize("news", [[1], [26, 1, 64, 33], [0, 5, 32, 0, 31], [300, 7, 1024, 65]])
def test_masks(gpu, news, window):
    rng = np.random.default_rng(sum(news) + window)
    b = Batch(gpu, [(5000 + m, m) for m in news], 16, rng, pad=2)
    parents = [_spec.random_tree(rng, m, back=rng.integers(1, 40), roots=0.1) for m in news]
    # some parents that are no rows before: roots, too
    for ps in parents:
        for j in range(len(ps)):
            if ps[j] < 0 and rng.random() < 0.5:
                ps[j] = int(rng.choice([j, j + 1, 2**31 - 1, -2**31]))
    words = -(-max(news) // 32) + 1
    flat = np.array(sum(parents, []) + [0, 0], np.int32)
    mask, pos = torch.full((b.rows, words), 77, dtype=torch.int32, device=gpu), torch.full((b.rows,), 77, dtype=torch.int32, device=gpu)
    kq.kv_tree(b.c, dev(flat, gpu), mask, pos, window=window)
    torch.cuda.synchronize()
    got, at = mask.cpu().numpy().view(np.uint32), pos.cpu().numpy()
    for i, (m, ps) in enumerate(zip(news, parents)):
        rows = slice(b.starts[i], b.starts[i + 1])
        if m:
            assert np.array_equal(got[rows], _spec.words_of(_spec.masks(ps, window), words)), i
            assert np.array_equal(at[rows], 5000 + _spec.depths(ps)), i
    assert (got[-2:] == 77).all() and (at[-2:] == 77).all(), "rows behind the last sequence"
    only = torch.full((b.rows, words), 77, dtype=torch.int32, device=gpu)
    kq.kv_tree(b.c, dev(flat, gpu), only, window=window)
    torch.cuda.synchronize()
    assert torch.equal(only, mask), "without positions"


# ---- attention

def tree_case(gpu, seqs, heads, group, dim, kind="i8", dtype="f16", page=16, block=16, window=0, sinks=False, lse=True, q_start=True,
              pad=0, seed=0, nan=False, max_len=None, trees=None, pos=None, words=None, scale=None, spoil=None):
    """One call against the oracle. trees: parents of each sequence's rows, or bool [n][n]; drawn where there are none.
    pos: the rows' positions, or their trees'. nan: codes that are no values wherever no sequence has a token."""
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
    sees, at = [], []
    for i, (n, m) in enumerate(seqs):
        t = _spec.random_tree(rng, m) if trees is None else trees[i]
        sees.append(np.asarray(t, bool).reshape(m, m) if m and np.ndim(t) == 2 else _spec.masks(t))
        at.append(n - m + (np.zeros(m, np.int64) if np.ndim(t) == 2 else _spec.depths(t)) if pos is None else pos[i])
    words = words or -(-b.max_q // 32)
    bits = np.full((b.rows, words), 0xFFFFFFFF, np.uint32)  # bits behind a sequence's rows name nothing
    for i, (n, m) in enumerate(seqs):
        own = _spec.words_of(sees[i], words) if m else np.zeros((0, words), np.uint32)
        behind = ~_spec.words_of(np.ones((1, m), bool), words) if m else 0
        bits[b.starts[i]:b.starts[i + 1]] = own | behind
    where = np.full(b.rows, -5, np.int32)
    for i in range(len(seqs)):
        where[b.starts[i]:b.starts[i + 1]] = at[i]
    tree = kq.KVTree(dev(bits, gpu), dev(where, gpu) if window else None)
    qt, q64 = to(rng.normal(0, 1, (b.rows, q_heads, dim)) * np.exp(rng.normal(0, 0.7, (b.rows, q_heads, 1))), dtype, gpu)
    s = rng.normal(0, 3, q_heads).astype(np.float32) if sinks is True else np.float32(sinks) if sinks else None
    out = torch.full((b.rows, q_heads, dim), 7.0, dtype=DTYPES[dtype], device=gpu)
    ls = torch.full((b.rows, q_heads), 7.0, device=gpu) if lse else None
    n = kq.kv_attn_tree_workspace_size(cache, b.c, q_heads)
    ws = torch.full((n + 4096,), 0xA5, dtype=torch.uint8, device=gpu)
    args = dict(scale=scale, window=window, sinks=None if s is None else torch.from_numpy(s).to(gpu), lse=ls)
    print(f"tree {seqs} heads {heads} x {group} dim {dim} {kind} {dtype} page {page}/{block} window {window}", flush=True)
    kq.kv_attn_tree(cache, b.c, tree, qt, out, ws, n, **args)
    torch.cuda.synchronize()
    assert (ws[n:] == 0xA5).all(), "behind the workspace"
    first, first_lse = out.clone(), None if ls is None else ls.clone()
    eps, tiny = EPS[dtype]
    for i, (length, m) in enumerate(seqs):
        if not m:
            continue
        rows = slice(b.starts[i], b.starts[i + 1])
        want = _spec.attend(oracle, b.table[i], length, q64[rows], dim**-0.5 if scale is None else scale, sees[i], at[i], window, s)
        tol, tol_lse = _spec.attend_tolerance(want, dim, eps, tiny)
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
    kq.kv_attn_tree(cache, b.c, tree, qt, out, ws, n, **args)
    torch.cuda.synchronize()
    assert torch.equal(out, first) and (ls is None or torch.equal(ls, first_lse)), "a second run differs"
    return b, cache, qt, out, ls


# lengths and nodes: no prefix, one token, nothing, nodes over several blocks, pages and tiles, more rows than tokens
FEW = [(1, 1), (5, 5), (0, 0), (20, 4), (64, 3), (65, 5), (127, 5), (300, 2), (17, 0), (3, 5), (513, 4), (0, 2)]
MANY = [(70, 70), (1, 1), (200, 33), (64, 64), (5, 9), (0, 3), (129, 2), (40, 0), (17, 16), (300, 111), (97, 64), (640, 26)]


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("dim,group", [(64, 8), (96, 3), (128, 4), (192, 1), (256, 2), (128, 1)])
def test_few_rows(gpu, dim, group, kind, dtype):
    tree_case(gpu, FEW, 2, group, dim, kind, dtype, pad=2, nan=True, sinks=group == 3)


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("dim,group", [(64, 8), (96, 3), (128, 4), (192, 1), (256, 2)])
def test_many_rows(gpu, dim, group, kind, dtype):
    tree_case(gpu, MANY, 2, group, dim, kind, dtype, pad=5, nan=True, sinks=group == 8)


@pytest.mark.parametrize("window", [1, 2, 16, 63, 64, 65, 128, 600, 2**32 - 1])
def test_window(gpu, window):
    tree_case(gpu, [(n + 5, 5) for n in (0, 1, 64, 127, 128, 129, 1000)] + [(3, 5), (0, 5)], 2, 3, 64, window=window, sinks=window % 2 == 0, nan=True)
    tree_case(gpu, MANY, 2, 4, 128, window=window, sinks=window % 2 == 0, nan=True, kind="e4m3")


def test_window_positions(gpu):
    """Positions of the caller's own: before the first row (they count as that), and far behind any token."""
    seqs = [(200, 6), (40, 6), (6, 6)]
    pos = [np.array([194, 0, -7, 199, 230, 2**31 - 2**16 - 1]), np.array([34, 35, 36, 60, 70, 20]), np.array([0, 1, 2, 3, 4, 9])]
    for group in (2, 16):
        for window in (1, 30, 100, 2**32 - 1):
            tree_case(gpu, seqs, 2, group, 64, window=window, pos=pos)


@pytest.mark.parametrize("group", [1, 4, 16])
def test_masks_of_any_kind(gpu, group):
    """Rows that see nothing, everything, or rows behind them, with and without tokens before and sinks."""
    rng = np.random.default_rng(group)
    seqs = [(6, 6), (30, 6), (6, 6), (80, 40), (40, 40), (45, 40)]
    trees = [np.zeros((6, 6)), np.zeros((6, 6)), np.ones((6, 6)), rng.random((40, 40)) < 0.5, np.zeros((40, 40)), np.tri(40).T]
    for sinks in (False, True, [-np.inf] * (2 * group)):
        tree_case(gpu, seqs, 2, group, 64, trees=trees, sinks=sinks, nan=True)
    tree_case(gpu, seqs, 2, group, 128, trees=trees, window=3, words=4)


@pytest.mark.parametrize("page,block", [(16, 16), (32, 16), (64, 64), (256, 256), (1024, 16)])
def test_pages(gpu, page, block):
    tree_case(gpu, [(1500, 7), (100, 3), (1, 1)], 2, 4, 128, "i8", "bf16", page, block, sinks=True, nan=True)
    tree_case(gpu, [(700, 60), (100, 33), (64, 64)], 2, 4, 64, "e4m3", "f16", page, block, nan=True)


def test_chain_is_causal(gpu):
    """A chain's rows see what kv_attn's do: the same sums, and the same bits."""
    for seqs, group in (([(500, 7), (65, 7), (7, 7)], 4), ([(500, 70), (90, 70), (70, 70)], 4)):
        b, cache, q, out, lse = tree_case(gpu, seqs, 2, group, 128, trees=[list(range(-1, m - 1)) for _, m in seqs])
        want, want_lse = torch.empty_like(out), torch.empty_like(lse)
        n = kq.kv_attn_workspace_size(cache, b.c, 2 * group)
        kq.kv_attn(cache, b.c, q, want, torch.empty(n, dtype=torch.uint8, device=gpu), n, lse=want_lse)
        torch.cuda.synchronize()
        assert (out.float() - want.float()).abs().max() <= 2.0**-9 * want.float().abs().max()
        assert (lse - want_lse).abs().max() <= 2.0**-19 * (want_lse.abs().max() + 1)


def ragged(n, longest, seed, new):
    rng = np.random.default_rng(seed)
    lens = rng.integers(0, 40, n)
    lens[rng.integers(0, n, 4)] = rng.integers(longest // 2, longest, 4)
    lens[n // 3] = longest
    return [(int(x) + int(m), int(m)) for x, m in zip(lens, rng.integers(0, new + 1, n))]


# the ways to share out few rows, and splits of many
@pytest.mark.parametrize("n,heads,group,longest,new,kw", [
    (40, 2, 4, 2700, 4, {}), (70, 1, 16, 2500, 3, dict(kind="e4m3")), (300, 1, 2, 2700, 5, {}), (280, 1, 3, 2600, 2, dict(window=2200, sinks=True)),
    (1100, 1, 2, 2500, 2, {}), (20, 8, 8, 2100, 8, dict(dim=192)), (5, 1, 8, 3000, 64, dict(dim=128)), (2, 2, 4, 4000, 100, dict(kind="e4m3")),
    (30, 2, 8, 900, 20, dict(dim=128, window=700)), (3, 1, 1, 3000, 300, {})])
def test_shares(gpu, n, heads, group, longest, new, kw):
    tree_case(gpu, ragged(n, longest, n, new), heads, group, **{"dim": 64, "nan": True, "pad": 1, **kw})


# shares of many rows: a cut for each row of work, and for each workgroup; tiles of 128 and 256 rows, one and two
@pytest.mark.parametrize("n,heads,group,longest,kw", [
    (300, 1, 16, 2300, {}), (150, 4, 16, 2300, dict(kind="e4m3")), (150, 1, 32, 2200, dict(dim=128)), (100, 3, 32, 2200, dict(dim=128, kind="e4m3")),
    (150, 2, 32, 2300, dict(window=2100, sinks=True)), (140, 2, 16, 2200, dict(dim=192)), (90, 2, 24, 2400, dict(dim=96, page=64, block=32))])
def test_shares_of_many_rows(gpu, n, heads, group, longest, kw):
    tree_case(gpu, ragged(n, longest, n + group, 8), heads, group, **{"dim": 64, "nan": True, "pad": 1, **kw})


def test_long_and_bounds_above(gpu):
    tree_case(gpu, [(9001, 9), (30, 4)], 1, 4, 64, max_len=20000)
    tree_case(gpu, [(4000, 70), (71, 70)], 1, 2, 64, max_len=50000, page=64, block=32)
    tree_case(gpu, [(2600, 1000), (1100, 1024)], 1, 1, 64)


def test_without_q_start_and_strides(gpu):
    tree_case(gpu, [(100, 5), (400, 5), (4, 5)], 2, 4, 128, "e4m3", q_start=False, scale=-0.3)
    tree_case(gpu, [(100, 40), (400, 40), (39, 40)], 2, 4, 64, "e4m3", q_start=False, lse=False)


def test_pages_that_are_none(gpu):
    def spoil(b, gpu):
        b.table[0, 2], b.table[1, 0], b.table[2, 3] = -1, 2**31 - 1, b.n_pages
        b.c.pages.copy_(torch.from_numpy(b.table))

    tree_case(gpu, [(100, 5), (40, 5), (70, 5)], 2, 4, 64, spoil=spoil)
    tree_case(gpu, [(100, 50), (40, 40), (70, 65)], 2, 4, 64, spoil=spoil)


def test_graph(gpu):
    """Masks and attention in one graph, on lengths and parents that change between replays."""
    rng = np.random.default_rng(1)
    for new, group in ((4, 4), (40, 4)):
        b = Batch(gpu, [(150, new), (90, new)], 16, rng, q_start=False, max_len=4000)
        oracle = _kv.Cache(b.n_pages, 2, 64)
        oracle.fill(rng)
        cache = upload(oracle, gpu)
        q, _ = to(rng.normal(0, 1, (b.rows, 2 * group, 64)), "f16", gpu)
        out, lse = torch.empty_like(q), torch.empty((b.rows, 2 * group), device=gpu)
        parent = dev(np.array(_spec.random_tree(rng, new) * 2, np.int32), gpu)
        mask, pos = torch.empty((b.rows, 2), dtype=torch.int32, device=gpu), torch.empty(b.rows, dtype=torch.int32, device=gpu)
        n = kq.kv_attn_tree_workspace_size(cache, b.c, 2 * group)
        ws = torch.empty(n, dtype=torch.uint8, device=gpu)

        def step():
            tree = kq.kv_tree(b.c, parent, mask, pos)
            kq.kv_attn_tree(cache, b.c, tree, q, out, ws, n, window=70, lse=lse)

        replay_check(step, [out, lse])
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            step()
        parent.copy_(torch.from_numpy(np.array(_spec.random_tree(rng, new, back=2) * 2, np.int32)))
        b.c.kv_len -= 33
        g.replay()
        torch.cuda.synchronize()
        got = out.clone()
        step()
        torch.cuda.synchronize()
        assert torch.equal(got, out)


@pytest.mark.parametrize("seqs", [[(3000, 40), (500, 33)], [(3000, 5), (500, 3)]])
def test_two_streams_and_two_graphs(gpu, seqs):
    """Two calls at once, each with a workspace of its own; then two graphs that share one, replayed in turn."""
    b, cache, q, out, lse = tree_case(gpu, seqs, 2, 4, 64, trees=[list(range(-1, m - 1)) for _, m in seqs])
    parent = dev(np.concatenate([np.arange(-1, m - 1) for _, m in seqs]).astype(np.int32), gpu)
    tree = kq.kv_tree(b.c, parent, torch.zeros((b.rows, 2), dtype=torch.int32, device=gpu))
    n = kq.kv_attn_tree_workspace_size(cache, b.c, 8)
    ws = [torch.full((n,), 0xA5, dtype=torch.uint8, device=gpu) for _ in range(2)]
    qs = [q, -q]
    outs = [torch.full_like(out, 7.0) for _ in range(2)]

    def call(i, w):
        kq.kv_attn_tree(cache, b.c, tree, qs[i], outs[i], ws[w], n)

    call(1, 1)
    torch.cuda.synchronize()
    want = [out, outs[1].clone()]
    streams = [torch.cuda.Stream() for _ in range(2)]
    for _ in range(3):
        for o in outs:
            o.fill_(7.0)
        torch.cuda.synchronize()
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                call(i, i)
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(outs, want)), "two streams"
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for i, g in enumerate(graphs):
        with torch.cuda.graph(g):
            call(i, 0)
    for _ in range(3):
        for o in outs:
            o.fill_(7.0)
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, c) for a, c in zip(outs, want)), "two graphs"


@pytest.mark.parametrize("dim,kind", [(192, "i8"), (256, "e4m3"), (128, "i8"), (64, "e4m3")])
@pytest.mark.parametrize("max_q", [520, 1024])
def test_bounds_of_many_tiles(gpu, dim, kind, max_q):
    """A bound of rows far above what the sequences have: more tiles than workgroups that the device holds at once (of 128
    rows, at 64 heads a key), one group, the largest workspaces."""
    def bound(b, gpu):
        b.max_q = max_q
        b.c = kq.KVBatch(b.c.pages, b.c.kv_len, b.max_len, q_start=b.c.q_start, max_q=max_q)

    tree_case(gpu, [(700, 5), (0, 0), (80, 1), (9, 3)], 2, 64, dim, kind, nan=True, pad=1, max_len=5000, spoil=bound)
    tree_case(gpu, [(300, 3), (90, 2)], 1, 64, dim, kind, "bf16", window=70, sinks=True, spoil=bound)


def test_most_sequences(gpu):
    """65535 sequences: masks, positions, and a tree's attention of equal values, which is that value."""
    n = 65535
    cache = kq.kv_cache(n, 1, 64, device=gpu)
    cache.v.fill_(3)
    cache.v_exp.fill_(127)
    pages = torch.arange(n, dtype=torch.int32, device=gpu).flip(0)[:, None].contiguous()
    kv_len = torch.arange(n, dtype=torch.int32, device=gpu) % 14 + 3
    b = kq.KVBatch(pages, kv_len, 16, max_q=3)
    mask, pos = torch.full((3 * n, 1), 77, dtype=torch.int32, device=gpu), torch.full((3 * n,), 77, dtype=torch.int32, device=gpu)
    tree = kq.kv_tree(b, torch.tensor([-1, 0, 0], dtype=torch.int32, device=gpu).repeat(n), mask, pos)
    torch.cuda.synchronize()
    assert torch.equal(mask.view(n, 3).cpu(), torch.tensor([[1, 3, 5]], dtype=torch.int32).repeat(n, 1))
    assert torch.equal(pos.view(n, 3), kv_len[:, None] - 3 + torch.tensor([0, 1, 1], dtype=torch.int32, device=gpu))
    q = torch.randn((3 * n, 2, 64), device=gpu).half()
    out, lse = torch.zeros_like(q), torch.zeros((3 * n, 2), device=gpu)
    size = kq.kv_attn_tree_workspace_size(cache, b, 2)
    kq.kv_attn_tree(cache, b, tree, q, out, torch.empty(size, dtype=torch.uint8, device=gpu), size, lse=lse)
    torch.cuda.synchronize()
    assert (out == 3).all()
    seen = (kv_len[:, None] - 3 + torch.tensor([1, 2, 2], device=gpu)).view(-1, 1).float()
    # keys of zero: lse is the logarithm of the tokens' number, below 4: four roundings of 2^-22 (sum, logarithm, factor, torch's)
    assert ((lse - seen.log()).abs() <= 2.0**-20).all()
