"""Verification of drafted tokens, the kept rows moved together in the cache, and a whole step
of speculative decoding, on the GPU through the C ABI, against 64 bits (tests/_spec.py).

Decisions are compared exactly. They are taken in 64 bits: sums of up to 2^18 values differ by 2^-52 times their
number at most however they are added up, 2^-34, so inputs whose nearest decision lies within 2^-30 of its border are
not used (none of these seeds' do)."""
import numpy as np
import pytest
import torch

from kernels_amd import kq
from tests import _kv, _rope, _spec
from tests._util import dev
from tests.test_gpu_graphs import replay_check
from tests.test_gpu_kv import Batch, codes_of, same_cache, to, upload

pytestmark = pytest.mark.gpu
NEAR = 2.0**-30


def softmax(z):
    w = np.exp(z - z.max(-1, keepdims=True))
    return (w / w.sum(-1, keepdims=True)).astype(np.float32)


def draft_of(rng, parents, vocab, spread, near, draft):
    """p, tokens, u, q and q_rows of a sequence: drafts drawn from a model `near` the target."""
    n = len(parents)
    z = rng.normal(0, spread, (n, vocab))
    zq = z + rng.normal(0, near, (n, vocab))
    p, q = softmax(z), softmax(zq)
    tokens, rows = np.zeros(n, np.int32), np.full(n, -1, np.int32)
    rank = [sum(a == b for a in parents[:j]) for j, b in enumerate(parents)]
    for j in range(1, n):
        a = parents[j] if 0 <= parents[j] < j else 0
        if draft == "none" or (draft == "mixed" and rng.random() < 0.4):
            tokens[j] = np.argsort(-zq[a], kind="stable")[min(rank[j], vocab - 1)]
        else:
            rows[j] = a
            w = q[a].astype(np.float64)
            tokens[j] = rng.choice(vocab, p=w / w.sum())
    return p, tokens, rng.random(n).astype(np.float32), (None if draft == "none" else q), rows


def verify_case(gpu, trees, vocab, draft="none", spread=3.0, near=1.0, seed=0, chain=False, use_start=True, pad=0, stride=0, edit=None,
                margin=NEAR):
    """trees: parents of each sequence's rows."""
    rng = np.random.default_rng(seed + vocab + sum(map(len, trees)))
    news = [len(t) for t in trees]
    starts = np.concatenate([[0], np.cumsum(news)]).astype(np.int32)
    rows, max_q = int(starts[-1]) + pad, max(max(news), 1)
    p, q = np.full((rows, vocab), np.nan, np.float32), np.full((rows, vocab), np.nan, np.float32)
    tokens, u, parent, q_rows = (np.full(rows, 5, t) for t in (np.int32, np.float32, np.int32, np.int32))
    want = []
    for i, t in enumerate(trees):
        if not t:
            want.append(([], [], np.inf))
            continue
        at = slice(starts[i], starts[i + 1])
        pp, tok, uu, qq, qr = draft_of(rng, t, vocab, spread, near, draft)
        if edit is not None:
            edit(i, pp, tok, uu, qq, qr)
        want.append(_spec.verify(pp, tok, uu, t, qq, qr))
        assert want[-1][2] > margin, "too near a border"
        p[at], tokens[at], u[at], parent[at] = pp, tok, uu, t
        q_rows[at] = np.where(qr < 0, qr, qr + starts[i])
        if qq is not None:
            q[at] = qq
    wide = vocab + stride
    pd = torch.full((rows, wide), float("nan"), device=gpu)[:, :vocab]
    pd.copy_(torch.from_numpy(p))
    qd = torch.full((rows, wide), float("nan"), device=gpu)[:, :vocab]
    qd.copy_(torch.from_numpy(q))
    n_seq = len(trees)
    keep, out = (torch.full((n_seq, max_q), 77, dtype=torch.int32, device=gpu) for _ in "ko")
    n_keep = torch.full((n_seq,), 77, dtype=torch.int32, device=gpu)
    size = kq.draft_verify_workspace_size(n_seq, max_q, vocab)
    ws = torch.full((size + 4096,), 0xA5, dtype=torch.uint8, device=gpu)
    args = dict(q=None if draft == "none" else qd, q_index=None if draft == "none" else dev(q_rows, gpu),
                parent=None if chain else dev(parent, gpu), start=dev(starts, gpu) if use_start else None)
    if draft == "own":  # a row of q for each row
        args["q"], args["q_index"] = qd[torch.from_numpy(q_rows).clamp(min=0).to(gpu).long()].contiguous(), None
    td, ud = dev(tokens, gpu), dev(u, gpu)
    print(f"verify {news} of {vocab} draft {draft}", flush=True)

    def call():
        kq.draft_verify(pd, td, ud, keep, n_keep, out, ws, size, **args)

    call()
    torch.cuda.synchronize()
    assert (ws[size:] == 0xA5).all(), "behind the workspace"
    k, n, o = keep.cpu().numpy(), n_keep.cpu().numpy(), out.cpu().numpy()
    for i, (rows_kept, toks, _) in enumerate(want):
        assert n[i] == len(rows_kept), (i, n[i], rows_kept)
        assert k[i].tolist() == rows_kept + [-1] * (max_q - len(rows_kept)), i
        assert o[i].tolist() == toks + [-1] * (max_q - len(toks)), (i, o[i], toks)
    return call, [keep, n_keep, out], want


def chain(n):
    return list(range(-1, n - 1))


@pytest.mark.parametrize("vocab", [1, 2, 7, 100, 4095, 4096, 4097, 12289, 32000])
def test_chains(gpu, vocab):
    for draft in ("none", "own", "shared"):
        for seed in range(3):
            verify_case(gpu, [chain(n) for n in (1, 2, 5, 3, 0, 9)], vocab, draft, seed=seed, chain=draft != "shared", pad=1, stride=seed)
    verify_case(gpu, [chain(4)] * 3, vocab, "own", use_start=False, chain=True)


@pytest.mark.parametrize("draft", ["none", "shared", "mixed"])
@pytest.mark.parametrize("vocab", [3, 50, 5000, 20000])
def test_trees(gpu, vocab, draft):
    rng = np.random.default_rng(vocab)
    for seed in range(4):
        trees = [_spec.random_tree(rng, n, back=4 + 6 * seed, roots=0.05) for n in (1, 26, 0, 64, 65, 2)]
        verify_case(gpu, trees, vocab, draft, seed=seed, near=0.5, spread=[0.5, 2, 4, 8][seed])


def test_wide_and_deep(gpu):
    """A row that many continue, and the most rows of a sequence."""
    verify_case(gpu, [[-1] + [0] * 200, [-1] + [0] * 30], 3000, "none", spread=0.1)
    verify_case(gpu, [[-1] + [0] * 40, [-1] + [0] * 10], 3000, "mixed", spread=0.3)
    verify_case(gpu, [chain(1024)], 300, "none", spread=30.0, near=0.01)
    verify_case(gpu, [chain(500)], 64, "shared", spread=2.0, near=0.001)


def test_large_vocabulary(gpu):
    verify_case(gpu, [chain(5)] * 3, 201088, "own", chain=True)
    verify_case(gpu, [_spec.random_tree(np.random.default_rng(0), 40)] * 2, 131073, "mixed")


def test_numbers_that_are_none(gpu):
    """Negative, infinite and NaN probabilities count as 0; tokens outside the vocabulary are never kept."""
    def edit(i, p, tok, u, q, q_rows):
        p[:, 3], p[:, 7], p[:, 11], p[:, 13] = np.nan, np.inf, -1.0, -np.inf
        if q is not None:
            q[:, 3], q[:, 20], q[:, 21] = 0.5, np.nan, np.inf
        if len(tok) > 4:
            tok[1], tok[2], tok[3] = -1, 50, 2**31 - 1

    for draft in ("none", "shared", "mixed"):
        verify_case(gpu, [chain(2), [-1] + [0] * 6 + [2, 3, 4, 5], chain(1)], 50, draft, edit=edit)


def test_nothing_left(gpu):
    """Rows of no probability, and rows whose all is turned down: the first of the largest."""
    def zeros(i, p, tok, u, q, q_rows):
        p[:] = 0.0
        if i == 1:
            p[:, [9, 4990]] = 0.25
            tok[1:] = [9, 4990]
            u[:] = 0.9999999
            u[2] = 1.0  # a number that keeps nothing

    verify_case(gpu, [chain(2), [-1, 0, 0], chain(1)], 5000, "none", edit=zeros, margin=-1.0)


def test_borders_of_the_draw(gpu):
    """u = 0 draws the first place of any probability, the largest u the last; sums that pass chunks."""
    for at in (0, 1, 4095, 4096, 8191, 9000):
        def edit(i, p, tok, u, q, q_rows, at=at):
            p[:] = 0.0
            p[:, at] = 0.5
            p[:, 9999] = 0.5
            u[:] = [0.0, 1.0 - 2.0**-24, 0.25, 0.5][i % 4]

        verify_case(gpu, [chain(1)] * 4, 10000, "none", edit=edit, margin=-1.0)


def test_certain_tokens(gpu):
    """Probabilities of 1 (greedy decoding): a draft is kept where it is the target's token."""
    def edit(i, p, tok, u, q, q_rows):
        best = p.argmax(1)
        p[:] = 0.0
        p[np.arange(len(p)), best] = 1.0

    for seed in range(3):
        verify_case(gpu, [chain(6), _spec.random_tree(np.random.default_rng(seed), 30, back=4)], 1000, "none", spread=4.0, near=0.5, edit=edit, seed=seed,
                    margin=-1.0)


def test_verify_distribution(gpu):
    """What comes first is distributed as the target's draws are: 4096 sequences of one drafted token, and of three
    siblings, each token's share within six standard deviations."""
    vocab, n_seq = 6, 4096
    rng = np.random.default_rng(0)
    p, q = softmax(rng.normal(0, 1, (1, vocab))), softmax(rng.normal(0, 1, (1, vocab)))
    for parents in ([-1, 0], [-1, 0, 0, 0]):
        m = len(parents)
        tok = rng.choice(vocab, (n_seq, m), p=q[0].astype(np.float64) / q[0].astype(np.float64).sum()).astype(np.int32)
        keep, out = (torch.empty((n_seq, m), dtype=torch.int32, device=gpu) for _ in "ko")
        n_keep = torch.empty(n_seq, dtype=torch.int32, device=gpu)
        size = kq.draft_verify_workspace_size(n_seq, m, vocab)
        ws = torch.empty(size, dtype=torch.uint8, device=gpu)
        kq.draft_verify(dev(p, gpu).expand(n_seq * m, vocab), dev(tok.reshape(-1), gpu), torch.from_numpy(rng.random(n_seq * m).astype(np.float32)).to(gpu),
                        keep, n_keep, out, ws, size, q=dev(q, gpu), q_index=torch.zeros(n_seq * m, dtype=torch.int32, device=gpu),
                        parent=dev(np.tile(np.array(parents, np.int32), n_seq), gpu))
        torch.cuda.synchronize()
        share = np.bincount(out[:, 0].cpu().numpy(), minlength=vocab) / n_seq
        assert (np.abs(share - p[0]) <= 6 * np.sqrt(p[0] * (1 - p[0]) / n_seq)).all(), (share, p)


def test_verify_graph(gpu):
    for draft in ("none", "shared"):
        call, outs, _ = verify_case(gpu, [_spec.random_tree(np.random.default_rng(3), 20)] * 3, 9000, draft)
        s = torch.cuda.Stream()
        with torch.cuda.stream(s):
            call()
        torch.cuda.synchronize()
        want = [o.clone() for o in outs]
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            call()
        for _ in range(4):
            for o in outs:
                o.fill_(55)
            g.replay()
            torch.cuda.synchronize()
            assert all(torch.equal(a, b) for a, b in zip(outs, want))
            call()
            torch.cuda.synchronize()


# ---- the kept rows

KEEP = [(20, 5, [0, 2, 4]), (17, 9, [0, 1, 2]), (0, 0, []), (100, 64, [0, 3, 17, 40, 41, 63]), (90, 90, [0, 5, 11, 30, 50, 70, 71, 72, 88]),
        (33, 2, [1]), (64, 33, [0]), (5, 5, []), (130, 40, [20, 21, 22, 23, 24, 25, 26, 27, 28, 29, 30, 31, 32, 33, 34, 35, 36, 37, 38, 39]),
        (3, 5, [0, 1, 3, 4]), (300, 200, list(range(0, 200, 3))), (50, 20, list(range(20))), (70, 30, [0, 2, 2, 5]), (70, 30, [0, 3, 30, 4]),
        (70, 30, [0, 1, 4, 2, 9]), (70, 30, [2, 0]), (2, 1, [0])]


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("dim,heads,page,block", [(64, 3, 16, 16), (128, 2, 64, 16), (96, 1, 32, 32), (192, 2, 64, 64), (256, 1, 16, 16),
                                                  (128, 1, 256, 128), (96, 5, 16, 16), (64, 2, 512, 256)])
def test_keep(gpu, dim, heads, page, block, kind):
    rng = np.random.default_rng(dim + heads + page + block)
    seqs = [(n, m) for n, m, _ in KEEP]
    b = Batch(gpu, seqs, page, rng)
    oracle = _kv.Cache(b.n_pages, heads, dim, page, block, kind)
    oracle.fill(rng)
    for w in "kv":  # exponents that differ by much more than codes have bits, too
        oracle.exps[w] = np.where(rng.random(oracle.exps[w].shape) < 0.1, rng.integers(63, 180, oracle.exps[w].shape), oracle.exps[w]).astype(np.uint8)
    cache = upload(oracle, gpu)
    keep = np.full((len(KEEP), b.max_q), 9, np.int32)
    for i, (_, _, rows) in enumerate(KEEP):
        keep[i, :len(rows)] = rows
    n_keep = np.array([len(rows) for _, _, rows in KEEP], np.int32)
    kq.kv_keep(cache, b.c, dev(keep, gpu), dev(n_keep, gpu))
    torch.cuda.synchronize()
    for i, (n, m, rows) in enumerate(KEEP):
        for w in "kv":
            _spec.keep_rows(oracle, w, b.table[i], n, m, rows)
    same_cache(cache, oracle, "keep")


def test_keep_counts_and_pages(gpu):
    """Counts beyond the rows, pages that are none (as sources: zeros; as places: not written), no q_start."""
    rng = np.random.default_rng(1)
    seqs = [(40, 12), (50, 12), (60, 12), (45, 12), (90, 12)]
    b = Batch(gpu, seqs, 16, rng, q_start=False)
    b.table[1, 3], b.table[2, 2 + 1], b.table[4, 5] = -1, b.n_pages, 2**31 - 1
    b.c.pages.copy_(torch.from_numpy(b.table))
    oracle = _kv.Cache(b.n_pages, 2, 64)
    oracle.fill(rng)
    cache = upload(oracle, gpu)
    keep = np.sort(np.stack([rng.permutation(12) for _ in seqs]), 1).astype(np.int32)
    keep[:, 2:8] += 4
    keep[:, 8:] = 12
    n_keep = np.array([100, 8, 7, -3, 2**31 - 1], np.int32)
    kq.kv_keep(cache, b.c, dev(keep, gpu), dev(n_keep, gpu))
    torch.cuda.synchronize()
    for i, (n, m) in enumerate(seqs):
        for w in "kv":
            _spec.keep_rows(oracle, w, b.table[i], n, m, keep[i, :max(0, min(n_keep[i], m))].tolist())
    same_cache(cache, oracle, "keep")


# ---- a whole step

@pytest.mark.parametrize("kind,dtype,page,block", [("i8", "f16", 16, 16), ("e4m3", "bf16", 64, 32)])
def test_step(gpu, kind, dtype, page, block):
    """Trees' masks, keys turned into the cache, attention, verification, the kept rows together, and the next step's single
    token over what is left, all in a graph: against the same from the oracles, the cache bit for bit."""
    rng = np.random.default_rng(page)
    heads, group, dim, vocab, new = 2, 4, 64, 777, 12
    lens = [70, 33, 12, 150]
    seqs = [(n, new) for n in lens]
    b = Batch(gpu, seqs, page, rng, q_start=False, max_len=200)
    oracle = _kv.Cache(b.n_pages, heads, dim, page, block, kind)
    oracle.fill(rng)
    cache = upload(oracle, gpu)
    q_heads = heads * group
    parents = [_spec.random_tree(rng, new, back=3) for _ in seqs]
    x, x64 = to(rng.normal(0, 1, (b.rows, q_heads + 2 * heads, dim)), dtype, gpu)
    nxt, n64 = to(rng.normal(0, 1, (len(seqs), q_heads + 2 * heads, dim)), dtype, gpu)
    drafts = [draft_of(rng, t, vocab, 2.0, 0.7, "none") for t in parents]
    p, tokens, u = (np.concatenate([d[i] for d in drafts]) for i in range(3))
    freqs = np.array([10000.0 ** (-2 * i / dim) for i in range(dim // 2)], np.float32)
    rope = kq.Rope(torch.from_numpy(freqs).to(gpu))
    pd, td, ud, par = dev(p, gpu), dev(tokens, gpu), dev(u, gpu), dev(np.concatenate(parents).astype(np.int32), gpu)
    mask, pos = torch.zeros((b.rows, 1), dtype=torch.int32, device=gpu), torch.zeros(b.rows, dtype=torch.int32, device=gpu)
    q, out = (torch.zeros((b.rows, q_heads, dim), dtype=x.dtype, device=gpu) for _ in "qo")
    q1, out1 = (torch.zeros((len(seqs), q_heads, dim), dtype=x.dtype, device=gpu) for _ in "qo")
    keep, toks = (torch.zeros((len(seqs), new), dtype=torch.int32, device=gpu) for _ in "ko")
    n_keep = torch.zeros(len(seqs), dtype=torch.int32, device=gpu)
    kv_len = b.c.kv_len.clone()
    then = kq.KVBatch(b.c.pages, kv_len, 200)
    sizes = (kq.kv_attn_tree_workspace_size(cache, b.c, q_heads), kq.kv_attn_workspace_size(cache, then, q_heads),
             kq.draft_verify_workspace_size(len(seqs), new, vocab))
    ws = [torch.empty(n, dtype=torch.uint8, device=gpu) for n in sizes]

    def step():
        tree = kq.kv_tree(b.c, par, mask, pos)
        kq.kv_write_rope(cache, b.c, rope, x[:, q_heads:q_heads + heads], x[:, q_heads + heads:], q=x[:, :q_heads], q_out=q, pos=pos)
        kq.kv_attn_tree(cache, b.c, tree, q, out, ws[0], sizes[0])
        kq.draft_verify(pd, td, ud, keep, n_keep, toks, ws[2], sizes[2], parent=par)
        kq.kv_keep(cache, b.c, keep, n_keep)
        torch.add(b.c.kv_len, n_keep - new + 1, out=kv_len)
        kq.kv_write_rope(cache, then, rope, nxt[:, q_heads:q_heads + heads], nxt[:, q_heads + heads:], q=nxt[:, :q_heads], q_out=q1)
        kq.kv_attn(cache, then, q1, out1, ws[1], sizes[1])

    s = torch.cuda.Stream()
    with torch.cuda.stream(s):  # on another stream, and on a copy of the cache's bytes
        saved = [t.clone() for t in (cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_exp, cache.v_exp)]
        step()
        for t, w in zip((cache.k.view(torch.uint8), cache.v.view(torch.uint8), cache.k_exp, cache.v_exp), saved):
            t.copy_(w)
    torch.cuda.synchronize()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        step()
    g.replay()
    torch.cuda.synchronize()

    eps, tiny = {"f16": (2.0**-10, 2.0**-25), "bf16": (2.0**-7, 2.0**-134)}[dtype]
    dt = x.dtype
    for i, (n, m) in enumerate(seqs):
        rows = slice(i * new, (i + 1) * new)
        first, depth = n - m, _spec.depths(parents[i])
        turned = _rope.turned(x64[rows], first + depth, freqs)
        turned = torch.from_numpy(turned).float().to(dt).double().numpy()
        oracle.write("k", turned[:, q_heads:q_heads + heads], b.table[i], n, m)
        oracle.write("v", x64[rows, q_heads + heads:], b.table[i], n, m)
        assert np.array_equal(q[rows].double().cpu().numpy(), turned[:, :q_heads]), "queries"
        want = _spec.attend(oracle, b.table[i], n, turned[:, :q_heads], dim**-0.5, _spec.masks(parents[i]))
        tol, _ = _spec.attend_tolerance(want, dim, eps, tiny)
        assert (np.abs(out[rows].double().cpu().numpy() - want[0]) <= tol).all(), i
        kept, came, margin = _spec.verify(*drafts[i][:3], parents[i])
        assert margin > NEAR
        assert keep[i, :n_keep[i]].tolist() == kept and toks[i, :n_keep[i]].tolist() == came
        for w in "kv":
            _spec.keep_rows(oracle, w, b.table[i], n, m, kept)
        length = first + len(kept) + 1
        assert int(kv_len[i]) == length
        one = torch.from_numpy(_rope.turned(n64[i:i + 1], [length - 1], freqs)).float().to(dt).double().numpy()
        oracle.write("k", one[:, q_heads:q_heads + heads], b.table[i], length, 1)
        oracle.write("v", n64[i:i + 1, q_heads + heads:], b.table[i], length, 1)
        want = _kv.attend(oracle, b.table[i], length, one[:, :q_heads], dim**-0.5)
        tol, _ = _kv.attend_tolerance(*want, dim, eps, tiny)
        assert (np.abs(out1[i:i + 1].double().cpu().numpy() - want[0]) <= tol).all(), i
    same_cache(cache, oracle, "step")


@pytest.mark.parametrize("kind", ["i8", "e4m3"])
@pytest.mark.parametrize("dim,page,block", [(64, 16, 16), (96, 32, 16), (256, 64, 32)])
def test_keep_of_no_page(gpu, dim, page, block, kind):
    """Rows whose page is none come as codes of zero, whatever the cache's other pages hold (negative values here, and
    codes that are no values)."""
    rng = np.random.default_rng(dim)
    n, m = 6 * page, 3 * page
    b = Batch(gpu, [(n, m), (n, m)], page, rng)
    b.table[0, 4], b.table[1, 5] = -1, b.n_pages
    b.c.pages.copy_(torch.from_numpy(b.table))
    oracle = _kv.Cache(b.n_pages, 2, dim, page, block, kind)
    oracle.fill(rng)
    for w in "kv":
        oracle.codes[w] |= 0x80
        oracle.codes[w][(oracle.codes[w] & 0x7F) == (0x7F if kind == "e4m3" else 0)] ^= 1
    rows = list(range(1, m, 2))
    none = [int(p) for p in b.table[:, 3:].ravel() if 0 <= p < b.n_pages]
    oracle.codes["k"][[p for p in range(b.n_pages) if p not in b.table]] = 0xFF  # pages of no sequence
    assert none and len(rows) < b.max_q
    cache = upload(oracle, gpu)
    keep = np.full((2, b.max_q), -1, np.int32)
    keep[:, :len(rows)] = rows
    kq.kv_keep(cache, b.c, dev(keep, gpu), dev(np.full(2, len(rows), np.int32), gpu))
    torch.cuda.synchronize()
    for i in range(2):
        for w in "kv":
            _spec.keep_rows(oracle, w, b.table[i], n, m, rows)
    same_cache(cache, oracle, "keep")
    codes, _ = codes_of(cache)
    for w in "kv":
        assert np.array_equal(codes[w], oracle.codes[w]), f"{w}: the bytes"


def test_verify_most_sequences(gpu):
    """65535 chains of one token picked outright, in a vocabulary of 7."""
    n, vocab, rng = 65535, 7, np.random.default_rng(0)
    p = softmax(rng.normal(0, 1.5, (2 * n, vocab)))
    token = rng.integers(0, vocab, 2 * n).astype(np.int32)
    u = rng.random(2 * n).astype(np.float32)
    keep, out = (torch.full((n, 2), 77, dtype=torch.int32, device=gpu) for _ in "ko")
    n_keep = torch.full((n,), 77, dtype=torch.int32, device=gpu)
    size = kq.draft_verify_workspace_size(n, 2, vocab)
    kq.draft_verify(dev(p, gpu), dev(token, gpu), dev(u, gpu), keep, n_keep, out, torch.empty(size, dtype=torch.uint8, device=gpu), size)
    torch.cuda.synchronize()
    i, x, u0, u1 = np.arange(n), token[1::2], u[0::2].astype(np.float64), u[1::2].astype(np.float64)
    there = p[0::2][i, x].astype(np.float64)
    kept = u1 < there
    left = p[0::2].astype(np.float64)
    left[i, x] = 0.0
    left[kept] = p[1::2][kept]
    up = left.cumsum(1)
    aim = u0 * up[:, -1]
    last = (up <= aim[:, None]).sum(1)
    sure = np.abs(up - aim[:, None]).min(1) > NEAR  # nearer to a border either place is right
    assert sure.mean() > 0.999
    got = out.cpu().numpy()
    assert np.array_equal(n_keep.cpu().numpy(), 1 + kept)
    assert np.array_equal(keep.cpu().numpy(), np.stack([np.zeros(n), np.where(kept, 1, -1)], 1))
    assert np.array_equal(got[kept, 0], x[kept]) and (got[~kept, 1] == -1).all()
    assert np.array_equal(got[i, kept.astype(int)][sure], last[sure])


def test_keep_most_sequences(gpu):
    """65535 sequences of a page each, two rows of four moved, exponents all the same: codes as they were."""
    n = 65535
    cache = kq.kv_cache(n, 1, 64, device=gpu)
    g = torch.Generator(device=gpu)
    g.manual_seed(0)
    for t in (cache.k, cache.v):
        t.copy_(torch.randint(-127, 128, t.shape, generator=g, device=gpu, dtype=torch.int8))
    pages = torch.arange(n, dtype=torch.int32, device=gpu).flip(0)[:, None].contiguous()
    kv_len = torch.full((n,), 16, dtype=torch.int32, device=gpu)
    k, v = cache.k.clone(), cache.v.clone()
    k[:, :, 12:14], v[..., 12:14] = k[:, :, 13::2].clone(), v[..., 13::2].clone()
    kq.kv_keep(cache, kq.KVBatch(pages, kv_len, 16, max_q=4), torch.tensor([1, 3, -1, -1], dtype=torch.int32, device=gpu).repeat(n, 1),
               torch.full((n,), 2, dtype=torch.int32, device=gpu))
    torch.cuda.synchronize()
    assert torch.equal(cache.k, k) and torch.equal(cache.v, v)
    assert (cache.k_exp == 63).all() and (cache.v_exp == 63).all()


@pytest.mark.parametrize("draft", ["none", "shared"])
def test_verify_two_streams_and_two_graphs(gpu, draft):
    """Two calls at once, each with a workspace of its own; then two graphs that share one, replayed in turn, with
    other numbers between the replays."""
    rng = np.random.default_rng(11)
    trees = [_spec.random_tree(rng, n) for n in (20, 33, 5)]
    starts = np.concatenate([[0], np.cumsum([len(t) for t in trees])]).astype(np.int32)
    vocab, rows, max_q = 9000, int(starts[-1]), 33
    size = kq.draft_verify_workspace_size(3, max_q, vocab)
    ws = [torch.full((size,), 0xA5, dtype=torch.uint8, device=gpu) for _ in range(2)]
    parent, start = dev(np.concatenate(trees).astype(np.int32), gpu), dev(starts, gpu)
    calls, outs, us, ins = [], [], [], []
    for i in range(2):
        parts = [draft_of(rng, t, vocab, 3.0, 0.5, draft) for t in trees]
        p, tok, u = (np.concatenate([d[k] for d in parts]) for k in range(3))
        rows_of = np.concatenate([np.where(d[4] < 0, -1, d[4] + s) for d, s in zip(parts, starts)]).astype(np.int32)
        q = None if draft == "none" else dev(np.concatenate([d[3] for d in parts]), gpu)
        out = [torch.full((3, max_q), 77, dtype=torch.int32, device=gpu) for _ in "ko"] + [torch.full((3,), 77, dtype=torch.int32, device=gpu)]
        args = dict(q=q, q_index=None if q is None else dev(rows_of, gpu), parent=parent, start=start)
        pd, td, ud = dev(p, gpu), dev(tok, gpu), dev(u, gpu)
        calls.append(lambda w, pd=pd, td=td, ud=ud, out=out, args=args: kq.draft_verify(pd, td, ud, out[0], out[2], out[1], ws[w], size, **args))
        outs.append(out), us.append(ud), ins.append(parts)

    def check(i):
        u = us[i].cpu().numpy()
        for s, (t, d) in enumerate(zip(trees, ins[i])):
            kept, toks, margin = _spec.verify(d[0], d[1], u[starts[s]:starts[s + 1]], t, d[3], d[4])
            assert margin > NEAR
            n = int(outs[i][2][s])
            assert n == len(kept) and outs[i][0][s].tolist() == kept + [-1] * (max_q - n) and outs[i][1][s].tolist() == toks + [-1] * (max_q - n)

    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(3):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                calls[i](i)
        torch.cuda.synchronize()
        check(0), check(1)
    graphs = [torch.cuda.CUDAGraph() for _ in range(2)]
    for i, g in enumerate(graphs):
        with torch.cuda.graph(g):
            calls[i](0)
    for _ in range(3):
        for u in us:
            u.copy_(torch.from_numpy(rng.random(rows).astype(np.float32)))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        check(0), check(1)


def test_keep_graph(gpu):
    """kq_kv_keep captured, replayed on lengths, rows and codes that change between replays."""
    rng = np.random.default_rng(4)
    seqs = [(150, 20), (90, 20), (33, 20)]
    b = Batch(gpu, seqs, 32, rng, q_start=False)
    first = _kv.Cache(b.n_pages, 2, 128, 32, 32, "e4m3")
    first.fill(rng)
    cache = upload(first, gpu)
    keep, n_keep = torch.zeros((3, 20), dtype=torch.int32, device=gpu), torch.zeros(3, dtype=torch.int32, device=gpu)
    kq.kv_keep(cache, b.c, keep, n_keep)
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        kq.kv_keep(cache, b.c, keep, n_keep)
    torch.cuda.synchronize()
    oracle = first.copy()
    for r in range(4):
        rows = [sorted(rng.permutation(20)[:rng.integers(1, 20)].tolist()) for _ in seqs]
        lens = [n - 3 * r for n, _ in seqs]
        b.c.kv_len.copy_(torch.tensor(lens, dtype=torch.int32))
        keep.copy_(torch.tensor([x + [-1] * (20 - len(x)) for x in rows], dtype=torch.int32))
        n_keep.copy_(torch.tensor([len(x) for x in rows], dtype=torch.int32))
        g.replay()
        torch.cuda.synchronize()
        for i, n in enumerate(lens):
            for w in "kv":
                _spec.keep_rows(oracle, w, b.table[i], n, 20, rows[i])
        same_cache(cache, oracle, f"replay {r}")
