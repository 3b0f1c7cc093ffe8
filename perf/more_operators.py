"""A step of speculative decoding over the 8-bit key/value cache, operator by operator, as cases to be timed and compared.

Kinds of case (the "kind" of the dict):

  rope    rotary positions of queries and keys (rope); with "grad" the rotation and the
          gradient of its input
  append  a step's keys rotated on their way into the cache, the values beside them, the queries
          rotated (kv_write_rope), and the blocks that the step touched read back (kv_read)
  tree    attention of a tree of drafted tokens, each over the cached tokens and its own
          ancestors (kv_attn_tree)
  verify  drafted tokens against the target's probabilities, with given random numbers
          (draft_verify): which are kept, and the token behind them
  keep    the kept tokens of a tree moved together in the cache (kv_keep), and read back

The cache is paged. A page holds `page` tokens of every head:

  k      [pages][heads][page][dim]          8-bit codes (int8 or e4m3)
  v      [pages][heads][page/16][dim][16]   the same, 16 tokens of a column together
  k_exp, v_exp  uint8 [pages][heads][page/block]: a code c of block b stands
         for c * 2^(exp - 127)

A step's rows are a sequence's newest tokens. In a tree row 0 is the last token that is certain and the
others are drafted: row j continues row parent[j] < j, and stands at the position of row 0 plus its depth.
"""
import math
import random

import torch

own = False

DEV = "cuda"
LOWEST = -64  # exponents that the cache uses: from here
HIGHEST = {"i8": 121, "e4m3": 119}  # to here
LARGEST = {"i8": 127.0, "e4m3": 448.0}
FLOAT = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}


def _rope_case(name, rows, heads, dim, dtype, rot=0, pairs=False, far=8192, amplitude=1.0, grad=False):
    return {"name": name, "kind": "rope", "rows": rows, "heads": heads, "dim": dim, "dtype": dtype, "rot": rot or dim,
            "pairs": pairs, "far": far, "amplitude": amplitude, "grad": grad}


def _cache_case(name, kind, seqs, lens, new, q_heads, heads, dim, store, dtype, page=16, block=16, window=0, sinks=False,
                rot=0, pairs=False, amplitude=1.0, tree=False):
    """lens, new: the shortest and longest length, and number of newest tokens, of a sequence."""
    return {"name": name, "kind": kind, "seqs": seqs, "len_lo": lens[0], "len_hi": lens[1], "new_lo": new[0],
            "new_hi": new[1], "q_heads": q_heads, "heads": heads, "dim": dim, "store": store, "dtype": dtype,
            "page": page, "block": block, "window": window, "sinks": sinks, "rot": rot or dim, "pairs": pairs,
            "amplitude": amplitude, "tree": tree}


def _verify_case(name, seqs, new, vocab, draft, tree):
    """draft: "none" (candidates picked outright), "rows" (a row of probabilities for each drafted token) or "shared"
    (one for all that continue the same token, and some picked outright)."""
    return {"name": name, "kind": "verify", "seqs": seqs, "new_lo": new[0], "new_hi": new[1], "vocab": vocab,
            "draft": draft, "tree": tree}


def listed():
    return [
        # the smallest call: one token's queries and keys (Llama-3-8B heads), at a far position
        _rope_case("rope_b1", 1, 40, 128, "f16", far=131072),
        # a training step's rotation of two sequences of 4096, there and back
        _rope_case("rope_grad", 8192, 40, 128, "bf16", far=4096, grad=True),
        # one sequence's new token into a block that other tokens began
        _cache_case("append_b1", "append", 1, (777, 777), (1, 1), 32, 8, 128, "i8", "f16"),
        # trees of many sequences, 70B-class heads, half of each head rotated in pairs
        _cache_case("append_b48", "append", 48, (40, 8191), (9, 26), 64, 8, 128, "e4m3", "bf16", page=64, block=32,
                    rot=64, pairs=True, tree=True),
        # prefill of a few prompts of odd lengths, positions stretched for long contexts
        _cache_case("append_prefill", "append", 5, (1201, 9001), (1201, 5003), 32, 8, 128, "i8", "bf16", amplitude=1.1386),
        # one sequence's tree: latency
        _cache_case("tree_b1", "tree", 1, (701, 701), (26, 26), 32, 8, 128, "i8", "f16", tree=True),
        # a busy server's step: trees behind sequences of very different lengths
        _cache_case("tree_b16", "tree", 16, (300, 12000), (33, 64), 64, 8, 128, "e4m3", "bf16", page=64, tree=True),
        # a tree over one long context
        _cache_case("tree_long", "tree", 1, (131071, 131071), (60, 60), 32, 8, 128, "i8", "bf16", tree=True),
        # one sequence's tree of outright candidates, a Llama-3 vocabulary
        _verify_case("verify_b1", 1, (60, 60), 128256, "none", True),
        # chains of four drafted tokens with the draft model's probabilities
        _verify_case("verify_b64", 64, (5, 5), 128256, "rows", False),
        # an accepted path moved together
        _cache_case("keep_b1", "keep", 1, (1501, 1501), (60, 60), 32, 8, 128, "i8", "f16", tree=True),
        _cache_case("keep_b64", "keep", 64, (300, 9000), (26, 64), 64, 8, 64, "e4m3", "bf16", page=64, block=32, tree=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def _draw_rope(rng):
    dim = rng.choice([32, 64, 64, 80, 96, 128, 128, 128, 192, 256])
    heads, dtype, grad = _log_int(rng, 1, 96), rng.choice(["f16", "bf16", "bf16", "f32"]), rng.random() < 0.4
    rows = _log_int(rng, 1, max(1, 8192 * 40 * 128 // (heads * dim * (2 if dtype == "f32" else 1) * (1 if grad else 1))))
    rot = dim if rng.random() < 0.6 else 2 * rng.randint(1, dim // 2)
    return _rope_case("", min(rows, 16384), heads, dim, dtype, rot, rng.random() < 0.4, _log_int(rng, 16, 2**20),
                      rng.choice([1.0, 1.0, rng.uniform(0.8, 1.5)]), grad)


def _draw_verify(rng):
    vocab, tree = _log_int(rng, 100, 201088), rng.random() < 0.5
    draft = rng.choice(["none", "rows", "shared"])
    seqs = _log_int(rng, 1, 64)
    new = rng.randint(1, 64) if tree and draft == "none" else rng.randint(1, 16) if tree else rng.randint(1, 9)
    new = max(1, min(new, 64 * 5 * 128256 // (seqs * vocab)))
    return _verify_case("", max(1, min(seqs, 64 * 5 * 128256 // (new * vocab))), (rng.randint(1, new), new), vocab, draft, tree)


def draw(rng):
    kind = rng.choice(["rope", "append", "append", "tree", "tree", "tree", "verify", "verify", "keep"])
    if kind in ("rope", "verify"):
        c = _draw_rope(rng) if kind == "rope" else _draw_verify(rng)
        del c["name"]
        return c
    heads = rng.choice([1, 2, 4, 8, 8, 8, 16])
    group = rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 8, 16])
    dim = rng.choice([64, 64, 96, 128, 128, 128, 192, 256])
    block = rng.choice([16, 16, 32, 64])
    page = block * rng.choice([1, 1, 2, 4])
    store, dtype = rng.choice(["i8", "e4m3"]), rng.choice(["f16", "bf16"])
    seqs = _log_int(rng, 1, 64)
    hi = max(1, min(_log_int(rng, 16, 131072), 2**27 // (heads * dim * seqs)))
    lo = _log_int(rng, 1, hi)
    tree, window, sinks = True, 0, False
    if kind == "append":
        tree = rng.random() < 0.5
        new = _log_int(rng, 1, min(hi, 64 if tree else 8192))
        seqs = max(1, min(seqs, 2**24 // (heads * (group + 2) * dim * new)))
    elif kind == "tree":
        new = rng.randint(1, min(hi, rng.choice([8, 32, 64, 128])))
        window = rng.choice([0, 0, _log_int(rng, 1, 4096)])
        sinks = rng.random() < 0.3
        group = max(1, min(group, 2**33 // (new * hi * heads * dim)))
        seqs = max(1, min(seqs, 2**33 // (new * hi * heads * group * dim)))
    else:
        new = rng.randint(1, min(hi, 64))
    rot = dim if rng.random() < 0.5 else 16 * rng.randint(1, dim // 16)
    c = _cache_case("", kind, seqs, (lo, hi), (_log_int(rng, 1, new), new), heads * group, heads, dim, store, dtype, page,
                    block, window, sinks, rot, rng.random() < 0.4, rng.choice([1.0, rng.uniform(0.8, 1.5)]), tree)
    del c["name"]
    return c


# ---------------------------------------------------------------------------

def _spread(lo, hi, i, by):
    """The i-th of numbers spread over lo..hi by their logarithm; the first is hi."""
    return lo if lo >= hi else int(round(lo * (hi / lo) ** ((1.0 - i * by) % 1.0 or 1.0)))


def _news(case):
    return [_spread(case["new_lo"], case["new_hi"], i, 0.7548776662) for i in range(case["seqs"])]


def _lengths(case):
    """(tokens, newest tokens) of each sequence."""
    ns = [_spread(case["len_lo"], case["len_hi"], i, 0.6180339887) for i in range(case["seqs"])]
    return [(n, min(n, m)) for n, m in zip(ns, _news(case))]


def _parents(case, news):
    """Of each sequence's nodes: a tree of its own shape, or a chain."""
    got = []
    for i, m in enumerate(news):
        r = random.Random(64 * m + i)
        got.append([-1] + [r.randrange(max(0, j - 8), j) if case["tree"] else j - 1 for j in range(1, m)] if m else [])
    return got


def _depths(parents):
    got = []
    for p in parents:
        got.append(0 if p < 0 else got[p] + 1)
    return got


def _kept(case, news):
    """Rows of each sequence that are kept: row 0, the next few where they are, and a few from behind."""
    got = []
    for i, m in enumerate(news):
        r = random.Random(64 * m + i)
        n = min(m, r.randint(1, 8))
        stay = r.randint(1, n)
        behind = sorted(r.sample(range(n, m), min(n - stay, m - n)))
        got.append(list(range(stay)) + behind)
    return got


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _starts(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return at


def _freqs(rot):
    return torch.tensor([500000.0 ** (-2.0 * i / rot) for i in range(rot // 2)], dtype=torch.float32, device=DEV)


def _pow2(e):
    """2^e in float32, exactly (below 2^-126: 2^-126, where every code's product rounds to zero too)."""
    return ((e.clamp(-126, 127) + 127) << 23).view(torch.float32)


def _exponent(a, store):
    """The smallest e with a <= largest code * 2^e, within the cache's range."""
    m, e = torch.frexp(a.double() / LARGEST[store])  # m in [0.5, 1); 64 bits keep a quotient from rounding to a power of two
    e = e - (m == 0.5).int()
    return torch.where(a > 0, e, LOWEST).clamp(LOWEST, HIGHEST[store])


def _encode(x, store):
    """Codes of float32 values already divided by their scale: half to even, saturated."""
    x = x.clamp(-LARGEST[store], LARGEST[store])
    return x.round().to(torch.int8) if store == "i8" else x.to(torch.float8_e4m3fn).view(torch.int8)


def _decode(c, store):
    return c.float() if store == "i8" else c.view(torch.float8_e4m3fn).float()


def _fill(n_pages, case, g, seen):
    """Codes [pages][heads][page][dim] and exponent bytes of random keys or values; seen [pages][page]: tokens that are
    in the cache (the others are zero)."""
    heads, page, dim, block = case["heads"], case["page"], case["dim"], case["block"]
    codes = torch.empty((n_pages, heads, page, dim), dtype=torch.int8, device=DEV)
    exps = torch.empty((n_pages, heads, page // block), dtype=torch.uint8, device=DEV)
    channel = torch.empty((heads, 1, dim), device=DEV).normal_(0.0, 0.5, generator=g).exp()
    step = max(1, 2**27 // (heads * page * dim))
    for p in range(0, n_pages, step):
        n = min(step, n_pages - p)
        x = torch.empty((n, heads, page, dim), device=DEV).normal_(generator=g) * channel
        x = x * (torch.empty((n, heads, page, 1), device=DEV).normal_(0.0, 0.3, generator=g).exp())
        x = (x * seen[p:p + n, None, :, None]).view(n, heads, page // block, block, dim)
        e = _exponent(x.abs().amax((3, 4)), case["store"])
        codes[p:p + n] = _encode(x * _pow2(-e)[..., None, None], case["store"]).view(n, heads, page, dim)
        exps[p:p + n] = (e + 127).to(torch.uint8)
    return codes, exps


def _columns(v):
    """[pages][heads][page][dim] into the values' order [pages][heads][page/16][dim][16]."""
    n, heads, page, dim = v.shape
    return v.view(n, heads, page // 16, 16, dim).transpose(3, 4).contiguous()


def _prepare_rope(case, g):
    shape, dtype = (case["rows"], case["heads"], case["dim"]), FLOAT[case["dtype"]]
    state = {"x": torch.empty(shape, device=DEV).normal_(generator=g).to(dtype), "freqs": _freqs(case["rot"])}
    state["pos"] = torch.randint(0, case["far"], (case["rows"],), generator=g, device=DEV).int()
    state["y"] = torch.empty(shape, dtype=dtype, device=DEV)
    if case["grad"]:
        state["dy"] = torch.empty(shape, device=DEV).normal_(generator=g).to(dtype)
        state["dx"] = torch.empty(shape, dtype=dtype, device=DEV)
    return state


def _prepare_verify(case, g):
    news = _news(case)
    parents, starts, rows, vocab = _parents(case, news), _starts(news), sum(news), case["vocab"]
    z = torch.empty((rows, vocab), device=DEV).normal_(0.0, 3.0, generator=g)
    state = {"p": torch.softmax(z, 1), "u": torch.rand(rows, generator=g, device=DEV), "start": _ints(starts),
             "parent": _ints(sum(parents, [])), "max_q": max(news), "q": None, "q_index": None}
    before = _ints([starts[i] + max(p, 0) for i, ps in enumerate(parents) for p in ps]).long()  # row of what a row continues
    z += torch.empty((rows, vocab), device=DEV).normal_(0.0, 1.5, generator=g)
    if case["draft"] == "none":
        rank = [sum(q == p for q in ps[:j]) for ps in parents for j, p in enumerate(ps)]
        state["token"] = torch.topk(z, min(16, vocab), 1)[1][before, _ints(rank).long().clamp(max=min(16, vocab) - 1)].int()
    else:
        q = torch.softmax(z, 1)
        drawn = []
        for r in range(0, rows, 64):  # a token of q for each row
            w = torch.rand((min(64, rows - r), vocab), generator=g, device=DEV).clamp(min=1e-20)
            drawn.append((-w.log() / q[before[r:r + 64]].clamp(min=1e-35)).argmin(1))
        state["token"] = torch.cat(drawn).int()
        if case["draft"] == "rows":
            state["q"] = q[before]
        else:
            state["q"], state["q_index"] = q, before.int()
            state["q_index"][torch.rand(rows, generator=g, device=DEV) < 0.1] = -1
    state["keep"], state["out"] = (torch.zeros((case["seqs"], max(news)), dtype=torch.int32, device=DEV) for _ in "ko")
    state["n_keep"] = torch.zeros(case["seqs"], dtype=torch.int32, device=DEV)
    return state


def _masks(parents, words):
    """int32 [rows][words]: bit t of a row: it is row t of its sequence, or continues it."""
    got = []
    for ps in parents:
        bits = []
        for j, p in enumerate(ps):
            bits.append((bits[p] if p >= 0 else 0) | 1 << j)
        for b in bits:
            w = [b >> 32 * k & 0xFFFFFFFF for k in range(words)]
            got.append([v - 2**32 if v >= 2**31 else v for v in w])
    return _ints(got).view(-1, words)


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    if case["kind"] == "rope":
        return {"case": dict(case), **_prepare_rope(case, g)}
    if case["kind"] == "verify":
        return {"case": dict(case), **_prepare_verify(case, g)}
    kind, lengths = case["kind"], _lengths(case)
    news = [m for _, m in lengths]
    page, heads, dim, q_heads = case["page"], case["heads"], case["dim"], case["q_heads"]
    needed = [-(-n // page) for n, _ in lengths]
    n_pages, wide = sum(needed) + 3, max(max(needed), 1)
    order = list(range(n_pages))
    random.Random(seed).shuffle(order)
    table, at = [], 0
    in_cache = [0] * n_pages  # tokens of each page that are there before the call
    for (n, new), k in zip(lengths, needed):
        mine = order[at:at + k]
        at += k
        table.append(mine + [-1] * (wide - k))
        for j, p in enumerate(mine):
            in_cache[p] = max(0, min(page, n - (new if kind == "append" else 0) - j * page))
    seen = torch.arange(page, device=DEV) < _ints(in_cache)[:, None]
    (k, k_exp), (v, v_exp) = _fill(n_pages, case, g, seen), _fill(n_pages, case, g, seen)
    code = torch.int8 if case["store"] == "i8" else torch.float8_e4m3fn
    rows, dtype = sum(news), FLOAT[case["dtype"]]
    state = {"case": dict(case), "k": k.view(code), "v": _columns(v).view(code), "k_exp": k_exp, "v_exp": v_exp,
             "pages": _ints(table), "kv_len": _ints([n for n, _ in lengths]), "max_len": max(n for n, _ in lengths),
             "q_start": _ints(_starts(news)), "max_q": max(news)}
    parents = _parents(case, news)
    if kind == "keep":
        kept = _kept(case, news)
        state["keep"] = _ints([r + [-1] * (max(news) - len(r)) for r in kept])
        state["n_keep"] = _ints([len(r) for r in kept])
        # read back: from the block of the first row on
        ends = [n - m + len(r) for (n, m), r in zip(lengths, kept)]
        back = [e - (n - m) // case["block"] * case["block"] for e, (n, m) in zip(ends, lengths)]
        state["back_len"], state["back_start"], state["max_back"] = _ints(ends), _ints(_starts(back)), max(back)
        state["out_k"], state["out_v"] = (torch.zeros((sum(back), heads, dim), dtype=dtype, device=DEV) for _ in "kv")
        return state
    # one row of a fused projection: q of every head, then k, then v
    x = torch.empty((rows, q_heads + 2 * heads, dim), device=DEV).normal_(generator=g)
    x *= torch.empty((rows, q_heads + 2 * heads, 1), device=DEV).normal_(0.0, 0.5, generator=g).exp()
    x = x.to(dtype)
    state["q"], state["new_k"], state["new_v"] = x[:, :q_heads], x[:, q_heads:q_heads + heads], x[:, q_heads + heads:]
    state["out"] = torch.zeros((rows, q_heads, dim), dtype=dtype, device=DEV)
    depth = sum([[n - m + d for d in _depths(p)] for (n, m), p in zip(lengths, parents)], [])
    state["pos"] = _ints(depth) if case["tree"] else None
    if kind == "tree":
        state["mask"] = _masks(parents, -(-max(news) // 32))
        state["lse"] = torch.zeros((rows, q_heads), dtype=torch.float32, device=DEV)
        state["sinks"] = torch.empty(q_heads, device=DEV).normal_(0.0, 2.0, generator=g) if case["sinks"] else None
        return state
    state["freqs"] = _freqs(case["rot"])
    back = [n - (n - m) // case["block"] * case["block"] for n, m in lengths]  # the touched blocks
    state["back_len"], state["back_start"], state["max_back"] = state["kv_len"], _ints(_starts(back)), max(back)
    state["out_k"], state["out_v"] = (torch.zeros((sum(back), heads, dim), dtype=dtype, device=DEV) for _ in "kv")
    return state


# ---- the plain forms

def _turned(x, pos, freqs, case, sign=1.0):
    """Rotated in 64 bits, for the angles of far positions and the blocks' exponents; [rows][heads][dim]."""
    rot = case["rot"]
    angle = pos.double()[:, None, None] * freqs.double()
    c, s = torch.cos(angle) * case["amplitude"], torch.sin(angle) * (case["amplitude"] * sign)
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if case["pairs"] else (slice(0, rot // 2), slice(rot // 2, rot))
    x64, y = x.double(), x.double()
    y[..., a] = x64[..., a] * c - x64[..., b] * s
    y[..., b] = x64[..., b] * c + x64[..., a] * s
    return y.float().to(x.dtype)


def _rows(start, kv_len, width):
    """For `width` newest tokens of each sequence: (row, position, whether there is one)."""
    start = start.long()
    n = (start[1:] - start[:-1])[:, None]
    j = torch.arange(width, device=DEV)[None]
    return start[:-1, None] + j, kv_len.long()[:, None] - n + j, j < n


def _slots(pages, pos, page):
    """(page, token in it) of positions [seqs][...]."""
    flat = pos.clamp(min=0).reshape(len(pos), -1)
    p = pages.long().gather(1, (flat // page).clamp(max=pages.shape[1] - 1)).clamp(min=0)
    return p.view(pos.shape), (flat % page).view(pos.shape)


def _codes(state, which, p, t):
    codes = state[which].view(torch.int8)
    return codes[p, :, t] if which == "k" else codes[p, :, t // 16, :, t % 16]


def _values(state, which, p, t):
    """float32 values [...][heads][dim] of the cache's tokens (p, t)."""
    c = state["case"]
    e = state[which + "_exp"][p, :, t // c["block"]].int() - 127
    return _decode(_codes(state, which, p, t), c["store"]) * _pow2(e)[..., None]


def _put(state, which, p, t, codes):
    if which == "k":
        state["k"].view(torch.int8)[p, :, t] = codes
    else:
        state["v"].view(torch.int8)[p, :, t // 16, :, t % 16] = codes


def _plain_write(state, which, new):
    c = state["case"]
    block, store = c["block"], c["store"]
    q_start, kv_len = state["q_start"].long(), state["kv_len"].long()
    n = q_start[1:] - q_start[:-1]
    first = kv_len - n
    touched = (state["max_q"] + block - 2) // block + 1
    b = first[:, None] // block + torch.arange(touched, device=DEV)  # [seqs][touched]
    pos = b[..., None] * block + torch.arange(block, device=DEV)
    here = pos < kv_len[:, None, None]
    fresh = here & (pos >= first[:, None, None])
    i, j = here[..., 0].nonzero(as_tuple=True)  # the blocks that there are
    pos, here, fresh = pos[i, j], here[i, j], fresh[i, j]
    row = (q_start[i, None] + pos - first[i, None]).clamp(0, len(new) - 1)
    x = torch.where(fresh[..., None, None], new[row].float(), 0.0)  # [blocks][block][heads][dim]
    e = _exponent(x.abs().amax((1, 3)), store)
    p, t = _slots(state["pages"][i], pos, c["page"])
    before = state[which + "_exp"][p[:, 0], :, t[:, 0] // block].int() - 127
    e = torch.where((pos[:, :1] < first[i, None]), torch.maximum(e, before), e)
    # exact: a float32 holds every code, and a power of two changes its exponent alone
    old = _decode(_codes(state, which, p, t), store) * _pow2(before - e)[:, None, :, None]
    both = _encode(torch.where(fresh[..., None, None], x * _pow2(-e)[:, None, :, None], old), store)
    _put(state, which, p[here], t[here], both[here])
    state[which + "_exp"][p[:, 0], :, t[:, 0] // block] = (e + 127).to(torch.uint8)


def _plain_keep(state, which):
    """Blocks of the kept tokens' new places: a block's exponent is the largest of its own and of those that tokens
    come from, and all of its tokens go by it."""
    c = state["case"]
    block, store, page = c["block"], c["store"], c["page"]
    q_start, kv_len = state["q_start"].long(), state["kv_len"].long()
    first, n_keep = kv_len - (q_start[1:] - q_start[:-1]), state["n_keep"].long()
    touched = (state["max_q"] + block - 2) // block + 1
    pos = (first[:, None] // block + torch.arange(touched, device=DEV))[..., None] * block + torch.arange(block, device=DEV)
    j = pos - first[:, None, None]
    moves = (j >= 0) & (j < n_keep[:, None, None])
    row = state["keep"].long().gather(1, j.clamp(0, state["max_q"] - 1).flatten(1)).view(j.shape)
    src = torch.where(moves, first[:, None, None] + row, pos)
    moves &= src != pos
    i, b = (pos[..., 0] < (first + n_keep)[:, None]).nonzero(as_tuple=True)
    pos, src, moves = pos[i, b], src[i, b], moves[i, b]
    here = pos < kv_len[i, None]
    p, t = _slots(state["pages"][i], pos, page)
    ps, ts = _slots(state["pages"][i], torch.where(here, src, pos), page)
    exps = state[which + "_exp"]
    from_e = exps[ps, :, ts // block].int() - 127  # [blocks][block][heads]
    own_e = exps[p[:, 0], :, t[:, 0] // block].int() - 127
    e = torch.maximum(own_e, torch.where(moves[..., None], from_e, own_e[:, None]).amax(1))
    codes = _encode(_decode(_codes(state, which, ps, ts), store) * _pow2(from_e - e[:, None])[..., None], store)
    _put(state, which, p[here], t[here], codes[here])
    exps[p[:, 0], :, t[:, 0] // block] = (e + 127).to(torch.uint8)


def _plain_read(state, which, out):
    row, pos, there = _rows(state["back_start"], state["back_len"], state["max_back"])
    i, j = there.nonzero(as_tuple=True)
    p, t = _slots(state["pages"][i], pos[i, j][:, None], state["case"]["page"])
    top = torch.finfo(out.dtype).max
    out[row[i, j]] = _values(state, which, p[:, 0], t[:, 0]).clamp(-top, top).to(out.dtype)


def _plain_tree(state):
    c = state["case"]
    heads, group, dim, width = c["heads"], c["q_heads"] // c["heads"], c["dim"], state["max_q"]
    row, pos, there = _rows(state["q_start"], state["kv_len"], width)
    seqs, kv_len, first = len(row), state["kv_len"].long()[:, None], pos[:, :1]
    row = row.clamp(max=len(state["q"]) - 1)
    # with a window from the first token that some row can see on
    span = min(state["max_len"], c["window"] + width - 1) if c["window"] else state["max_len"]
    key = torch.arange(span, device=DEV) + ((kv_len - span).clamp(min=0) if c["window"] else torch.zeros_like(kv_len))
    p, t = _slots(state["pages"], key, c["page"])
    k, v = (_values(state, w, p, t).permute(0, 2, 1, 3).contiguous() for w in "kv")  # [seqs][heads][keys][dim]
    q = state["q"][row].float().view(seqs, width, heads, group, dim).permute(0, 2, 3, 1, 4)
    s = torch.matmul(q.reshape(seqs, heads, group * width, dim), k.transpose(2, 3)) * (1.0 / math.sqrt(dim))
    s = s.view(seqs, heads, group, width, -1)
    node = (key - first).clamp(0, 32 * state["mask"].shape[1] - 1)
    bits = state["mask"][row].gather(2, (node // 32)[:, None].expand(-1, width, -1)) >> (node % 32)[:, None]
    sees = (key < first)[:, None].expand(-1, width, -1)
    if c["window"]:
        sees = sees & (key[:, None] > state["pos"].long()[row][..., None] - c["window"])
    sees = sees | ((key >= first) & (key < kv_len))[:, None] & (bits & 1).bool()
    s = torch.where(sees[:, None, None], s, -math.inf)
    v = torch.where((key < kv_len)[:, None, :, None], v, 0.0)
    sink = torch.full((1, heads, group, 1, 1), -math.inf, device=DEV)
    if state["sinks"] is not None:
        sink = state["sinks"].view(1, heads, group, 1, 1)
    m = torch.maximum(s.amax(-1, keepdim=True), sink)
    m = torch.where(torch.isinf(m), 0.0, m)
    w = torch.exp(s - m)
    total = w.sum(-1, keepdim=True) + torch.exp(sink - m)
    o = torch.matmul(w.view(seqs, heads, group * width, -1), v).view(seqs, heads, group, width, dim)
    o = torch.where(total > 0, o / total, 0.0)
    lse = (torch.log(total) + m)[..., 0]
    i, j = there.nonzero(as_tuple=True)
    o = o.permute(0, 3, 1, 2, 4).reshape(seqs, width, heads * group, dim)
    state["out"][row[i, j]] = o[i, j].to(state["out"].dtype)
    state["lse"][row[i, j]] = lse.permute(0, 3, 1, 2).reshape(seqs, width, heads * group)[i, j]


def _plain_verify(state):
    """In 64 bits: acceptances and draws lie next to borders. All sequences a row at a time: a row continues only
    rows before it, so one pass in order takes every step of the way."""
    p, u, token, q = state["p"], state["u"].double(), state["token"].long(), state["q"]
    start = state["start"].long()
    n, seqs = start[1:] - start[:-1], torch.arange(len(start) - 1, device=DEV)
    at, left, mass = torch.zeros_like(n), p[start[:-1]].double(), torch.ones(len(n), dtype=torch.float64, device=DEV)
    keep, out = torch.full_like(state["keep"], -1), torch.full_like(state["out"], -1)
    keep[:, 0] = 0
    count = torch.ones_like(n)
    for j in range(1, state["max_q"]):
        row = (start[:-1] + j).clamp(max=len(p) - 1)
        tries, tok = (j < n) & (state["parent"].long()[row] == at), token[row]
        has = torch.zeros_like(tries)
        if q is not None:
            which = row if state["q_index"] is None else state["q_index"].long()[row]
            has, which = which >= 0, which.clamp(min=0)
        drawn = torch.where(has, q[which, tok].double(), 1.0) if q is not None else 1.0
        there = left[seqs, tok]
        taken = tries & (u[row] * mass * drawn < there)
        turned_down = tries & ~taken
        if q is not None:
            rest = (left - mass[:, None] * q[which].double()).clamp(min=0.0)
            left = torch.where((turned_down & has)[:, None], rest, left)
        outright = turned_down & ~has
        left[seqs, tok] = torch.where(outright, 0.0, left[seqs, tok])
        mass = torch.where(outright, mass - there, torch.where(turned_down, left.sum(1), mass))
        left = torch.where(taken[:, None], p[row].double(), left)
        mass = torch.where(taken, 1.0, mass)
        at = torch.where(taken, j, at)
        last = (seqs, (count - 1).clamp(max=state["max_q"] - 1))
        out[last] = torch.where(taken, tok, out[last].long()).int()
        nxt = (seqs, count.clamp(max=state["max_q"] - 1))
        keep[nxt] = torch.where(taken, j, keep[nxt].long()).int()
        count = count + taken
    up = left.cumsum(1)
    aim = u[start[:-1]][:, None] * up[:, -1:]
    drawn = (up <= aim).sum(1).clamp(max=p.shape[1] - 1)
    drawn = torch.where(up[:, -1] > 0, drawn, p[start[:-1] + at].argmax(1))
    out[seqs, count - 1] = drawn.int()
    state["keep"].copy_(keep)
    state["out"].copy_(out)
    state["n_keep"].copy_(count)


def _plain(state):
    c = state["case"]
    kind = c["kind"]
    if kind == "rope":
        state["y"] = _turned(state["x"], state["pos"], state["freqs"], c)
        if c["grad"]:
            state["dx"] = _turned(state["dy"], state["pos"], state["freqs"], c, -1.0)
    elif kind == "tree":
        _plain_tree(state)
    elif kind == "verify":
        _plain_verify(state)
    else:
        if kind == "append":
            pos = state["pos"]
            if pos is None:
                row, at, there = _rows(state["q_start"], state["kv_len"], state["max_q"])
                pos = torch.empty(len(state["q"]), dtype=torch.int64, device=DEV)
                pos[row[there]] = at[there]
            state["out"] = _turned(state["q"], pos, state["freqs"], c)
            _plain_write(state, "k", _turned(state["new_k"], pos, state["freqs"], c))
            _plain_write(state, "v", state["new_v"])
        else:
            _plain_keep(state, "k")
            _plain_keep(state, "v")
        _plain_read(state, "k", state["out_k"])
        _plain_read(state, "v", state["out_v"])


# ---- the framework's calls

def _handles(state):
    """What a program keeps: the rotation, the cache's handle, the step's batch and tree, the workspace."""
    from kernels_amd import kq
    c = state["case"]
    if c["kind"] in ("rope", "append"):
        state["rope"] = kq.Rope(state["freqs"], pairs=c["pairs"], amplitude=c["amplitude"])
        state["back_rope"] = kq.Rope(state["freqs"], pairs=c["pairs"], amplitude=c["amplitude"], inverse=True)
    if c["kind"] == "verify":
        n = kq.draft_verify_workspace_size(c["seqs"], state["max_q"], c["vocab"])
        state["ws"], state["ws_bytes"] = torch.empty(n, dtype=torch.uint8, device=DEV), n
    elif c["kind"] != "rope":
        state["cache"] = kq.KVCache(state["k"], state["v"], state["k_exp"], state["v_exp"])
        state["batch"] = kq.KVBatch(state["pages"], state["kv_len"], state["max_len"], q_start=state["q_start"],
                                    max_q=state["max_q"])
    if "back_start" in state:
        state["back"] = kq.KVBatch(state["pages"], state["back_len"], state["max_len"], q_start=state["back_start"],
                                   max_q=state["max_back"])
    if c["kind"] == "tree":
        state["nodes"] = kq.KVTree(state["mask"], state["pos"])
        n = kq.kv_attn_tree_workspace_size(state["cache"], state["batch"], c["q_heads"])
        state["ws"], state["ws_bytes"] = torch.empty(n, dtype=torch.uint8, device=DEV), n
    state["kq"] = kq


def _own(state):
    if "kq" not in state:
        _handles(state)
    kq, c = state["kq"], state["case"]
    kind = c["kind"]
    if kind == "rope":
        kq.rope(state["x"], state["y"], state["pos"], state["rope"])
        if c["grad"]:
            kq.rope(state["dy"], state["dx"], state["pos"], state["back_rope"])
    elif kind == "tree":
        kq.kv_attn_tree(state["cache"], state["batch"], state["nodes"], state["q"], state["out"], state["ws"],
                        state["ws_bytes"], window=c["window"], sinks=state["sinks"], lse=state["lse"])
    elif kind == "verify":
        kq.draft_verify(state["p"], state["token"], state["u"], state["keep"], state["n_keep"], state["out"], state["ws"],
                        state["ws_bytes"], q=state["q"], q_index=state["q_index"],
                        parent=state["parent"] if c["tree"] else None, start=state["start"])
    elif kind == "append":
        kq.kv_write_rope(state["cache"], state["batch"], state["rope"], state["new_k"], state["new_v"], q=state["q"],
                         q_out=state["out"], pos=state["pos"])
        kq.kv_read(state["cache"], state["back"], state["out_k"], state["out_v"])
    else:
        kq.kv_keep(state["cache"], state["batch"], state["keep"], state["n_keep"])
        kq.kv_read(state["cache"], state["back"], state["out_k"], state["out_v"])


def run(state):
    if own:
        _own(state)
    else:
        _plain(state)
    kind = state["case"]["kind"]
    if kind == "rope":
        return {"y": state["y"], "dx": state["dx"]} if state["case"]["grad"] else {"y": state["y"]}
    if kind == "tree":
        return {"out": state["out"], "lse": state["lse"]}
    if kind == "verify":
        return {"keep": state["keep"], "n_keep": state["n_keep"], "out": state["out"]}
    got = {"k": state["out_k"], "v": state["out_v"], "k_exp": state["k_exp"], "v_exp": state["v_exp"]}
    return got | {"q": state["out"]} if kind == "append" else got


# ---------------------------------------------------------------------------

def work(case):
    kind = case["kind"]
    if kind == "rope":
        n = case["rows"] * case["heads"] * case["dim"] * (2.0 if case["grad"] else 1.0)
        return {"bytes": 2 * n * (4 if case["dtype"] == "f32" else 2), "flops": 3.0 * n * case["rot"] / case["dim"]}
    if kind == "verify":
        # the rows that the last token is drawn from, and a few numbers for each drafted one
        n = case["seqs"] * case["vocab"] * (1.0 if case["draft"] == "none" else 2.0)
        return {"bytes": 4 * n + 24 * sum(_news(case)), "flops": 2 * n}
    lengths, wide = _lengths(case), case["heads"] * case["dim"]
    rows = sum(m for _, m in lengths)
    if kind == "append":
        new = 2.0 * wide * rows
        old = 2.0 * wide * sum((n - m) % case["block"] for n, m in lengths)
        turned = 4.0 * rows * case["q_heads"] * case["dim"]
        # the new values and the blocks' older codes in, the new codes and the values read back out; the queries
        return {"bytes": new * 3 + old + (new + old) * 2 + turned, "flops": 4.0 * (new + old) + 3 * turned / 4}
    if kind == "keep":
        kept = _kept(case, [m for _, m in lengths])
        moved = 2.0 * wide * sum(r != j for rs in kept for j, r in enumerate(rs))
        back = 2.0 * wide * sum((n - m) % case["block"] + len(r) for (n, m), r in zip(lengths, kept))
        return {"bytes": 2 * moved + 3 * back, "flops": 2 * back}
    codes = pairs = 0.0
    for (n, m), ps in zip(lengths, _parents(case, [m for _, m in lengths])):
        codes += min(n, case["window"] + m - 1) if case["window"] else n
        before = [min(n - m, max(0, case["window"] - d - 1)) if case["window"] else n - m for d in _depths(ps)]
        pairs += sum(before) + sum(d + 1 for d in _depths(ps))
    return {"bytes": codes * 2 * wide + rows * case["q_heads"] * (4 * case["dim"] + 4),
            "flops": 4.0 * pairs * case["q_heads"] * case["dim"]}


# ---- the same from the definition, in 64 bits

def _pow2_64(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


def _turned64(x, pos, freqs, case, sign=1.0):
    """By complex numbers: (a + ib) e^(i angle) amplitude; float64."""
    rot, x = case["rot"], x.double()
    angle = torch.outer(pos.double(), freqs.double()) * sign
    by = torch.polar(torch.full_like(angle, case["amplitude"]), angle)[:, None]
    part = x[..., :rot]
    if case["pairs"]:
        z = torch.view_as_complex(part.reshape(*part.shape[:-1], rot // 2, 2).contiguous()) * by
        z = torch.view_as_real(z).flatten(-2)
    else:
        z = torch.complex(part[..., :rot // 2].contiguous(), part[..., rot // 2:].contiguous()) * by
        z = torch.cat([z.real, z.imag], -1)
    return torch.cat([z, x[..., rot:]], -1)


def _tokens64(state, which, i, n):
    """The first n tokens of sequence i: float64 [n][heads][dim]."""
    c = state["case"]
    ids = state["pages"][i, :-(-n // c["page"])].long()
    codes = state[which][ids]
    if which == "v":
        codes = codes.view(torch.int8).transpose(3, 4).reshape(len(ids), c["heads"], c["page"], c["dim"])
        codes = codes.view(state[which].dtype)
    scale = _pow2_64(state[which + "_exp"][ids].long() - 127)
    x = codes.double() * scale.repeat_interleave(c["block"], 2)[..., None]
    return x.transpose(1, 2).reshape(-1, c["heads"], c["dim"])[:n]


def _round64(x, store):
    """The nearest codes' values, half to even: int8, or e4m3's 4 significant bits down to multiples of 2^-9."""
    step = 1.0 if store == "i8" else _pow2_64((torch.frexp(x).exponent - 4).clamp(min=-9))
    return ((x / step).round() * step).clamp(-LARGEST[store], LARGEST[store])


def _scale64(a, store):
    """e, from the quotient's logarithm, put right by one where that was rounded."""
    big = LARGEST[store]
    e = torch.log2(a.clamp(min=1e-300) / big).ceil().clamp(LOWEST, HIGHEST[store]).long()
    e = e + ((a > big * _pow2_64(e)) & (e < HIGHEST[store])).long()
    return e - ((a <= big * _pow2_64(e - 1)) & (e > LOWEST)).long()


def _exact_blocks(state, which, i, n, first, end, place):
    """Tokens from first's block to `end` (float64 [tokens][heads][dim]) of sequence i of n tokens, where
    place(tokens [n][heads][dim], block's first token, its exponents) gives a block's new values and exponents; the
    exponents go into the state."""
    c = state["case"]
    block, was, got = c["block"], _tokens64(state, which, i, n), []
    new = []
    for t0 in range(first // block * block, end, block):
        page, s = state["pages"][i, t0 // c["page"]].long(), t0 % c["page"] // block
        e = state[which + "_exp"][page, :, s].long() - 127
        x, e = place(was, t0, e)
        new.append((page, s, e))
        scale = _pow2_64(e)[:, None]
        got.append(_round64(x / scale, c["store"]) * scale)
    for page, s, e in new:
        state[which + "_exp"][page, :, s] = (e + 127).to(torch.uint8)
    return torch.cat(got)[:end - first // block * block]


def _exact_write(state, which, new, i, n, first):
    c = state["case"]
    block = c["block"]

    def place(was, t0, e):
        t1, old = min(t0 + block, n), max(first - t0, 0)
        fresh = new[max(t0, first) - first:t1 - first]
        wanted = _scale64(fresh.abs().amax((0, 2)), c["store"])
        return torch.cat([was[t0:t0 + old], fresh]), torch.maximum(wanted, e) if old else wanted

    return _exact_blocks(state, which, i, n, first, n, place)


def _exact_keep(state, which, i, n, first, kept):
    c = state["case"]
    block = c["block"]
    before = state[which + "_exp"].clone()

    def place(was, t0, e):
        src = [first + kept[t - first] if first <= t < first + len(kept) else t for t in range(t0, min(t0 + block, n))]
        for t, s in zip(range(t0, t0 + block), src):
            if s != t:
                e = torch.maximum(e, before[state["pages"][i, s // c["page"]].long(), :, s % c["page"] // block].long() - 127)
        return was[torch.tensor(src, device=DEV)], e

    return _exact_blocks(state, which, i, n, first, first + len(kept), place)


def _exact_verify(state):
    case = state["case"]
    news, starts = _news(case), state["start"].tolist()
    parents = _parents(case, news)
    got = {k: torch.full_like(state[k], -1) for k in ("keep", "n_keep", "out")}
    token, index = state["token"].tolist(), None if state["q_index"] is None else state["q_index"].tolist()
    for i, (m, r0) in enumerate(zip(news, starts)):
        at, path, toks = 0, [0], []
        while True:
            left, mass, went = state["p"][r0 + at].double(), 1.0, -1
            for j in [j for j in range(1, m) if parents[i][j] == at]:
                tok, r = token[r0 + j], r0 + j
                f = r if index is None else index[r]
                draft = state["q"][f].double() if state["q"] is not None and f >= 0 else None
                prob = 1.0 if draft is None else float(draft[tok])
                if float(state["u"][r]) * mass * prob < float(left[tok]):
                    went = j
                    break
                if draft is None:
                    mass -= float(left[tok])
                    left[tok] = 0.0
                else:
                    left = torch.relu(left - mass * draft)
                    mass = float(left.sum())
            if went < 0:
                break
            at = went
            path.append(went)
            toks.append(token[r0 + went])
        up = torch.cumsum(left, 0)
        hit = (up > float(state["u"][r0]) * float(up[-1])).nonzero()
        toks.append(int(hit[0]) if len(hit) else int(state["p"][r0 + at].argmax()))
        got["keep"][i, :len(path)], got["out"][i, :len(toks)] = _ints(path), _ints(toks)
        got["n_keep"][i] = len(path)
    return got


def exact(case, seed):
    state, kind = prepare(case, seed), case["kind"]
    if kind == "rope":
        got = {"y": _turned64(state["x"], state["pos"], state["freqs"], case)}
        return got | {"dx": _turned64(state["dy"], state["pos"], state["freqs"], case, -1.0)} if case["grad"] else got
    if kind == "verify":
        return _exact_verify(state)
    lengths = _lengths(case)
    starts = _starts([m for _, m in lengths])
    if kind in ("append", "keep"):
        got = {}
        if kind == "append":
            pos = state["pos"]
            if pos is None:
                pos = torch.cat([torch.arange(n - m, n, device=DEV) for n, m in lengths])
            got["q"] = _turned64(state["q"], pos, state["freqs"], case)
            # the cache takes keys as a rotation of their own leaves them: of their type
            k = _turned64(state["new_k"], pos, state["freqs"], case).float().to(FLOAT[case["dtype"]]).double()
            new = {"k": k, "v": state["new_v"].double()}
        kept = _kept(case, [m for _, m in lengths])
        for w in "kv":
            parts = []
            for i, (n, m) in enumerate(lengths):
                if kind == "append":
                    parts.append(_exact_write(state, w, new[w][starts[i]:starts[i + 1]], i, n, n - m))
                else:
                    parts.append(_exact_keep(state, w, i, n, n - m, kept[i]))
            got[w] = torch.cat(parts)
        return got | {"k_exp": state["k_exp"], "v_exp": state["v_exp"]}
    group, dim = case["q_heads"] // case["heads"], case["dim"]
    out = torch.zeros_like(state["out"], dtype=torch.float64)
    lse = torch.full_like(state["lse"], -math.inf, dtype=torch.float64)
    none = torch.full((case["q_heads"],), -math.inf, dtype=torch.float64, device=DEV)
    sinks = state["sinks"].double() if state["sinks"] is not None else none
    for i, ((n, m), ps) in enumerate(zip(lengths, _parents(case, [m for _, m in lengths]))):
        first, up = n - m, [[] for _ in ps]
        for j, p in enumerate(ps):
            up[j] = (up[p] if p >= 0 else []) + [j]
        sees = torch.zeros((m, n), dtype=torch.bool)
        for j, line in enumerate(up):
            lo = max(0, first + len(line) - case["window"]) if case["window"] else 0
            sees[j, lo:first] = True
            sees[j, [first + a for a in line]] = True
        sees = sees.to(DEV)
        k, v = (_tokens64(state, w, i, n) for w in "kv")
        for h in range(case["q_heads"]):
            kh, vh = k[:, h // group], v[:, h // group]
            s = (state["q"][starts[i]:starts[i + 1], h].double() @ kh.t().contiguous()) / math.sqrt(dim)
            s = torch.cat([torch.where(sees, s, -math.inf), sinks[h].expand(m, 1)], 1)
            total = torch.logsumexp(s, 1)
            lse[starts[i]:starts[i + 1], h] = total
            w = torch.exp(s[:, :-1] - total[:, None])
            out[starts[i]:starts[i + 1], h] = torch.where(torch.isfinite(total)[:, None], w @ vh.contiguous(), 0.0)
    return {"out": out, "lse": lse}
