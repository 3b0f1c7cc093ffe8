"""The 8-bit key/value cache and the attention that reads it, as cases to be timed and compared.

Kinds of case (the "kind" of the dict):

  write  the new keys and values of a step into the cache (kv_write), and the
         blocks that it touched read back (kv_read)
  read   whole sequences out of the cache (kv_read), as for moving them to
         another server or a plain attention
  attn   attention of the newest tokens over their sequences (kv_attn): one
         token each in decode, a few in speculative decoding, many in prefill

The cache is paged. A page holds `page` tokens of every head:

  k      [pages][heads][page][dim]          8-bit codes (int8 or e4m3)
  v      [pages][heads][page/16][dim][16]   the same, 16 tokens of a column together
  k_exp, v_exp  uint8 [pages][heads][page/block]: a code c of block b stands
         for c * 2^(exp - 127)

The sequences of a case have lengths of their own, spread over a range, and
their pages lie anywhere in the pool. The newest tokens' q, k and v are slices
of one projection's output, as a fused q/k/v projection leaves them.
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


def _case(name, kind, seqs, lens, new, q_heads, heads, dim, store, dtype, page=16, block=16, causal=True,
          window=0, sinks=False, empty=False):
    """lens, new: the shortest and longest length, and number of newest tokens, of a sequence."""
    return {"name": name, "kind": kind, "seqs": seqs, "len_lo": lens[0], "len_hi": lens[1],
            "new_lo": new[0], "new_hi": new[1], "q_heads": q_heads, "heads": heads, "dim": dim, "store": store,
            "dtype": dtype, "page": page, "block": block, "causal": causal, "window": window,
            "sinks": sinks, "empty": empty}


def listed():
    return [
        # the smallest call: one sequence's new token (Llama-3-8B heads) into
        # a block that other tokens began
        _case("write_b1", "write", 1, (777, 777), (1, 1), 32, 8, 128, "i8", "f16"),
        # a decode step of many sequences, 70B-class heads, larger pages
        _case("write_b96", "write", 96, (40, 8191), (1, 1), 64, 8, 128, "e4m3", "bf16", page=64, block=32),
        # prefill of a few prompts of odd lengths, some behind a cached prefix
        _case("write_prefill", "write", 5, (1201, 9001), (1201, 5003), 32, 8, 128, "i8", "bf16"),
        # a batch's sequences out of the cache, for a move to another server
        _case("read_b24", "read", 24, (7, 6007), (1, 1), 64, 8, 64, "i8", "bf16", page=32, block=32),
        # one long sequence
        _case("read_long", "read", 1, (131072, 131072), (1, 1), 32, 8, 128, "e4m3", "f16", page=64, block=64),
        # one short sequence, one token: latency
        _case("attn_b1_short", "attn", 1, (113, 113), (1, 1), 32, 8, 128, "i8", "f16"),
        # one token over a long context, 70B-class heads
        _case("attn_b1_long", "attn", 1, (131071, 131071), (1, 1), 64, 8, 128, "e4m3", "bf16"),
        # the decode step of a busy server: many sequences of very different lengths
        _case("attn_b64", "attn", 64, (100, 12000), (1, 1), 32, 8, 128, "i8", "f16"),
        # gpt-oss heads: 64 wide, 128-token window and a sink for each head
        _case("attn_window_sinks", "attn", 48, (50, 30000), (1, 1), 64, 8, 64, "i8", "bf16", page=32, block=32,
              window=128, sinks=True),
        # speculative decoding: up to five proposed tokens a sequence
        _case("attn_draft", "attn", 12, (500, 8000), (3, 5), 64, 8, 128, "e4m3", "f16", page=64),
        # a prompt's chunk behind what is already cached
        _case("attn_chunk", "attn", 1, (16384, 16384), (2048, 2048), 32, 8, 128, "i8", "bf16"),
        # prefill of several prompts of odd lengths, gpt-oss heads with sinks
        _case("attn_prefill", "attn", 4, (331, 3001), (331, 3001), 64, 8, 64, "e4m3", "f16", page=128, block=64,
              sinks=True),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["write", "read", "attn", "attn", "attn"])
    heads = rng.choice([1, 2, 4, 8, 8, 8, 16])
    group = rng.choice([1, 2, 3, 4, 4, 5, 7, 8, 8, 16])
    dim = rng.choice([64, 64, 96, 128, 128, 128, 192, 256])
    block = rng.choice([16, 16, 32, 64])
    page = block * rng.choice([1, 1, 2, 4])
    store, dtype = rng.choice(["i8", "e4m3"]), rng.choice(["f16", "bf16"])
    seqs = _log_int(rng, 1, 96)
    # tokens in all: what the largest listed cases read
    room = 2**27 // (heads * dim)
    hi = max(1, min(_log_int(rng, 16, 131072), room // seqs))
    lo = _log_int(rng, 1, hi)
    new = (1, 1)
    causal, window, sinks = True, 0, False
    if kind == "write":
        if rng.random() < 0.5:
            new = (1, _log_int(rng, 1, min(hi, 8192)))
            seqs = max(1, min(seqs, 2**23 // (heads * dim * new[1])))
    elif kind == "read":
        if rng.random() < 0.2:
            dtype, seqs = "f32", (seqs + 1) // 2
    else:
        form = rng.choice(["decode", "decode", "few", "chunk"])
        if form == "few":
            new = (1, min(hi, rng.randint(2, 8)))
        elif form == "chunk":
            hi = min(hi, 16384)
            lo = min(lo, hi)
            new = (1, min(hi, _log_int(rng, 9, 2048)))
            # products in all
            group = max(1, min(group, 2**36 // (new[1] * hi * heads * dim)))
            seqs = max(1, min(seqs, 2**36 // (new[1] * hi * heads * group * dim)))
        window = rng.choice([0, 0, _log_int(rng, 1, 4096)])
        sinks = rng.random() < 0.3
        causal = window > 0 or rng.random() < 0.85
    c = _case("", kind, seqs, (lo, hi), new, heads * group, heads, dim, store, dtype, page, block, causal, window,
              sinks, kind == "attn" and rng.random() < 0.15)
    del c["name"]
    return c


# ---------------------------------------------------------------------------

def _spread(lo, hi, i, by):
    """The i-th of numbers spread over lo..hi by their logarithm; the first is hi."""
    return lo if lo >= hi else int(round(lo * (hi / lo) ** ((1.0 - i * by) % 1.0 or 1.0)))


def _lengths(case):
    """(tokens, newest tokens) of each sequence."""
    got = []
    for i in range(case["seqs"]):
        n = _spread(case["len_lo"], case["len_hi"], i, 0.6180339887)
        if case["empty"] and i % 5 == 1:
            n = 0
        new = _spread(case["new_lo"], case["new_hi"], i, 0.7548776662)
        got.append((n, min(n, new) if case["kind"] != "attn" or n else new))
    return got


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
    x = torch.nan_to_num(x, nan=0.0, posinf=LARGEST[store], neginf=-LARGEST[store])
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


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device=DEV)


def _starts(counts):
    at = [0]
    for n in counts:
        at.append(at[-1] + n)
    return at


def prepare(case, seed):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed)
    lengths = _lengths(case)
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
            in_cache[p] = max(0, min(page, n - (new if case["kind"] == "write" else 0) - j * page))
    seen = torch.arange(page, device=DEV) < _ints(in_cache)[:, None]
    (k, k_exp), (v, v_exp) = _fill(n_pages, case, g, seen), _fill(n_pages, case, g, seen)
    code = torch.int8 if case["store"] == "i8" else torch.float8_e4m3fn
    state = {"case": dict(case), "k": k.view(code), "v": _columns(v).view(code), "k_exp": k_exp, "v_exp": v_exp,
             "pages": _ints(table), "kv_len": _ints([n for n, _ in lengths]), "max_len": max(n for n, _ in lengths)}
    new = [n for n, _ in lengths] if case["kind"] == "read" else [n for _, n in lengths]
    state["q_start"], state["max_q"], rows = _ints(_starts(new)), max(max(new), 1), sum(new)
    dtype = FLOAT[case["dtype"]]
    if case["kind"] != "read":
        # one row of a fused projection: q of every head, then k, then v
        x = torch.empty((rows, q_heads + 2 * heads, dim), device=DEV).normal_(generator=g)
        x *= torch.empty((rows, q_heads + 2 * heads, 1), device=DEV).normal_(0.0, 0.5, generator=g).exp()
        x = x.to(dtype)
        state["q"], state["new_k"], state["new_v"] = x[:, :q_heads], x[:, q_heads:q_heads + heads], x[:, q_heads + heads:]
    if case["kind"] == "write":
        # the touched blocks, from their first token on
        back = [n - (n - m) // case["block"] * case["block"] for n, m in lengths]
        state["back_start"], state["max_back"], rows = _ints(_starts(back)), max(back), sum(back)
    if case["kind"] == "attn":
        state["out"] = torch.zeros((rows, q_heads, dim), dtype=dtype, device=DEV)
        state["lse"] = torch.zeros((rows, q_heads), dtype=torch.float32, device=DEV)
        state["sinks"] = torch.empty(q_heads, device=DEV).normal_(0.0, 2.0, generator=g) if case["sinks"] else None
    else:
        state["out_k"], state["out_v"] = (torch.zeros((rows, heads, dim), dtype=dtype, device=DEV) for _ in "kv")
    return state


# ---- the plain forms

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


def _values(state, which, p, t):
    """float32 values [...][heads][dim] of the cache's tokens (p, t)."""
    c = state["case"]
    codes = state[which].view(torch.int8)
    codes = codes[p, :, t] if which == "k" else codes[p, :, t // 16, :, t % 16]
    e = state[which + "_exp"][p, :, t // c["block"]].int() - 127
    return _decode(codes, c["store"]) * _pow2(e)[..., None]


def _plain_write(state, which, new):
    c = state["case"]
    block, store = c["block"], c["store"]
    q_start, kv_len = state["q_start"].long(), state["kv_len"].long()
    n = q_start[1:] - q_start[:-1]
    first = kv_len - n
    touched = (state["max_q"] + block - 2) // block + 1
    b = first[:, None] // block + torch.arange(touched, device=DEV)  # [seqs][touched]
    pos = b[..., None] * block + torch.arange(block, device=DEV)
    pos = pos.masked_fill((n == 0)[:, None, None], 2**40)
    here = pos < kv_len[:, None, None]
    fresh = here & (pos >= first[:, None, None])
    i, j = here[..., 0].nonzero(as_tuple=True)  # the blocks that there are
    pos, here, fresh = pos[i, j], here[i, j], fresh[i, j]
    row = (q_start[i, None] + pos - first[i, None]).clamp(0, len(new) - 1)
    x = new[row].float() * fresh[..., None, None]  # [blocks][block][heads][dim]
    x = torch.where(fresh[..., None, None], x, 0.0)
    a = torch.where(torch.isfinite(x), x, 0.0).abs().amax((1, 3))
    e = _exponent(a, store)
    p, t = _slots(state["pages"][i], pos, c["page"])
    exps = state[which + "_exp"]
    before = exps[p[:, 0], :, t[:, 0] // block].int() - 127
    e = torch.where((pos[:, :1] < first[i, None]), torch.maximum(e, before), e)
    codes = state[which].view(torch.int8)
    old = codes[p, :, t] if which == "k" else codes[p, :, t // 16, :, t % 16]
    # exact: a float32 holds every code, and a power of two changes its exponent alone
    old = _decode(old, store) * _pow2(before - e)[:, None, :, None]
    both = torch.where(fresh[..., None, None], x * _pow2(-e)[:, None, :, None], old)
    both = _encode(both, store)[here]
    p, t = p[here], t[here]
    if which == "k":
        codes[p, :, t] = both
    else:
        codes[p, :, t // 16, :, t % 16] = both
    exps[state["pages"].long()[i, pos[:, 0] // c["page"]], :, pos[:, 0] % c["page"] // block] = (e + 127).to(torch.uint8)


def _plain_read(state, which, start, width, out):
    row, pos, there = _rows(start, state["kv_len"], width)
    i, j = there.nonzero(as_tuple=True)
    p, t = _slots(state["pages"][i], pos[i, j][:, None], state["case"]["page"])
    top = torch.finfo(out.dtype).max
    out[row[i, j]] = _values(state, which, p[:, 0], t[:, 0]).clamp(-top, top).to(out.dtype)


def _plain_attn(state):
    c = state["case"]
    heads, group, dim, width = c["heads"], c["q_heads"] // c["heads"], c["dim"], state["max_q"]
    row, pos, there = _rows(state["q_start"], state["kv_len"], width)
    seqs = len(row)
    at = torch.arange(state["max_len"], device=DEV)
    lo = 0
    if c["window"]:
        # the keys that some row can see, counted from the first of them
        span = min(state["max_len"], c["window"] + width - 1)
        lo = (state["kv_len"].long() - span).clamp(min=0)[:, None]
        at = at[:span]
    key = (at + lo).expand(seqs, -1)
    p, t = _slots(state["pages"], key, c["page"])
    k, v = (_values(state, w, p, t).permute(0, 2, 1, 3).contiguous() for w in "kv")  # [seqs][heads][keys][dim]
    q = state["q"][row.clamp(max=len(state["q"]) - 1)].float()  # [seqs][width][q_heads][dim]
    q = q.view(seqs, width, heads, group, dim).permute(0, 2, 3, 1, 4).reshape(seqs, heads, group * width, dim)
    s = torch.matmul(q, k.transpose(2, 3)) * (1.0 / math.sqrt(dim))
    s = s.view(seqs, heads, group, width, -1)
    sees = (key[:, None] < state["kv_len"].long()[:, None, None]) & there[..., None]
    if c["causal"]:
        sees = sees & (key[:, None] <= pos[..., None])
    if c["window"]:
        sees = sees & (key[:, None] > pos[..., None] - c["window"])
    sees = sees[:, None, None]
    s = torch.where(sees, s, -math.inf)
    v = torch.where((key < state["kv_len"].long()[:, None])[:, None, :, None], v, 0.0)
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


# ---- the framework's calls

def _handles(state):
    """What a serving program keeps: the cache's handle, the step's batch and the workspace."""
    from kernels_amd import kq
    cache = kq.KVCache(state["k"], state["v"], state["k_exp"], state["v_exp"])
    state["cache"] = cache
    state["batch"] = kq.KVBatch(state["pages"], state["kv_len"], state["max_len"], q_start=state["q_start"],
                                max_q=state["max_q"])
    if state["case"]["kind"] == "write":
        state["back"] = kq.KVBatch(state["pages"], state["kv_len"], state["max_len"], q_start=state["back_start"],
                                   max_q=state["max_back"])
    if state["case"]["kind"] == "attn":
        n = kq.kv_attn_workspace_size(cache, state["batch"], state["case"]["q_heads"])
        state["ws"], state["ws_bytes"] = torch.empty(n, dtype=torch.uint8, device=DEV), n
    state["kq"] = kq


def _own(state):
    if "kq" not in state:
        _handles(state)
    kq, c = state["kq"], state["case"]
    if c["kind"] == "write":
        kq.kv_write(state["cache"], state["batch"], state["new_k"], state["new_v"])
        kq.kv_read(state["cache"], state["back"], state["out_k"], state["out_v"])
    elif c["kind"] == "read":
        kq.kv_read(state["cache"], state["batch"], state["out_k"], state["out_v"])
    else:
        kq.kv_attn(state["cache"], state["batch"], state["q"], state["out"], state["ws"], state["ws_bytes"],
                   causal=c["causal"], window=c["window"], sinks=state["sinks"], lse=state["lse"])


def _plain(state):
    kind = state["case"]["kind"]
    if kind == "attn":
        _plain_attn(state)
        return
    start, width = state["q_start"], state["max_q"]
    if kind == "write":
        _plain_write(state, "k", state["new_k"])
        _plain_write(state, "v", state["new_v"])
        start, width = state["back_start"], state["max_back"]
    _plain_read(state, "k", start, width, state["out_k"])
    _plain_read(state, "v", start, width, state["out_v"])


def run(state):
    if own:
        _own(state)
    else:
        _plain(state)
    kind = state["case"]["kind"]
    if kind == "attn":
        return {"out": state["out"], "lse": state["lse"]}
    got = {"k": state["out_k"], "v": state["out_v"]}
    if kind == "write":
        got |= {"k_exp": state["k_exp"], "v_exp": state["v_exp"]}
    return got


# ---------------------------------------------------------------------------

def work(case):
    lengths = _lengths(case)
    wide = case["heads"] * case["dim"]
    size = 4 if case["dtype"] == "f32" else 2
    if case["kind"] == "read":
        n = 2.0 * wide * sum(n for n, _ in lengths)
        return {"bytes": n * (1 + size), "flops": n}
    if case["kind"] == "write":
        new = 2.0 * wide * sum(m for _, m in lengths)
        old = 2.0 * wide * sum((n - m) % case["block"] for n, m in lengths)
        # the new values and the blocks' older codes in, the new codes and the values read back out
        return {"bytes": new * (size + 1) + old + (new + old) * size, "flops": 4.0 * (new + old)}
    codes = pairs = rows = 0.0
    for n, m in lengths:
        rows += m
        if not n:
            continue
        most = min(n, case["window"] + m - 1) if case["window"] else n
        codes += most
        if not case["causal"]:
            pairs += m * n
        elif case["window"]:
            pairs += sum(min(case["window"], max(0, n - m + j + 1)) for j in range(m))
        else:
            pairs += m * n - m * (m - 1) / 2
    per_row = case["q_heads"] * (2 * case["dim"] * size + 4)
    return {"bytes": codes * 2 * wide + rows * per_row, "flops": 4.0 * pairs * case["q_heads"] * case["dim"]}


# ---- the same from the definition, in 64 bits

def _pow2_64(e):
    return ((e.long() + 1023) << 52).view(torch.float64)


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
    big = LARGEST[store]
    x = torch.nan_to_num(x, nan=0.0, posinf=big, neginf=-big)
    step = 1.0 if store == "i8" else _pow2_64((torch.frexp(x).exponent - 4).clamp(min=-9))
    return ((x / step).round() * step).clamp(-big, big)


def _scale64(a, store):
    """e, from the quotient's logarithm, put right by one where that was rounded."""
    big = LARGEST[store]
    e = torch.log2(a.clamp(min=1e-300) / big).ceil().clamp(LOWEST, HIGHEST[store]).long()
    e = e + ((a > big * _pow2_64(e)) & (e < HIGHEST[store])).long()
    return e - ((a <= big * _pow2_64(e - 1)) & (e > LOWEST)).long()


def _exact_write(state, which, new, i, n, first, row):
    """Sequence i's touched blocks, from the first of them: float64 [tokens][heads][dim]; the exponents go into the state."""
    c = state["case"]
    block = c["block"]
    was = _tokens64(state, which, i, n)
    b0 = first // block
    x = torch.zeros((-(-n // block) - b0) * block, c["heads"], c["dim"], dtype=torch.float64, device=DEV)
    old = x.clone()
    at = first - b0 * block
    x[at:at + n - first] = new[row:row + n - first].double()
    old[:at] = was[b0 * block:first]
    x, old = (y.view(-1, block, c["heads"], c["dim"]) for y in (x, old))
    a = torch.where(torch.isfinite(x), x, 0.0).abs().amax((1, 3))
    e = _scale64(a, c["store"])
    ids = state["pages"][i].long()
    blocks = torch.arange(b0, b0 + len(x), device=DEV)
    p, s = ids[blocks * block // c["page"]], blocks * block % c["page"] // block
    if at:
        e[0] = torch.maximum(e[0], state[which + "_exp"][p[0], :, s[0]].long() - 127)
    state[which + "_exp"][p, :, s] = (e + 127).to(torch.uint8)
    scale = _pow2_64(e)[:, None, :, None]
    fresh = (blocks[:, None] * block + torch.arange(block, device=DEV) >= first)[..., None, None]
    got = _round64(torch.where(fresh, x, old) / scale, c["store"]) * scale
    return got.view(-1, c["heads"], c["dim"])[:n - b0 * block]


def exact(case, seed):
    state = prepare(case, seed)
    lengths = _lengths(case)
    if case["kind"] == "read":
        k, v = ([_tokens64(state, w, i, n) for i, (n, _) in enumerate(lengths)] for w in "kv")
        top = torch.finfo(FLOAT[case["dtype"]]).max
        return {"k": torch.cat(k).clamp(-top, top), "v": torch.cat(v).clamp(-top, top)}
    starts = _starts([m for _, m in lengths])
    if case["kind"] == "write":
        top = torch.finfo(FLOAT[case["dtype"]]).max
        got = {}
        for w in "kv":
            parts = [_exact_write(state, w, state["new_" + w], i, n, n - m, starts[i]) for i, (n, m) in enumerate(lengths) if m]
            got[w] = torch.cat(parts).clamp(-top, top)
        return got | {"k_exp": state["k_exp"], "v_exp": state["v_exp"]}
    group, dim = case["q_heads"] // case["heads"], case["dim"]
    out = torch.zeros_like(state["out"], dtype=torch.float64)
    lse = torch.full_like(state["lse"], -math.inf, dtype=torch.float64)
    sinks = state["sinks"].double() if state["sinks"] is not None else torch.full((case["q_heads"],), -math.inf, dtype=torch.float64, device=DEV)
    for i, (n, m) in enumerate(lengths):
        if n == 0:
            lse[starts[i]:starts[i] + m] = sinks
            continue
        lo = max(0, n - m + 1 - case["window"]) if case["window"] else 0
        k, v = (_tokens64(state, w, i, n)[lo:] for w in "kv")
        j = torch.arange(lo, n, device=DEV)
        pos = torch.arange(n - m, n, device=DEV)[:, None]
        sees = torch.ones((m, n - lo), dtype=torch.bool, device=DEV)
        if case["causal"]:
            sees &= j <= pos
        if case["window"]:
            sees &= j > pos - case["window"]
        for h in range(case["q_heads"]):
            kh, vh = k[:, h // group], v[:, h // group]
            s = (state["q"][starts[i]:starts[i] + m, h].double() @ kh.t().contiguous()) / math.sqrt(dim)
            s = torch.cat([torch.where(sees, s, -math.inf), sinks[h].expand(m, 1)], 1)
            lse[starts[i]:starts[i] + m, h] = total = torch.logsumexp(s, 1)
            w = torch.exp(s[:, :-1] - total[:, None])
            out[starts[i]:starts[i] + m, h] = torch.where(torch.isfinite(total)[:, None], w @ vh.contiguous(), 0.0)
    return {"out": out, "lse": lse}
