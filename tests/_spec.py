"""A step of speculative decoding in 64 bits on the CPU (numpy): trees, their attention,
verification and the kept rows. Written from the rules in include/kq.h, row by row."""
import numpy as np

from tests import _kv


def lines(parents):
    """The rows that each row of a sequence continues, itself last: from a root on."""
    got = []
    for j, p in enumerate(parents):
        got.append((got[p] if 0 <= p < j else []) + [j])
    return got


def masks(parents, window=0):
    """[n][n] bool: what each row sees of its sequence's rows."""
    m = np.zeros((len(parents), len(parents)), bool)
    for j, line in enumerate(lines(parents)):
        m[j, line[-window:] if window else line] = True
    return m


def depths(parents):
    return np.array([len(line) - 1 for line in lines(parents)], np.int64)


def words_of(sees, words):
    """bool [rows][n] -> uint32 [rows][words]."""
    got = np.zeros((len(sees), words), np.uint32)
    for t in range(sees.shape[1]):
        got[:, t // 32] |= sees[:, t].astype(np.uint32) << np.uint32(t % 32)
    return got


def random_tree(rng, n, back=8, roots=0.0):
    """Parents of n rows, each one of the `back` rows before it; `roots`: the share of rows that are none's."""
    got = [-1]
    for j in range(1, n):
        got.append(-1 if rng.random() < roots else int(rng.integers(max(0, j - back), j)))
    return got[:n]


def attend(cache, table, length, q, scale, sees, pos=None, window=0, sinks=None):
    """_kv.attend of a tree's rows: sees [n][n] what each row sees of the sequence's rows."""
    n, q_heads, dim = q.shape
    group, first = q_heads // cache.heads, length - n
    there = [t for t in range(length) if 0 <= table[t // cache.page] < cache.n_pages]
    k = np.zeros((len(there), cache.heads, dim))
    v = k.copy()
    ev = np.zeros((len(there), cache.heads))
    for i, t in enumerate(there):
        k[i], v[i] = (cache.token(w, table[t // cache.page], t % cache.page) for w in "kv")
        ev[i] = cache.exps["v"][table[t // cache.page], :, t % cache.page // cache.block].astype(np.float64) - 127
    at = np.array(there, np.int64)
    o, spread, codes = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape)
    lse, reach = np.full((n, q_heads), -np.inf), np.zeros((n, q_heads))
    for j in range(n):
        seen = at < first
        if window:
            seen &= at > max(int(pos[j]), first) - window
        for t in np.flatnonzero(sees[j]):
            seen |= at == first + t
        for h in range(q_heads):
            kk, vv = k[seen, h // group], v[seen, h // group]
            s = kk @ q[j, h] * scale
            m = max([s.max() if len(s) else -np.inf, sinks[h] if sinks is not None else -np.inf])
            if np.isinf(m):
                lse[j, h] = m
                continue
            w = np.exp(s - m)
            total = w.sum() + (np.exp(sinks[h] - m) if sinks is not None else 0.0)
            lse[j, h] = np.log(total) + m
            if len(s):
                o[j, h] = w @ vv / total
                spread[j, h] = w @ np.abs(vv) / total
                e = ev[seen, h // group]
                codes[j, h] = (np.abs(vv) * 2.0 ** (e.max() - e)[:, None]).sum(0)
                reach[j, h] = (np.abs(kk) @ np.abs(q[j, h])).max() * abs(scale)
    return o, lse, spread, reach, codes


def attend_tolerance(want, dim, eps, tiny):
    """The arithmetic is kq_kv_attn's, and so is the bound."""
    return _kv.attend_tolerance(*want, dim, eps, tiny)


# ---- verification, and the kept rows

def verify(p, tokens, u, parents, q=None, q_rows=None):
    """A sequence: p [n][vocab], tokens, u and parents [n], q [n_q][vocab], q_rows [n] (below 0: picked outright), in
    64 bits -> (kept rows, tokens, margin): margin is how far, relative to what is compared, the nearest decision
    was from going the other way."""
    clean = lambda a: np.where(np.isfinite(a) & (a > 0), a, 0.0).astype(np.float64)  # noqa: E731
    n, vocab = p.shape
    at, kept, out, margin = 0, [0], [], np.inf

    def differs(a, b):
        nonlocal margin
        margin = min(margin, abs(a - b) / max(abs(a), abs(b), 1e-300))

    while True:
        left, mass, went = clean(p[at]), 1.0, None
        for c in [c for c in range(1, n) if 0 <= parents[c] < c and parents[c] == at]:
            x, outright = int(tokens[c]), q is None or q_rows[c] < 0
            real = 0 <= x < vocab
            prob = 1.0 if outright else float(clean(q[q_rows[c], x])) if real else 0.0
            there = float(left[x]) if real else 0.0
            if there or u[c] * mass * prob:
                differs(u[c] * mass * prob, there)
            if u[c] * mass * prob < there:
                went = c
                break
            if outright:
                mass -= there
                if real:
                    left[x] = 0.0
            else:
                left = np.maximum(left - mass * clean(q[q_rows[c]]), 0.0)
                mass = float(left.sum())
        if went is None:
            break
        at = went
        kept.append(went)
        out.append(int(tokens[went]))
    up = np.cumsum(left)
    if up[-1] > 0:
        aim = u[0] * up[-1]
        x = int(np.argmax(up > aim))
        differs(aim, up[x])
        if x and up[x - 1]:
            differs(aim, up[x - 1])
        out.append(x)
    else:
        out.append(int(np.argmax(clean(p[at]))))
    return kept, out, margin


def keep_rows(cache, which, table, length, n, kept):
    """kq_kv_keep of one sequence: the rows `kept` of its last n tokens, into a _kv.Cache."""
    first = length - n
    rows = []
    for j, k in enumerate(kept):
        if not (j <= k < n and (not rows or k > rows[-1])):
            break
        rows.append(k)
    block, page = cache.block, cache.page
    src = {first + j: first + k for j, k in enumerate(rows) if k != j and first + j >= 0}
    before = {w: x[which].copy() for w, x in (("codes", cache.codes), ("exps", cache.exps))}

    def of(t):
        """(codes [heads][dim], exponent bytes [heads]) of a token as it was, or None."""
        p = table[t // page]
        return (before["codes"][p, :, t % page], before["exps"][p, :, t % page // block].astype(int)) if 0 <= p < cache.n_pages else None

    for b in sorted({t // block for t in src}):
        t0 = b * block
        p, s = table[t0 // page], t0 % page
        if not 0 <= p < cache.n_pages:
            continue
        own = before["exps"][p, :, s // block].astype(int)
        e = own.copy()
        for t, a in src.items():
            if t // block == b and of(a) is not None:
                e = np.maximum(e, of(a)[1])
        for t in range(t0, min(t0 + block, length)):
            got = of(src.get(t, t))
            for h in range(cache.heads):
                if got is None:
                    codes = np.zeros(cache.dim, np.uint8)
                elif got[1][h] == e[h]:
                    codes = got[0][h]
                else:
                    codes = _kv.encode(_kv.decode(got[0][h], cache.kind) * 2.0 ** float(got[1][h] - e[h]), cache.kind)
                cache.codes[which][p, h, t % page] = codes
        cache.exps[which][p, :, s // block] = e
