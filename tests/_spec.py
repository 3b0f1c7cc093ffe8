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
