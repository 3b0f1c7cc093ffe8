"""The 8-bit key/value cache in 64 bits on the CPU (numpy): what kq_kv_write,
kq_kv_read and kq_kv_attn are compared with. Written from the format's rules
in include/kq.h, token by token."""
import numpy as np

LARGEST = {"i8": 127.0, "e4m3": 448.0}
MAX_EXP = {"i8": 121, "e4m3": 119}
MIN_EXP = -64


def e4m3_values():
    """The 256 values of e4m3 (NaN at 0x7F and 0xFF)."""
    got = np.zeros(256)
    for c in range(256):
        e, m = c >> 3 & 15, c & 7
        v = m * 2.0**-9 if e == 0 else (8 + m) * 2.0**(e - 10)
        got[c] = (-v if c & 128 else v) if c & 127 != 127 else np.nan
    return got


E4M3 = e4m3_values()
_POSITIVE = E4M3[:127]  # ascending, by code


def decode(codes, kind):
    """uint8 codes -> float64."""
    return codes.view(np.int8).astype(np.float64) if kind == "i8" else E4M3[codes]


def encode(y, kind):
    """float64 -> uint8 codes, to nearest even, saturated; NaN is 0."""
    y = np.where(np.isnan(y), 0.0, y)
    y = np.clip(y, -LARGEST[kind], LARGEST[kind])
    if kind == "i8":
        return np.rint(y).astype(np.int8).view(np.uint8)
    a = np.abs(y)
    hi = np.searchsorted(_POSITIVE, a).clip(0, 126)
    lo = (hi - 1).clip(0)
    up, down = _POSITIVE[hi] - a, a - _POSITIVE[lo]
    c = np.where(up < down, hi, np.where(down < up, lo, np.where(hi % 2 == 0, hi, lo)))
    return (c | np.where(np.signbit(y), 128, 0)).astype(np.uint8)


def exponent(a, kind):
    """The smallest e of the range with a <= largest code * 2^e."""
    e = MIN_EXP
    while a > LARGEST[kind] * 2.0**e and e < MAX_EXP[kind]:
        e += 1
    return e


class Cache:
    """codes uint8 k [pages][heads][page][dim], v likewise (rows, not the
    device's columns), exponent bytes uint8 [pages][heads][page/block]."""

    def __init__(self, n_pages, heads, dim, page=16, block=16, kind="i8"):
        self.n_pages, self.heads, self.dim, self.page, self.block, self.kind = n_pages, heads, dim, page, block, kind
        self.codes = {w: np.zeros((n_pages, heads, page, dim), np.uint8) for w in "kv"}
        self.exps = {w: np.full((n_pages, heads, page // block), 63, np.uint8) for w in "kv"}

    def copy(self):
        c = Cache(self.n_pages, self.heads, self.dim, self.page, self.block, self.kind)
        c.codes, c.exps = ({w: x[w].copy() for w in "kv"} for x in (self.codes, self.exps))
        return c

    def fill(self, rng, nan=False):
        """Random codes (NaN codes of e4m3 only where asked for) and moderate scales everywhere."""
        for w in "kv":
            c = rng.integers(0, 256, self.codes[w].shape, dtype=np.uint8)
            if self.kind == "e4m3" and not nan:
                c[(c & 127) == 127] ^= 1
            if self.kind == "i8":
                c[c == 128] = 129
            # values of about 1: largest code * 2^e
            mid = 127 - 6 if self.kind == "i8" else 127 - 8
            self.codes[w], self.exps[w] = c, rng.integers(mid - 1, mid + 2, self.exps[w].shape).astype(np.uint8)

    def token(self, which, page, t):
        """float64 [heads][dim] of token t of a page."""
        e = self.exps[which][page, :, t // self.block].astype(np.float64) - 127
        return decode(self.codes[which][page, :, t], self.kind) * 2.0 ** e[:, None]

    def write(self, which, x, table, length, new):
        """The last `new` of a sequence's `length` tokens: x float64 [new][heads][dim]."""
        first = length - new
        b = max(first, 0) // self.block
        while new and b * self.block < length:
            t0, t1 = b * self.block, min((b + 1) * self.block, length)
            page, s = table[t0 // self.page], t0 % self.page
            b += 1
            if not 0 <= page < self.n_pages:
                continue
            fresh = [t for t in range(t0, t1) if t >= max(first, 0)]
            for h in range(self.heads):
                y = np.stack([x[t - first, h] for t in fresh])
                a = np.abs(np.where(np.isfinite(y), y, 0.0)).max()
                e = exponent(a, self.kind)
                if fresh[0] > t0:
                    was = int(self.exps[which][page, h, s // self.block]) - 127
                    if e > was:
                        for t in range(t0, fresh[0]):
                            old = decode(self.codes[which][page, h, s + t - t0], self.kind)
                            self.codes[which][page, h, s + t - t0] = encode(old * 2.0 ** (was - e), self.kind)
                    e = max(e, was)
                self.exps[which][page, h, s // self.block] = e + 127
                for t, yt in zip(fresh, y):
                    self.codes[which][page, h, s + t - t0] = encode(yt * 2.0**-e, self.kind)

    def read(self, which, table, length, new):
        """float64 [new][heads][dim], NaN rows at negative positions."""
        got = np.full((new, self.heads, self.dim), np.nan)
        for j in range(new):
            t = length - new + j
            if t >= 0:
                page = table[t // self.page]
                got[j] = self.token(which, page, t % self.page) if 0 <= page < self.n_pages else 0.0
        return got


def attend(cache, table, length, q, scale, causal=True, window=0, sinks=None):
    """q float64 [n][q_heads][dim] -> (o, lse, spread, reach, codes): float64 results, sum p |v|, the largest
    sum |q k| * scale of a row, and sum |code of v| * the largest scale of v: what the tolerances go by."""
    n, q_heads, dim = q.shape
    group = q_heads // cache.heads
    seen = [t for t in range(length) if 0 <= table[t // cache.page] < cache.n_pages]
    k = np.zeros((len(seen), cache.heads, dim))
    v = k.copy()
    ev = np.zeros((len(seen), cache.heads))
    for i, t in enumerate(seen):
        k[i], v[i] = (cache.token(w, table[t // cache.page], t % cache.page) for w in "kv")
        ev[i] = cache.exps["v"][table[t // cache.page], :, t % cache.page // cache.block].astype(np.float64) - 127
    at = np.array(seen, np.int64)
    o, spread, codes = np.zeros(q.shape), np.zeros(q.shape), np.zeros(q.shape)
    lse, reach = np.full((n, q_heads), -np.inf), np.zeros((n, q_heads))
    for j in range(n):
        pos = length - n + j
        sees = np.ones(len(at), bool)
        if causal:
            sees &= at <= pos
        if window:
            sees &= at > pos - window
        for h in range(q_heads):
            kk, vv = k[sees, h // group], v[sees, h // group]
            s = kk @ q[j, h] * scale
            m = max([s.max() if len(s) else -np.inf, sinks[h] if sinks is not None else -np.inf])
            if np.isinf(m):  # nothing in sight, or a sink that takes all
                lse[j, h] = m
                continue
            w = np.exp(s - m)
            total = w.sum() + (np.exp(sinks[h] - m) if sinks is not None else 0.0)
            lse[j, h] = np.log(total) + m
            if len(s):
                o[j, h] = w @ vv / total
                spread[j, h] = w @ np.abs(vv) / total
                e = ev[sees, h // group]
                codes[j, h] = (np.abs(vv) * 2.0 ** (e.max() - e)[:, None]).sum(0)
                reach[j, h] = (np.abs(kk) @ np.abs(q[j, h])).max() * abs(scale)
    return o, lse, spread, reach, codes


def attend_tolerance(o, lse, spread, reach, codes, dim, eps, tiny):
    """How far (out, lse) may be off.

    A score is dim exact products summed in 32 bits, then times the scale (itself
    rounded), plus the exponent, minus the maximum (in steps of log2): off by at
    most E = (dim + 16) 2^-24 (reach + 96), 96 covering exponents and the lift.
    exp2 and the sums add a few 2^-23. A probability is then rounded to fp16
    (2^-11 of itself), so out is off by (2^-11 + 4 E) sum p |v|, and by the
    rounding of the result: eps / 2 of it, or half its type's smallest step.
    fp16 rounds no finer than 2^-24: w = 2^(t - m + 11), t = log2 p + e_v, is off by
    2^-25 where it is subnormal, and out = sum w code / sum w 2^-e_v by 2^-25 sum
    |code| / sum w 2^-e_v. The reference m is at most the largest t, whose token
    alone makes the denominator 2^11 2^-e_v at least: out is off by at most
    2^-36 sum |code| 2^(largest e_v).
    lse: E, and its own roundings."""
    E = (dim + 16) * 2.0**-24 * (reach + 96.0)
    out = (2.0**-11 + 4 * E)[..., None] * spread * 1.01 + eps / 2 * np.abs(o) * 1.01 + tiny + 2.0**-36 * codes
    with np.errstate(invalid="ignore"):
        size = np.where(np.isfinite(lse), np.abs(lse), 0.0)
    return out, 2 * E + 2.0**-21 * (size + 1.0)
