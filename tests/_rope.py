"""Rotary positions in 64 bits on the CPU (numpy), what kq_rope and kq_kv_write_rope are compared
with, and the bound on their differences. Written from the formulas in include/kq.h."""
import numpy as np


def turned(x, pos, freqs, pairs=False, amplitude=1.0, inverse=False):
    """x float64 [rows][heads][dim] turned by pos [rows] times freqs float32 [rot / 2], by complex numbers."""
    rot = 2 * len(freqs)
    angle = np.asarray(pos, np.float64)[:, None, None] * np.asarray(freqs, np.float64)
    by = amplitude * np.exp((-1j if inverse else 1j) * angle)
    y = np.array(x, np.float64)
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if pairs else (slice(0, rot // 2), slice(rot // 2, rot))
    z = (y[..., a] + 1j * y[..., b]) * by
    y[..., a], y[..., b] = z.real, z.imag
    return y


def tolerance(x, y, rot, pairs, amplitude, eps, tiny, far):
    """How far a turned value may be from y.

    The angle is exact to 2^-53 of itself (a product of 31 and 24 bits rounded
    once): 2^-52 far radians cover it and the oracle's own. The factors are off by 2^-50
    beside that, the products and their sum by 2^-52 of the pair's size |x_a| + |x_b|. Then y is
    rounded to 32 bits (2^-24 of itself, or half the smallest step of those, 2^-150) and to its type (eps / 2,
    or half its smallest step)."""
    size = np.zeros_like(x)
    a, b = (slice(0, rot, 2), slice(1, rot, 2)) if pairs else (slice(0, rot // 2), slice(rot // 2, rot))
    size[..., a] = size[..., b] = np.abs(x[..., a]) + np.abs(x[..., b])
    off = abs(amplitude) * size * (2.0**-52 * far + 2.0**-49)
    return off + np.abs(y) * (2.0**-24 + eps / 2) * 1.001 + 2.0**-150 + tiny
