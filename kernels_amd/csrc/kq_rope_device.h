// kq_rope_device.h -- rotary positions: what kq_rope and kq_kv_write_rope share.
//
// An angle pos * inv_freq of a far position needs 64 bits: at position 131072 a float holds the
// angle of the fastest pair to 0.008. MI355X runs float64 sums and products at the float32 rate, so cosines, sines
// and the rotation itself are 64-bit too, and what comes out (keys rounded once, blocks' exponents) does not
// depend on how it is computed.
// Rows of queries share their pairs' angles among up to 64 / (rot / 16) heads, through LDS; keys on their way into a cache
// compute them anew for each head, as one wave is at one head's block.
#pragma once
#include "kq_device.h"
#include "kq_internal.h"
#include "kq_kv_device.h"

namespace kq {
namespace rope {

// cos and sin of x radians, |x| < 2^32, to about 2^-52: the nearest multiple of pi / 2 taken off
// in two steps (its first 53 bits, and the next 53: each step is one fused multiply-add), then
// Taylor's series, whose next term is below 2^-54 for |r| <= pi / 4.
__device__ __forceinline__ void cos_sin(double x, double& c, double& s) {
    constexpr double kRound = 6755399441055744.0;  // 1.5 * 2^52: the sum's low bits are the integer
    const double t = __builtin_fma(x, 0.63661977236758134308, kRound);
    const uint32_t quarter = (uint32_t)__builtin_bit_cast(uint64_t, t);
    const double k = t - kRound;
    const double r = __builtin_fma(-k, 6.123233995736766e-17, __builtin_fma(-k, 1.5707963267948966, x));
    const double z = r * r;
    double p = -1.0 / 1307674368000.0;  // 1 / 15!
    p = __builtin_fma(p, z, 1.0 / 6227020800.0);
    p = __builtin_fma(p, z, -1.0 / 39916800.0);
    p = __builtin_fma(p, z, 1.0 / 362880.0);
    p = __builtin_fma(p, z, -1.0 / 5040.0);
    p = __builtin_fma(p, z, 1.0 / 120.0);
    p = __builtin_fma(p, z, -1.0 / 6.0);
    const double sn = __builtin_fma(r * z, p, r);
    double q = 1.0 / 20922789888000.0;  // 1 / 16!
    q = __builtin_fma(q, z, -1.0 / 87178291200.0);
    q = __builtin_fma(q, z, 1.0 / 479001600.0);
    q = __builtin_fma(q, z, -1.0 / 3628800.0);
    q = __builtin_fma(q, z, 1.0 / 40320.0);
    q = __builtin_fma(q, z, -1.0 / 720.0);
    q = __builtin_fma(q, z, 1.0 / 24.0);
    q = __builtin_fma(q, z, -0.5);
    const double cs = __builtin_fma(q, z, 1.0);
    const bool odd = quarter & 1;
    const double a = odd ? sn : cs, b = odd ? cs : sn;
    // quarters 1 and 2 have a negative cosine, 2 and 3 a negative sine
    c = (quarter + 1) & 2 ? -a : a;
    s = quarter & 2 ? -b : b;
}

// Times the amplitude, of pair i at a position.
__device__ __forceinline__ void factors(const Rope& r, int pos, uint32_t i, double& c, double& s) {
    cos_sin((double)pos * (double)r.freq[i], c, s);
    c *= r.amplitude;
    s *= r.amplitude_sin;
}

// Two values turned, and rounded to 32 bits: the compiler would make one rounding of this and of that to 16 bits,
// in several instructions more.
__device__ __forceinline__ void turn(float a, float b, double c, double s, float& ya, float& yb) {
    const double x = a, y = b;
    ya = (float)__builtin_fma(x, c, -(y * s));
    yb = (float)__builtin_fma(y, c, x * s);
    asm("" : "+v"(ya), "+v"(yb));
}

// Eight consecutive elements of type F (kq_dtype) as floats, and back.
template <int F>
struct Eight {
    static constexpr int kWords = F == KQ_F32 ? 8 : 4;
    u32x4 w[kWords / 4];
    __device__ __forceinline__ void load(const uint8_t* p) {
#pragma unroll
        for (int i = 0; i < kWords / 4; ++i) w[i] = *reinterpret_cast<const u32x4*>(p + 16 * i);
    }
    __device__ __forceinline__ void store(uint8_t* p) const {
#pragma unroll
        for (int i = 0; i < kWords / 4; ++i) *reinterpret_cast<u32x4*>(p + 16 * i) = w[i];
    }
    __device__ __forceinline__ float get(int i) const {
        if constexpr (F == KQ_F32) {
            const uint32_t u = w[i / 4][i % 4];
            return __builtin_bit_cast(float, u);
        } else {
            return kv::elem<F == KQ_BF16>(i % 2 ? w[0][i / 2] >> 16 : w[0][i / 2] & 0xFFFF);
        }
    }
    __device__ __forceinline__ void set(int i, float a, float b) {  // elements i and i + 1, i even
        if constexpr (F == KQ_F32) {
            w[i / 4][i % 4] = __builtin_bit_cast(uint32_t, a);
            w[i / 4][i % 4 + 1] = __builtin_bit_cast(uint32_t, b);
        } else {
            w[0][i / 2] = kv::pair16<F == KQ_BF16>(a, b);
        }
    }
};

// Eight pairs: of HALVES a holds the first values and b the second ones, of pairs in a row a and b follow
// one another. f(e, c, s): the factors of pair e.
template <int F, int PAIRS, class Fn>
__device__ __forceinline__ void turn_eight(Eight<F>& a, Eight<F>& b, Fn f) {
    if constexpr (PAIRS) {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            double c, s;
            f(e, c, s);
            Eight<F>& x = e < 4 ? a : b;
            float y0, y1;
            turn(x.get(2 * (e % 4)), x.get(2 * (e % 4) + 1), c, s, y0, y1);
            x.set(2 * (e % 4), y0, y1);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; e += 2) {
            double c0, s0, c1, s1;
            f(e, c0, s0);
            f(e + 1, c1, s1);
            float a0, a1, b0, b1;
            turn(a.get(e), b.get(e), c0, s0, a0, b0);
            turn(a.get(e + 1), b.get(e + 1), c1, s1, a1, b1);
            a.set(e, a0, a1);
            b.set(e, b0, b1);
        }
    }
}

// Sixteen columns of a head that are turned together, unit u: their first and second eight.
template <int PAIRS>
__device__ __forceinline__ uint32_t first_eight(uint32_t u) {
    return PAIRS ? 16 * u : 8 * u;
}
template <int PAIRS>
__device__ __forceinline__ uint32_t second_eight(uint32_t u, uint32_t rot) {
    return PAIRS ? 16 * u + 8 : rot / 2 + 8 * u;
}

struct Factor {
    double c, s;
};

// A wave turns heads h0 .. h1 - 1 of one row: the factors of its pairs into `table` (the wave's rot / 2
// places), then every lane keeps those of its eight pairs in registers for all the heads.
template <int F, int PAIRS>
__device__ __forceinline__ void turn_heads(const Rope& r, int pos, const uint8_t* x, uint8_t* y, int64_t x_head,
                                           int64_t y_head, uint32_t h0, uint32_t h1, uint32_t D, Factor* table) {
    constexpr int kSize = F == KQ_F32 ? 4 : 2;
    const uint32_t lane = threadIdx.x & 63, pairs = r.rot / 2;
    // whole vectors: asked for before the angles, and the next heads' before these are turned
    const bool vectors = r.rot % 16 == 0;
    const uint32_t units = vectors ? r.rot / 16 : 1, at_once = 64 / units, u = lane % units;
    const uint32_t ca = first_eight<PAIRS>(u) * kSize, cb = second_eight<PAIRS>(u, r.rot) * kSize;
    uint32_t h = vectors && lane < at_once * units ? h0 + lane / units : h1;
    Eight<F> a, b;
    auto load = [&](uint32_t head) {
        if (head >= h1) return;
        const uint8_t* const from = x + (int64_t)head * x_head * kSize;
        a.load(from + ca);
        b.load(from + cb);
    };
    load(h);
    for (uint32_t i = lane; i < pairs; i += 64) factors(r, pos, i, table[i].c, table[i].s);
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
    if (vectors) {
        if (h < h1) {
            Factor f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = table[8 * u + e];
            for (; h < h1; h += at_once) {
                uint8_t* const to = y + (int64_t)h * y_head * kSize;
                Eight<F> ya = a, yb = b;
                load(h + at_once);
                turn_eight<F, PAIRS>(ya, yb, [&](int e, double& c, double& s) { c = f[e].c, s = f[e].s; });
                ya.store(to + ca);
                yb.store(to + cb);
            }
        }
    } else {
        auto get = [&](const uint8_t* p) {
            if constexpr (F == KQ_F32) return *reinterpret_cast<const float*>(p);
            else return kv::elem<F == KQ_BF16>(*reinterpret_cast<const uint16_t*>(p));
        };
        auto put = [&](uint8_t* p, float v) {
            if constexpr (F == KQ_F32) *reinterpret_cast<float*>(p) = v;
            else *reinterpret_cast<uint16_t*>(p) = (uint16_t)kv::pair16<F == KQ_BF16>(v, 0.0f);
        };
        for (h = h0; h < h1; ++h) {
            const uint8_t* const from = x + (int64_t)h * x_head * kSize;
            uint8_t* const to = y + (int64_t)h * y_head * kSize;
            for (uint32_t i = lane; i < pairs; i += 64) {
                const uint32_t one = (PAIRS ? 2 * i : i) * kSize, two = (PAIRS ? 2 * i + 1 : pairs + i) * kSize;
                float ya, yb;
                turn(get(from + one), get(from + two), table[i].c, table[i].s, ya, yb);
                put(to + one, ya);
                put(to + two, yb);
            }
        }
    }
    if (x == y || r.rot == D) return;
    // columns that are not turned
    const uint32_t rest = D - r.rot;
    if (r.rot % 8 == 0) {
        for (uint32_t i = lane; i < (h1 - h0) * (rest / 8); i += 64) {
            const uint32_t head = h0 + i / (rest / 8), d = (r.rot + i % (rest / 8) * 8) * kSize;
            Eight<F> v;
            v.load(x + (int64_t)head * x_head * kSize + d);
            v.store(y + (int64_t)head * y_head * kSize + d);
        }
    } else {
        for (uint32_t i = lane; i < (h1 - h0) * rest; i += 64) {
            const uint32_t head = h0 + i / rest, d = (r.rot + i % rest) * kSize;
            const uint8_t* const from = x + (int64_t)head * x_head * kSize + d;
            uint8_t* const to = y + (int64_t)head * y_head * kSize + d;
            if constexpr (F == KQ_F32) *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(from);
            else *reinterpret_cast<uint16_t*>(to) = *reinterpret_cast<const uint16_t*>(from);
        }
    }
}

}  // namespace rope
}  // namespace kq
