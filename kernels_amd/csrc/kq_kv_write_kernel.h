// kq_kv_write_kernel.h -- the kernel that writes the 8-bit key/value cache (the layout
// and the rule of the scales: kq.h), of keys as they come (kq_kv_cache.hip) or turned
// by their position on the way (kq_kv_rope.hip).
#pragma once
#include "kq_kv_device.h"
#include "kq_rope_device.h"

namespace kq {
namespace kv {

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// Magnitude bits of both halves of pairs order as the magnitudes do; from kInf on they are no finite value's.
template <int BF>
constexpr uint32_t kInf = BF ? 0x7F80u : 0x7C00u;
__device__ __forceinline__ uint32_t pair_max(uint32_t pair, uint32_t m) {
    return __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(u16x2, pair & 0x7FFF7FFFu),
                                                                  __builtin_bit_cast(u16x2, m)));
}
// The larger half, and the same of finite values alone.
__device__ __forceinline__ uint32_t half_max(uint32_t m) { return max(m & 0xFFFFu, m >> 16); }
template <int BF>
__device__ __forceinline__ uint32_t finite_max(uint32_t pair, uint32_t m) {
    const uint32_t a = pair & 0x7FFFu, b = pair >> 16 & 0x7FFFu;
    return max(m, max(a < kInf<BF> ? a : 0u, b < kInf<BF> ? b : 0u));
}

// Four codes of a dword anew: the values they stand for times `keep`, rounded.
template <int TYPE>
__device__ __forceinline__ uint32_t rounded_anew(uint32_t w, float keep) {
    float y[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) y[q] = to_range<TYPE>(Code<TYPE>::value(w >> 8 * q & 0xFF), keep);
    return Code<TYPE>::code2(y[0], y[1]) | Code<TYPE>::code2(y[2], y[3]) << 16;
}
// Codes of four values times `scale`. PLAIN: all are finite and within the codes' range as they are.
// int8: adding 1.5 * 2^23 rounds to nearest even and leaves the integer's low byte in the sum's.
template <int TYPE, bool PLAIN>
__device__ __forceinline__ uint32_t four_codes(float a, float b, float c, float d, float scale) {
    if constexpr (!PLAIN) {
        return Code<TYPE>::code2(to_range<TYPE>(a, scale), to_range<TYPE>(b, scale)) |
               Code<TYPE>::code2(to_range<TYPE>(c, scale), to_range<TYPE>(d, scale)) << 16;
    } else if constexpr (TYPE == KQ_KV_I8) {
        auto low = [&](float x) { return __builtin_bit_cast(uint32_t, __builtin_fmaf(x, scale, 12582912.0f)); };
        return __builtin_amdgcn_perm(low(b), low(a), 0x0C0C0400u) | __builtin_amdgcn_perm(low(d), low(c), 0x04000C0Cu);
    } else {
        const int w = __builtin_amdgcn_cvt_pk_fp8_f32(a * scale, b * scale, 0, false);
        return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c * scale, d * scale, w, true);
    }
}

// One wave writes one block of one head's K or V: the largest new magnitude over the wave, the
// exponent, then the codes. Blocks of 16 tokens stay in registers in between (bf16 prefill of 13k
// tokens, 8 heads of 128: 28-35 us for 82 MB with a second read, 21-27 without); larger ones are read
// twice, 16 tokens at a time, the second time from a cache.
//
// TURN: the layout of the pairs that keys are turned by (0: HALVES, 1: PAIRS), or none
// (-1). A lane then holds units of 16 columns that are turned together, in place of
// chunks of 8 in order; everything behind is the same. Angles are computed anew by each head's
// wave, and once: blocks of up to kept_subs(D) x 16 tokens wait in LDS, turned, for their scale (48 trees of 9-26 rows into
// blocks of 32, 64 and 8 heads of 128: turned twice 22.0 us, so 16.6).
constexpr int kept_subs(int D) { return D <= 128 ? 256 / D : 1; }
template <int D, int TYPE, int BF, int TURN>
__device__ __forceinline__ void write_block(const Cache& c, const Batch& b, const Rows& K, const Rows& V, uint32_t groups, uint32_t block_x,
                                            const Turn& turn, u32x4* kept) {
    const int lane = threadIdx.x & 63;
    const uint32_t job = (block_x % groups) * 4 + (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    if (job >= 2 * c.heads) return;
    const uint32_t h = job >> 1;
    const bool is_v = job & 1;
    const Seq s = sequence(b, c.page_log2, blockIdx.y);
    const int first = s.len - s.n, first0 = max(first, 0), B = 1 << c.block_log2;
    // unsigned: blocks behind a sequence of nearly 2^31 tokens pass 31 bits
    const uint32_t t0u = (((uint32_t)first0 >> c.block_log2) + block_x / groups) << c.block_log2;
    if (s.n == 0 || t0u >= (uint32_t)s.len) return;
    const int t0 = (int)t0u;
    const int page = page_of(c, b.pages + (uint64_t)blockIdx.y * b.max_pages, t0);
    const int lo = max(first0 - t0, 0), hi = min(s.len - t0, B);  // the block's new tokens
    // field by field: from a reference to one of the two the compiler makes more offsets of rows ahead, and takes 268
    // registers at 192 columns and one wave a SIMD in place of 179 and two (five prompts of 331 to 5001 tokens, 8 heads,
    // bf16: 59 us in place of 38), 104 at 96 in place of 92 (17.1 and 15.7)
    const Rows R = {is_v ? V.p : K.p, is_v ? V.row : K.row, is_v ? V.head : K.head};
    const uint16_t* const x = static_cast<const uint16_t*>(R.p) + (int64_t)(s.row0 + t0 - first) * R.row +
                              (int64_t)h * R.head;  // token t0's values

    // 16 tokens in registers. K: 8 columns of a token a piece. V: two columns of 16 tokens, or of 8
    // where that fills the wave.
    constexpr int NK = TURN < 0 ? D / 32 : (D + 63) / 64 * 2, H = D == 64 ? 2 : 1, TL = 16 / H, NV = (D / 2 * H + 63) / 64;
    u32x4 xk[NK];
    // Token (of 16) and first column of chunk j of K; TURN: which unit's half, some lanes' last is none.
    auto chunk = [&](int j, int& t, int& col) __attribute__((always_inline)) {
        const int i = lane + 64 * (TURN < 0 ? j : j / 2);
        if constexpr (TURN < 0) {
            t = i / (D / 8), col = i % (D / 8) * 8;
            return true;
        } else {
            const uint32_t u = (uint32_t)i % (D / 16), rot = turn.rope.rot;
            t = i / (D / 16);
            col = (int)(TURN == 1 || u >= rot / 16 ? 16 * u + j % 2 * 8
                                                   : j % 2 ? rope::second_eight<0>(u, rot) : rope::first_eight<0>(u));
            return D % 64 == 0 || i < D;
        }
    };
    uint32_t xv[NV][TL];
    // (inlined by force: of functions of their own, which the compiler makes of the two at 192 and 256 wide, the
    // values' registers go through memory: five prompts of 331 to 5001 tokens, 8 heads of 256, written and
    // read 143 us so, 64 inlined)
    auto load = [&](int sub) __attribute__((always_inline)) {
        if (!is_v) {
#pragma unroll
            for (int j = 0; j < NK; ++j) {
                int t, col;
                const bool one = chunk(j, t, col);
                t += sub;
                xk[j] = one && t >= lo && t < hi ? *reinterpret_cast<const u32x4*>(x + (int64_t)t * R.row + col) : u32x4{};
            }
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int q = 0; q < TL; ++q) {
                    const int i = lane + 64 * j, t = sub + i / (D / 2) * TL + q;
                    const bool there = t >= lo && t < hi && (NV * 64 == D / 2 * H || i < D / 2 * H);
                    xv[j][q] = there ? *reinterpret_cast<const uint32_t*>(x + (int64_t)t * R.row + i % (D / 2) * 2) : 0u;
                }
        }
    };
    // ... and turned, as 16-bit values again
    auto rotate = [&](int sub) __attribute__((always_inline)) {
        if constexpr (TURN >= 0) {
            if (is_v) return;
            const rope::Rope& r = turn.rope;
#pragma unroll
            for (int j = 0; j < NK; j += 2) {
                int t, col;
                const bool one = chunk(j, t, col);
                const uint32_t u = (uint32_t)(lane + 32 * j) % (D / 16);
                t += sub;
                if (!one || t < lo || t >= hi || u >= r.rot / 16) continue;
                const int pos = turn.pos ? turn.pos[s.row0 + t0 + t - first] : t0 + t;
                rope::Eight<BF> p, q;
                p.w[0] = xk[j], q.w[0] = xk[j + 1];
                rope::turn_eight<BF, TURN>(p, q, [&](int e, double& cs, double& sn) { rope::factors(r, pos, 8 * u + e, cs, sn); });
                xk[j] = p.w[0], xk[j + 1] = q.w[0];
            }
        }
    };
    load(lo & ~15);  // on its way while the page id is
    if (page < 0) return;
    rotate(lo & ~15);
    // The tokens of `sub` once more, for the passes behind the first; put by: into LDS.
    const bool wait = TURN >= 0 && !is_v && B > 16 && B <= 16 * kept_subs(D);
    auto put_by = [&](int sub) __attribute__((always_inline)) {
        if constexpr (TURN >= 0)
            if (wait)
#pragma unroll
                for (int j = 0; j < NK; ++j) kept[(sub / 16 * NK + j) * 64 + lane] = xk[j];
    };
    auto again = [&](int sub) __attribute__((always_inline)) {
        if (wait && sub >= (lo & ~15)) {
#pragma unroll
            for (int j = 0; j < NK; ++j) xk[j] = kept[(sub / 16 * NK + j) * 64 + lane];
        } else {
            load(sub), rotate(sub);
        }
    };
    uint8_t* const codes = (is_v ? c.v : c.k) + code_offset(c, D, page, h, t0);
    uint8_t* const ep = (is_v ? c.v_exp : c.k_exp) + exp_offset(c, page, h, t0);
    const int was = lo > 0 ? (int)*ep - 127 : -127;
    uint32_t m = 0;
    for (int sub = lo & ~15; sub < hi; sub += 16) {
        if (sub > lo) load(sub), rotate(sub);
        put_by(sub);
        if (!is_v) {
#pragma unroll
            for (int j = 0; j < NK; ++j)
#pragma unroll
                for (int q = 0; q < 4; ++q) m = pair_max(xk[j][q], m);
        } else {
#pragma unroll
            for (int j = 0; j < NV; ++j)
#pragma unroll
                for (int q = 0; q < TL; ++q) m = pair_max(xv[j][q], m);
        }
    }
    m = wave_max(half_max(m));
    const bool finite = m < kInf<BF>;
    if (!finite) {  // once more, without infinities and NaN
        m = 0;
        for (int sub = lo & ~15; sub < hi; sub += 16) {
            if (B > 16) again(sub);
            if (!is_v) {
#pragma unroll
                for (int j = 0; j < NK; ++j)
#pragma unroll
                    for (int q = 0; q < 4; ++q) m = finite_max<BF>(xk[j][q], m);
            } else {
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int q = 0; q < TL; ++q) m = finite_max<BF>(xv[j][q], m);
            }
        }
        m = wave_max(m);
    }
    const int wanted = block_exponent<TYPE>(elem<BF>(m));
    const int e = max(wanted, was);
    const bool grew = lo > 0 && wanted > was;
    const float keep = pow2f(max(was - e, -126));  // what older codes are multiplied by
    // e >= kMinExp; up to 128 where a cache from elsewhere holds such a byte: a subnormal scale, exact too
    const float scale = __builtin_ldexpf(1.0f, -e);
    if (lane == 0) *ep = (uint8_t)(e + 127);
    auto write = [&](auto plain) __attribute__((always_inline)) {
        constexpr bool P = decltype(plain)::value;
        for (int sub = grew ? 0 : lo & ~15; sub < hi; sub += 16) {
            if (B > 16) again(sub);
            if (!is_v) {
#pragma unroll
                for (int j = 0; j < NK; ++j) {
                    int t, col;
                    if (!chunk(j, t, col)) continue;
                    t += sub;
                    u32x2* const at = reinterpret_cast<u32x2*>(codes + (uint32_t)(t * D + col));
                    if (t >= lo && t < hi) {
                        const u32x4 v = xk[j];
                        u32x2 w;
#pragma unroll
                        for (int q = 0; q < 2; ++q)
                            w[q] = four_codes<TYPE, P>(elem<BF>(v[2 * q] & 0xFFFF), elem<BF>(v[2 * q] >> 16),
                                                       elem<BF>(v[2 * q + 1] & 0xFFFF), elem<BF>(v[2 * q + 1] >> 16), scale);
                        *at = w;
                    } else if (t < lo && grew) {
                        const u32x2 old = *at;
                        *at = u32x2{rounded_anew<TYPE>(old.x, keep), rounded_anew<TYPE>(old.y, keep)};
                    }
                }
                continue;
            }
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int i = lane + 64 * j, t = sub + i / (D / 2) * TL;
                if (NV * 64 != D / 2 * H && i >= D / 2 * H) continue;
                uint32_t* const at = reinterpret_cast<uint32_t*>(codes + (uint32_t)(sub * D + i % (D / 2) * 32 + i / (D / 2) * TL));
                const bool part = t < lo || t + TL > hi;  // older tokens, or none, among them
                uint32_t out[2][TL / 4];
#pragma unroll
                for (int w = 0; w < TL / 4; ++w) {
                    const uint32_t* const v = xv[j] + 4 * w;
                    uint32_t col[2] = {four_codes<TYPE, P>(elem<BF>(v[0] & 0xFFFF), elem<BF>(v[1] & 0xFFFF), elem<BF>(v[2] & 0xFFFF),
                                                           elem<BF>(v[3] & 0xFFFF), scale),
                                       four_codes<TYPE, P>(elem<BF>(v[0] >> 16), elem<BF>(v[1] >> 16), elem<BF>(v[2] >> 16),
                                                           elem<BF>(v[3] >> 16), scale)};
                    if (part) {
                        // bytes of older tokens stay, or are rounded anew; those behind the last stay
                        uint32_t fresh = 0, older = 0;
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            fresh |= t + 4 * w + q >= lo && t + 4 * w + q < hi ? 0xFFu << 8 * q : 0u;
                            older |= t + 4 * w + q < lo ? 0xFFu << 8 * q : 0u;
                        }
#pragma unroll
                        for (int n = 0; n < 2; ++n) {
                            uint32_t old = at[4 * n + w];
                            if (grew) old = (rounded_anew<TYPE>(old, keep) & older) | (old & ~older);
                            col[n] = (col[n] & fresh) | (old & ~fresh);
                        }
                    }
                    out[0][w] = col[0];
                    out[1][w] = col[1];
                }
#pragma unroll
                for (int n = 0; n < 2; ++n)
                    if constexpr (TL == 16) *reinterpret_cast<u32x4*>(at + 4 * n) = u32x4{out[n][0], out[n][1], out[n][2], out[n][3]};
                    else *reinterpret_cast<u32x2*>(at + 4 * n) = u32x2{out[n][0], out[n][1]};
            }
        }
    };
    // at the range's end a finite value may still exceed the largest code
    if (finite && e < Code<TYPE>::kMaxExp) write(Int<1>());
    else write(Int<0>());
}

}  // namespace kv
}  // namespace kq
