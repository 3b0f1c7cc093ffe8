// kq_kv_attn_kernel.h -- attention over the 8-bit cache, few rows: the wave
// kernel of kq_kv_attn.hip.
//
// A wave takes 64 tokens at a time against 16 rows (query tokens x the heads of a
// group) of one sequence and head. Both products are 16x16x32 fp16 MFMAs on
// transposed results, so that nothing moves between lanes:
//   S^T = K Q^T: lane (r = lane % 16, g = lane / 16) receives tokens 4g..4g+3 of a
//         16-token operand, for row r. Which tokens stand in an operand is
//         free: operand t (of 4) holds token 16 (i / 4) + 4t + i % 4 at place i,
//         so that lane (r, g) ends with the tokens 16g..16g+15, one exponent.
//   O^T = V^T P^T: the lane's 16 probabilities are two operands as they are
//         (k place 8g + j <-> token 16g + 8h + j), and the matching V operand is
//         the 16 bytes that hold column d of the lane's 16 tokens.
// With t_p = log2(e) s_p + e_v(p), the probabilities and V's scale are one number
// w_p = 2^(t_p - m); the denominator is the sum of w_p 2^-e_v(p).
#pragma once
#include "kq_kv_device.h"

namespace kq {
namespace kv {

constexpr int kTile = 64;      // tokens a wave takes at a time
constexpr int kLift = 14;      // probabilities are scaled by 2^14: the fp16 ones stay normal down to 2^-28 of the largest
constexpr int kSegment = 8192;  // tokens whose page ids a workgroup holds at a time
constexpr float kLowest = -3.0e38f;  // running maximum before any token

// Tokens that a row tile sees: [lo, hi), lo a multiple of 64.
struct Span {
    int lo, hi;
};
__device__ __forceinline__ Span span_of(const Seq& s, const Attn& a, int row, int rows) {
    Span v = {0, s.len};
    if (a.causal) {
        const int pos = s.len - s.n, last = min(row + rows, (int)(s.n * a.group)) - 1;
        v.hi = max(pos + last / (int)a.group + 1, 0);
        if (a.window) v.lo = max(pos + row / (int)a.group - (int)a.window + 1, 0) & ~(kTile - 1);
    }
    return v;
}
__device__ __forceinline__ int splits_of(const Span& v, int chunk) {
    return v.hi > v.lo ? (v.hi - v.lo + chunk - 1) / chunk : 0;
}

// Of a value in lanes l, l ^ 16, l ^ 32, l ^ 48: one step of its largest or sum. (A bit cast of an
// element of the swap's result would take element 0 both times: values go through variables.)
template <bool HALVES>
__device__ __forceinline__ void swapped(float v, float& x, float& y) {
    const uint32_t u = __builtin_bit_cast(uint32_t, v);
    uint32_t p, q;
    if constexpr (HALVES) {
        const auto s = __builtin_amdgcn_permlane32_swap(u, u, false, false);
        p = s[0], q = s[1];
    } else {
        const auto s = __builtin_amdgcn_permlane16_swap(u, u, false, false);
        p = s[0], q = s[1];
    }
    x = __builtin_bit_cast(float, p);
    y = __builtin_bit_cast(float, q);
}
__device__ __forceinline__ float across_rows_maxf(float v) {
    float x, y;
    swapped<false>(v, x, y);
    swapped<true>(fmaxf(x, y), x, y);
    return fmaxf(x, y);
}
__device__ __forceinline__ float across_rows_sum(float v) {
    float x, y;
    swapped<false>(v, x, y);
    swapped<true>(x + y, x, y);
    return x + y;
}

// Four outputs of a row, from column d on.
__device__ __forceinline__ void store4(const Rows& O, int row, uint32_t head, int d, f32x4 y, bool bf) {
    uint16_t* const to = static_cast<uint16_t*>(O.p) + (int64_t)row * O.row + (int64_t)head * O.head + d;
    *reinterpret_cast<u32x2*>(to) = bf ? u32x2{pair16<1>(y[0], y[1]), pair16<1>(y[2], y[3])}
                                       : u32x2{pair16<0>(y[0], y[1]), pair16<0>(y[2], y[3])};
}

// The last step of a row: joins the sink, writes lse, and returns what the row's sums are
// multiplied by. m and l as the waves keep them: l = sum 2^(s log2e + kLift - m).
__device__ __forceinline__ float finish(const Attn& a, float m, float l, int row, uint32_t head, uint32_t q_heads,
                                        bool write_lse) {
    float total = l == 0.0f ? -__builtin_inff() : __builtin_amdgcn_logf(l) + (m - kLift);  // log2
    float y = l == 0.0f ? 0.0f : 1.0f / l;
    if (a.sinks) {
        const float own = total, sink = a.sinks[head] * 1.44269504f, top = fmaxf(own, sink);
        total = top + __builtin_amdgcn_logf(__builtin_amdgcn_exp2f(own - top) + __builtin_amdgcn_exp2f(sink - top));
        y *= __builtin_amdgcn_exp2f(own - total);
    }
    if (a.lse && write_lse) a.lse[(int64_t)row * q_heads + head] = total * 0.69314718f;
    return y;
}

// One workgroup: a row tile of 16 rows, one split of its tokens, four waves that take
// 64 tokens in turn and join their sums at the end.
template <int D, int TYPE>
__global__ __launch_bounds__(256, 2) void kv_attn_k(Cache c, Batch b, Attn a, Plan p, Rows Q, Rows O, int bf,
                                                    float* ws) {
    constexpr int C64 = D / 64, kHalf = D % 64 ? 1 : 0;  // 64-column pieces of a key, and a 32-column one
    constexpr int kPad = D + 4;
    __shared__ __attribute__((aligned(16))) float o_lds[4 * 16 * kPad];
    __shared__ float m_lds[4][16], l_lds[4][16];
    __shared__ int ids[kSegment / 16 + 1];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, g = lane >> 4;
    uint32_t id = blockIdx.x;
    const uint32_t h = id % c.heads;
    id /= c.heads;
    const uint32_t tile = id % p.tiles;
    id /= p.tiles;
    const uint32_t split = id % p.splits, seq = id / p.splits;
    const Seq s = sequence(b, c.page_log2, seq);
    const int row0 = (int)tile * 16, rows = s.n * (int)a.group;
    if (row0 >= rows) return;
    const Span sp = span_of(s, a, row0, 16);
    const int n_splits = splits_of(sp, (int)p.chunk);
    if ((int)split >= max(n_splits, 1)) return;
    const int lo = sp.lo + (int)(split * p.chunk), hi = (int)min((int64_t)sp.hi, (int64_t)lo + p.chunk);

    const int32_t* const table = b.pages + (uint64_t)seq * b.max_pages;

    // this lane's row
    const int row = row0 + r, tok = row / (int)a.group;
    const uint32_t head = h * a.group + (uint32_t)(row % (int)a.group), q_heads = c.heads * a.group;
    const bool there = row < rows;
    const int pos = s.len - s.n + tok;
    const int sees_hi = a.causal ? pos + 1 : s.len, sees_lo = a.window ? pos + 1 - (int)a.window : 0;

    // Q as the second operand of S^T, in fp16; bf16 rows go through a power of two
    f16x8 q[D / 32];
    float q_scale = a.scale_log2;
    {
        u32x4 raw[D / 32];
        const uint16_t* const x = static_cast<const uint16_t*>(Q.p) +
                                  (there ? (int64_t)(s.row0 + tok) * Q.row + (int64_t)head * Q.head : 0);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) {
            const int d = i < 2 * C64 ? i / 2 * 64 + g * 16 + i % 2 * 8 : C64 * 64 + g * 8;
            raw[i] = there ? *reinterpret_cast<const u32x4*>(x + d) : u32x4{};
        }
        if (bf) {
            uint32_t m = 0;
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) m = max(m, max(raw[i][j] & 0x7FFFu, raw[i][j] >> 16 & 0x7FFFu));
            m = across_rows_max(m);
            // largest magnitude into [2^14, 2^15); an infinity or NaN makes its row NaN anyway
            const int e = m >= 0x7F80u ? 0 : min(max(14 - ((int)(m >> 7) - 127), -126), 126);
            q_scale *= pow2f(-e);
            const float up = pow2f(e);
#pragma unroll
            for (int i = 0; i < D / 32; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    q[i][2 * j] = (_Float16)(bf2f((uint16_t)(raw[i][j] & 0xFFFF)) * up);
                    q[i][2 * j + 1] = (_Float16)(bf2f((uint16_t)(raw[i][j] >> 16)) * up);
                }
        } else {
#pragma unroll
            for (int i = 0; i < D / 32; ++i) q[i] = __builtin_bit_cast(f16x8, raw[i]);
        }
    }

    float m = kLowest, l = 0.0f;  // of the row; l: this lane's tokens alone
    f32x4 o[D / 16] = {};
    int page0 = 0;
    for (int base = lo; base < hi; base += 4 * kTile) {
        if (!((base - lo) % kSegment)) {  // the page ids of the next tokens
            __syncthreads();
            page0 = base >> c.page_log2;
            const int pages = ((min(hi, base + kSegment) - 1) >> c.page_log2) - page0 + 1;
            for (int i = tid; i < pages; i += 256) {
                const int v = table[page0 + i];
                ids[i] = (uint32_t)v < c.n_pages ? v : -1;
            }
            __syncthreads();
        }
        const int t0 = base + wave * kTile;
        if (t0 >= hi) continue;
        // the lane's blocks: of V and the scores, and of K
        const int tv = t0 + 16 * g, tk = t0 + 16 * (r >> 2);
        const int last = hi - 1;
        const int pv = ids[(min(tv, last) >> c.page_log2) - page0], pk = ids[(min(tk, last) >> c.page_log2) - page0];
        const uint8_t* const kp = c.k + code_offset(c, D, max(pk, 0), h, tk) + (r & 3) * D;
        const uint8_t* const vp = c.v + code_offset(c, D, max(pv, 0), h, tv) + r * 16;
        const uint64_t eo = exp_offset(c, max(pv, 0), h, tv);
        const int ke = (int)c.k_exp[eo] - 127, ve = (int)c.v_exp[eo] - 127;

        f32x4 st[4];
#pragma unroll
        for (int t = 0; t < 4; ++t) {
            st[t] = f32x4{0, 0, 0, 0};
#pragma unroll
            for (int i = 0; i < C64; ++i) {
                const u32x4 w = *reinterpret_cast<const u32x4*>(kp + t * 4 * D + i * 64 + g * 16);
                st[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_f16x8<TYPE>(w.x, w.y), q[2 * i], st[t], 0, 0, 0);
                st[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_f16x8<TYPE>(w.z, w.w), q[2 * i + 1], st[t], 0, 0, 0);
            }
            if constexpr (kHalf) {
                const u32x2 w = *reinterpret_cast<const u32x2*>(kp + t * 4 * D + C64 * 64 + g * 8);
                st[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_f16x8<TYPE>(w.x, w.y), q[2 * C64], st[t], 0, 0, 0);
            }
        }

        const float f = q_scale * pow2f(min(max(ke, -126), 127)), ev = (float)ve;
        float x[16], top = kLowest;
        // tokens in sight of the row, of the lane's 16
        const int from = sees_lo - tv, to = pv < 0 ? 0 : min(sees_hi, hi) - tv;
        const bool all = from <= 0 && to >= 16;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            x[i] = __builtin_fmaf(st[i / 4][i % 4], f, ev);
            if (!all && (i < from || i >= to)) x[i] = -__builtin_inff();
            top = fmaxf(top, x[i]);
        }
        top = fmaxf(across_rows_maxf(top), m);
        const float fade = __builtin_amdgcn_exp2f(m - top);
        m = top;
        float sum = 0.0f;
        f16x8 w[2];
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float y = __builtin_amdgcn_exp2f(x[i] - (m - kLift));
            sum += y;
            w[i / 8][i % 8] = (_Float16)y;
        }
        l = l * fade + sum * pow2f(min(max(-ve, -126), 127));
        // bytes of tokens that no length covers may hold anything, NaN among it
        const int valid = pv < 0 ? 0 : min(max(hi - tv, 0), 16);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) {
            u32x4 v = *reinterpret_cast<const u32x4*>(vp + i * 256);
            if (valid < 16) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int n = min(max(valid - 4 * j, 0), 4);
                    v[j] = n == 4 ? v[j] : v[j] & ((1u << 8 * n) - 1);
                }
            }
            o[i] *= fade;
            o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_f16x8<TYPE>(v.x, v.y), w[0], o[i], 0, 0, 0);
            o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes_f16x8<TYPE>(v.z, v.w), w[1], o[i], 0, 0, 0);
        }
    }

    // join the waves
    l = across_rows_sum(l);
    if (g == 0) {
        m_lds[wave][r] = m;
        l_lds[wave][r] = l;
    }
    __syncthreads();
    {
        float top = m_lds[0][r];
#pragma unroll
        for (int w = 1; w < 4; ++w) top = fmaxf(top, m_lds[w][r]);
        const float fade = __builtin_amdgcn_exp2f(m - top);
        float* const to = o_lds + (wave * 16 + r) * kPad;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) *reinterpret_cast<f32x4*>(to + i * 16 + g * 4) = o[i] * fade;
    }
    __syncthreads();
    for (int i = tid; i < 16 * (D / 4); i += 256) {
        const int rr = i / (D / 4), d = i % (D / 4) * 4, my_row = row0 + rr;
        if (my_row >= rows) break;
        f32x4 y = *reinterpret_cast<const f32x4*>(o_lds + rr * kPad + d);
        float top = m_lds[0][rr];
#pragma unroll
        for (int w = 1; w < 4; ++w) {
            y += *reinterpret_cast<const f32x4*>(o_lds + (w * 16 + rr) * kPad + d);
            top = fmaxf(top, m_lds[w][rr]);
        }
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) sum += l_lds[w][rr] * __builtin_amdgcn_exp2f(m_lds[w][rr] - top);
        const uint32_t hd = h * a.group + (uint32_t)(my_row % (int)a.group);
        const int at = s.row0 + my_row / (int)a.group;
        if (n_splits <= 1) {
            store4(O, at, hd, d, y * finish(a, top, sum, at, hd, q_heads, d == 0), bf);
        } else {
            // [row][split]: D sums, then m and l
            float* const part = ws + ((((uint64_t)seq * p.splits + split) * p.tiles + tile) * c.heads + h) * (16 * (D + 2)) + rr * D;
            *reinterpret_cast<f32x4*>(part + d) = y;
            if (d == 0) {
                float* const ml = part - rr * D + 16 * D + rr * 2;
                ml[0] = top;
                ml[1] = sum;
            }
        }
    }
}

// Joins the splits of one row and query head: four waves take every fourth split.
template <int D>
__global__ __launch_bounds__(256) void kv_join_k(Cache c, Batch b, Attn a, Plan p, Rows O, int bf, const float* ws) {
    __shared__ __attribute__((aligned(16))) float o_lds[4][D];
    __shared__ float l_lds[4];
    const uint32_t q_heads = c.heads * a.group, head = blockIdx.x % q_heads, h = head / a.group;
    const uint32_t j = blockIdx.x / q_heads % b.max_q, seq = blockIdx.x / q_heads / b.max_q;
    const Seq s = sequence(b, c.page_log2, seq);
    if ((int)j >= s.n) return;
    const int row = (int)(j * a.group + head % a.group), tile = row / 16;
    const int n = splits_of(span_of(s, a, tile * 16, 16), (int)p.chunk);
    if (n <= 1) return;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    constexpr int kPart = 16 * (D + 2);
    const float* const first = ws + (((uint64_t)seq * p.splits * p.tiles + tile) * c.heads + h) * kPart;
    const uint64_t step = (uint64_t)p.tiles * c.heads * kPart;
    float m = kLowest;
    for (int i = lane; i < n; i += 64) m = fmaxf(m, first[i * step + 16 * D + row % 16 * 2]);
#pragma unroll
    for (int i = 1; i < 64; i *= 2) m = fmaxf(m, __shfl_xor(m, i));
    float l = 0.0f, o[(D + 63) / 64] = {};
    for (int i = wave; i < n; i += 4) {
        const float* const part = first + i * step;
        const float f = __builtin_amdgcn_exp2f(part[16 * D + row % 16 * 2] - m);
        l += part[16 * D + row % 16 * 2 + 1] * f;
#pragma unroll
        for (int k = 0; k < (D + 63) / 64; ++k)
            if (k * 64 + lane < D) o[k] += part[row % 16 * D + k * 64 + lane] * f;
    }
#pragma unroll
    for (int k = 0; k < (D + 63) / 64; ++k)
        if (k * 64 + lane < D) o_lds[wave][k * 64 + lane] = o[k];
    if (lane == 0) l_lds[wave] = l;
    __syncthreads();
    if ((int)threadIdx.x < D / 4) {
        const int d = (int)threadIdx.x * 4, at = s.row0 + (int)j;
        f32x4 y = {0, 0, 0, 0};
        l = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            y += *reinterpret_cast<const f32x4*>(&o_lds[w][d]);
            l += l_lds[w];
        }
        store4(O, at, head, d, y * finish(a, m, l, at, head, q_heads, d == 0), bf);
    }
}

}  // namespace kv
}  // namespace kq
