// kq_kv_rows_kernel.h -- attention over the 8-bit cache, many rows: the kernel of
// kq_kv_attn_<D>.hip for prompts and chunks: calls of more than 64 rows a sequence and head.
//
// A workgroup of NW waves takes 32 NW rows (query tokens x the heads of a group) of a sequence
// and head, 64 tokens at a time. The tokens' codes become fp16 once for all its waves, in
// LDS, on their way to 32x32x16 MFMAs; like the kernel for few rows it computes S^T = K Q^T and
// O^T = V^T P^T, so that probabilities stay in the lanes that computed them: lane (n, g), n =
// lane % 32, g = lane / 32, receives of a 32-token operand the places 8a + 4g + b (a, b < 4),
// where tokens 16g + 4a + b stand -- 16 tokens with one exponent, in order.
#pragma once
#include "kq_kv_attn_kernel.h"

namespace kq {
namespace kv {

typedef float f32x16v __attribute__((ext_vector_type(16)));

constexpr int kRowIds = 1024;  // page ids held at a time

// Codes of 64 tokens in LDS as fp16. K: [D/8][64 + 1 places][8] (the odd place spreads the
// writers of a token over the banks); V: [64/8][D][8].
template <int D>
struct RowTile {
    _Float16 k[D / 8 * 65 * 8];
    _Float16 v[8 * D * 8];
    int exps[8];  // exponent bytes of the four 16-token blocks: K's (-1: no page), V's (kBase: no page or token)
};

template <int D, int TYPE, int NW>
__global__ __launch_bounds__(64 * NW, D >= 192 ? 1 : 2) void kv_rows_k(Cache c, Batch b, Attn a, RowPlan p, Rows Q, Rows O,
                                                                       int bf, float* ws) {
    constexpr int T = 64 * NW, RT = 32 * NW;
    constexpr int kPieces = 64 * D / 16, kEach = (kPieces + T - 1) / T;  // 16-byte pieces of K (and of V); a thread's
    __shared__ __attribute__((aligned(16))) RowTile<D> tiles[2];
    __shared__ int ids[kRowIds];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = lane & 31, g = lane >> 5;
    // heads fastest: the row tiles of a head meet in one XCD's cache where there are eight heads.
    // The last tiles, with the most tokens to see, first.
    uint32_t id = blockIdx.x;
    const uint32_t h = id % c.heads;
    id /= c.heads;
    const uint32_t tile = p.tiles - 1 - id % p.tiles;
    id /= p.tiles;
    const uint32_t split = id % p.splits, seq = id / p.splits;
    const Seq s = sequence(b, c.page_log2, seq);
    const int row0 = (int)tile * RT, rows = s.n * (int)a.group;
    if (row0 >= rows) return;
    const Span sp = span_of<false>(s, a, row0, RT);
    const int n_splits = row_splits(sp, (int)p.chunk);
    if ((int)split >= max(n_splits, 1)) return;
    const int lo = sp.lo + (int)(split * p.chunk), hi = (int)min((int64_t)sp.hi, (int64_t)lo + p.chunk);
    const int32_t* const table = b.pages + (uint64_t)seq * b.max_pages;

    // a row that there is not sees what the last one does: it takes no tile off the short way
    const int row = min(row0 + wave * 32 + n, rows - 1), tok = row / (int)a.group;
    const uint32_t q_heads = c.heads * a.group, head = h * a.group + (uint32_t)(row % (int)a.group);
    const bool there = row0 + wave * 32 + n < rows;
    const int pos = s.len - s.n + tok;
    const int sees_hi = row0 + wave * 32 < rows ? min(a.causal ? pos + 1 : s.len, hi) : 0, sees_lo = a.window ? pos + 1 - (int)a.window : 0;

    // Q as the second operand: 8 of each 16 columns
    f16x8 q[D / 16];
    int q_exp = 0;  // undoes the power of two of a bf16 row
    {
        u32x4 raw[D / 16];
        const uint16_t* const x = static_cast<const uint16_t*>(Q.p) +
                                  (there ? (int64_t)(s.row0 + tok) * Q.row + (int64_t)head * Q.head : 0);
#pragma unroll
        for (int i = 0; i < D / 16; ++i)
            raw[i] = there ? signed16(*reinterpret_cast<const u32x4*>(x + i * 16 + g * 8), a.scale_log2) : u32x4{};
        if (bf) {
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) top = max(top, max(raw[i][j] & 0x7FFFu, raw[i][j] >> 16 & 0x7FFFu));
            const auto both = __builtin_amdgcn_permlane32_swap(top, top, false, false);
            const int e = bf_lift(max(both[0], both[1]));
            const float up = pow2f(e);
            q_exp = -e;
#pragma unroll
            for (int i = 0; i < D / 16; ++i) q[i] = bf_f16x8(raw[i], up);
        } else {
#pragma unroll
            for (int i = 0; i < D / 16; ++i) q[i] = __builtin_bit_cast(f16x8, raw[i]);
        }
    }

    int page0 = 0, page1 = 0;  // ids holds the table's [page0, page1)
    u32x4 kc[kEach], vc[kEach];
    int valid[kEach];  // tokens of the piece's block that there are
    int ex = 0;
    auto page_at = [&](int t) { return ids[(min(t, hi - 1) >> c.page_log2) - page0]; };
    // Tokens t0 .. t0 + 63 on their way into registers.
    auto load = [&](int t0) {
        const int last = (min(t0 + 64, hi) - 1) >> c.page_log2;
        if (last >= page1) {  // the next page ids (the same for every thread)
            __syncthreads();
            page0 = t0 >> c.page_log2;
            page1 = min(page0 + kRowIds, ((hi - 1) >> c.page_log2) + 1);
            for (int i = page0 + tid; i < page1; i += T) {
                const int v = table[i];
                ids[i - page0] = (uint32_t)v < c.n_pages ? v : -1;
            }
            __syncthreads();
        }
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int i = tid + e * T;
            if (kPieces % T == 0 || i < kPieces) {
                // 16-byte piece i % D of block i / D, of K and of V; the block is the wave's, but for 96 columns
                const int in = i / D * 16, t = t0 + (D % 64 ? in : __builtin_amdgcn_readfirstlane(in));
                int page = page_at(t);
                if (D % 64 == 0) page = __builtin_amdgcn_readfirstlane(page);
                const uint64_t off = code_offset(c, D, max(page, 0), h, t);
                kc[e] = *reinterpret_cast<const u32x4*>(c.k + off + i % D * 16);
                vc[e] = *reinterpret_cast<const u32x4*>(c.v + off + i % D * 16);
                valid[e] = page < 0 ? 0 : hi - t;
            }
        }
        if (tid < 8) {
            const int t = t0 + (tid & 3) * 16, page = page_at(t);
            const uint64_t at = exp_offset(c, max(page, 0), h, t);
            ex = tid < 4 ? page < 0 ? -1 : (int)c.k_exp[at] : page < 0 || t >= hi ? kBase : (int)c.v_exp[at];
        }
    };
    // ... and out of them.
    auto store = [&](RowTile<D>& to) {
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int i = tid + e * T;
            if (kPieces % T == 0 || i < kPieces) {
                const int t = i / (D / 16), col = i % (D / 16);
                // token 16g + 4a + b of 32 stands at place 8a + 4g + b
                const int place = (t & 32) + (t >> 2 & 3) * 8 + (t >> 4 & 1) * 4 + (t & 3);
                _Float16* const k = to.k + (2 * col * 65 + place) * 8;
                *reinterpret_cast<f16x8*>(k) = codes_f16x8<TYPE>(kc[e].x, kc[e].y);
                *reinterpret_cast<f16x8*>(k + 65 * 8) = codes_f16x8<TYPE>(kc[e].z, kc[e].w);
                // bytes of tokens that no length covers, or of no page, may hold anything, NaN among it
                if (valid[e] < 16) {
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int keep = min(max(valid[e] - 4 * j, 0), 4);
                        vc[e][j] = keep == 4 ? vc[e][j] : vc[e][j] & ((1u << 8 * keep) - 1);
                    }
                }
                _Float16* const v = to.v + (i / D * 2 * D + i % D) * 8;
                *reinterpret_cast<f16x8*>(v) = codes_f16x8<TYPE>(vc[e].x, vc[e].y);
                *reinterpret_cast<f16x8*>(v + D * 8) = codes_f16x8<TYPE>(vc[e].z, vc[e].w);
            }
        }
        if (tid < 8) to.exps[tid] = ex;
    };

    float m = kLowest, l = 0.0f;
    int base = kBase;  // of l
    f32x16v o[D / 32] = {};
    auto compute = [&](int t0, const RowTile<D>& in) {
        if (!__any(t0 < sees_hi && t0 + 64 > sees_lo)) return;  // no token of it in sight of the wave
        f32x16v st[2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            st[u] = f32x16v{};
#pragma unroll
            for (int i = 0; i < D / 16; ++i)
                st[u] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                    *reinterpret_cast<const f16x8*>(in.k + ((2 * i + g) * 65 + u * 32 + n) * 8), q[i], st[u], 0, 0, 0);
        }
        const int k0 = in.exps[g], k1 = in.exps[2 + g], v0 = in.exps[4 + g], v1 = in.exps[6 + g];
        // t = f s + e with f >= 0: the largest t of a block is its largest s's
        float f[2] = {score_factor(a, k0, q_exp), score_factor(a, k1, q_exp)};
        float e[2] = {(float)(v0 - 127), (float)(v1 - 127)};
        if (!__all(t0 + 64 <= sees_hi && t0 >= sees_lo && k0 >= 0 && k1 >= 0)) {
            // only the few tiles that need it: nothing of this is computed ahead of the branch
            int first = sees_lo - t0 - 16 * g;
            asm volatile("" : "+v"(first));
            const int end = first + sees_hi - sees_lo;
#pragma unroll
            for (int u = 0; u < 2; ++u) {
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    const int t = 32 * u + i;
                    st[u][i] = t < first || t >= end || (u ? k1 : k0) < 0 ? -__builtin_inff()
                                                                         : __builtin_fmaf(st[u][i], f[u], e[u]);
                }
                f[u] = 1.0f;
                e[u] = 0.0f;
            }
        }
        float top = m;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float most = st[u][0];
#pragma unroll
            for (int i = 1; i < 16; ++i) most = fmaxf(most, st[u][i]);
            top = fmaxf(top, __builtin_fmaf(most, f[u], e[u]));
        }
        {
            float x, y;
            swapped<true>(top, x, y);
            top = fmaxf(x, y);
        }
        if (__any(top > m + kSlack)) {
            const float fade = __builtin_amdgcn_exp2f(m - top);
            m = top;
            l *= fade;
#pragma unroll
            for (int i = 0; i < D / 32; ++i) o[i] *= fade;
        }
        if (__any(base_far(base, v0) || base_far(base, v1))) {
            const int to = base_near(base, min(v0, v1), max(v0, v1));
            l = __builtin_ldexpf(l, to - base);
            base = to;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const float down = e[u] - (m - kLift);
            f16x8 w[2];
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(st[u][i], f[u], down));
                sum += y;
                w[i / 8][i % 8] = (_Float16)y;
            }
            l += sum * pow2f(base - (u ? v1 : v0));
#pragma unroll
            for (int hh = 0; hh < 2; ++hh)
#pragma unroll
                for (int i = 0; i < D / 32; ++i)
                    o[i] = __builtin_amdgcn_mfma_f32_32x32x16_f16(
                        *reinterpret_cast<const f16x8*>(in.v + ((4 * u + 2 * g + hh) * D + 32 * i + n) * 8), w[hh], o[i], 0, 0, 0);
        }
    };

    if (lo < hi) {
        load(lo);
        store(tiles[0]);
        if (lo + 64 < hi) load(lo + 64);
        __syncthreads();
        int cur = 0;
        for (int t0 = lo; t0 < hi; t0 += 64, cur ^= 1) {
            compute(t0, tiles[cur]);
            if (t0 + 64 < hi) {
                store(tiles[cur ^ 1]);
                if (t0 + 128 < hi) load(t0 + 128);
            }
            __syncthreads();
        }
    }

    if (!there) return;
    {
        float x, y;
        swapped<true>(l, x, y);
        l = x + y;
    }
    const int at = s.row0 + tok;
    if (n_splits <= 1) {
        const float y = finish(a, m, l, base, at, head, q_heads, g == 0);
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                store4(O, at, head, i * 32 + j * 8 + g * 4,
                       from_base(f32x4{o[i][4 * j] * y, o[i][4 * j + 1] * y, o[i][4 * j + 2] * y, o[i][4 * j + 3] * y}, base), bf);
    } else {
        float* const part = ws + ((((uint64_t)seq * p.splits + split) * p.tiles + tile) * c.heads + h) * (RT * (D + kRowSum));
        float* const to = part + (row - row0) * D;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<f32x4*>(to + i * 32 + j * 8 + g * 4) =
                    f32x4{o[i][4 * j], o[i][4 * j + 1], o[i][4 * j + 2], o[i][4 * j + 3]};
        if (g == 0) *reinterpret_cast<RowSum*>(part + RT * D + (row - row0) * kRowSum) = {m, l, base, 0};
    }
}

// Adds up the splits of kv_rows_k: a wave takes one (token, query head).
template <int D>
__global__ __launch_bounds__(256) void kv_rows_join_k(Cache c, Batch b, Attn a, RowPlan p, Rows O, int bf, const float* ws) {
    const uint32_t q_heads = c.heads * a.group, id = blockIdx.x * 4 + (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t head = id % q_heads, h = head / a.group, j = id / q_heads % b.max_q, seq = id / q_heads / b.max_q;
    if (seq >= b.n_seq) return;
    const Seq s = sequence(b, c.page_log2, seq);
    if ((int)j >= s.n) return;
    const int RT = (int)p.rows, row = (int)(j * a.group + head % a.group), tile = row / RT, in = row % RT;
    const int n = row_splits(span_of<false>(s, a, tile * RT, RT), (int)p.chunk);
    if (n <= 1) return;
    const uint64_t size = (uint64_t)RT * (D + kRowSum);
    const float* const first = ws + (((uint64_t)seq * p.splits * p.tiles + tile) * c.heads + h) * size;
    const uint64_t step = (uint64_t)p.tiles * c.heads * size;
    join_row<D, 1>(a, n, [&](int i) { return first + i * step + in * D; },
                   [&](int i) { return first + i * step + RT * D + in * kRowSum; }, nullptr, O, bf, s.row0 + (int)j, head, q_heads);
}

template <int D, int TYPE>
hipError_t rows_d(const Cache& c, const Batch& b, const Attn& a, const RowPlan& p, const Rows& Q, const Rows& O, bool bf,
                  float* ws, hipStream_t s) {
    const uint32_t wgs = b.n_seq * p.splits * p.tiles * c.heads;
    if constexpr (row_most(D) > 128) {
        if (p.rows > 128) kv_rows_k<D, TYPE, 8><<<wgs, 512, 0, s>>>(c, b, a, p, Q, O, bf, ws);
        else kv_rows_k<D, TYPE, 4><<<wgs, 256, 0, s>>>(c, b, a, p, Q, O, bf, ws);
    } else {
        kv_rows_k<D, TYPE, 4><<<wgs, 256, 0, s>>>(c, b, a, p, Q, O, bf, ws);
    }
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits == 1) return e;
    kv_rows_join_k<D><<<(b.n_seq * b.max_q * c.heads * a.group + 3) / 4, 256, 0, s>>>(c, b, a, p, O, bf, ws);
    return hipGetLastError();
}

}  // namespace kv
}  // namespace kq
