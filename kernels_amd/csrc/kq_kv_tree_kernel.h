// kq_kv_tree_kernel.h -- attention of trees over the 8-bit cache, many rows: what kq_kv_tree_<D>.hip runs where a
// sequence and head has more than 64 rows (few rows: kv_few_k).
//
// A tree's rows all see the whole of their sequence, and there are few of them for its length: a row of work (a
// sequence and head) is one or a few tiles of 128 or 256 rows over thousands of tokens. So the tokens are shared out
// as they are for few rows: equal parts or shares of all units of 64 tokens, whatever the lengths.
//
// The products are laid out as in kv_rows_k (32 rows a wave, S^T = K Q^T, O^T = V^T P^T, codes made fp16 once for all
// waves, in LDS). Unlike there no lane is ever masked off on the way: a row that there is not computes what the tile's last
// one does, loads beyond an end are of the last element again. (Copies that the compiler makes of registers where
// lanes meet again behind a branch have been of the masked lanes alone, in kernels that need more than 256 registers.)
//
// What bounds it is time that two waves a SIMD (some 220 registers) leave open. By counters, of a wave's time a half is waits for loads,
// for LDS and for the others at each tile's barrier (60 rows over 131072 tokens: 50%, 16 trees of 33 to 64 rows: 56), a seventh
// waits for the issue, a third issues (35, 29). No unit is full: matrix products 39% of a SIMD's time (30), vector instructions 50 (40), LDS
// 28 (24, a tenth of it bank conflicts). Those 16 trees, over 300 to 12000 tokens, 64 heads over 8 of 128, take 177 us, 27 of
// them the join (96 GFLOP; a large matrix product's rate would take 77; of their waves 22%, weighted by tokens, have no rows); 60 rows over
// 131072 tokens, 32 heads over 8 of 128: 176, 8 of them the join (129 GFLOP, 103). A 32x32x16 product keeps its unit for 32 cycles and
// the issue for 11, a vector instruction the issue for 4, an exponential 8.
//
// Probabilities are rounded to fp16 for their product with V (2^-11 of each at most), as in kv_rows_k: codes are exact in fp16, whose products run
// at sixteen times the rate of 32-bit ones. Sums, statistics and the denominator, which adds up what was not rounded, are 32 bits. Against 64 bits outputs
// are off by 0.16390% of their size over those 16 trees, bf16, of which the output's own rounding is 0.1636; 0.16074 over the long sequence, of 0.1607;
// in fp16 (26 rows over 701 tokens) 0.0207, of 0.0205.
// Left out one at a time, products, loads from LDS and loads from memory are worth about a tenth each, exponentials
// nothing. No faster: the next keys' product beside the exponentials (180 us against 182), three tiles in LDS, half of
// the waves half a tile ahead, 64 rows a wave with one wave a SIMD (250).
#pragma once
#include "kq_kv_rows_kernel.h"

namespace kq {
namespace kv {

// Rows row0 .. of a sequence and head (of its `rows`), 32 a wave, over the tokens [lo, hi), lo a multiple of 64. Then, in
// the waves that have rows, then(row, tok, head, g, m, l, base, o): the lane's row, with the reference, the denominator,
// its base, and the lane's share of the sums.
template <int D, int TYPE, int NW, class Then>
__device__ __forceinline__ void tree_piece(const Cache& c, const Batch& b, const Attn& a, const Rows& Q, int bf, const Seq& s, int seq,
                                           uint32_t h, int row0, int rows, int lo, int hi, RowTile<D>* tiles, int* ids, Then then) {
    constexpr int T = 64 * NW;
    constexpr int kPieces = 64 * D / 16, kEach = (kPieces + T - 1) / T;  // 16-byte pieces of K (and of V); a thread's
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), n = lane & 31, g = lane >> 5;
    const int32_t* const table = b.pages + (uint64_t)seq * b.max_pages;
    const bool busy = row0 + wave * 32 < rows;  // the same for all lanes
    const int row = min(row0 + wave * 32 + n, rows - 1), tok = row / (int)a.group;
    const uint32_t head = h * a.group + (uint32_t)(row % (int)a.group);
    // the tokens before the first row, from a window on; of those from it on the row's bits
    const int first_row = s.len - s.n, before = min(max(first_row, 0), hi);
    const uint32_t* const mask = a.mask + (uint64_t)(uint32_t)(s.row0 + tok) * a.words;
    const int32_t at_pos = a.window ? a.pos[s.row0 + tok] : 0;

    int page0 = 0, page1 = 0;  // ids holds the table's [page0, page1)
    u32x4 kc[kEach], vc[kEach];
    int valid[kEach];  // tokens of the piece's block that there are
    constexpr int kOwn = -2;
    int ex = 0, instead = kOwn;  // an exponent's byte, and what stands in its place
    auto page_at = [&](int t) { return ids[(min(t, hi - 1) >> c.page_log2) - page0]; };
    // Tokens t0 .. t0 + 63 on their way into registers.
    auto load = [&](int t0) {
        const int last = (min(t0 + 64, hi) - 1) >> c.page_log2;
        if (last >= page1) {  // the next page ids (the same for every thread)
            __syncthreads();
            page0 = t0 >> c.page_log2;
            page1 = min(page0 + kRowIds, ((hi - 1) >> c.page_log2) + 1);
            for (int from = page0; from < page1; from += T) {
                const int i = min(from + tid, page1 - 1), id = table[i];
                ids[i - page0] = (uint32_t)id < c.n_pages ? id : -1;
            }
            __syncthreads();
        }
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            // 16-byte piece i % D of block i / D, of K and of V; the block is the wave's, but for 96 columns
            const int i = min(tid + e * T, kPieces - 1), in = i / D * 16, t = t0 + (D % 64 ? in : __builtin_amdgcn_readfirstlane(in));
            int page = page_at(t);
            if (D % 64 == 0) page = __builtin_amdgcn_readfirstlane(page);
            const uint64_t off = code_offset(c, D, max(page, 0), h, t);
            kc[e] = *reinterpret_cast<const u32x4*>(c.k + off + i % D * 16);
            vc[e] = *reinterpret_cast<const u32x4*>(c.v + off + i % D * 16);
            valid[e] = page < 0 ? 0 : hi - t;
        }
        if (wave == 0) {
            // eight exponents: four blocks' of K (-1: no page), then of V (kBase: no page or token)
            const int t = t0 + (tid & 3) * 16, page = page_at(t);
            ex = (tid & 4 ? c.v_exp : c.k_exp)[exp_offset(c, max(page, 0), h, t)];
            const bool none = page < 0, neither = none | (t >= hi);
            const int for_k = none ? -1 : kOwn, for_v = neither ? kBase : kOwn;
            instead = tid & 4 ? for_v : for_k;
        }
    };
    // ... and out of them.
    auto store = [&](RowTile<D>& to) {
#pragma unroll
        for (int e = 0; e < kEach; ++e) {
            const int i = min(tid + e * T, kPieces - 1), t = i / (D / 16), col = i % (D / 16);
            // token 16g + 4a + b of 32 stands at place 8a + 4g + b
            const int place = (t & 32) + (t >> 2 & 3) * 8 + (t >> 4 & 1) * 4 + (t & 3);
            _Float16* const k = to.k + (2 * col * 65 + place) * 8;
            *reinterpret_cast<f16x8*>(k) = codes_f16x8<TYPE>(kc[e].x, kc[e].y);
            *reinterpret_cast<f16x8*>(k + 65 * 8) = codes_f16x8<TYPE>(kc[e].z, kc[e].w);
            // bytes of tokens that no length covers, or of no page, may hold anything, NaN among it
            if (D % 64 ? __any(valid[e] < 16) : valid[e] < 16) {
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
        if (wave == 0) to.exps[tid & 7] = instead == kOwn ? ex : instead;
    };

    // Q as the second operand, 8 of each 16 columns: asked for all at once, while the first codes are on their way
    f16x8 q[D / 16];
    int q_exp = 0;  // undoes the power of two of a bf16 row
    auto load_q = [&]() {
        u32x4 raw[D / 16];
        const uint16_t* const x = static_cast<const uint16_t*>(Q.p) + (int64_t)(s.row0 + tok) * Q.row + (int64_t)head * Q.head + g * 8;
#pragma unroll
        for (int i = 0; i < D / 16; ++i) raw[i] = *reinterpret_cast<const u32x4*>(x + i * 16);
#pragma unroll
        for (int i = 0; i < D / 16; ++i) raw[i] = signed16(raw[i], a.scale_log2);
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
    };

    float m = kLowest, l = 0.0f;
    int base = kBase;  // of l
    f32x16v o[D / 32] = {};
    const int sees_lo = a.window ? max(at_pos, first_row) + 1 - (int)a.window : 0;
    auto compute = [&](int t0, const RowTile<D>& in) {
        if (!busy || !__any(t0 + 64 > min(sees_lo, first_row))) return;  // no token of it in sight of the wave
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
        if (!__all(t0 + 64 <= before && t0 >= sees_lo && k0 >= 0 && k1 >= 0)) {
            // only the few tiles that need it: nothing of this is computed ahead of the branch
            int t = t0 + 16 * g;
            asm volatile("" : "+v"(t));
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint32_t any = tree_bits(mask, (int)a.words, t + 32 * u, first_row, sees_lo, hi);
                const uint32_t sees = (u ? k1 : k0) < 0 ? 0u : any;
#pragma unroll
                for (int i = 0; i < 16; ++i) st[u][i] = sees >> i & 1 ? __builtin_fmaf(st[u][i], f[u], e[u]) : -__builtin_inff();
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
                w[i / 8][i % 8] = (_Float16)y;  // what the product takes (above)
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
        load_q();
        store(tiles[0]);
        load(lo + 64);  // beyond the end: blocks of the last page, which nothing takes out of the registers
        __syncthreads();
        int cur = 0, t0 = lo;
        for (; t0 + 64 < hi; t0 += 64, cur ^= 1) {
            compute(t0, tiles[cur]);
            store(tiles[cur ^ 1]);
            load(t0 + 128);
            __syncthreads();
        }
        compute(t0, tiles[cur]);
    }
    if (!busy) return;
    float x, y;
    swapped<true>(l, x, y);
    then(row, tok, head, g, m, x + y, base, o);
}

template <int D, int TYPE, int NW>
__global__ __launch_bounds__(64 * NW, D >= 192 ? 1 : 2) void kv_tree_rows_k(Cache c, Batch b, Attn a, FewPlan p, Rows Q, Rows O, int bf,
                                                                            float* ws) {
    constexpr int RT = 32 * NW;
    __shared__ __attribute__((aligned(16))) RowTile<D> tiles[2];
    __shared__ int ids[kRowIds];
    static_assert(kRowIds >= kScan, "units of the sequences");
    const uint32_t q_heads = c.heads * a.group;
    // an eighth of the groups, one behind the other, in each of eight XCDs, and a group's workgroups side by side
    const uint32_t group = blockIdx.x % 8 * ((p.groups + 7) / 8) + blockIdx.x / 8 / p.tiles, tile = blockIdx.x / 8 % p.tiles;
    const int row0 = (int)tile * RT;
    const Share share = share_of<true, 1>(c, b, a, p, group, 0, ids);
    Cut* const cuts = reinterpret_cast<Cut*>(ws);
    if (p.mode == FewPlan::kShares && !p.by_row && group < p.groups && tile == 0 && threadIdx.x == 0) cuts[group].parts = 0;
    int left = share.units, unit = share.unit, seq = share.seq;
    uint32_t h = share.head;
    uint64_t at = share.at;
    while (left > 0) {
        seq = __builtin_amdgcn_readfirstlane(seq);
        h = (uint32_t)__builtin_amdgcn_readfirstlane((int)h);
        const Seq s = sequence(b, c.page_log2, (uint32_t)seq);
        const Span sp = span_of<true>(s, a, 0, 0);
        const int units = units_of<true>(s, a, 0, (int)p.start), mine = min(left, units - unit);
        if (mine <= 0) {  // a sequence without rows
            ++seq;
            continue;
        }
        const int rows = s.n * (int)a.group, tail = (int)p.start;
        const int lo = sp.lo + max(unit - tail, 0) * kTile;
        const int hi = (int)min((int64_t)sp.hi, (int64_t)sp.lo + (int64_t)max(unit + mine - tail, 0) * kTile);
        const bool whole = mine == units;
        if (row0 < rows) {
            __syncthreads();  // the piece before is done with what LDS holds
            float* const part = slot_of<D, RT / 16>(ws, p, 2 * group + (unit == 0), tile);
            tree_piece<D, TYPE, NW>(c, b, a, Q, bf, s, seq, h, row0, rows, lo, hi, tiles, ids,
                                    [&](int row, int tok, uint32_t head, int g, float m, float l, int base, const f32x16v (&o)[D / 32]) {
                const int at_row = s.row0 + tok;
                float* const to = part + (row - row0) * D;
                if (whole) {
                    const float y = finish(a, m, l, base, at_row, head, q_heads, g == 0);
#pragma unroll
                    for (int i = 0; i < D / 32; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            store4(O, at_row, head, i * 32 + j * 8 + g * 4,
                                   from_base(f32x4{o[i][4 * j] * y, o[i][4 * j + 1] * y, o[i][4 * j + 2] * y, o[i][4 * j + 3] * y}, base), bf);
                } else {
#pragma unroll
                    for (int i = 0; i < D / 32; ++i)
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            *reinterpret_cast<f32x4*>(to + i * 32 + j * 8 + g * 4) =
                                f32x4{o[i][4 * j], o[i][4 * j + 1], o[i][4 * j + 2], o[i][4 * j + 3]};
                    *reinterpret_cast<RowSum*>(part + RT * D + (row - row0) * kRowSum) = {m, l, base, 0};
                }
            });
        }
        if (unit == 0 && tile == 0 && threadIdx.x == 0 && p.mode != FewPlan::kRows && (p.by_row || mine < units)) {
            int parts = share.parts;
            if (p.mode == FewPlan::kShares) parts = (int)(((at + (uint64_t)units) * share.groups - 1) / share.total) - (int)group + 1;
            cuts[p.by_row ? (uint32_t)seq * c.heads + h : group] = {seq, (int)h, (int)group, whole ? 0 : parts};
        }
        left -= mine;
        at += (uint64_t)mine;
        unit = 0;
        if (++h == c.heads) h = 0, ++seq;
    }
}

template <int D, int TYPE, int NW>
hipError_t tree_rows_n(const Cache& c, const Batch& b, const Attn& a, const FewPlan& p, const Rows& Q, const Rows& O, bool bf,
                       float* ws, hipStream_t s) {
    constexpr int R = 2 * NW;
    kv_tree_rows_k<D, TYPE, NW><<<(p.groups + 7) / 8 * 8 * p.tiles, 64 * NW, 0, s>>>(c, b, a, p, Q, O, bf, ws);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.mode == FewPlan::kRows) return e;
    const uint32_t rows = b.max_q * a.group;
    // many parts a row of work, and rows few enough: four waves for each of its rows
    if (p.groups >= 8 * p.cuts && rows <= 65535) kv_join_k<D, R, 4><<<dim3(p.cuts, rows), 256, 0, s>>>(c, b, a, p, O, bf, ws);
    else kv_join_k<D, R, 1><<<dim3(p.cuts, (rows + 3) / 4), 256, 0, s>>>(c, b, a, p, O, bf, ws);
    return hipGetLastError();
}

template <int D, int TYPE>
hipError_t tree_rows_d(const Cache& c, const Batch& b, const Attn& a, const FewPlan& p, const Rows& Q, const Rows& O, bool bf,
                       float* ws, hipStream_t s) {
    if constexpr (row_most(D) > 128)
        if (p.sixteens > 8) return tree_rows_n<D, TYPE, 8>(c, b, a, p, Q, O, bf, ws, s);
    return tree_rows_n<D, TYPE, 4>(c, b, a, p, Q, O, bf, ws, s);
}

}  // namespace kv
}  // namespace kq
