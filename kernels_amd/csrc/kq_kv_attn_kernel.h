// kq_kv_attn_kernel.h -- attention over the 8-bit cache, few rows: the wave
// kernel of kq_kv_attn.hip.
//
// A wave takes 64 tokens at a time against 16 or 32 rows (query tokens x the heads of a
// group) of one sequence and head, of up to 64. Both products are 16x16x32 fp16 MFMAs on
// transposed results, so that nothing moves between lanes:
//   S^T = K Q^T: lane (r = lane % 16, g = lane / 16) receives tokens 4g..4g+3 of a
//         16-token operand, for row r. Which tokens stand in an operand is
//         free: operand t (of 4) holds token 16 (i / 4) + 4t + i % 4 at place i,
//         so that lane (r, g) ends with the tokens 16g..16g+15, one exponent.
//   O^T = V^T P^T: the lane's 16 probabilities are two operands as they are
//         (k place 8g + j <-> token 16g + 8h + j), and the matching V operand is
//         the 16 bytes that hold column d of the lane's 16 tokens.
// With t_p = log2(e) s_p + e_v(p), the probabilities and V's scale are one number
// w_p = 2^(t_p - m); the denominator is the sum of w_p 2^-e_v(p), kept times a power of two
// where float32's range asks for it.
#pragma once
#include "kq_kv_device.h"

namespace kq {
namespace kv {

constexpr int kTile = 64;      // tokens a wave takes at a time
constexpr int kRound = 256;    // ... and four waves do
// A row's sums go by a reference m that its largest t exceeds by kSlack at most: it moves, and the sums with
// it, only where it would be by more (with every new maximum the sums of 32 rows moved in most
// tiles of 64 tokens). Probabilities are scaled by 2^kLift, so that the fp16 ones lie below 2^15 and stay
// normal down to 2^-25 of the reference.
constexpr int kLift = 11;
constexpr float kSlack = 4.0f;
constexpr int kIds = 4096;     // page ids that a workgroup holds at a time
constexpr int kScan = 1024;    // most sequences whose lengths a workgroup adds up
constexpr float kLowest = -3.0e38f;  // reference before any token

// The denominator's terms w 2^(127 - byte), of V's bytes, lie between 2^11 2^-128 and 2^15 2^127, which float32 does not
// hold: a wave keeps their sums l times 2^(base - 127), the base a byte. It is 127, and moves, l with it, only where a
// block's byte is more than 64 below it (2^31 such tokens' sum is finite) or more than 110 above (a term of the row's largest
// is normal): never for bytes from 63 to 237, and to 64 or 145 at most. What that costs: up to 1% (131071 tokens, 64 / 8
// heads of 128: 56.9 us in a graph, 56.7 without; a prefill of 4 prompts, 64 wide: 167, 167), but 3% for many short
// sequences 64 wide, whose kernel goes from 126 to 130 registers (73 of 100 to 1795 tokens: 28.4 us, 27.5 without).
constexpr int kBase = 127;
__device__ __forceinline__ bool base_far(int base, int byte) { return (uint32_t)(base + 110 - byte) > 174u; }
// The base that suits the bytes low .. high of the wave's lanes (which differ by 100 at most).
__device__ __forceinline__ int base_near(int base, int low, int high) {
    low = (int)~wave_max(~(uint32_t)low);
    high = (int)wave_max((uint32_t)high);
    return __builtin_amdgcn_readfirstlane(min(max(base, high - 110), low + 64));
}
// What a row's parts are joined by.
struct alignas(16) RowSum {
    float m, l;
    int base, unused;
};
constexpr int kRowSum = sizeof(RowSum) / sizeof(float);

// Tokens that rows row .. row + rows - 1 of a sequence and head see: [lo, hi), lo a multiple of 64.
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

__device__ __forceinline__ int row_splits(const Span& v, int chunk) {
    return v.hi > v.lo ? (v.hi - v.lo - 1) / chunk + 1 : 0;
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
// multiplied by, before 2^(base - 127). m, l and base as the waves keep them: l = 2^(base - 127) sum 2^(s log2e + kLift - m).
__device__ __forceinline__ float finish(const Attn& a, float m, float l, int base, int row, uint32_t head, uint32_t q_heads,
                                        bool write_lse) {
    float total = l == 0.0f ? -__builtin_inff() : __builtin_amdgcn_logf(l) + (m - kLift) - (float)(base - 127);  // log2
    float y = l == 0.0f ? 0.0f : 1.0f / l;
    float lse = total * 0.69314718f;
    if (a.sinks) {
        const float own = total, given = a.sinks[head], sink = given * 1.44269504f, top = fmaxf(own, sink);
        // no token in sight and a sink of (about) -inf, or a sink that takes all; a NaN stays one
        if (__builtin_isinf(top) && own == own) {
            lse = given;
            y = 0.0f;
        } else {
            total = top + __builtin_amdgcn_logf(__builtin_amdgcn_exp2f(own - top) + __builtin_amdgcn_exp2f(sink - top));
            lse = total * 0.69314718f;
            y *= __builtin_amdgcn_exp2f(own - total);
        }
    }
    if (a.lse && write_lse) a.lse[(int64_t)row * q_heads + head] = lse;
    return y;
}

__device__ __forceinline__ f32x4 from_base(f32x4 y, int base) {
#pragma unroll
    for (int i = 0; i < 4; ++i) y[i] = __builtin_ldexpf(y[i], base - 127);
    return y;
}

// The power of two that brings a row's largest bf16 magnitude (bits m) into [2^14, 2^15). Of rows with an infinity or a
// NaN none helps: their scores are infinite or NaN.
__device__ __forceinline__ int bf_lift(uint32_t m) {
    return m >= 0x7F80u ? 0 : min(max(14 - ((int)(m >> 7) - 127), -126), 126);
}
__device__ __forceinline__ f16x8 bf_f16x8(u32x4 raw, float up) {
    f16x8 q;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        q[2 * j] = (_Float16)(bf2f((uint16_t)(raw[j] & 0xFFFF)) * up);
        q[2 * j + 1] = (_Float16)(bf2f((uint16_t)(raw[j] >> 16)) * up);
    }
    return q;
}

// Eight elements of q, with the scale's sign: the kernels multiply scores by its size, so that larger
// scores stay larger.
__device__ __forceinline__ u32x4 signed16(u32x4 v, float scale) {
    return v ^ (scale < 0.0f ? 0x80008000u : 0u);
}

// What sums of products are multiplied by for scores in log2: finite, so that keys of zero give zeros whatever their byte.
__device__ __forceinline__ float score_factor(const Attn& a, int byte, int q_exp) {
    return fminf(__builtin_ldexpf(fabsf(a.scale_log2), byte - 127 + q_exp), 3.402823466e38f);
}

// A row's query as the second operand of S^T, in fp16: 16 columns a lane of each 64, 8 of a
// last 32. bf16 rows go through a power of two; returns the exponent that undoes it.
template <int D>
__device__ __forceinline__ int load_q(const Rows& Q, bool there, int row, uint32_t head, int g, int bf, float scale,
                                        f16x8 (&q)[D / 32]) {
    constexpr int C64 = D / 64;
    u32x4 raw[D / 32];
    const uint16_t* const x =
        static_cast<const uint16_t*>(Q.p) + (there ? (int64_t)row * Q.row + (int64_t)head * Q.head : 0);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) {
        const int d = i < 2 * C64 ? i / 2 * 64 + g * 16 + i % 2 * 8 : C64 * 64 + g * 8;
        raw[i] = there ? signed16(*reinterpret_cast<const u32x4*>(x + d), scale) : u32x4{};
    }
    if (!bf) {
#pragma unroll
        for (int i = 0; i < D / 32; ++i) q[i] = __builtin_bit_cast(f16x8, raw[i]);
        return 0;
    }
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) m = max(m, max(raw[i][j] & 0x7FFFu, raw[i][j] >> 16 & 0x7FFFu));
    const int e = bf_lift(across_rows_max(m));
    const float up = pow2f(e);
#pragma unroll
    for (int i = 0; i < D / 32; ++i) q[i] = bf_f16x8(raw[i], up);
    return -e;
}

// Token of one of the few rows: row / group by a multiplication, exact below 64 x 64.
__device__ __forceinline__ int token_of(const Attn& a, int row) { return (int)((uint32_t)row * a.group_inv >> 16); }

template <bool ONCE, class T>
__device__ __forceinline__ T load_codes(const T* p) {
    return ONCE ? ldg_nt(p) : *p;
}

// ---- the work of a call of few rows, shared out evenly
//
// A row of work (a sequence and head) is ceil(tokens / kTile) units, and p.start more at its beginning, the
// price of beginning it: asking for its length, page ids, query and first codes one after
// the other takes about as long as 768 / D units do.
// kParts: rows of work are cut into parts of at most c units (a round's, at least), with the smallest c that
// gives no more parts than groups (or near it). kShares: all rows' units in order of sequence and head are cut
// into equal shares, one for each group, however the lengths differ.
// A row of work that a cut goes through leaves partial sums: a group's first piece, if it continues a
// row, in slot 2k, a last piece that begins a row and does not end it in slot 2k + 1 (k the group);
// kv_join_k adds the row's parts up.
__device__ __forceinline__ int units_of(const Seq& s, const Attn& a, int rows, int start) {
    const Span v = span_of(s, a, 0, rows);
    return s.n == 0 ? 0 : max((v.hi - v.lo + kTile - 1) / kTile, 1) + start;
}

struct Share {
    int seq;
    uint32_t head;
    int unit;        // first unit, within its row of work
    int units;       // in all
    int parts;       // of its row of work (kParts)
    uint64_t at;     // of the first unit, among all (kShares)
    uint64_t total;
    uint32_t groups; // that have some
};

// Inclusive sum over the wave, in DPP steps (six exchanges through the LDS unit take 0.3 us, and a
// share takes up to seven sums): 1, 2, 4 and 8 lanes within rows of 16, then the rows before.
template <int CTRL, int ROWS>
__device__ __forceinline__ int plus_dpp(int v) {
    return v + __builtin_amdgcn_update_dpp(0, v, CTRL, ROWS, 0xF, false);
}
__device__ __forceinline__ int prefix64(int v) {
    v = plus_dpp<0x111, 0xF>(v);
    v = plus_dpp<0x112, 0xF>(v);
    v = plus_dpp<0x114, 0xF>(v);
    v = plus_dpp<0x118, 0xF>(v);
    v = plus_dpp<0x142, 0xA>(v);
    return plus_dpp<0x143, 0xC>(v);
}

// What group k does; each wave works it out for itself from the units of all sequences.
// lds: kScan ints.
__device__ inline Share share_of(const Cache& c, const Batch& b, const Attn& a, const FewPlan& p, uint32_t k, int rows,
                                 int* lds) {
    const int lane = threadIdx.x & 63, n = (int)b.n_seq;
    Share w = {0, 0, 0, 0, 1, 0, 0, p.groups};
    if (k >= p.groups) return w;
    if (p.mode == FewPlan::kRows) {
        w.seq = (int)(k / c.heads);
        w.head = k % c.heads;
        w.units = units_of(sequence(b, c.page_log2, w.seq), a, rows, (int)p.start);
        return w;
    }
    int u0;  // of sequence `lane`
    if (n <= 64) {
        u0 = lane < n ? units_of(sequence(b, c.page_log2, lane), a, rows, (int)p.start) : 0;
    } else {
        for (int i = threadIdx.x; i < n; i += 256) lds[i] = units_of(sequence(b, c.page_log2, i), a, rows, (int)p.start);
        __syncthreads();
        u0 = lds[lane];
    }
    // sum over all sequences of f(units)
    auto sum = [&](auto f) {
        int v = 0;
        for (int i = lane; i < n; i += 64) v += f(i < 64 ? u0 : lds[i]);
        return (uint64_t)(uint32_t)__builtin_amdgcn_readlane(prefix64(v), 63);
    };
    // the sequence i with sum_{j < i} f <= x < sum_{j <= i} f; x becomes what is left, u its units
    auto find = [&](uint32_t& x, int& u, auto f) {
        int before = 0;
        for (int i0 = 0; i0 < n; i0 += 64) {
            const int mine = i0 + lane < n ? i0 ? lds[i0 + lane] : u0 : 0, v = f(mine);
            const int up = prefix64(v) + before;
            const uint64_t hit = __ballot((uint32_t)(up - v) <= x && x < (uint32_t)up);
            if (hit) {
                const int l = __ffsll((unsigned long long)hit) - 1;
                x -= (uint32_t)__builtin_amdgcn_readlane(up - v, l);
                u = __builtin_amdgcn_readlane(mine, l);
                return i0 + l;
            }
            before = __builtin_amdgcn_readlane(up, 63);
        }
        return 0;
    };
    const uint64_t all = sum([](int u) { return u; });
    if (all == 0) return w;
    int u = 0;
    if (p.mode == FewPlan::kParts) {
        // c from the mean on; the last is enough for any lengths: sum ceil(u / c) <= sum u / c + rows of work
        const uint32_t most = p.groups / c.heads;
        uint32_t size = max((uint32_t)((all + most - 1) / most), (uint32_t)(kRound / kTile)), count = 0;
        for (int tries = 0; tries < 4; ++tries, ++size) {
            count = (uint32_t)sum([&](int v) { return (int)(((uint32_t)v + size - 1) / size); });
            if (count <= most) break;
        }
        if (count > most) {
            size = max(size, (uint32_t)((all + most - n - 1) / (most - n)));
            count = (uint32_t)sum([&](int v) { return (int)(((uint32_t)v + size - 1) / size); });
        }
        if (k >= count * c.heads) return w;
        // parts in order of head, then sequence
        w.head = k / count;
        uint32_t x = k % count;
        w.seq = find(x, u, [&](int v) { return (int)(((uint32_t)v + size - 1) / size); });
        w.parts = (int)(((uint32_t)u + size - 1) / size);
        // the first u % parts of them are a unit longer
        const int each = u / w.parts, more = u - each * w.parts;
        w.unit = (int)x * each + min((int)x, more);
        w.units = each + ((int)x < more);
        return w;
    }
    w.total = all * c.heads;
    if (w.total < w.groups) w.groups = (uint32_t)w.total;
    if (k >= w.groups) return w;
    if (w.total < 0xFFFFFFFFu / w.groups) {  // short divisions where they do
        w.at = (uint32_t)w.total * k / w.groups;
        w.units = (int)((uint32_t)w.total * (k + 1) / w.groups - (uint32_t)w.at);
    } else {
        w.at = w.total * k / w.groups;
        w.units = (int)(w.total * (k + 1) / w.groups - w.at);
    }
    // in order of sequence, then head
    uint32_t x = (uint32_t)(w.total <= 0xFFFFFFFFu ? (uint32_t)w.at / c.heads : w.at / c.heads);
    const uint32_t odd = (uint32_t)(w.at - (uint64_t)x * c.heads);
    w.seq = find(x, u, [](int v) { return v; });
    const uint64_t in = (uint64_t)x * c.heads + odd;
    w.head = (uint32_t)(in <= 0xFFFFFFFFu ? (uint32_t)in / (uint32_t)u : in / (uint32_t)u);
    w.unit = (int)(in - (uint64_t)w.head * (uint32_t)u);
    return w;
}

// A row of work that is cut: the group of its first part, and how many parts (0: it is whole).
// By row of work where those are no more than the groups, else by group.
struct Cut {
    int seq, head, first, parts;
};
// The partial results of slot i and row tile t: [16 R][D] sums, then [16 R] of RowSum.
template <int D, int R>
__device__ __forceinline__ float* slot_of(float* ws, const FewPlan& p, uint32_t i, uint32_t t) {
    return ws + p.cuts * 4 + ((uint64_t)i * p.tiles + t) * (16 * R * (D + kRowSum));
}

// Few rows (tokens x heads of a group) of a sequence and head, 16 R a workgroup. Four waves take 64 tokens
// of a piece in turn and join their sums at its end. What bounds it is the stream of codes:
// a wave asks for its next keys as soon as the present ones are multiplied, and for its
// next values after the product with the present ones, so that most of 16 KiB a wave
// (128 wide) is always on its way. ONCE: no other workgroup reads the codes, and they are loaded past the
// caches' other lines (64 sequences of 2486 tokens 69 us without, 64 with); with two row tiles to
// share them that costs more than it saves (28 us without, 31 with).
template <int D, int TYPE, int R, bool ONCE>
__global__ __launch_bounds__(256, few_waves(D)) void kv_few_k(Cache c, Batch b, Attn a, FewPlan p, Rows Q, Rows O, int bf,
                                                              float* ws) {
    constexpr int C64 = D / 64, kHalf = D % 64 ? 1 : 0;  // 64-column pieces of a key, and a 32-column one
    constexpr int kPad = D + 4;
    __shared__ __attribute__((aligned(16))) float o_lds[4 * 16 * R * kPad];
    __shared__ float m_lds[4][16 * R], l_lds[4][16 * R];
    __shared__ int base_lds[4];
    static_assert(sizeof(o_lds) >= kIds * sizeof(int) && kIds >= kScan, "page ids, units of the sequences");
    int* const ids = reinterpret_cast<int*>(o_lds);  // page ids of the piece, until the waves join
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, r = lane & 15, g = lane >> 4;
    const uint32_t q_heads = c.heads * a.group;

    // the workgroups of a group side by side in one of eight XCDs: 8 groups' first tiles, their second, ...
    const uint32_t group = blockIdx.x / (8 * p.tiles) * 8 + blockIdx.x % 8, tile = blockIdx.x / 8 % p.tiles;
    const int all_rows = (int)(b.max_q * a.group), row0 = (int)tile * 16 * R;
    const Share share = share_of(c, b, a, p, group, all_rows, ids);
    Cut* const cuts = reinterpret_cast<Cut*>(ws);
    if (p.mode == FewPlan::kShares && !p.by_row && group < p.groups && tile == 0 && tid == 0) cuts[group].parts = 0;
    int left = share.units, unit = share.unit;
    int seq = share.seq;
    uint32_t h = share.head;
    uint64_t at = share.at;
    while (left > 0) {
        seq = __builtin_amdgcn_readfirstlane(seq);
        h = (uint32_t)__builtin_amdgcn_readfirstlane((int)h);
        const Seq s = sequence(b, c.page_log2, (uint32_t)seq);
        const Span sp = span_of(s, a, 0, all_rows);  // the same for all row tiles
        const int units = units_of(s, a, all_rows, (int)p.start), mine = min(left, units - unit);
        if (mine <= 0) {  // a sequence without rows
            ++seq;
            continue;
        }
        const int rows = s.n * (int)a.group - row0, tail = (int)p.start;  // from this tile on
        const int lo = sp.lo + max(unit - tail, 0) * kTile;
        const int hi = (int)min((int64_t)sp.hi, (int64_t)sp.lo + (int64_t)max(unit + mine - tail, 0) * kTile);
        const int32_t* const table = b.pages + (uint64_t)seq * b.max_pages;

        if (rows > 0) {
            // this lane's row of each sixteen
            f16x8 q[R][D / 32];
            float m[R], l[R];  // of the row; l: this lane's tokens alone
            int q_exp[R], sees_lo[R], sees_hi[R], base = kBase;
            f32x4 o[R][D / 16];
#pragma unroll
            for (int k = 0; k < R; ++k) {
                // a row that there is not sees what the last one does: it takes no tile off the short way
                const bool there = 16 * k + r < rows;
                const int row = there ? row0 + 16 * k + r : row0 + rows - 1, tok = token_of(a, row);
                const int pos = s.len - s.n + tok;
                sees_hi[k] = min(a.causal ? pos + 1 : s.len, hi);
                sees_lo[k] = a.window ? pos + 1 - (int)a.window : 0;
                q_exp[k] = load_q<D>(Q, there, s.row0 + tok, h * a.group + (uint32_t)(row - tok * (int)a.group),
                                                             g, bf, a.scale_log2, q[k]);
                m[k] = kLowest;
                l[k] = 0.0f;
#pragma unroll
                for (int i = 0; i < D / 16; ++i) o[k][i] = f32x4{0, 0, 0, 0};
            }

            int page0 = 0;
            u32x4 kw[4 * C64 + 1], vw[D / 16];
            u32x2 kx[4];  // the 32-column pieces
            int ke = 0, ve = 0, pv = 0;
            // Codes of the wave's 64 tokens from t0 on: the lane's row of K operand t, and its columns of V
            // with the exponents of its 16 tokens.
            auto page_at = [&](int t) { return ids[(min(t, hi - 1) >> c.page_log2) - page0]; };
            auto load_k = [&](int t0) {
                const int tk = t0 + 16 * (r >> 2);
                const uint8_t* const kp = c.k + code_offset(c, D, max(page_at(tk), 0), h, tk) + (r & 3) * D;
#pragma unroll
                for (int t = 0; t < 4; ++t) {
#pragma unroll
                    for (int i = 0; i < C64; ++i) kw[t * C64 + i] = load_codes<ONCE>(reinterpret_cast<const u32x4*>(kp + t * 4 * D + i * 64 + g * 16));
                    if constexpr (kHalf) kx[t] = load_codes<ONCE>(reinterpret_cast<const u32x2*>(kp + t * 4 * D + C64 * 64 + g * 8));
                }
            };
            auto load_v = [&](int t0) {
                const int tv = t0 + 16 * g;
                pv = page_at(tv);
                const uint64_t eo = exp_offset(c, max(pv, 0), h, tv);
                ke = c.k_exp[eo];
                ve = c.v_exp[eo];
                const uint8_t* const vp = c.v + code_offset(c, D, max(pv, 0), h, tv) + r * 16;
#pragma unroll
                for (int i = 0; i < D / 16; ++i) vw[i] = load_codes<ONCE>(reinterpret_cast<const u32x4*>(vp + i * 256));
            };
            auto step = [&](int t0, auto more) {
                // products on the same sums stand apart: each waits for the one before
                f32x4 st[R][4];
#pragma unroll
                for (int t = 0; t < 4; ++t)
#pragma unroll
                    for (int k = 0; k < R; ++k) st[k][t] = f32x4{0, 0, 0, 0};
#pragma unroll
                for (int i = 0; i < 2 * C64 + kHalf; ++i)
#pragma unroll
                    for (int t = 0; t < 4; ++t) {
                        const u32x4 w = kw[t * C64 + min(i / 2, C64 - 1)];
                        const f16x8 x = i == 2 * C64 ? codes_f16x8<TYPE>(kx[t].x, kx[t].y)
                                        : i % 2      ? codes_f16x8<TYPE>(w.z, w.w)
                                                     : codes_f16x8<TYPE>(w.x, w.y);
#pragma unroll
                        for (int k = 0; k < R; ++k) st[k][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, q[k][i], st[k][t], 0, 0, 0);
                    }
                __builtin_amdgcn_sched_barrier(0);  // into the registers just read, not beside them
                if constexpr (decltype(more)::value) load_k(t0 + kRound);
                __builtin_amdgcn_sched_barrier(0);

                const int tv = t0 + 16 * g;
                const bool part = t0 + kTile > hi || __any(pv < 0);  // blocks among them that hold anything
                int byte = ve;
                if (part && (tv >= hi || pv < 0)) byte = kBase;
                if (__any(base_far(base, byte))) {
                    const int to = base_near(base, byte, byte);
#pragma unroll
                    for (int k = 0; k < R; ++k) l[k] = __builtin_ldexpf(l[k], to - base);
                    base = to;
                }
                const float un_v = pow2f(base - byte);
                f16x8 w[R][2];
#pragma unroll
                for (int k = 0; k < R; ++k) {
                    // t = f s + e with f >= 0: the largest t is the largest s's
                    float f = score_factor(a, ke, q_exp[k]), e = (float)(ve - 127);
                    // tokens in sight of the row, of the lane's 16
                    const int from = sees_lo[k] - tv, to = pv < 0 ? 0 : sees_hi[k] - tv;
                    if (!__all(from <= 0 && to >= 16)) {
                        // only the few tiles that need it: nothing of this is computed ahead of the branch
                        int first = from;
                        asm volatile("" : "+v"(first));
#pragma unroll
                        for (int i = 0; i < 16; ++i)
                            st[k][i / 4][i % 4] = i < first || i >= to ? -__builtin_inff() : __builtin_fmaf(st[k][i / 4][i % 4], f, e);
                        f = 1.0f;
                        e = 0.0f;
                    }
                    float top = st[k][0][0];
#pragma unroll
                    for (int i = 1; i < 16; ++i) top = fmaxf(top, st[k][i / 4][i % 4]);
                    top = across_rows_maxf(fmaxf(m[k], __builtin_fmaf(top, f, e)));
                    if (__any(top > m[k] + kSlack)) {
                        const float fade = __builtin_amdgcn_exp2f(m[k] - top);
                        m[k] = top;
                        l[k] *= fade;
#pragma unroll
                        for (int i = 0; i < D / 16; ++i) o[k][i] *= fade;
                    }
                    const float down = e - (m[k] - kLift);
                    float sum = 0.0f;
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        const float y = __builtin_amdgcn_exp2f(__builtin_fmaf(st[k][i / 4][i % 4], f, down));
                        sum += y;
                        w[k][i / 8][i % 8] = (_Float16)y;
                    }
                    l[k] += sum * un_v;
                }
                if (part) {
                    // bytes of tokens that no length covers may hold anything, NaN among it
                    const int valid = pv < 0 ? 0 : min(max(hi - tv, 0), 16);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int n = min(max(valid - 4 * j, 0), 4);
                        const uint32_t keep = n == 4 ? 0xFFFFFFFFu : (1u << 8 * n) - 1;
#pragma unroll
                        for (int i = 0; i < D / 16; ++i) vw[i][j] &= keep;
                    }
                }
#pragma unroll
                for (int i0 = 0; i0 < D / 16; i0 += 4)
#pragma unroll
                    for (int hh = 0; hh < 2; ++hh)
#pragma unroll
                        for (int i = i0; i < i0 + 4 && i < D / 16; ++i) {
                            const f16x8 x = hh ? codes_f16x8<TYPE>(vw[i].z, vw[i].w) : codes_f16x8<TYPE>(vw[i].x, vw[i].y);
#pragma unroll
                            for (int k = 0; k < R; ++k) o[k][i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(x, w[k][hh], o[k][i], 0, 0, 0);
                        }
                __builtin_amdgcn_sched_barrier(0);
                if constexpr (decltype(more)::value) load_v(t0 + kRound);
                __builtin_amdgcn_sched_barrier(0);
            };
            // the piece, or as much of it as there is room for page ids
            const int most = ((kIds - 1) << c.page_log2) & ~(kRound - 1);
            for (int from = lo; from < hi;) {
                const int to = hi - from > most ? from + most : hi;
                __syncthreads();
                page0 = from >> c.page_log2;
                const int pages = ((to - 1) >> c.page_log2) - page0 + 1;
                for (int i = tid; i < pages; i += 256) {
                    const int v = table[page0 + i];
                    ids[i] = (uint32_t)v < c.n_pages ? v : -1;
                }
                __syncthreads();
                int t0 = from + wave * kTile;
                if (t0 < to) {
                    load_k(t0);
                    load_v(t0);
                    for (; t0 < to - kRound; t0 += kRound) step(t0, Int<1>());
                    step(t0, Int<0>());
                }
                from = to;
            }

            // join the waves
            const bool whole = mine == units;
            float* const part = slot_of<D, R>(ws, p, 2 * group + (unit == 0), tile);
            __syncthreads();
#pragma unroll
            for (int k = 0; k < R; ++k) {
                l[k] = across_rows_sum(l[k]);
                if (g == 0) {
                    m_lds[wave][16 * k + r] = m[k];
                    l_lds[wave][16 * k + r] = l[k];
                }
            }
            if (lane == 0) base_lds[wave] = base;
            __syncthreads();
#pragma unroll
            for (int k = 0; k < R; ++k) {
                float top = m_lds[0][16 * k + r];
#pragma unroll
                for (int w = 1; w < 4; ++w) top = fmaxf(top, m_lds[w][16 * k + r]);
                const float fade = __builtin_amdgcn_exp2f(m[k] - top);
                float* const to = o_lds + ((wave * R + k) * 16 + r) * kPad;
#pragma unroll
                for (int i = 0; i < D / 16; ++i) *reinterpret_cast<f32x4*>(to + i * 16 + g * 4) = o[k][i] * fade;
            }
            __syncthreads();
            const int one = min(min(base_lds[0], base_lds[1]), min(base_lds[2], base_lds[3]));
            for (int i = tid; i < min(rows, 16 * R) * (D / 4); i += 256) {
                const int row = i / (D / 4), d = i % (D / 4) * 4;
                f32x4 y = *reinterpret_cast<const f32x4*>(o_lds + row * kPad + d);
                float best = m_lds[0][row];
#pragma unroll
                for (int w = 1; w < 4; ++w) {
                    y += *reinterpret_cast<const f32x4*>(o_lds + (w * 16 * R + row) * kPad + d);
                    best = fmaxf(best, m_lds[w][row]);
                }
                float sum = 0.0f;
#pragma unroll
                for (int w = 0; w < 4; ++w) sum += __builtin_ldexpf(l_lds[w][row], one - base_lds[w]) * __builtin_amdgcn_exp2f(m_lds[w][row] - best);
                if (whole) {
                    const int tok = token_of(a, row0 + row), out = s.row0 + tok;
                    const uint32_t head = h * a.group + (uint32_t)(row0 + row - tok * (int)a.group);
                    store4(O, out, head, d, from_base(y * finish(a, best, sum, one, out, head, q_heads, d == 0), one), bf);
                } else {
                    *reinterpret_cast<f32x4*>(part + row * D + d) = y;
                    if (d == 0) *reinterpret_cast<RowSum*>(part + 16 * R * D + row * kRowSum) = {best, sum, one, 0};
                }
            }
            __syncthreads();
        }
        if (unit == 0 && tile == 0 && tid == 0 && p.mode != FewPlan::kRows && (p.by_row || mine < units)) {
            int parts = share.parts;
            if (p.mode == FewPlan::kShares)  // the last unit's group: shares begin at floor(k total / groups)
                parts = (int)(((at + (uint64_t)units) * share.groups - 1) / share.total) - (int)group + 1;
            cuts[p.by_row ? (uint32_t)seq * c.heads + h : group] = {seq, (int)h, (int)group, mine == units ? 0 : parts};
        }
        left -= mine;
        at += (uint64_t)mine;
        unit = 0;
        if (++h == c.heads) h = 0, ++seq;
    }
}

// Adds up the n parts of a row: sums(i) and row_sum(i) are part i's sums and RowSum. W waves of a workgroup
// share the parts (lds: W (D + kRowSum) floats), or one does it alone.
template <int D, int W, class Sums, class Of>
__device__ __forceinline__ void join_row(const Attn& a, int n, Sums sums, Of row_sum, float* lds, const Rows& O, int bf,
                                         int at, uint32_t head, uint32_t q_heads) {
    constexpr int N = (D + 63) / 64;
    const int lane = threadIdx.x & 63, wave = W > 1 ? __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)) : 0;
    float m = kLowest, l = 0.0f, o[N] = {};
    int base = kBase;
    for (int i0 = 0; i0 < n; i0 += 16 * W) {
        const int here = min((n - i0 - wave + W - 1) / W, 16);  // this wave's: i0 + wave, and every W-th
        // the sums are asked for along with what scales them
        float v[16][N];
        RowSum own = {kLowest, 0.0f, kBase, 0};
        if (lane < here) own = *reinterpret_cast<const RowSum*>(row_sum(i0 + wave + lane * W));
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i < here) {
                const float* const from = sums(i0 + wave + i * W);
#pragma unroll
                for (int k = 0; k < N; ++k) v[i][k] = D % 64 == 0 || k * 64 + lane < D ? from[k * 64 + lane] : 0.0f;
            }
        float top = fmaxf(m, own.m);
#pragma unroll
        for (int d = 1; d < 16; d *= 2) top = fmaxf(top, __shfl_xor(top, d));
        top = __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, top)));
        const int one = min(base, __builtin_amdgcn_readfirstlane((int)~wave_max(~(uint32_t)own.base)));
        const float fade = __builtin_amdgcn_exp2f(m - top), f = __builtin_amdgcn_exp2f(own.m - top);
        m = top;
        l = __builtin_ldexpf(l, one - base) * fade + wave_sum(__builtin_ldexpf(own.l, one - own.base) * f);
        base = one;
#pragma unroll
        for (int k = 0; k < N; ++k) o[k] *= fade;
#pragma unroll
        for (int i = 0; i < 16; ++i)
            if (i < here) {
                const float fi = __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), i));
#pragma unroll
                for (int k = 0; k < N; ++k) o[k] += v[i][k] * fi;
            }
    }
    if constexpr (W > 1) {
        RowSum* const all = reinterpret_cast<RowSum*>(lds + W * D);
        if (lane == 0) all[wave] = {m, l, base, 0};
        __syncthreads();
        float top = all[0].m;
        base = all[0].base;
#pragma unroll
        for (int w = 1; w < W; ++w) {
            top = fmaxf(top, all[w].m);
            base = min(base, all[w].base);
        }
        const float fade = __builtin_amdgcn_exp2f(m - top);
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (D % 64 == 0 || k * 64 + lane < D) lds[wave * D + k * 64 + lane] = o[k] * fade;
        l = 0.0f;
#pragma unroll
        for (int w = 0; w < W; ++w) l += __builtin_ldexpf(all[w].l, base - all[w].base) * __builtin_amdgcn_exp2f(all[w].m - top);
        m = top;
        __syncthreads();
        if (wave) return;
#pragma unroll
        for (int k = 0; k < N; ++k)
            if (D % 64 == 0 || k * 64 + lane < D) {
                o[k] = 0.0f;
#pragma unroll
                for (int w = 0; w < W; ++w) o[k] += lds[w * D + k * 64 + lane];
            }
    }
    const float y = finish(a, m, l, base, at, head, q_heads, lane == 0);
    uint16_t* const to = static_cast<uint16_t*>(O.p) + (int64_t)at * O.row + (int64_t)head * O.head;
#pragma unroll
    for (int k = 0; k < N; ++k)
        if (D % 64 == 0 || k * 64 + lane < D) {
            const float v = __builtin_ldexpf(o[k] * y, base - 127);
            to[k * 64 + lane] = (uint16_t)(bf ? pair16<1>(v, 0.0f) : pair16<0>(v, 0.0f));
        }
}

// The cut rows of work of kv_few_k, one of their (token, head) rows for each W waves.
template <int D, int R, int W>
__global__ __launch_bounds__(256) void kv_join_k(Cache c, Batch b, Attn a, FewPlan p, Rows O, int bf, float* ws) {
    __shared__ __attribute__((aligned(16))) float lds[W > 1 ? W * (D + kRowSum) : 1];
    const int row = W > 1 ? (int)blockIdx.y : (int)blockIdx.y * 4 + __builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    // by row of work: a sequence without rows has written nothing
    const Cut cut = reinterpret_cast<const Cut*>(ws)[blockIdx.x];
    const Seq own = sequence(b, c.page_log2, p.by_row ? blockIdx.x / c.heads : 0);
    if (p.by_row && own.n == 0) return;
    if (cut.parts == 0) return;
    const Seq s = p.by_row ? own : sequence(b, c.page_log2, (uint32_t)cut.seq);
    if (row >= s.n * (int)a.group) return;
    // part 0 begins the row of work, the others continue it: slots 2k + 1, then 2 (k + i)
    const int in = row % (16 * R);
    auto part = [&](int i) { return slot_of<D, R>(ws, p, 2 * (cut.first + i) + (i == 0), (uint32_t)(row / (16 * R))); };
    join_row<D, W>(a, cut.parts, [&](int i) { return part(i) + in * D; },
                   [&](int i) { return part(i) + 16 * R * D + in * kRowSum; }, lds, O, bf, s.row0 + row / (int)a.group,
                   (uint32_t)cut.head * a.group + (uint32_t)(row % (int)a.group), c.heads * a.group);
}

template <int D, int TYPE, int R>
hipError_t few_r(const Cache& c, const Batch& b, const Attn& a, const FewPlan& p, const Rows& Q, const Rows& O, bool bf,
                 float* ws, hipStream_t s) {
    const uint32_t wgs = (p.groups + 7) / 8 * 8 * p.tiles;
    if (p.tiles == 1) kv_few_k<D, TYPE, R, true><<<wgs, 256, 0, s>>>(c, b, a, p, Q, O, bf, ws);
    else if constexpr (R == few_sixteens(D)) kv_few_k<D, TYPE, R, false><<<wgs, 256, 0, s>>>(c, b, a, p, Q, O, bf, ws);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.mode == FewPlan::kRows) return e;
    const uint32_t rows = b.max_q * a.group;
    // many parts a row of work: four waves for each of its rows
    if (p.groups >= 8 * p.cuts) kv_join_k<D, R, 4><<<dim3(p.cuts, rows), 256, 0, s>>>(c, b, a, p, O, bf, ws);
    else kv_join_k<D, R, 1><<<dim3(p.cuts, (rows + 3) / 4), 256, 0, s>>>(c, b, a, p, O, bf, ws);
    return hipGetLastError();
}

template <int D, int TYPE>
hipError_t few_d(const Cache& c, const Batch& b, const Attn& a, const FewPlan& p, const Rows& Q, const Rows& O, bool bf,
                 float* ws, hipStream_t s) {
    if constexpr (few_sixteens(D) > 1)
        if (p.sixteens == 2) return few_r<D, TYPE, 2>(c, b, a, p, Q, O, bf, ws, s);
    return few_r<D, TYPE, 1>(c, b, a, p, Q, O, bf, ws, s);
}

}  // namespace kv
}  // namespace kq
