// kq_kv_keep.hip -- the kept rows of drafted tokens moved together in the 8-bit cache (kq_kv_keep).
#include "kq_kv_write_kernel.h"

namespace kq {
namespace kv {
namespace {

// Where the tokens of 16 places come from.
struct Sources {
    uint64_t code[16];  // offset of the source's 16-token block
    int exp[16];        // byte; of no page: -1
    int in[16];         // token of its block; -1: the place's own token stays
};

// One wave moves the rows of one head's K or V. A row moves down, or stays: blocks of 16 places are taken in
// order, and everything that comes into one is in registers before any of it is written, so that no source
// is overwritten before it is read. Exponent bytes are written after their block. What bounds it is
// one way to memory after the other: lengths, rows, page ids, exponents, codes; of V, whose columns hold 16 tokens each, then a moved token's
// byte in each column, waited for before the next token's is asked for. (One sequence of 60 rows, 8 heads of 128, every eighth of
// the rows kept: 6.6 us; 64 trees of 26 to 64 rows, 8 heads of 64: 7.4, where what it moves would take 0.9. Rows that
// all stay, and the wave has nothing to do: 1.6.)
template <int D, int TYPE>
__global__ __launch_bounds__(256) void kv_keep_k(Cache c, Batch b, const int32_t* keep, const int32_t* n_keep) {
    __shared__ int rows[kMostNodes];
    __shared__ Sources sources[4];
    const int tid = threadIdx.x, lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const Seq s = sequence(b, c.page_log2, blockIdx.y);
    const int32_t* const table = b.pages + (uint64_t)blockIdx.y * b.max_pages;
    int n = min(min(max(n_keep[blockIdx.y], 0), (int)b.max_q), s.n);
    for (int j = tid; j < n; j += 256) rows[j] = keep[(uint64_t)blockIdx.y * b.max_q + j];
    __syncthreads();
    // rows that stay come first; the list ends before what is no row, or not in order
    int stay = n;
    for (int j0 = 0; j0 < n; j0 += 64) {
        const int j = j0 + lane, k = j < n ? rows[j] : 0, before = j > 0 && j < n ? rows[j - 1] : -1;
        const uint64_t bad = __ballot(j < n && (k < j || k <= before || k >= s.n));
        if (bad) n = j0 + __ffsll((unsigned long long)bad) - 1;
        const uint64_t moves = __ballot(j < n && k != j);
        if (moves && stay > j0) stay = min(stay, j0 + __ffsll((unsigned long long)moves) - 1);
    }
    stay = min(stay, n);
    const uint32_t job = blockIdx.x * 4 + (uint32_t)wave;
    if (job >= 2 * c.heads || stay >= n) return;
    const uint32_t h = job >> 1;
    const bool is_v = job & 1;
    const int first = s.len - s.n, from = max(first + stay, 0), end = first + n;  // places from .. end - 1 are moved into
    const int B = 1 << c.block_log2;
    uint8_t* const codes = is_v ? c.v : c.k;
    uint8_t* const exps = is_v ? c.v_exp : c.k_exp;
    Sources& src = sources[wave];
    for (int t0 = from & ~(B - 1); t0 < end; t0 += B) {
        const int page = page_of(c, table, t0);
        if (page < 0) continue;
        uint8_t* const ep = exps + exp_offset(c, page, h, t0);
        const int was = *ep, hi = min(t0 + B, s.len);
        int e = was;
        for (int t = max(t0, from) + lane; t < min(t0 + B, end); t += 64) {
            const int at = first + rows[t - first], p = page_of(c, table, at);
            if (p >= 0) e = max(e, (int)exps[exp_offset(c, p, h, at)]);
        }
        e = (int)wave_max((uint32_t)e);
        const bool grew = e > was;
        for (int sub = grew ? t0 : max(t0, from) & ~15; sub < (grew ? hi : min(t0 + B, end)); sub += 16) {
            if (lane < 16) {
                const int t = sub + lane;
                const bool moved = t >= from && t < end;
                const int at = moved ? first + rows[t - first] : t, p = moved ? page_of(c, table, at) : page;
                src.code[lane] = code_offset(c, D, max(p, 0), h, at);
                src.exp[lane] = p < 0 ? -1 : moved ? (int)exps[exp_offset(c, p, h, at)] : was;
                src.in[lane] = moved ? at & 15 : -1;
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            // 2^(its exponent - e) of a token (below 2^-126 every code rounds to zero all the same). Of no page: codes of
            // zero, whatever was read in their place (times zero a negative e4m3 value would leave its sign)
            auto keeps = [&](int exp) { return pow2f(max(exp - e, -126)); };
            uint8_t* const to = codes + code_offset(c, D, page, h, sub);
            if (!is_v) {
                constexpr int N = D / 32;
                u32x2 w[N];
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const int i = lane + 64 * j, t = i / (D / 8), in = src.in[t];
                    w[j] = *reinterpret_cast<const u32x2*>(codes + src.code[t] + (uint32_t)((in < 0 ? t : in) * D + i % (D / 8) * 8));
                }
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
                for (int j = 0; j < N; ++j) {
                    const int i = lane + 64 * j, t = i / (D / 8), exp = src.exp[t];
                    if (sub + t >= hi || (src.in[t] < 0 && !grew)) continue;
                    const float f = keeps(exp);
                    u32x2 y = exp == e ? w[j] : u32x2{rounded_anew<TYPE>(w[j].x, f), rounded_anew<TYPE>(w[j].y, f)};
                    if (exp < 0) y = u32x2{0, 0};
                    *reinterpret_cast<u32x2*>(to + i * 8) = y;
                }
                continue;
            }
            constexpr int N = (D + 63) / 64;
            u32x4 w[N];
#pragma unroll
            for (int j = 0; j < N; ++j) {
                const int col = min(lane + 64 * j, D - 1);
                w[j] = *reinterpret_cast<const u32x4*>(to + col * 16);
#pragma unroll
                for (int t = 0; t < 16; ++t) {
                    const int in = src.in[t];
                    if (in < 0 && !grew) continue;  // the same for all lanes
                    const int exp = src.exp[t];
                    uint32_t byte = in < 0 ? w[j][t / 4] >> 8 * (t % 4) & 0xFF : codes[src.code[t] + (uint32_t)(col * 16 + in)];
                    if (sub + t >= hi) continue;
                    if (exp != e) byte = exp < 0 ? 0 : rounded_anew<TYPE>(byte, keeps(exp)) & 0xFF;
                    w[j][t / 4] = (w[j][t / 4] & ~(0xFFu << 8 * (t % 4))) | byte << 8 * (t % 4);
                }
            }
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
#pragma unroll
            for (int j = 0; j < N; ++j)
                if (D % 64 == 0 || lane + 64 * j < D) *reinterpret_cast<u32x4*>(to + (lane + 64 * j) * 16) = w[j];
        }
        if (grew && lane == 0) *ep = (uint8_t)e;
    }
}

}  // namespace
}  // namespace kv

hipError_t launch_kv_keep(const kv::Cache& c, const kv::Batch& b, uint32_t D, int type, const int32_t* keep, const int32_t* n_keep,
                          hipStream_t s) {
    const dim3 grid((2 * c.heads + 3) / 4, b.n_seq);
    return kv::by_dim(D, type, [&](auto d, auto t) {
        kv::kv_keep_k<decltype(d)::value, decltype(t)::value><<<grid, 256, 0, s>>>(c, b, keep, n_keep);
        return hipGetLastError();
    });
}

}  // namespace kq
