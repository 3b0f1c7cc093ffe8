// kq_kv_attn.hip -- attention over the 8-bit key/value cache (kq_kv_attn):
// launch plan and launches.
#include <algorithm>

#include "kq_kv_attn_kernel.h"

namespace kq {
namespace kv {
namespace {

uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

uint64_t splits_wanted(const Cache& c, const Batch& b, uint64_t tiles) {
    return ceil_div((uint64_t)cu_count() * 8, b.n_seq * tiles * c.heads);
}

template <int D, int TYPE>
hipError_t attn_d(const Cache& c, const Batch& b, const Attn& a, const Plan& p, const Rows& Q, const Rows& O, bool bf,
                  float* ws, hipStream_t s) {
    const uint32_t wgs = b.n_seq * p.splits * p.tiles * c.heads;
    kv_attn_k<D, TYPE><<<wgs, 256, 0, s>>>(c, b, a, p, Q, O, bf, ws);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits == 1) return e;
    kv_join_k<D><<<b.n_seq * b.max_q * c.heads * a.group, 256, 0, s>>>(c, b, a, p, O, bf, ws);
    return hipGetLastError();
}

}  // namespace
}  // namespace kv

// Splits: enough workgroups to fill the device several times over, each of 256 tokens (64
// a wave) at least.
kv::Plan kv_attn_plan(const kv::Cache& c, const kv::Batch& b, uint32_t group, uint32_t window) {
    kv::Plan p;
    p.tiles = (uint32_t)kv::ceil_div((uint64_t)b.max_q * group, 16);
    // a row tile's tokens: the window of its first row to its last row, from a multiple of 64 on
    uint64_t longest = b.max_len;
    if (window) longest = std::min<uint64_t>(longest, (uint64_t)window + 15 + kv::kTile - 1);
    p.chunk = (uint32_t)kv::ceil_div(kv::ceil_div(longest, kv::splits_wanted(c, b, p.tiles)), 256) * 256;
    p.splits = (uint32_t)kv::ceil_div(longest, p.chunk);
    return p;
}

// Of a split: 16 rows of sums, m and l. No window makes more splits than
// splits_wanted, nor than 256-token pieces of max_len.
size_t kv_attn_ws_bytes(const kv::Cache& c, const kv::Batch& b, uint32_t D, uint32_t group) {
    const uint64_t tiles = kv::ceil_div((uint64_t)b.max_q * group, 16);
    const uint64_t splits = std::min(kv::splits_wanted(c, b, tiles), kv::ceil_div(b.max_len, 256));
    return splits > 1 ? b.n_seq * tiles * c.heads * splits * 16 * (D + 2) * 4 : 0;
}

hipError_t launch_kv_attn(const kv::Cache& c, const kv::Batch& b, uint32_t D, int type, const kv::Attn& a,
                          const kv::Plan& p, const kv::Rows& Q, const kv::Rows& O, bool bf, void* ws, hipStream_t s) {
    return kv::by_dim(D, type, [&](auto d, auto t) {
        return kv::attn_d<decltype(d)::value, decltype(t)::value>(c, b, a, p, Q, O, bf, static_cast<float*>(ws), s);
    });
}

}  // namespace kq
