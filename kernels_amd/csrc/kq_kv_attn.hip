// kq_kv_attn.hip -- attention over the 8-bit key/value cache (kq_kv_attn): launch
// plans, and the launches of the kernel for few rows.
#include <algorithm>

#include "kq_kv_attn_kernel.h"

#ifndef KV_WGS
#define KV_WGS 2
#endif

namespace kq {
namespace kv {
namespace {

uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

// Tokens that `rows` rows of a sequence and head see at most, from a multiple of 64 on.
uint64_t longest_span(const Batch& b, uint64_t rows, uint32_t window) {
    return window ? std::min<uint64_t>(b.max_len, (uint64_t)window + rows - 1 + kTile - 1) : b.max_len;
}

// Few rows: the kernel of kq_kv_attn_kernel.h.
bool few(const Batch& b, uint32_t group) { return (uint64_t)b.max_q * group <= 16; }

// Its workgroups: all that the device holds at once (their registers allow two a compute unit, one
// at 256 columns), or one for each unit or row of work where there is less, or where
// the sequences are too many to add up their lengths in each workgroup.
struct FewPlan {
    uint32_t wgs;
    bool balanced, join;
};
FewPlan few_plan(const Cache& c, const Batch& b, uint32_t D, uint32_t window) {
    FewPlan p;
    const uint64_t units = ceil_div(longest_span(b, 16, window), kUnit), rows = (uint64_t)b.n_seq * c.heads;
    p.balanced = b.n_seq <= kScan && b.n_seq * units < 0x7FFFFFFF;
    p.wgs = (uint32_t)(p.balanced ? std::min<uint64_t>((uint64_t)cu_count() * (D == 256 ? 1 : KV_WGS), rows * units) : rows);
    p.join = p.balanced && units > 1;
    return p;
}
size_t few_ws_bytes(const FewPlan& p, uint32_t D) {
    return p.balanced ? (size_t)p.wgs * (sizeof(Cut) + 2 * 16 * (D + 2) * 4) : 0;
}

template <int D, int TYPE>
hipError_t few_d(const Cache& c, const Batch& b, const Attn& a, const FewPlan& p, const Rows& Q, const Rows& O, bool bf,
                 float* ws, hipStream_t s) {
    kv_attn_k<D, TYPE><<<p.wgs, 256, 0, s>>>(c, b, a, p.balanced, Q, O, bf, ws);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || !p.join) return e;
    kv_join_k<D><<<dim3(p.wgs, (b.max_q * a.group + 3) / 4), 256, 0, s>>>(c, b, a, p.wgs, O, bf, ws);
    return hipGetLastError();
}

uint64_t row_splits_wanted(const Cache& c, const Batch& b, const RowPlan& p) {
    return ceil_div((uint64_t)cu_count() * (p.rows == 256 ? 1 : 2), (uint64_t)b.n_seq * p.tiles * c.heads);
}
RowPlan row_plan(const Cache& c, const Batch& b, uint32_t group, uint32_t window) {
    RowPlan p;
    const uint64_t rows = (uint64_t)b.max_q * group;
    p.rows = rows <= 32 ? 32 : rows <= 64 ? 64 : rows <= 128 ? 128 : 256;
    p.tiles = (uint32_t)ceil_div(rows, p.rows);
    const uint64_t longest = longest_span(b, p.rows, window);
    p.chunk = (uint32_t)std::max<uint64_t>(ceil_div(ceil_div(longest, row_splits_wanted(c, b, p)), kTile) * kTile, kUnit);
    p.splits = (uint32_t)ceil_div(longest, p.chunk);
    return p;
}
// Of any window: a split has kUnit tokens at least.
size_t row_ws_bytes(const Cache& c, const Batch& b, uint32_t group, uint32_t D) {
    const RowPlan p = row_plan(c, b, group, 0);
    const uint64_t splits = std::min(row_splits_wanted(c, b, p), ceil_div(b.max_len, kUnit));
    return splits > 1 ? (size_t)b.n_seq * splits * p.tiles * c.heads * p.rows * (D + 2) * 4 : 0;
}

}  // namespace
}  // namespace kv

size_t kv_attn_ws_bytes(const kv::Cache& c, const kv::Batch& b, uint32_t D, uint32_t group) {
    const size_t n = kv::few(b, group) ? kv::few_ws_bytes(kv::few_plan(c, b, D, 0), D) : kv::row_ws_bytes(c, b, group, D);
    return n > 256 ? (n + 255) / 256 * 256 : 256;
}

bool kv_attn_fits(const kv::Cache& c, const kv::Batch& b, uint32_t group) {
    return (uint64_t)b.n_seq * b.max_q * c.heads * group < 0x7FFF0000ull;
}

hipError_t launch_kv_attn(const kv::Cache& c, const kv::Batch& b, uint32_t D, int type, const kv::Attn& a,
                          const kv::Rows& Q, const kv::Rows& O, bool bf, void* ws, hipStream_t s) {
    float* const w = static_cast<float*>(ws);
    if (kv::few(b, a.group)) {
        const kv::FewPlan p = kv::few_plan(c, b, D, a.window);
        return kv::by_dim(D, type, [&](auto d, auto t) {
            return kv::few_d<decltype(d)::value, decltype(t)::value>(c, b, a, p, Q, O, bf, w, s);
        });
    }
    const kv::RowPlan p = kv::row_plan(c, b, a.group, a.window);
    switch (D) {
        case 64: return kv::launch_rows<64>(type, c, b, a, p, Q, O, bf, w, s);
        case 96: return kv::launch_rows<96>(type, c, b, a, p, Q, O, bf, w, s);
        case 128: return kv::launch_rows<128>(type, c, b, a, p, Q, O, bf, w, s);
        case 192: return kv::launch_rows<192>(type, c, b, a, p, Q, O, bf, w, s);
        default: return kv::launch_rows<256>(type, c, b, a, p, Q, O, bf, w, s);
    }
}

}  // namespace kq
