// kq_rope.hip -- rotary positions (kq_rope): rows of heads turned by their position's angles.
//
// Memory bounds it: 8192 rows of 40 heads of 128 in bf16 take 33 us (168 MB, 5.1 TB/s: what a copy reaches). One
// row's 40 heads take 2.5 us, less than the host needs for the call.
#include "kq_rope_device.h"

namespace kq {
namespace rope {
namespace {

// A wave for a row and up to `each` of its heads; blockIdx.x = the waves, four of them.
template <int F, int PAIRS>
__global__ __launch_bounds__(256) void rope_k(Rope r, const int32_t* pos, kv::Rows X, kv::Rows Y, uint32_t n_rows,
                                              uint32_t heads, uint32_t D, uint32_t parts, uint32_t each) {
    __shared__ Factor tables[4][kMostHead / 2];
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint64_t id = (uint64_t)blockIdx.x * 4 + wave;
    const uint32_t row = (uint32_t)(id / parts), part = (uint32_t)(id % parts);
    if (row >= n_rows) return;
    constexpr int kSize = F == KQ_F32 ? 4 : 2;
    turn_heads<F, PAIRS>(r, pos[row], static_cast<const uint8_t*>(X.p) + (int64_t)row * X.row * kSize,
                         static_cast<uint8_t*>(Y.p) + (int64_t)row * Y.row * kSize, X.head, Y.head, part * each,
                         min(heads, (part + 1) * each), D, tables[wave]);
}

template <int F>
hipError_t rope_f(const Rope& r, const int32_t* pos, const kv::Rows& X, const kv::Rows& Y, uint32_t n_rows, uint32_t heads,
                  uint32_t D, uint32_t parts, uint32_t each, uint32_t wgs, hipStream_t s) {
    if (r.pairs) rope_k<F, 1><<<wgs, 256, 0, s>>>(r, pos, X, Y, n_rows, heads, D, parts, each);
    else rope_k<F, 0><<<wgs, 256, 0, s>>>(r, pos, X, Y, n_rows, heads, D, parts, each);
    return hipGetLastError();
}

}  // namespace
}  // namespace rope

// Heads of a row that a wave turns, in registers as many as its lanes take at once, and twice that where there are rows
// enough for the device's SIMDs: the angles count for more then (8192 rows of 40 x 128 bf16: 32.8 us, one time as many 34.1, all
// heads 34.5; 2048 rows: 9.0, 10.1, 8.5; 64 rows: 2.8 one time, 3.1 twice, 3.8 all). Value by value a wave is
// at one head for long: one head a wave, or all of them (rot 40 of 128 columns, 40 heads, 512 rows: 8.8 us, all heads
// 12.6; 2048 rows: 32.1, all heads 23.7). Its accesses of two bytes bound it: 2.8 times what a copy of those rows takes (rot 64: 8.5).
static uint32_t rope_heads_each(uint64_t n_rows, uint32_t heads, uint32_t rot) {
    const bool many = n_rows > 1024;
    if (rot % 16 == 0) return 64 / (rot / 16) << many;
    return many ? heads : 1;
}

bool rope_fits(uint32_t n_rows, uint32_t heads, uint32_t rot) {
    const uint32_t each = rope_heads_each(n_rows, heads, rot);
    return ((uint64_t)n_rows * ((heads + each - 1) / each) + 3) / 4 <= kv::kMostGroups;
}

hipError_t launch_rope(const rope::Rope& r, const int32_t* pos, const kv::Rows& X, const kv::Rows& Y, uint32_t n_rows,
                       uint32_t heads, uint32_t D, kq_dtype f, hipStream_t s) {
    const uint32_t each = rope_heads_each(n_rows, heads, r.rot), parts = (heads + each - 1) / each;
    const uint32_t wgs = (uint32_t)(((uint64_t)n_rows * parts + 3) / 4);
    return f == KQ_F16    ? rope::rope_f<KQ_F16>(r, pos, X, Y, n_rows, heads, D, parts, each, wgs, s)
           : f == KQ_BF16 ? rope::rope_f<KQ_BF16>(r, pos, X, Y, n_rows, heads, D, parts, each, wgs, s)
                          : rope::rope_f<KQ_F32>(r, pos, X, Y, n_rows, heads, D, parts, each, wgs, s);
}

}  // namespace kq
