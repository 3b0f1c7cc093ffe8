// kq_kv_rope.hip -- writing the 8-bit key/value cache with the rotary positions on the way
// (kq_kv_write_rope): keys turned before their block's scale is taken, queries turned beside them.
//
// Long prompts are bound by the writes and by 64-bit sums for the angles of keys, which each head's wave computes for itself
// (five prompts of 1201 to 5003 new tokens, 8 heads of 128 and 32 of queries: 78 us, as long as kq_rope and then kq_kv_write take, 75).
// At 192 and 256 columns the two calls are faster (blocks of 16: 120 and 154 us, in one call 153 and 177; blocks of 64, whose keys
// are turned twice, 122 and 182 at 192): the queries' waves hold the keys' registers and LDS, two waves a SIMD.
// Single tokens are bound by a chain of accesses (5.3 us), as kv_write_k's are; batches of trees by that chain with the angles in it and by the
// queries' rows, a wave each: 48 trees of 9 to 26 rows, 64 heads of queries over 8 of 128, 64 columns turned, 15.3 us, without
// queries 11.3 (kq_kv_write 9.3), with all columns turned 13.0: those that are not turned come last, a load, a wait and a store at a time.
#include "kq_kv_write_kernel.h"

namespace kq {
namespace kv {
namespace {

// blockIdx.x: first the blocks of keys and values, as in kv_write_k, then the rows of queries, q_each
// heads of one for each wave; .y = the sequence.
template <int D, int TYPE, int BF, int TURN>
__global__ __launch_bounds__(256) void kv_write_rope_k(Cache c, Batch b, Rows K, Rows V, uint32_t groups, uint32_t blocks, Turn turn,
                                                       Rows Q, Rows Qo, uint32_t q_heads, uint32_t q_parts, uint32_t q_each) {
    // a wave's turned keys, or the factors of a row
    constexpr int kKept = (D + 63) / 64 * 2 * 64 * kept_subs(D);
    static_assert(kKept * sizeof(u32x4) >= D / 2 * sizeof(rope::Factor));
    __shared__ u32x4 kept[4][kKept];
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    if (blockIdx.x < blocks) {
        write_block<D, TYPE, BF, TURN>(c, b, K, V, groups, blockIdx.x, turn, kept[wave]);
        return;
    }
    const uint32_t id = (blockIdx.x - blocks) * 4 + wave;
    const Seq s = sequence(b, c.page_log2, blockIdx.y);
    const int j = (int)(id / q_parts);
    if (j >= s.n) return;
    const uint32_t h0 = id % q_parts * q_each;
    const int row = s.row0 + j, pos = turn.pos ? turn.pos[row] : s.len - s.n + j;
    rope::turn_heads<BF, TURN>(turn.rope, pos, static_cast<const uint8_t*>(Q.p) + (int64_t)row * Q.row * 2,
                               static_cast<uint8_t*>(Qo.p) + (int64_t)row * Qo.row * 2, Q.head, Qo.head, h0,
                               min(q_heads, h0 + q_each), D, reinterpret_cast<rope::Factor*>(kept[wave]));
}

template <int D, int TYPE, int BF>
hipError_t write_rope_d(const Cache& c, const Batch& b, const Turn& turn, const Rows* Q, const Rows* Qo, uint32_t q_heads,
                        const Rows& K, const Rows& V, hipStream_t s) {
    const uint32_t groups = (2 * c.heads + 3) / 4, blocks = spans(b.max_q, 1u << c.block_log2) * groups;
    // heads of a row of queries a wave: four times as many as its lanes take at once. Waves are few beside the keys' (whose
    // registers and LDS they share), so that angles saved count for more than in kq_rope (32 heads of 128, bf16: 4
    // sequences of 2048 rows 42.8 us, one time as many 48.6; 48 of 20 rows 12.0, 15.7; one row 5.1 both)
    const uint32_t each = 4 * (64 / (turn.rope.rot / 16));
    const uint32_t parts = Q ? (q_heads + each - 1) / each : 0;
    const dim3 grid(blocks + (uint32_t)(((uint64_t)b.max_q * parts + 3) / 4), b.n_seq);
    const Rows q = Q ? *Q : Rows{}, qo = Q ? *Qo : Rows{};
    if (turn.rope.pairs) kv_write_rope_k<D, TYPE, BF, 1><<<grid, 256, 0, s>>>(c, b, K, V, groups, blocks, turn, q, qo, q_heads, parts, each);
    else kv_write_rope_k<D, TYPE, BF, 0><<<grid, 256, 0, s>>>(c, b, K, V, groups, blocks, turn, q, qo, q_heads, parts, each);
    return hipGetLastError();
}

}  // namespace
}  // namespace kv

hipError_t launch_kv_write_rope(const kv::Cache& c, const kv::Batch& b, uint32_t D, int type, const kv::Turn& turn,
                                const kv::Rows* Q, const kv::Rows* Qo, uint32_t q_heads, const kv::Rows& K, const kv::Rows& V,
                                bool bf, hipStream_t s) {
    return kv::by_dim(D, type, [&](auto d, auto t) {
        constexpr int N = decltype(d)::value, T = decltype(t)::value;
        return bf ? kv::write_rope_d<N, T, 1>(c, b, turn, Q, Qo, q_heads, K, V, s)
                  : kv::write_rope_d<N, T, 0>(c, b, turn, Q, Qo, q_heads, K, V, s);
    });
}

}  // namespace kq
