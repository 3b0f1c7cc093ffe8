// kq_spec.hip -- trees of drafted tokens (kq_kv_tree): their rows' masks and positions.
#include "kq_kv_device.h"

namespace kq {
namespace kv {
namespace {

// The rows that row j of n continues, itself first: f(row) for each, until there is no more or f says so. A parent
// is less than its row, so the way ends.
template <class Fn>
__device__ __forceinline__ void each_ancestor(const int* parent, int j, Fn f) {
    while (f(j)) {
        const int p = parent[j];
        if (p < 0 || p >= j) return;
        j = p;
    }
}

// A workgroup a sequence, a thread a row: it walks up its own ancestors. They come in falling order, so
// that each word of the mask is whole before the next begins. Latency bounds it: a step of
// the way is one read of LDS (one tree of 60 rows 2.7 us, 64 of 64 rows 3.8, 16 of 1024 rows, up to 130 deep, 44).
__global__ __launch_bounds__(256) void kv_tree_k(Batch b, const int32_t* parents, uint32_t* mask, uint32_t words, int32_t* pos,
                                                 uint32_t window) {
    __shared__ int parent[kMostNodes];
    const Seq s = sequence(b, 0, blockIdx.x);
    for (int j = threadIdx.x; j < s.n; j += 256) parent[j] = parents[s.row0 + j];
    __syncthreads();
    for (int j = threadIdx.x; j < s.n; j += 256) {
        uint32_t* const bits = mask + (uint64_t)(uint32_t)(s.row0 + j) * words;
        int at = (int)words - 1, depth = -1;
        uint32_t word = 0;
        each_ancestor(parent, j, [&](int t) {
            ++depth;
            if (window && (uint32_t)depth >= window) return true;
            for (; at > t >> 5; --at) {
                bits[at] = word;
                word = 0;
            }
            word |= 1u << (t & 31);
            return true;
        });
        for (; at >= 0; --at) {
            bits[at] = word;
            word = 0;
        }
        if (pos) pos[s.row0 + j] = s.len - s.n + depth;
    }
}

}  // namespace
}  // namespace kv

hipError_t launch_kv_tree(const kv::Batch& b, const int32_t* parent, uint32_t* mask, uint32_t words, int32_t* pos,
                          uint32_t window, hipStream_t s) {
    kv::kv_tree_k<<<b.n_seq, 256, 0, s>>>(b, parent, mask, words, pos, window);
    return hipGetLastError();
}

}  // namespace kq
