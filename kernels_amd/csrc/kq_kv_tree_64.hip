// kq_kv_tree_64.hip -- attention of trees over the 8-bit cache, heads 64 wide.
#include "kq_kv_tree_kernel.h"

namespace kq {
namespace kv {

template <>
hipError_t TreeKernels<64>::few(int type, const Cache& c, const Batch& b, const Attn& a, const FewPlan& p, const Rows& Q,
                              const Rows& O, bool bf, float* ws, hipStream_t s) {
    return type == KQ_KV_I8 ? few_d<64, KQ_KV_I8, true>(c, b, a, p, Q, O, bf, ws, s)
                            : few_d<64, KQ_KV_E4M3, true>(c, b, a, p, Q, O, bf, ws, s);
}

template <>
hipError_t TreeKernels<64>::rows(int type, const Cache& c, const Batch& b, const Attn& a, const FewPlan& p, const Rows& Q,
                               const Rows& O, bool bf, float* ws, hipStream_t s) {
    return type == KQ_KV_I8 ? tree_rows_d<64, KQ_KV_I8>(c, b, a, p, Q, O, bf, ws, s)
                            : tree_rows_d<64, KQ_KV_E4M3>(c, b, a, p, Q, O, bf, ws, s);
}

}  // namespace kv
}  // namespace kq
