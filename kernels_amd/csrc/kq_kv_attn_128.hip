// kq_kv_attn_128.hip -- attention over the 8-bit cache, heads 128 wide.
#include "kq_kv_rows_kernel.h"

namespace kq {
namespace kv {

template <>
hipError_t AttnKernels<128>::few(int type, const Cache& c, const Batch& b, const Attn& a, const FewPlan& p, const Rows& Q,
                              const Rows& O, bool bf, float* ws, hipStream_t s) {
    return type == KQ_KV_I8 ? few_d<128, KQ_KV_I8, false>(c, b, a, p, Q, O, bf, ws, s)
                            : few_d<128, KQ_KV_E4M3, false>(c, b, a, p, Q, O, bf, ws, s);
}

template <>
hipError_t AttnKernels<128>::rows(int type, const Cache& c, const Batch& b, const Attn& a, const RowPlan& p, const Rows& Q,
                               const Rows& O, bool bf, float* ws, hipStream_t s) {
    return type == KQ_KV_I8 ? rows_d<128, KQ_KV_I8>(c, b, a, p, Q, O, bf, ws, s)
                            : rows_d<128, KQ_KV_E4M3>(c, b, a, p, Q, O, bf, ws, s);
}

}  // namespace kv
}  // namespace kq
