// kq_kv_rows_64.hip -- many-row attention over the 8-bit cache, heads 64 wide.
#include "kq_kv_rows_kernel.h"

namespace kq {
namespace kv {

template <>
hipError_t launch_rows<64>(int type, const Cache& c, const Batch& b, const Attn& a, const RowPlan& p, const Rows& Q,
                           const Rows& O, bool bf, float* ws, hipStream_t s) {
    return type == KQ_KV_I8 ? rows_d<64, KQ_KV_I8>(c, b, a, p, Q, O, bf, ws, s)
                            : rows_d<64, KQ_KV_E4M3>(c, b, a, p, Q, O, bf, ws, s);
}

}  // namespace kv
}  // namespace kq
