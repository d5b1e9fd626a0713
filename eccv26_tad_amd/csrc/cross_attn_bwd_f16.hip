// Cross attention, backward, for float16 (cross_attn_bwd.h).
#include "cross_attn_bwd.h"

namespace svtad {
template void cross_bwd_q<f16>(const CrossArgs&, int, hipStream_t);
template void cross_bwd_kv<f16>(const CrossArgs&, hipStream_t);
}  // namespace svtad
