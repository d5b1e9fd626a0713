// Cross attention, backward, for bfloat16 (cross_attn_bwd.h).
#include "cross_attn_bwd.h"

namespace svtad {
template void cross_bwd_q<bf16>(const CrossArgs&, int, hipStream_t);
template void cross_bwd_kv<bf16>(const CrossArgs&, hipStream_t);
}  // namespace svtad
