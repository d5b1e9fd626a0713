// Cross attention, forward, for bfloat16 (cross_attn_fwd.h).
#include "cross_attn_fwd.h"

namespace svtad {
template void cross_fwd<bf16>(const CrossArgs&, int, hipStream_t);
}  // namespace svtad
