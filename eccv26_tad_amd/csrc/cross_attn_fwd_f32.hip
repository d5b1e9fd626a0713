// Cross attention, forward, for float32 (cross_attn_fwd.h).
#include "cross_attn_fwd.h"

namespace svtad {
template void cross_fwd<float>(const CrossArgs&, int, hipStream_t);
}  // namespace svtad
