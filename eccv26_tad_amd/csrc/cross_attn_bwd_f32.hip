// Cross attention, backward, for float32 (cross_attn_bwd.h).
#include "cross_attn_bwd.h"

namespace svtad {
template void cross_bwd_q<float>(const CrossArgs&, int, hipStream_t);
template void cross_bwd_kv<float>(const CrossArgs&, hipStream_t);
}  // namespace svtad
