// Launch interface of the cross-attention kernels; one file per type and
// direction instantiates it.
#pragma once

#include "sv_attn.h"

namespace svtad {

// wave_rows: waves of a workgroup along the rows (4: 128 rows, 2: 64, 1: 16)
template <typename T> void cross_fwd(const CrossArgs& p, int wave_rows, hipStream_t st);
template <typename T> void cross_bwd_q(const CrossArgs& p, int wave_rows, hipStream_t st);
template <typename T> void cross_bwd_kv(const CrossArgs& p, hipStream_t st);

// Keys of a workgroup of the dk, dv kernel
inline int cross_kv_keys(int d) { return d <= 64 ? 128 : 64; }

}  // namespace svtad
