// Launch interface of the cross-attention kernels; one file per type and
// direction instantiates it.
#pragma once

#include "sv_attn.h"

namespace svtad {

// wave_rows: waves of a workgroup along the rows (4: 128 rows, 2: 64, 1: 16)
template <typename T> void cross_fwd(const CrossArgs& p, int wave_rows, hipStream_t st);
template <typename T> void cross_bwd_q(const CrossArgs& p, int wave_rows, hipStream_t st);
template <typename T> void cross_bwd_kv(const CrossArgs& p, hipStream_t st);

// Workgroups of 4 waves that a compute unit is to hold, by what a kernel keeps in
// registers. At 64 channels (ViT-L training case, two / three of them): forward
// 570 / 538 us, dq 650 / 658, dk and dv 798 / 913 (three spill).
template <typename T, int DP> constexpr int kResidentFwd = sizeof(T) == 2 && DP <= 64 ? 3 : 1;
template <typename T, int DP> constexpr int kResidentBwd = sizeof(T) == 2 && DP <= 64 ? 2 : 1;

// Keys of a workgroup of the dk, dv kernel
constexpr int kCrossKvKeys = 128;

}  // namespace svtad
