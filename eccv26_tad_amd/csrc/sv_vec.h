// Vector loads and stores of rows whose start is aligned to an element only,
// and the wave reductions of the row kernels (gfx950, wave64).
#pragma once

#include "sv_common.h"

namespace svtad {

// N consecutive elements, moved by 16-byte instructions at any element
// alignment (global memory takes unaligned vector accesses on gfx950).
template <typename T, int N>
struct __attribute__((packed, aligned(sizeof(T)))) Pack {
    T e[N];
};

// Elements of 16 bytes.
template <typename T> constexpr int kVec = 16 / (int)sizeof(T);

template <int CTRL>
__device__ __forceinline__ float dpp_move(float v) {
    return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true));
}

// Sum over the aligned group of `lanes` (a power of two, uniform) lanes that
// holds the caller, in every lane of it, in a fixed order.
__device__ __forceinline__ float group_sum(float v, int lanes) {
    if (lanes > 1) v += dpp_move<0xB1>(v);   // quad_perm: lane ^ 1
    if (lanes > 2) v += dpp_move<0x4E>(v);   // quad_perm: lane ^ 2
    if (lanes > 4) v += dpp_move<0x141>(v);  // row_half_mirror: the other quad of 8
    if (lanes > 8) v += dpp_move<0x140>(v);  // row_mirror: the other half of 16
    if (lanes > 16) v += __shfl_xor(v, 16, 64);
    if (lanes > 32) v += __shfl_xor(v, 32, 64);
    return v;
}

// Sum of count float4 at p, p + stride, ... (floats), in order, four loads in
// flight
__device__ __forceinline__ void add_strided(float (&acc)[4], const float* p, int64_t stride, int count) {
    for (int i = 0; i < count; i += 4) {
        Pack<float, 4> v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) v[u] = *(const Pack<float, 4>*)(p + (i + u < count ? i + u : count - 1) * stride);
#pragma unroll
        for (int u = 0; u < 4; ++u)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[e] += i + u < count ? v[u].e[e] : 0.f;
    }
}

}  // namespace svtad
