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

// 8 or 16 bytes of global memory that are read, or written, once: they are not
// kept in the caches (1 GiB read through: 7.0 against 6.1 TB/s; copied: 5.6
// against 5.3). A wave's stores should fill whole lines: nothing merges them. The
// address space is given because pointers that were kept in LDS do not tell.
template <int BYTES> struct OnceType;
template <> struct OnceType<16> {
    typedef unsigned int type __attribute__((ext_vector_type(4), aligned(2)));
};
template <> struct OnceType<8> {
    typedef unsigned int type __attribute__((ext_vector_type(2), aligned(2)));
};
template <typename P>
__device__ __forceinline__ P load_once(const void* p) {
    typedef __attribute__((address_space(1))) const typename OnceType<sizeof(P)>::type* global;
    return __builtin_bit_cast(P, __builtin_nontemporal_load((global)p));
}
template <typename P>
__device__ __forceinline__ void store_once(void* p, const P& v) {
    typedef typename OnceType<sizeof(P)>::type U;
    typedef __attribute__((address_space(1))) U* global;
    __builtin_nontemporal_store(__builtin_bit_cast(U, v), (global)p);
}

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
