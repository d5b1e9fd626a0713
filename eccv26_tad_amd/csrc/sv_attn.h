// Pieces shared by the cross-attention kernels (gfx950).
//
// All products run on 16 x 16 matrix-core tiles whose left operand comes from
// LDS and whose right operand is in registers. A score tile is computed
// transposed, S^T = K Q^T: each lane then holds scores of ONE query (lane %
// 16) for 4 consecutive keys per tile, so the softmax runs in the lane (two
// lane exchanges join the 4 lane groups), and the tile is, without any
// movement, the right operand of the next product O^T = V^T P^T. That
// product's 32 reduction values are the keys of two score tiles: lane group g
// holds keys 4g .. 4g+3 of each, and V^T's operand is read to match, as two
// transposing LDS reads of 4 keys. The backward kernels use the same two
// patterns.
#pragma once

#include "sv_internal.h"
#include "sv_mfma.h"
#include "sv_vec.h"

namespace svtad {

// 8 reduction values of a 16 x 16 x 32 product per lane; float32 runs it as
// eight 16 x 16 x 4 products, whose operands pair values of equal position, so
// the same layout serves.
template <typename T> struct Frag8 {
    T e[8] __attribute__((aligned(16)));
};
template <> struct Frag8<f16> {
    u32x4 v;
};
template <> struct Frag8<bf16> {
    u32x4 v;
};

template <typename T>
__device__ __forceinline__ f32x4 mma(const Frag8<T>& a, const Frag8<T>& b, f32x4 c) {
    if constexpr (sizeof(T) == 2) {
        return MfmaOp<T>::run(a.v, b.v, c);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.e[j], b.e[j], c, 0, 0, 0);
        return c;
    }
}

template <typename T> __device__ __forceinline__ Frag8<T> zero_frag() {
    return __builtin_bit_cast(Frag8<T>, Pack<T, 8>{});
}

// 8 elements of a row of d in global memory from column c on, 0 past its end
template <typename T>
__device__ __forceinline__ Frag8<T> load_frag(const T* row, int c, int d) {
    if (c + 8 <= d) return __builtin_bit_cast(Frag8<T>, *(const Pack<T, 8>*)(row + c));
    Pack<T, 8> v;
#pragma unroll
    for (int e = 0; e < 8; ++e) v.e[e] = c + e < d ? row[c + e] : (T)0.f;
    return __builtin_bit_cast(Frag8<T>, v);
}

// The right operand of a 32-value product from two score tiles of a lane
template <typename T>
__device__ __forceinline__ Frag8<T> pack_frag(const f32x4& a, const f32x4& b) {
    Pack<T, 8> v;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        v.e[e] = (T)a[e];
        v.e[4 + e] = (T)b[e];
    }
    return __builtin_bit_cast(Frag8<T>, v);
}

// LDS tile of rows of DP elements; the pad spreads the 16 rows that a fragment
// read touches over all banks.
template <typename T, int DP> constexpr int kPitch = DP + 16 / (int)sizeof(T);

template <typename T>
__device__ __forceinline__ Frag8<T> lds_frag(const T* p) {  // 8 consecutive elements
    Frag8<T> f;
    if constexpr (sizeof(T) == 2) {
        f.v = *(const u32x4*)p;
    } else {
        const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
        for (int e = 0; e < 4; ++e) f.e[e] = a[e], f.e[4 + e] = b[e];
    }
    return f;
}

// Transposed: column `col0 + lane % 16` of rows 4g .. 4g+3 and 16 + 4g ..
// 16 + 4g+3 below `tile` (g = lane / 16): the left operand that pairs with
// pack_frag. For 16-bit types the transposing read: the 16 lanes of a group
// give the addresses of 4 rows' 4 chunks and receive a column each.
typedef short s16x4 __attribute__((ext_vector_type(4)));
template <typename T, int PITCH_>
__device__ __forceinline__ Frag8<T> lds_frag_t(const T* tile, int col0, int lane) {
    const int g = lane >> 4, i = lane & 15;
    Frag8<T> f;
    if constexpr (sizeof(T) == 2) {
        typedef __attribute__((address_space(3))) s16x4* lds4;
        const T* p = tile + (4 * g + (i >> 2)) * PITCH_ + col0 + 4 * (i & 3);
        union {
            s16x4 h[2];
            u32x4 v;
        } u;
        u.h[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)p);
        u.h[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds4)(p + 16 * PITCH_));
        f.v = u.v;
    } else {
        const T* p = tile + 4 * g * PITCH_ + col0 + i;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            f.e[e] = p[e * PITCH_];
            f.e[4 + e] = p[(16 + e) * PITCH_];
        }
    }
    return f;
}

__device__ __forceinline__ float across_groups_max(float v) {  // over lanes of equal lane % 16
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}
__device__ __forceinline__ float across_groups_sum(float v) {
    v += __shfl_xor(v, 16, 64);
    return v + __shfl_xor(v, 32, 64);
}

// Stores 4 consecutive float32 values as T; the row's end may fall inside.
template <typename T>
__device__ __forceinline__ void store4(T* row, int c, int d, f32x4 v) {
    if (c + 4 <= d) {
        Pack<T, 4> o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o.e[e] = (T)v[e];
        *(Pack<T, 4>*)(row + c) = o;
    } else {
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + e < d) row[c + e] = (T)v[e];
    }
}

// ---------------------------------------------------------------------------

struct CrossArgs {
    const void *q, *k, *v, *o, *dout;
    void *out, *dk, *dv;   // out: the forward's output, or dq
    float* lse;            // [B KH][M]: log2 of a row's sum of 2^(c s), +inf for a row that sees no key
    float* delta;          // [B KH][M]: sum over d of dout out
    const int32_t* lengths;   // [B] or NULL
    const uint8_t* mask;      // [B, Nk] by mask_b, mask_n, or NULL; nonzero: the key is seen
    float* part;           // partial results of the splits (NULL: none)
    int64_t qb, qn, qh, kb, kn, kh, vb, vn, vh, ob, on, oh, gb, gn, gh;  // element strides of q, k, v, o, dout
    int64_t mask_b, mask_n;
    int B, H, KH, G, D;    // G = H / KH query heads per key head
    int64_t Nq, Nk, M;     // M = Nq G rows per key head: row r is query r / G, head (key head) G + r % G
    int splits;            // of the reduced axis
    float c, scale;        // scale log2(e)
};

// Row r of the M rows of key head `j`: its query and head
__device__ __forceinline__ int64_t row_at(const CrossArgs& p, int64_t r, int64_t sn, int64_t sh, int j) {
    if (p.G == 1) return r * sn + j * sh;
    const uint64_t n = (uint64_t)r / (uint32_t)p.G;
    return n * sn + (int64_t)(j * p.G + (int)(r - n * p.G)) * sh;
}

__device__ __forceinline__ int64_t seen_length(const CrossArgs& p, int b) {
    if (!p.lengths) return p.Nk;
    const int64_t n = p.lengths[b];
    return n < 0 ? 0 : n > p.Nk ? p.Nk : n;
}

}  // namespace svtad
