// Pieces shared by the cross-attention kernels (gfx950).
//
// All products run on the matrix cores with the left operand from LDS and the
// right operand in registers. A score tile is computed transposed, S^T = K Q^T:
// each lane then holds scores of ONE query (lane % S, tiles of S x S, S 32 or
// 16), so that the softmax runs in the lane and a row's sum takes one or two
// lane exchanges, and the tile is, without any movement, the right operand of
// the next product O^T = V^T P^T: V^T is read from LDS in the order in which
// the lanes hold the keys. The backward kernels use the same two patterns.
#pragma once

#include <type_traits>

#include "sv_internal.h"
#include "sv_mfma.h"
#include "sv_vec.h"

namespace svtad {

template <typename I>
__device__ __forceinline__ I lesser(I a, I b) {  // in integers (an overloaded min may go by way of double)
    return a < b ? a : b;
}

// 8 reduction values of a product, per lane
template <typename T> struct Frag8 {
    T e[8] __attribute__((aligned(16)));
};
template <> struct Frag8<f16> {
    u32x4 v;
};
template <> struct Frag8<bf16> {
    u32x4 v;
};

template <typename T> __device__ __forceinline__ Frag8<T> zero_frag() {
    return __builtin_bit_cast(Frag8<T>, Pack<T, 8>{});
}

// 8 elements of a row of d in global memory from column c on, 0 past its end.
// VEC: d is a multiple of 8 and rows start at 16 bytes.
template <typename T, bool VEC>
__device__ __forceinline__ Frag8<T> load_frag(const T* row, int c, int d) {
    if constexpr (VEC) {
        return c < d ? *(const Frag8<T>*)(row + c) : zero_frag<T>();
    } else {
        Pack<T, 8> v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v.e[e] = c + e < d ? row[c + e] : (T)0.f;
        return __builtin_bit_cast(Frag8<T>, v);
    }
}

// A tile of rows of W elements in LDS, in pieces of 16 bytes without padding
// (so that a wave's loads may land there directly, 64 consecutive pieces at a
// time). Row r keeps its piece c at place c ^ swizzle(r), which spreads both
// kinds of reads over all banks: the same piece of 16 rows (frag), and 2 or 4
// neighbouring pieces of 8 or 4 rows (frag_t). For both the swizzle is the row's
// number, in units of the rows that fill all banks (256 bytes), with its bits
// reversed: neighbouring rows differ in the highest bit.
template <typename T, int W>
struct LdsTile {
    static constexpr int kRow = W * (int)sizeof(T), kPieces = kRow / 16, kElems = 16 / (int)sizeof(T);
    static constexpr int kBits = kRow >= 256 ? 4 : kRow == 128 ? 3 : 2, kShift = 4 - kBits;

    static __device__ __forceinline__ int swizzle(int r) {
        return (int)(__builtin_bitreverse32((uint32_t)((r & 15) >> kShift)) >> (32 - kBits));
    }
};

typedef float f32x16 __attribute__((ext_vector_type(16)));

// Products of S x S tiles, 64 lanes: lane l has column l % S of the right operand
// and of the result and row l % S of the left one, with 8 reduction values at
// slot l / S of K = 512 / S. Its 4 Q result values are rows row4(q) .. + 3 of
// group q. float32 runs as eight products whose operands pair values of equal
// position, so the same layout serves. S 32 takes fewer operand reads per
// product and more issue slots are free beside it (random operands, one or two
// waves per SIMD: 1850 TFLOP/s against 1150 and 1540 with S 16); S 16 wastes
// less on a few rows.
template <typename T, int S>
struct Shape {
    typedef float Acc __attribute__((ext_vector_type(S * S / 64)));
    static constexpr int K = 512 / S, Q = S * S / 256;

    static __device__ __forceinline__ int col(int lane) { return lane % S; }
    static __device__ __forceinline__ int slot(int lane) { return lane / S; }
    static __device__ __forceinline__ int row4(int q, int lane) { return S == 32 ? 8 * q + 4 * slot(lane) : 4 * slot(lane); }

    static __device__ __forceinline__ Acc mma(const Frag8<T>& a, const Frag8<T>& b, Acc c) {
        if constexpr (sizeof(T) == 4) {
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                if constexpr (S == 32) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.e[j], b.e[j], c, 0, 0, 0);
                else c = __builtin_amdgcn_mfma_f32_16x16x4f32(a.e[j], b.e[j], c, 0, 0, 0);
            }
            return c;
        } else if constexpr (S == 16) {
            return MfmaOp<T>::run(a.v, b.v, c);
        } else if constexpr (std::is_same_v<T, f16>) {
            return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a.v), __builtin_bit_cast(f16x8, b.v), c, 0, 0, 0);
        } else {
            return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a.v), __builtin_bit_cast(bf16x8, b.v), c, 0, 0, 0);
        }
    }
    // Whether product ks of a row of d elements has any: float32 products are slow
    // enough for the branch, in 16 bits the zeros are multiplied.
    static __device__ __forceinline__ bool step_in(int ks, int d) { return sizeof(T) == 2 || ks * K < d; }
    static __device__ __forceinline__ Acc fill(float v) {
        Acc a;
#pragma unroll
        for (int e = 0; e < 4 * Q; ++e) a[e] = v;
        return a;
    }
    static __device__ __forceinline__ f32x4 quad(const Acc& a, int q) { return f32x4{a[4 * q], a[4 * q + 1], a[4 * q + 2], a[4 * q + 3]}; }

    // The right operand of product kk (rows kk K .. of a column of tiles) from the
    // lane's own results
    static __device__ __forceinline__ Frag8<T> pack(const Acc* tiles, int kk) {
        typedef T tx8 __attribute__((ext_vector_type(8)));
        typedef float f32x8 __attribute__((ext_vector_type(8)));
        f32x8 v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = S == 32 ? tiles[kk / 2][(8 * (kk & 1) + e) % (4 * Q)] : tiles[2 * kk + e / 4][e % 4];
        return __builtin_bit_cast(Frag8<T>, __builtin_convertvector(v, tx8));
    }

    // From an LDS tile of rows of W elements: elements ks K + 8 slot .. of row r0 +
    // lane % S
    template <int W>
    static __device__ __forceinline__ Frag8<T> frag(const unsigned char* tile, int r0, int ks, int lane) {
        typedef LdsTile<T, W> L;
        const unsigned char* const row = tile + (r0 + col(lane)) * L::kRow;
        const int sw = L::swizzle(col(lane));
        if constexpr (sizeof(T) == 2) {
            Frag8<T> f;
            f.v = *(const u32x4*)(row + (((ks * (K / 8)) ^ (slot(lane) ^ sw)) << 4));
            return f;
        } else {
            union {
                u32x4 q[2];
                Frag8<T> f;
            } u;
            const int at = (ks * (K / 4)) ^ ((2 * slot(lane)) ^ sw);
            u.q[0] = *(const u32x4*)(row + (at << 4));
            u.q[1] = *(const u32x4*)(row + ((at ^ 1) << 4));
            return u.f;
        }
    }
    // Transposed, column db S + lane % S of the K rows from r0 on in the order of
    // `pack`: rows 4 slot .. + 3 and K / 2 + 4 slot .. + 3. For 16-bit types the
    // transposing read: the 16 lanes of a group give the addresses of 4 rows'
    // 4 chunks of 8 bytes and receive a column each.
    template <int W>
    static __device__ __forceinline__ Frag8<T> frag_t(const unsigned char* tile, int r0, int db, int lane) {
        typedef LdsTile<T, W> L;
        Frag8<T> f;
        if constexpr (sizeof(T) == 2) {
            typedef short s16x4 __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) s16x4* lds4;
            const int i = lane & 15, r = 4 * slot(lane) + (i >> 2);
            const int piece = (S == 32 ? 2 * ((lane >> 4) & 1) : 0) + ((i >> 1) & 1);  // of the S columns
            union {
                s16x4 h[2];
                u32x4 v;
            } u;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int rh = r + h * (K / 2);
                u.h[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                    (lds4)(tile + (r0 + rh) * L::kRow + (((db * (S / 8)) ^ (piece ^ L::swizzle(rh))) << 4) + 8 * (i & 1)));
            }
            f.v = u.v;
        } else {
            const int i = col(lane);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int r = 4 * slot(lane) + e % 4 + e / 4 * (K / 2);
                f.e[e] = *(const T*)(tile + (r0 + r) * L::kRow + (((db * (S / 4)) ^ ((i >> 2) ^ L::swizzle(r))) << 4) + 4 * (i & 3));
            }
        }
        return f;
    }

    // Over the lanes of one column
    static __device__ __forceinline__ float col_max(float v) {
        if constexpr (S == 16) v = fmaxf(v, __shfl_xor(v, 16, 64));
        return fmaxf(v, __shfl_xor(v, 32, 64));
    }
    static __device__ __forceinline__ float col_sum(float v) {
        if constexpr (S == 16) v += __shfl_xor(v, 16, 64);
        return v + __shfl_xor(v, 32, 64);
    }
};

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

// Stores 4 values as T, and with `rest` what the rounding took from them, as T
template <typename T>
__device__ __forceinline__ void store4_rest(T* row, T* rest, int c, int d, f32x4 v) {
    store4<T>(row, c, d, v);
    if (rest) {
#pragma unroll
        for (int e = 0; e < 4; ++e) v[e] -= (float)(T)v[e];
        store4<T>(rest, c, d, v);
    }
}

// A buffer from `base` (the same for the wave) on, as the builtins and as the
// instruction take it. Loads check their rows themselves and give kOOB where
// there is none; valid offsets are below 2^31.
struct Buffer {
    rsrc_t r;
    u32x4 q;
};
__device__ __forceinline__ Buffer open_buffer(const void* base) {
    const uint64_t at = (uint64_t)base;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)at), hi = __builtin_amdgcn_readfirstlane((uint32_t)(at >> 32));
    return {make_rsrc(base, 0x7fffffffu), u32x4{lo, hi & 0xffffu, 0x7fffffffu, 0x00020000u}};
}

// Where in LDS a pointer into it points: the low half of its flat address (the
// high half is the aperture). The same for the wave.
__device__ __forceinline__ uint32_t lds_offset(const void* p) {
    return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)p);
}

// 16 bytes per lane from `offset` in the buffer to 16 lane + `to` in LDS (`to` is
// the same for the wave). Written as the instruction itself: before any read of
// LDS the compiler waits for the loads to LDS that it knows of, as it cannot
// tell which of two tiles they go to, and no load would be in flight during the
// work on the tile before. There is no output register; `landed` waits. m0, which
// holds the LDS address, is set in the same statement. The compiler cannot see into
// it either: a descriptor's words may come from a vector instruction
// (v_readfirstlane) right before the statement, and a load may read them 5 wait
// states later at the earliest. The write of m0 is one, the s_nop the other 4.
// ONCE: memory that nobody reads again, not kept in the caches.
template <bool ONCE>
__device__ __forceinline__ void load_to_lds(u32x4 r, uint32_t offset, const unsigned char* to) {
    const uint32_t base = lds_offset(to);
    if constexpr (ONCE)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen nt lds"
                     :
                     : "s"(base), "v"(offset), "s"(r)
                     : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                     :
                     : "s"(base), "v"(offset), "s"(r)
                     : "memory", "m0");
}

// The same for 4 bytes per lane.
__device__ __forceinline__ void load_word_to_lds(u32x4 r, uint32_t offset, const void* to) {
    const uint32_t base = lds_offset(to);
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 3\n\tbuffer_load_dword %1, %2, 0 offen lds"
                 :
                 : "s"(base), "v"(offset), "s"(r)
                 : "memory", "m0");
}

// One thread's share of loading a tile of TILE rows by W elements to LDS through
// a buffer descriptor: rows that do not exist, and columns past d, arrive as
// zeros without a branch. VEC: straight to LDS, without registers; a barrier
// after `landed` makes the tile readable. Otherwise element by element through
// registers, which `store` empties into the tile.
template <typename T, int TILE, int W, bool VEC, bool ONCE = false>
struct Stage {
    typedef LdsTile<T, W> Tile;
    static constexpr int kCount = TILE * Tile::kPieces / 256, kBytes = TILE * Tile::kRow, E = Tile::kElems;
    static_assert(TILE * Tile::kPieces % 256 == 0, "whole pieces per thread");
    u32x4 v[VEC ? 1 : kCount];

    static __device__ __forceinline__ int row(int i) { return (threadIdx.x + i * 256) / Tile::kPieces; }
    static __device__ __forceinline__ int col(int i) {
        return (((threadIdx.x + i * 256) % Tile::kPieces) ^ Tile::swizzle(row(i))) * E;
    }

    // piece i, of a row that starts `at` bytes from the descriptor's (kOOB: none)
    __device__ __forceinline__ void load(int i, const Buffer& r, uint32_t at, int d, unsigned char* tile) {
        constexpr int S = (int)sizeof(T);
        const int c = col(i);
        if constexpr (VEC) {
            load_to_lds<ONCE>(r.q, c < d ? at + c * S : kOOB, tile + (i * 256 + (threadIdx.x & ~63)) * 16);
        } else {
            Pack<T, E> p;
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const uint32_t off = c + e < d ? at + (c + e) * S : kOOB;
                if constexpr (S == 2) p.e[e] = __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b16(r.r, off, 0, 0));
                else p.e[e] = __builtin_bit_cast(T, __builtin_amdgcn_raw_buffer_load_b32(r.r, off, 0, 0));
            }
            v[i] = __builtin_bit_cast(u32x4, p);
        }
    }
    __device__ __forceinline__ void store(unsigned char* tile) const {
        if constexpr (!VEC) {
#pragma unroll
            for (int i = 0; i < kCount; ++i) *(u32x4*)(tile + (threadIdx.x + i * 256) * 16) = v[i];
        }
    }
};

// Waits for this wave's loads to LDS (which the compiler does not know of), by
// the builtin, from which the compiler sees that its own loads are done as well:
// else it would wait for those made before a loop inside it, and with them for
// the loads to LDS.
__device__ __forceinline__ void landed() {
    asm volatile("" ::: "memory");
    __builtin_amdgcn_s_waitcnt(0x0f70);  // vmcnt(0)
    asm volatile("" ::: "memory");
}

// ---------------------------------------------------------------------------

struct CrossArgs {
    const void *q, *k, *v, *o, *dout;
    void *out, *dk, *dv;   // out: the forward's output, or dq
    void* rest;            // like the forward's output: what its rounding took (NULL: not kept)
    float* lse;            // [B KH][M]: log2 of a row's sum of 2^(c s), +inf for a row that sees no key
    float* delta;          // [B KH][M]: minus the sum over d of dout out
    const int32_t* lengths;   // [B] or NULL
    const uint8_t* mask;      // [B, Nk] by mask_b, mask_n, or NULL; nonzero: the key is seen
    float* part;           // partial results of the splits (NULL: none)
    int64_t qb, qn, qh, kb, kn, kh, vb, vn, vh, ob, on, oh, gb, gn, gh;  // element strides of q, k, v, o, dout
    int64_t mask_b, mask_n;
    int B, H, KH, G, D;    // G = H / KH query heads per key head
    int64_t Nq, Nk, M;     // M = Nq G rows per key head (below 2^31): row r is query r / G, head (key head) G + r % G
    int splits;            // of the reduced axis
    float c, scale;        // c = scale log2(e)
    float inv_g;           // 1 / G
    float up, down;        // a power of two and its inverse: what float16 probabilities are scaled by in dv
    bool vec;              // D and all strides are multiples of 8 elements, all starts of 16 bytes
};

__device__ __forceinline__ int64_t seen_length(const CrossArgs& p, int b) {
    if (!p.lengths) return p.Nk;
    const int64_t n = p.lengths[b];
    return n < 0 ? 0 : n > p.Nk ? p.Nk : n;
}

// Splits are joined by workgroups of 256 / G chunks of 4 values by G thread
// groups, each of which takes consecutive splits; the groups' sums are added in
// order. Few splits take one group, whose loads are all in flight at once. No more
// than 1024 workgroups write partial results, so that all chunks together are far
// from 2^31: their divisions are 32 bits (24000 rows of 64 in two splits, the
// forward with its join: 23.8 us so, 30.7 by four groups and with 64 bits).
constexpr int kJoinGroups = 4, kOneGroup = 8, kMaxSplits = 64;  // groups, the most splits that one takes, and all take
template <int G>
struct JoinChunk {
    static constexpr int kChunks = 256 / G;
    uint32_t e;  // of all chunks
    int chunk, g;
    __device__ __forceinline__ JoinChunk() : e(blockIdx.x * kChunks + threadIdx.x % kChunks), chunk(threadIdx.x % kChunks), g(threadIdx.x / kChunks) {}
};
template <int G>
__device__ __forceinline__ f32x4 join_groups(f32x4 v, const JoinChunk<G>& j) {
    if constexpr (G == 1) return v;
    else {
        __shared__ f32x4 red[G - 1][JoinChunk<G>::kChunks];
        if (j.g > 0) red[j.g - 1][j.chunk] = v;
        __syncthreads();
#pragma unroll
        for (int q = 1; q < G; ++q) v += red[q - 1][j.chunk];
        return v;
    }
}
// This thread's share of a chunk's splits, `stride` floats apart, from p on
template <int G>
__device__ __forceinline__ f32x4 split_sum(const float* p, int64_t stride, int splits, int g) {
    const int per = (splits + G - 1) / G, s0 = lesser(splits, g * per), n = lesser(splits, s0 + per) - s0;
    float a[4] = {0.f, 0.f, 0.f, 0.f};
    add_strided(a, p + s0 * stride, stride, n);
    return f32x4{a[0], a[1], a[2], a[3]};
}

// Workgroup -> (sample and key head, tile): the n tiles of a head stay on one
// XCD, whose L2 then holds its keys (workgroup w runs on XCD w % 8), and
// neighbouring heads go to different XCDs, so that samples of unequal length
// load all XCDs alike. The heads beyond a multiple of 8 are cut across XCDs.
struct HeadTile {
    int bh;
    uint32_t tile;
};
__device__ __forceinline__ HeadTile head_tile(uint32_t w, uint32_t grid, uint32_t n) {
    const uint32_t eights = grid / n / 8, whole = eights * 8 * n;
    if (w < whole) {
        const uint32_t k = w >> 3, q = k / n;
        return {(int)(q * 8 + (w & 7)), k - q * n};
    }
    const uint32_t t = (uint32_t)xcd_tile(w - whole, grid - whole), q = t / n;
    return {(int)(eights * 8 + q), t - q * n};
}

// The sample whose length has this rank, the longest first: workgroups start in
// order, and those of long samples must not start last. Up to 64 samples, each
// lane ranks one (equal lengths by number); others keep their order.
__device__ __forceinline__ int sample_of_rank(const CrossArgs& p, int rank) {
    if (!p.lengths || p.B > 64 || p.B == 1) return rank;
    const int lane = threadIdx.x & 63;
    const int64_t own = lane < p.B ? seen_length(p, lane) : -1;
    const int n = (int)lesser<int64_t>(own, 0x7fffffff);
    int r = 0;
    for (int b = 0; b < p.B; ++b) {
        const int other = __builtin_amdgcn_readlane(n, b);
        r += other > n || (other == n && b < lane);
    }
    return __builtin_ctzll(__ballot(lane < p.B && r == rank));
}

// Row r of the M rows of key head `j`: the offset of its query and head
__device__ __forceinline__ int64_t row_at(const CrossArgs& p, int64_t r, int64_t sn, int64_t sh, int j) {
    if (p.G == 1) return r * sn + j * sh;
    const uint32_t n = (uint32_t)r / (uint32_t)p.G;
    return n * sn + (int64_t)(j * p.G + (int)(r - n * p.G)) * sh;
}

// The tile of rows r0 .. r0 + 63 as offsets from its first query's address: row
// i's bytes from there (without key head j's own offset)
struct RowTile {
    int64_t n0;  // first query
    int rem;     // r0 - n0 G
};
__device__ __forceinline__ RowTile row_tile(const CrossArgs& p, int64_t r0) {
    if (p.G == 1) return {r0, 0};
    const uint32_t n = (uint32_t)r0 / (uint32_t)p.G;
    return {(int64_t)n, (int)(r0 - n * p.G)};
}
__device__ __forceinline__ uint32_t row_tile_at(const CrossArgs& p, const RowTile& t, int i, int64_t sn, int64_t sh, int size) {
    if (p.G == 1) return (uint32_t)(i * (int)sn) * size;
    const int x = i + t.rem, n = (int)((x + 0.5f) * p.inv_g);  // x below 2^20: exact
    return (uint32_t)(n * (int)sn + (x - n * p.G) * (int)sh) * size;
}

}  // namespace svtad
