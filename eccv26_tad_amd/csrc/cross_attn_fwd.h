// Cross attention, forward: kernels and launch.
//
//   s = scale q . k,  p = softmax of s over the seen keys,  out = sum p v
//
// One pass over the keys with each row's running maximum and sum (float32).
// A workgroup of 4 waves owns WM R 16 rows of one key head (R row tiles of 16
// per wave) and walks over key tiles staged in LDS, the next tile's loads in
// flight in registers meanwhile; with WM < 4 the waves of equal rows share a
// tile's keys and are joined at the end. Rows are queries times the G query
// heads of the key head, so shared key heads are read once for all of them.
// With few rows the keys are split over workgroups, whose partial sums
// k_cross_join adds in a fixed order.
//
// Probabilities are rounded to T for the product with v (the matrix units'
// operand type); their sum, the maximum and the output's sums stay float32.
// Keys that are not seen are staged as zeros and their scores replaced, so
// neither infinities nor NaN in their places reach a result.
#pragma once

#include <type_traits>

#include "cross_attn.h"

namespace svtad {

constexpr float kNegInf = -__builtin_huge_valf();

// The sums keep the scale of an earlier maximum until a score is 2^kSlack above
// it: after the first tiles of a row they are hardly rescaled again (32 products
// per tile and lane otherwise), and the powers stay below 2^kSlack.
constexpr float kSlack = 8.f;

// Keys of a staged tile: 64, or 32 per wave where the waves share a tile.
template <int WM> constexpr int kTileKeys = WM == 1 ? 128 : 64;

// The keys of one sample and key head as a workgroup walks over them: tiles of
// TK keys and values in LDS, two of them where they fit (one is read while the
// next arrives), and which keys are seen.
template <typename T, int TK, int W, bool VEC>
struct KeyTiles {
    typedef Stage<T, TK, W, VEC> S;
    static constexpr int kTile = 2 * S::kBytes, kBuffers = 2 * kTile <= 128 * 1024 ? 2 : 1;
    static constexpr size_t kBytes = (size_t)kBuffers * kTile;
    S sk, sv;
    const T *k, *v;
    const uint8_t* mask;
    int64_t len, t0, t1;
    unsigned char* mem;     // [kBuffers][K, V]
    uint8_t* seen_mem;      // [kBuffers][TK]
    uint8_t next[S::kCount];  // the mask at the next tile's rows
    uint8_t own, own_next;    // and at row threadIdx.x

    __device__ __forceinline__ KeyTiles(const CrossArgs& p, int b, int j, int split, unsigned char* mem, uint8_t* seen_mem)
        : k((const T*)p.k + b * p.kb + j * p.kh), v((const T*)p.v + b * p.vb + j * p.vh),
          mask(p.mask ? p.mask + b * p.mask_b : nullptr), len(seen_length(p, b)), mem(mem), seen_mem(seen_mem) {
        const uint32_t tiles = (uint32_t)cdiv(len, TK), per = (tiles + p.splits - 1) / p.splits;
        t0 = split * per, t1 = lesser(tiles, split * per + per);
    }

    __device__ __forceinline__ int left(int64_t tile) const { return (int)lesser<int64_t>(len - tile * TK, TK); }
    __device__ __forceinline__ unsigned char* keys(int64_t tile) const { return mem + (kBuffers == 2 ? (int)(tile & 1) * kTile : 0); }
    __device__ __forceinline__ unsigned char* values(int64_t tile) const { return keys(tile) + S::kBytes; }
    __device__ __forceinline__ uint8_t* seen(int64_t tile) const { return seen_mem + (kBuffers == 2 ? (int)(tile & 1) * TK : 0); }

    // The mask is read a tile ahead of the rows whose loads depend on it.
    __device__ __forceinline__ void fetch_mask(const CrossArgs& p, int64_t tile) {
        if (!mask || tile >= t1) return;
        const int n = left(tile);
        const uint8_t* const m = mask + tile * TK * p.mask_n;
#pragma unroll
        for (int i = 0; i < S::kCount; ++i) next[i] = S::row(i) < n ? m[S::row(i) * p.mask_n] : 0;
        own = (int)threadIdx.x < n ? m[threadIdx.x * p.mask_n] : 0;  // n is at most TK
    }
    template <bool MASK>  // false: there is no mask
    __device__ __forceinline__ void fetch(const CrossArgs& p, int64_t tile) {
        const int n = left(tile);
        const Buffer rk = open_buffer(k + tile * TK * p.kn), rv = open_buffer(v + tile * TK * p.vn);
#pragma unroll
        for (int i = 0; i < S::kCount; ++i) {
            const int r = S::row(i);
            const bool in = r < n && (!MASK || !mask || next[i]);
            sk.load(i, rk, in ? (uint32_t)(r * (int)p.kn) * (int)sizeof(T) : kOOB, p.D, keys(tile));
            sv.load(i, rv, in ? (uint32_t)(r * (int)p.vn) * (int)sizeof(T) : kOOB, p.D, values(tile));
        }
        if constexpr (MASK) {
            own_next = own;
            fetch_mask(p, tile + 1);
        }
    }
    template <bool MASK>
    __device__ __forceinline__ void arrive(int64_t tile) {
        if (MASK && mask && threadIdx.x < TK) seen(tile)[threadIdx.x] = own_next;
        sk.store(keys(tile));
        sv.store(values(tile));
        landed();
    }

    // All tiles of this split: whole(tile) on those whose keys are all seen,
    // part(tile) on the others (the last one, or with a mask any), in loops of
    // their own, so that neither carries the other's cases.
    template <typename F, typename G>
    __device__ __forceinline__ void walk(const CrossArgs& p, F whole, G part) {
        if (t0 >= t1) return;
        const int64_t tw = mask ? t0 : max<int64_t>(t0, lesser(t1, len / TK));
        fetch_mask(p, t0);
        if constexpr (kBuffers == 2) {
            fetch<true>(p, t0);
            arrive<true>(t0);
        }
        for (int64_t tile = t0; tile < tw; ++tile) step<false>(p, tile, whole);
        for (int64_t tile = tw; tile < t1; ++tile) step<true>(p, tile, part);
    }
    template <bool MASK, typename F>
    __device__ __forceinline__ void step(const CrossArgs& p, int64_t tile, F use) {
        __syncthreads();  // this tile has arrived, and nobody reads the other any more
        if constexpr (kBuffers == 2) {
            if (tile + 1 < t1) fetch<MASK>(p, tile + 1);
            use(tile);
            if (tile + 1 < t1) arrive<MASK>(tile + 1);
        } else {
            fetch<MASK>(p, tile);
            arrive<MASK>(tile);
            __syncthreads();
            use(tile);
        }
    }
};

template <typename T, int DP, int WM, int R, bool VEC>
__global__ __launch_bounds__(256) void k_cross_fwd(CrossArgs p) {
    constexpr int W = DP < 32 ? 32 : DP, KS = W / 32, DB = DP / 16;
    constexpr int WK = 4 / WM, TK = kTileKeys<WM>, KW = TK / WK, NB = KW / 16, ROWS = WM * R * 16;
    static_assert(KW % 32 == 0, "a wave's keys fill whole products");
    typedef LdsTile<T, W> Tile;
    typedef KeyTiles<T, TK, W, VEC> Keys;
    constexpr size_t kJoin = WK > 1 ? (size_t)WK * ROWS * (DP + 2) * 4 : 0;
    __shared__ __attribute__((aligned(16))) unsigned char mem[Keys::kBytes > kJoin ? Keys::kBytes : kJoin];
    __shared__ __attribute__((aligned(16))) uint8_t seen_mem[Keys::kBuffers * TK];

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave % WM, wk = wave / WM;
    const int g = lane >> 4, li = lane & 15;
    const uint32_t row_tiles = ((uint32_t)p.M + ROWS - 1) / ROWS;
    const HeadTile ht = head_tile(blockIdx.x, gridDim.x, row_tiles * p.splits);
    const int bh = ht.bh, b = bh / p.KH, j = bh - b * p.KH, split = (int)(ht.tile / row_tiles);
    const int64_t r0 = (int64_t)(ht.tile - split * row_tiles) * ROWS;
    Keys keys(p, b, j, split, mem, seen_mem);

    Frag8<T> qf[R][KS];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int64_t r = r0 + (wm * R + i) * 16 + li;
        const T* const q = (const T*)p.q + b * p.qb + (r < p.M ? row_at(p, r, p.qn, p.qh, j) : 0);
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[i][s] = load_frag<T, VEC>(q, s * 32 + g * 8, r < p.M ? p.D : 0);
    }

    f32x4 acc[DB][R];
    float m[R], l[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        m[i] = kNegInf, l[i] = 0.f;
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[db][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    auto use = [&](int64_t tile, auto part) __attribute__((always_inline)) {
        const unsigned char *const lk = keys.keys(tile), *const lv = keys.values(tile);
        f32x4 s[NB][R];
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
#pragma unroll
            for (int i = 0; i < R; ++i) s[nb][i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                const Frag8<T> a = Tile::frag(lk, wk * KW + nb * 16, ks, lane);
#pragma unroll
                for (int i = 0; i < R; ++i) s[nb][i] = mma<T>(a, qf[i][ks], s[nb][i]);
            }
        }
        if constexpr (part.value) {
            const int left = keys.left(tile) - wk * KW - 4 * g;
#pragma unroll
            for (int nb = 0; nb < NB; ++nb) {
                const uint32_t w = keys.mask ? *(const uint32_t*)(keys.seen(tile) + wk * KW + nb * 16 + 4 * g) : 0x01010101u;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const bool in = nb * 16 + e < left && ((w >> (8 * e)) & 0xff);
#pragma unroll
                    for (int i = 0; i < R; ++i) s[nb][i][e] = in ? s[nb][i][e] : kNegInf;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            float mx = s[0][i][0];
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int e = 0; e < 4; ++e) mx = fmaxf(mx, s[nb][i][e]);
            mx = across_groups_max(mx);
            if (__any((mx - m[i]) * p.c > kSlack)) {
                const float top = fmaxf(mx, m[i]), f = top == kNegInf ? 1.f : __builtin_amdgcn_exp2f((m[i] - top) * p.c);
                m[i] = top;
                l[i] *= f;
#pragma unroll
                for (int db = 0; db < DB; ++db) acc[db][i] *= f;
            }
            const float mc = m[i] == kNegInf ? 0.f : m[i] * p.c;  // no key seen so far: every power is 0
#pragma unroll
            for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[nb][i][e] = __builtin_amdgcn_exp2f(fmaf(s[nb][i][e], p.c, -mc));
                    l[i] += s[nb][i][e];
                }
        }
#pragma unroll
        for (int kg = 0; kg < NB / 2; ++kg) {
            Frag8<T> pf[R];
#pragma unroll
            for (int i = 0; i < R; ++i) pf[i] = pack_frag<T>(s[2 * kg][i], s[2 * kg + 1][i]);
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                const Frag8<T> a = Tile::frag_t(lv, wk * KW + kg * 32, db, lane);
#pragma unroll
                for (int i = 0; i < R; ++i) acc[db][i] = mma<T>(a, pf[i], acc[db][i]);
            }
        }
    };
    keys.walk(p, [&](int64_t t) { use(t, std::false_type()); }, [&](int64_t t) { use(t, std::true_type()); });
#pragma unroll
    for (int i = 0; i < R; ++i) l[i] = across_groups_sum(l[i]);

    if constexpr (WK > 1) {  // join the waves of equal rows, in order
        float* const jo = (float*)mem;               // [WK][ROWS][DP]
        float* const jm = jo + WK * ROWS * DP;       // [WK][ROWS][2]
        __syncthreads();
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int r = (wm * R + i) * 16 + li;
            if (g == 0) {
                jm[(wk * ROWS + r) * 2] = m[i];
                jm[(wk * ROWS + r) * 2 + 1] = l[i];
            }
#pragma unroll
            for (int db = 0; db < DB; ++db) *(f32x4*)(jo + (wk * ROWS + r) * DP + db * 16 + 4 * g) = acc[db][i];
        }
        __syncthreads();
        if (wk != 0) return;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const int r = (wm * R + i) * 16 + li;
            float top = m[i];
#pragma unroll
            for (int w = 1; w < WK; ++w) top = fmaxf(top, jm[(w * ROWS + r) * 2]);
            if (top == kNegInf) continue;
            float f = __builtin_amdgcn_exp2f((m[i] - top) * p.c);
            l[i] *= f;
#pragma unroll
            for (int db = 0; db < DB; ++db) acc[db][i] *= f;
#pragma unroll
            for (int w = 1; w < WK; ++w) {
                f = __builtin_amdgcn_exp2f((jm[(w * ROWS + r) * 2] - top) * p.c);
                l[i] += f * jm[(w * ROWS + r) * 2 + 1];
#pragma unroll
                for (int db = 0; db < DB; ++db) acc[db][i] += *(const f32x4*)(jo + (w * ROWS + r) * DP + db * 16 + 4 * g) * f;
            }
            m[i] = top;
        }
    }

#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int64_t r = r0 + (wm * R + i) * 16 + li;
        if (r >= p.M) continue;
        if (p.splits > 1) {
            const int64_t at = ((int64_t)split * p.B * p.KH + bh) * p.M + r;
            const int dp = (p.D + 3) & ~3;
            float* const po = p.part + at * dp;
            float* const pm = p.part + (int64_t)p.splits * p.B * p.KH * p.M * dp + at * 2;
#pragma unroll
            for (int db = 0; db < DB; ++db)
                if (db * 16 + 4 * g < p.D) *(f32x4*)(po + db * 16 + 4 * g) = acc[db][i];
            if (g == 0) {
                pm[0] = m[i];
                pm[1] = l[i];
            }
            continue;
        }
        T* const o = (T*)p.out + (int64_t)b * p.Nq * p.H * p.D + row_at(p, r, (int64_t)p.H * p.D, p.D, j);
        const float inv = l[i] == 0.f ? 0.f : 1.f / l[i];
#pragma unroll
        for (int db = 0; db < DB; ++db) store4<T>(o, db * 16 + 4 * g, p.D, acc[db][i] * inv);
        if (p.lse && g == 0)
            p.lse[bh * p.M + r] = l[i] == 0.f ? -kNegInf : m[i] * p.c + __builtin_amdgcn_logf(l[i]);
    }
}

// The splits of a row joined in order: one thread per 4 output values.
template <typename T>
__global__ __launch_bounds__(256) void k_cross_join(CrossArgs p) {
    const int dp = (p.D + 3) & ~3, nd = dp / 4;
    const int64_t rows = (int64_t)p.B * p.KH * p.M, e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (e >= rows * nd) return;
    const int64_t at = e / nd;
    const int c = (int)(e - at * nd) * 4;
    const float* const pm = p.part + (int64_t)p.splits * rows * dp;
    float top = kNegInf;
    for (int s = 0; s < p.splits; ++s) top = fmaxf(top, pm[(s * rows + at) * 2]);
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    float l = 0.f;
    if (top != kNegInf)
        for (int s = 0; s < p.splits; ++s) {
            const float f = __builtin_amdgcn_exp2f((pm[(s * rows + at) * 2] - top) * p.c);
            l += f * pm[(s * rows + at) * 2 + 1];
            acc += *(const f32x4*)(p.part + (s * rows + at) * dp + c) * f;
        }
    const int64_t bh = at / p.M, r = at - bh * p.M, b = bh / p.KH;
    const int j = (int)(bh - b * p.KH);
    T* const o = (T*)p.out + b * p.Nq * p.H * p.D + row_at(p, r, (int64_t)p.H * p.D, p.D, j);
    store4<T>(o, c, p.D, acc * (l == 0.f ? 0.f : 1.f / l));
    if (p.lse && c == 0) p.lse[at] = l == 0.f ? -kNegInf : top * p.c + __builtin_amdgcn_logf(l);
}

template <typename T, int WM, int R>
static void launch_cross_fwd(const CrossArgs& p, hipStream_t st) {
    const unsigned grid = (unsigned)(cdiv(p.M, WM * R * 16) * p.B * p.KH * p.splits);
    if (!p.vec) {
        if (p.D <= 32) k_cross_fwd<T, 32, WM, R, false><<<grid, 256, 0, st>>>(p);
        else k_cross_fwd<T, 128, WM, R, false><<<grid, 256, 0, st>>>(p);
    } else if (p.D <= 16) k_cross_fwd<T, 16, WM, R, true><<<grid, 256, 0, st>>>(p);
    else if (p.D <= 32) k_cross_fwd<T, 32, WM, R, true><<<grid, 256, 0, st>>>(p);
    else if (p.D <= 64) k_cross_fwd<T, 64, WM, R, true><<<grid, 256, 0, st>>>(p);
    else k_cross_fwd<T, 128, WM, R, true><<<grid, 256, 0, st>>>(p);
}

template <typename T>
void cross_fwd(const CrossArgs& p, int wave_rows, hipStream_t st) {
    if (wave_rows == 4) launch_cross_fwd<T, 4, 2>(p, st);
    else if (wave_rows == 2) launch_cross_fwd<T, 2, 2>(p, st);
    else launch_cross_fwd<T, 1, 1>(p, st);
    if (p.splits > 1) {
        const int64_t n = (int64_t)p.B * p.KH * p.M * ((p.D + 3) / 4);
        k_cross_join<T><<<(unsigned)cdiv(n, 256), 256, 0, st>>>(p);
    }
}

}  // namespace svtad
