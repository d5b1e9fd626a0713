// Cross attention, forward: kernels and launch.
//
//   s = scale q . k,  p = softmax of s over the seen keys,  out = sum p v
//
// One pass over the keys with each row's running scale and sum (float32). A
// workgroup of 4 waves owns WM S rows of one key head (S rows per wave) and walks
// over key tiles staged in LDS, the next tile's loads in flight meanwhile; with
// WM < 4 the waves of equal rows share a tile's keys and are joined at the end.
// Rows are queries times the G query heads of the key head, so shared key heads
// are read once for all of them. With few rows the keys are split over
// workgroups, whose partial sums k_cross_join adds in a fixed order.
//
// Probabilities are rounded to T for the product with v (the matrix units'
// operand type); their sum, the scale and the output's sums stay float32. Over the
// keys of a lone tile a second product adds what that rounding took: the backward's
// delta is made from the output, and with few keys its error would reach the
// gradients unaveraged. Past one tile it averages out: bfloat16 dq is off by 1.43 times
// as much as a result that is rounded once with the product at any number of keys,
// without it by 1.50 at 2 keys and 1.47 at 39.
// Bound by the issue of products and exponentials where there are many rows (16
// heads of 64, 2 x 4917 queries over 12289 keys of unequal length, bfloat16: 497 to
// 620 us, 0.81 to 0.65 PFLOP/s with the clock), by memory where there are few (one
// query over 8 x 31361 keys of 4 heads: 36 us, 4.8 TB/s).
// Keys that are not seen are staged as zeros and their scores replaced, so
// neither infinities nor NaN in their places reach a result. A sample's rows whose
// keys are all unseen are set to zero at the end: a product of zeros with a row's
// own infinities or NaN is no zero.
#pragma once

#include "cross_attn.h"

namespace svtad {

constexpr float kNegInf = -__builtin_huge_valf();

// A row's powers are taken relative to the largest score seen when its scale was
// last set. The scale is set again only when a score is 2^kSlack above it, which
// each lane sees from its own scores: after a row's first tiles neither the lane
// exchange of the maximum nor the rescaling of the sums runs (ViT-L training case:
// 541 us when a tile was computed twice instead, on sums that had grown too large,
// to save the maximum as well; 497 us so). Powers stay below 2^kSlack, which
// float32 sums and the operand types hold as well as those below 1.
constexpr float kSlack = 8.f;

// In float16 all powers are times 2^kLift besides, up to 2^15: a key whose weight is
// 2^-21 of the largest is a normal value still. Below those values the roundings of
// keys that are alike are large, alike too, and add up: where one token in 64 takes
// nearly all of the weight and the others 7e-7 of it each, what these add to the result
// is off by 4 % without the lift.
template <typename T> constexpr float kLift = std::is_same_v<T, f16> ? 7.f : 0.f;

// What sums relative to the maximum m are multiplied by to be relative to `top`, at
// least m. Parts with one maximum are added as they are, -inf included: no score of
// theirs was above it, but one may be NaN, and so may their sums.
__device__ __forceinline__ float power_of(float m, float top, float c) {
    return m == top ? 1.f : __builtin_amdgcn_exp2f((m - top) * c);
}

// Keys of a staged tile: 64, or 32 per wave where the waves share a tile.
template <int WM> constexpr int kTileKeys = WM == 1 ? 128 : 64;

// The keys of one sample and key head as a workgroup walks over them: tiles of
// TK keys and values in LDS, two of them where they fit (one is read while the
// next arrives). With a tile that has unseen keys comes what their scores start
// from, -inf (0 for the others): as the sum's initial value in the product that
// makes the scores it costs nothing, and unseen keys and values are zeros.
template <typename T, int TK, int W, bool VEC, bool ONCE = false>
struct KeyTiles {
    typedef Stage<T, TK, W, VEC, ONCE> S;
    static constexpr int kTile = 2 * S::kBytes, kBuffers = 2 * kTile <= 128 * 1024 ? 2 : 1;
    static constexpr size_t kBytes = (size_t)kBuffers * kTile;
    S sk, sv;
    const T *k, *v;
    const uint8_t* mask;
    int64_t len, t0, t1, tw;  // tiles t0 .. t1, of which those below tw are whole
    unsigned char* mem;       // [kBuffers][K, V]
    float* start_mem;         // [kBuffers][TK]
    uint8_t next[S::kCount];  // the mask at the next tile's rows
    uint8_t own, own_next;    // and at row threadIdx.x

    __device__ __forceinline__ KeyTiles(const CrossArgs& p, int b, int j, int split, unsigned char* mem, float* start_mem)
        : k((const T*)p.k + b * p.kb + j * p.kh), v((const T*)p.v + b * p.vb + j * p.vh),
          mask(p.mask ? p.mask + b * p.mask_b : nullptr), len(seen_length(p, b)), mem(mem), start_mem(start_mem) {
        const uint32_t tiles = (uint32_t)cdiv(len, TK), per = (tiles + p.splits - 1) / p.splits;
        t0 = split * per, t1 = lesser(tiles, split * per + per);
        // a tile alone goes the way of those with unseen keys
        tw = mask || tiles < 2 ? t0 : max<int64_t>(t0, lesser<int64_t>(t1, len / TK));
    }

    __device__ __forceinline__ int left(int64_t tile) const { return (int)lesser<int64_t>(len - tile * TK, TK); }
    __device__ __forceinline__ unsigned char* keys(int64_t tile) const { return mem + (kBuffers == 2 ? (int)(tile & 1) * kTile : 0); }
    __device__ __forceinline__ unsigned char* values(int64_t tile) const { return keys(tile) + S::kBytes; }
    __device__ __forceinline__ float* start(int64_t tile) const { return start_mem + (kBuffers == 2 ? (int)(tile & 1) * TK : 0); }

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
        if (tile >= tw && threadIdx.x < TK)
            start(tile)[threadIdx.x] = (int)threadIdx.x < left(tile) && (!MASK || !mask || own_next) ? 0.f : kNegInf;
        sk.store(keys(tile));
        sv.store(values(tile));
        landed();
    }

    // Whether the mask shows any key of this split (the same for the wave). It is read
    // again where that matters: a flag kept through the walk cost the kernel of many
    // rows 6 spilled registers.
    __device__ __forceinline__ bool any(const CrossArgs& p) const {
        const int64_t end = lesser<int64_t>(len, t1 * TK);
        bool in = false;
        for (int64_t n = t0 * TK + (threadIdx.x & 63); n < end; n += 64) in |= mask[n * p.mask_n] != 0;
        return __any(in);
    }

    // All tiles of this split: whole(tile) on those whose keys are all seen,
    // part(tile) on the others (the last one, or with a mask any), in loops of
    // their own, so that neither carries the other's cases.
    template <typename F, typename G>
    __device__ __forceinline__ void walk(const CrossArgs& p, F whole, G part) {
        if (t0 >= t1) return;
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

// What the scores of a tile of S keys from `at` on start from
template <typename M>
__device__ __forceinline__ typename M::Acc start_scores(const float* at, int lane) {
    typename M::Acc a;
#pragma unroll
    for (int q = 0; q < M::Q; ++q) {
        const f32x4 v = *(const f32x4*)(at + M::row4(q, lane));
#pragma unroll
        for (int e = 0; e < 4; ++e) a[4 * q + e] = v[e];
    }
    return a;
}

template <typename T, int DP, int WM, int S, bool VEC>
__global__ __launch_bounds__(256, (kResidentFwd<T, DP>)) void k_cross_fwd(CrossArgs p) {
    typedef Shape<T, S> M;
    typedef typename M::Acc Acc;
    constexpr int W = DP < 32 ? 32 : DP, KS = W / M::K, DB = DP < S ? 1 : DP / S;
    constexpr int WK = 4 / WM, TK = kTileKeys<WM>, KW = TK / WK, NB = KW / S, ROWS = WM * S;
    // Up to 16 rows (WM 1) are one row tile: each key is read by one workgroup (8 x
    // 31361 keys, one query each, a pass: 40.7 us past the caches, 44.0 through).
    typedef KeyTiles<T, TK, W, VEC, WM == 1> Keys;
    constexpr size_t kJoin = WK > 1 ? (size_t)WK * ROWS * (DB * S + 2) * 4 : 0;
    __shared__ __attribute__((aligned(16))) unsigned char mem[Keys::kBytes > kJoin ? Keys::kBytes : kJoin];
    __shared__ __attribute__((aligned(16))) float start_mem[Keys::kBuffers * TK];

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave % WM, wk = wave / WM;
    const int li = M::col(lane), slot = M::slot(lane);
    const uint32_t row_tiles = ((uint32_t)p.M + ROWS - 1) / ROWS;
    const HeadTile ht = head_tile(blockIdx.x, gridDim.x, row_tiles * p.splits);
    const int j = ht.bh % p.KH, b = sample_of_rank(p, ht.bh / p.KH), bh = b * p.KH + j, split = (int)(ht.tile / row_tiles);
    const int64_t r = (int64_t)(ht.tile - split * row_tiles) * ROWS + wm * S + li;  // this lane's row
    Keys keys(p, b, j, split, mem, start_mem);

    Frag8<T> qf[KS];
    {
        const T* const q = (const T*)p.q + b * p.qb + (r < p.M ? row_at(p, r, p.qn, p.qh, j) : 0);
#pragma unroll
        for (int s = 0; s < KS; ++s) qf[s] = load_frag<T, VEC>(q, s * M::K + slot * 8, r < p.M ? p.D : 0);
    }
    Acc acc[DB];
    float m = kNegInf, l = 0.f;
#pragma unroll
    for (int db = 0; db < DB; ++db) acc[db] = M::fill(0.f);
    auto values = [&](const unsigned char* lv, const Acc* s) __attribute__((always_inline)) {
#pragma unroll
        for (int kk = 0; kk < KW / M::K; ++kk) {
            const Frag8<T> pf = M::pack(s, kk);
#pragma unroll
            for (int db = 0; db < DB; ++db)
                acc[db] = M::mma(M::template frag_t<W>(lv, wk * KW + kk * M::K, db, lane), pf, acc[db]);
        }
    };
    auto use = [&](int64_t tile, auto part) __attribute__((always_inline)) {
        const unsigned char *const lk = keys.keys(tile), *const lv = keys.values(tile);
        Acc s[NB];
        float top = m;
#pragma unroll
        for (int nb = 0; nb < NB; ++nb) {
            if constexpr (part.value) s[nb] = start_scores<M>(keys.start(tile) + wk * KW + nb * S, lane);
            else s[nb] = M::fill(0.f);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                if (M::step_in(ks, p.D)) s[nb] = M::mma(M::template frag<W>(lk, wk * KW + nb * S, ks, lane), qf[ks], s[nb]);
        }
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < 4 * M::Q; ++e) top = fmaxf(top, s[nb][e]);
        if (__any((top - m) * p.c > kSlack)) {
            top = M::col_max(top);
            const float f = top == kNegInf ? 1.f : __builtin_amdgcn_exp2f((m - top) * p.c);
            m = top;
            l *= f;
#pragma unroll
            for (int db = 0; db < DB; ++db) acc[db] *= f;
        }
        const float mc = (m == kNegInf ? 0.f : m * p.c) - kLift<T>;  // no key seen so far: every power is 0
#pragma unroll
        for (int nb = 0; nb < NB; ++nb)
#pragma unroll
            for (int e = 0; e < 4 * M::Q; ++e) {
                s[nb][e] = __builtin_amdgcn_exp2f(fmaf(s[nb][e], p.c, -mc));
                l += s[nb][e];
            }
        values(lv, s);
        if constexpr (part.value && sizeof(T) == 2)
            if (keys.len <= TK) {
#pragma unroll
                for (int nb = 0; nb < NB; ++nb)
#pragma unroll
                    for (int e = 0; e < 4 * M::Q; ++e) s[nb][e] -= (float)(T)s[nb][e];
                values(lv, s);
            }
    };
    keys.walk(p, [&](int64_t t) { use(t, std::false_type()); }, [&](int64_t t) { use(t, std::true_type()); });
    l = M::col_sum(l);
    if (keys.mask && __any(l != l) && !keys.any(p)) {
        m = kNegInf, l = 0.f;
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[db] = M::fill(0.f);
    }

    if constexpr (WK > 1) {  // join the waves of equal rows, in order
        constexpr int DA = DB * S;
        float* const jo = (float*)mem;            // [WK][ROWS][DA]
        float* const jm = jo + WK * ROWS * DA;    // [WK][ROWS][2]
        const int at = wm * S + li;
        __syncthreads();
        if (slot == 0) {
            jm[(wk * ROWS + at) * 2] = m;
            jm[(wk * ROWS + at) * 2 + 1] = l;
        }
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int q = 0; q < M::Q; ++q)
                *(f32x4*)(jo + (wk * ROWS + at) * DA + db * S + M::row4(q, lane)) = M::quad(acc[db], q);
        __syncthreads();
        if (wk != 0) return;
        float top = m;
#pragma unroll
        for (int w = 1; w < WK; ++w) top = fmaxf(top, jm[(w * ROWS + at) * 2]);
        float f = power_of(m, top, p.c);
        l *= f;
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[db] *= f;
#pragma unroll
        for (int w = 1; w < WK; ++w) {
            f = power_of(jm[(w * ROWS + at) * 2], top, p.c);
            l += f * jm[(w * ROWS + at) * 2 + 1];
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int q = 0; q < M::Q; ++q) {
                    const f32x4 v = *(const f32x4*)(jo + (w * ROWS + at) * DA + db * S + M::row4(q, lane));
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[db][4 * q + e] += v[e] * f;
                }
        }
        m = top;
    }

    if (r >= p.M) return;
    if (p.splits > 1) {
        const int64_t at = ((int64_t)split * p.B * p.KH + bh) * p.M + r;
        const int dp = (p.D + 3) & ~3;
        float* const po = p.part + at * dp;
        float* const pm = p.part + (int64_t)p.splits * p.B * p.KH * p.M * dp + at * 2;
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int q = 0; q < M::Q; ++q) {
                const int c = db * S + M::row4(q, lane);
                if (c < p.D) *(f32x4*)(po + c) = M::quad(acc[db], q);
            }
        if (slot == 0) {
            pm[0] = m;
            pm[1] = l;
        }
        return;
    }
    const int64_t o = (int64_t)b * p.Nq * p.H * p.D + row_at(p, r, (int64_t)p.H * p.D, p.D, j);
    const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int q = 0; q < M::Q; ++q)
            store4_rest<T>((T*)p.out + o, p.rest ? (T*)p.rest + o : nullptr, db * S + M::row4(q, lane), p.D,
                           M::quad(acc[db], q) * inv);
    if (p.lse && slot == 0) p.lse[bh * p.M + r] = l == 0.f ? -kNegInf : m * p.c - kLift<T> + __builtin_amdgcn_logf(l);
}

// The splits of a row joined in order, a chunk of 4 output values per thread of
// each group
template <typename T, int G>
__global__ __launch_bounds__(256) void k_cross_join(CrossArgs p) {
    __shared__ float red[G][256 / G][2];
    const JoinChunk<G> j;
    const uint32_t nd = (p.D + 3) / 4, rows = (uint32_t)(p.B * p.KH * p.M), at = j.e < rows * nd ? j.e / nd : 0;
    const bool in = j.e < rows * nd;
    const int dp = nd * 4, c = in ? (int)(j.e - at * nd) * 4 : 0;
    const int per = (p.splits + G - 1) / G, s0 = lesser(p.splits, j.g * per), s1 = lesser(p.splits, s0 + per);
    const float* const pm = p.part + ((int64_t)p.splits * rows * dp + (int64_t)at * 2);
    const float* const po = p.part + ((int64_t)at * dp + c);
    constexpr int kMost = G == 1 ? kOneGroup : kMaxSplits / G;  // splits of a group
    float m[kMost], w[kMost], top = kNegInf, l = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f}, v[kMost];
#pragma unroll
    for (int i = 0; i < kMost; ++i)
        if (s0 + i < s1) {  // uniform
            m[i] = pm[(int64_t)(s0 + i) * rows * 2];
            w[i] = pm[(int64_t)(s0 + i) * rows * 2 + 1];
            v[i] = *(const f32x4*)(po + (int64_t)(s0 + i) * rows * dp);
        }
#pragma unroll
    for (int i = 0; i < kMost; ++i)
        if (s0 + i < s1) top = fmaxf(top, m[i]);
    if constexpr (G > 1) {
        red[j.g][j.chunk][0] = top;
        __syncthreads();
#pragma unroll
        for (int q = 0; q < G; ++q) top = fmaxf(top, red[q][j.chunk][0]);
    }
#pragma unroll
    for (int i = 0; i < kMost; ++i)
        if (s0 + i < s1) {
            const float f = power_of(m[i], top, p.c);
            l += f * w[i];
            acc += v[i] * f;
        }
    if constexpr (G > 1) red[j.g][j.chunk][1] = l;
    acc = join_groups<G>(acc, j);  // its barrier covers red
    if (j.g != 0 || !in) return;
#pragma unroll
    for (int q = 1; q < G; ++q) l += red[q][j.chunk][1];
    const uint32_t bh = at / (uint32_t)p.M, r = at - bh * (uint32_t)p.M, b = bh / p.KH, head = bh - b * p.KH;
    const int64_t o = b * p.Nq * p.H * p.D + row_at(p, r, (int64_t)p.H * p.D, p.D, head);
    store4_rest<T>((T*)p.out + o, p.rest ? (T*)p.rest + o : nullptr, c, p.D, acc * (l == 0.f ? 0.f : 1.f / l));
    if (p.lse && c == 0) p.lse[at] = l == 0.f ? -kNegInf : top * p.c - kLift<T> + __builtin_amdgcn_logf(l);
}

template <typename T, int WM, int S>
static void launch_cross_fwd(const CrossArgs& p, hipStream_t st) {
    const unsigned grid = (unsigned)(cdiv(p.M, WM * S) * p.B * p.KH * p.splits);
    if (!p.vec) {
        if (p.D <= 32) k_cross_fwd<T, 32, WM, S, false><<<grid, 256, 0, st>>>(p);
        else k_cross_fwd<T, 128, WM, S, false><<<grid, 256, 0, st>>>(p);
    } else if (p.D <= 32) k_cross_fwd<T, 32, WM, S, true><<<grid, 256, 0, st>>>(p);
    else if (p.D <= 64) k_cross_fwd<T, 64, WM, S, true><<<grid, 256, 0, st>>>(p);
    else k_cross_fwd<T, 128, WM, S, true><<<grid, 256, 0, st>>>(p);
}

template <typename T>
void cross_fwd(const CrossArgs& p, int wave_rows, hipStream_t st) {
    if (wave_rows == 4) launch_cross_fwd<T, 4, 32>(p, st);
    else if (wave_rows == 2) launch_cross_fwd<T, 2, 32>(p, st);
    else launch_cross_fwd<T, 1, 16>(p, st);
    if (p.splits > 1) {
        const int64_t n = (int64_t)p.B * p.KH * p.M * ((p.D + 3) / 4);
        if (p.splits <= kOneGroup) k_cross_join<T, 1><<<(unsigned)cdiv(n, 256), 256, 0, st>>>(p);
        else k_cross_join<T, kJoinGroups><<<(unsigned)cdiv(n, 256 / kJoinGroups), 256, 0, st>>>(p);
    }
}

}  // namespace svtad
