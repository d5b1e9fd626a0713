// Cross attention, backward: kernels and launch.
//
//   p = 2^(c s - lse),  dp = dout . v,  delta = sum over d of dout out
//   ds = p (dp - delta),  dq = scale sum over keys ds k
//   dk = scale sum over rows ds q,  dv = sum over rows p dout
//
// Two kernels, each the owner of what it writes, so that no sum needs an
// atomic and every run gives the same bits: one over row tiles that walks the
// keys (dq, and delta on the way), one over key tiles that walks the rows (dk
// and dv; the rows of a key head are those of all its query heads). Both
// recompute the scores, which costs two of the seven products and saves the
// score matrix in memory; bound like the forward (its case of many rows: dq 650 to
// 745 us, dk and dv 780 to 953, 0.93 to 0.81 and 1.03 to 0.85 PFLOP/s). p and ds are rounded to T as operands of the second
// products; all sums are float32. delta takes the output together with what its
// rounding took: among few keys that moves every ds of a row alike (bfloat16, 64
// wide, against a result that is rounded once: dq off by 1.50 times as much instead
// of 2.21 at 2 keys, 1.49 instead of 1.63 at 8, 1.47 instead of 1.51 at 39; 1.43 at
// all of them with the forward's second product). A probability among n keys is
// near 1 / n, which float16 holds with few bits (below 2^-14 fewer with every
// halving): for dv they are scaled up by a power of two, at most n, and the sum
// down again. A score gradient is as small times what dout and v are, or past
// float16's largest value where those are large: GradScale.
#pragma once

#include "cross_attn_fwd.h"

namespace svtad {

// Score gradients in float16: those of a row (in the dq kernel) or of a key (in the
// other), a column of the tile, are scaled by a power of two, which their sums in
// float32 give back at the end. It starts above any that could matter and falls to
// where the largest so far is near 2^kSet whenever one passes 2^kTop: so a sum's
// addends have all of float16's bits down to 2^-20 of its largest, whatever the
// size of dout (70 queries over 20000 keys of 32 channels, dq is off by 0.03 % with a
// dout of 1 or 1e-2 and 0.15 % with 1e-3, of which all but a little is the result's own
// rounding; rounded as they are 0.03, 0.35 and 3.4 %). It costs the two kernels 8 % at
// 2 x 16 heads of 64, 4917 queries and 12289 keys (dq 872 us, 805 without; dk and dv
// 1117, 1030) and nothing to 7 % at smaller sizes.
struct GradScale {
    static constexpr int kStart = 60, kTop = 15, kSet = 7;
    int e = kStart;

    // Over a tile's N scaled gradients; what the lane's own and its sums are to be
    // multiplied by where any lane's `change` says so.
    template <typename M, int N>
    static __device__ __forceinline__ float top(const typename M::Acc (&g)[N]) {
        float v = 0.f;
#pragma unroll
        for (int h = 0; h < N; ++h)
#pragma unroll
            for (int i = 0; i < 4 * M::Q; ++i) v = fmaxf(v, fabsf(g[h][i]));
        return v;
    }
    static __device__ __forceinline__ bool passed(float top) { return __any(top > (float)(1 << kTop)); }
    template <typename M>
    __device__ __forceinline__ float lower(float top) {
        top = M::col_max(top);
        const int d = top > (float)(1 << kTop) && top < __builtin_huge_valf() ? kSet - __builtin_amdgcn_frexp_expf(top) : 0;
        e += d;
        return __builtin_ldexpf(1.f, d);
    }
    __device__ __forceinline__ float undo() const { return __builtin_ldexpf(1.f, -e); }
};

template <typename T, int DP, int WM, int S, bool VEC>
__global__ __launch_bounds__(256, (kResidentBwd<T, DP>)) void k_cross_bwd_q(CrossArgs p) {
    typedef Shape<T, S> M;
    typedef typename M::Acc Acc;
    constexpr int W = DP < 32 ? 32 : DP, KS = W / M::K, DB = DP < S ? 1 : DP / S;
    constexpr int WK = 4 / WM, TK = kTileKeys<WM>, KW = TK / WK, ROWS = WM * S, NP = M::K > S ? M::K / S : 1;
    typedef KeyTiles<T, TK, W, VEC> Keys;
    constexpr size_t kJoin = WK > 1 ? (size_t)WK * ROWS * DB * S * 4 : 0;
    __shared__ __attribute__((aligned(16))) unsigned char mem[Keys::kBytes > kJoin ? Keys::kBytes : kJoin];
    __shared__ __attribute__((aligned(16))) float start_mem[Keys::kBuffers * TK];

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave % WM, wk = wave / WM;
    const int li = M::col(lane), slot = M::slot(lane);
    const uint32_t row_tiles = ((uint32_t)p.M + ROWS - 1) / ROWS;
    const HeadTile ht = head_tile(blockIdx.x, gridDim.x, row_tiles * p.splits);
    const int j = ht.bh % p.KH, b = sample_of_rank(p, ht.bh / p.KH), bh = b * p.KH + j, split = (int)(ht.tile / row_tiles);
    const int64_t r = (int64_t)(ht.tile - split * row_tiles) * ROWS + wm * S + li;  // this lane's row
    const bool in = r < p.M;

    Frag8<T> qf[KS], df[KS];
    float delta = 0.f;
    {
        const T* const q = (const T*)p.q + b * p.qb + (in ? row_at(p, r, p.qn, p.qh, j) : 0);
        const int64_t at = b * p.ob + (in ? row_at(p, r, p.on, p.oh, j) : 0);
        const T* const d = (const T*)p.dout + b * p.gb + (in ? row_at(p, r, p.gn, p.gh, j) : 0);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int c = ks * M::K + slot * 8;
            qf[ks] = load_frag<T, VEC>(q, c, in ? p.D : 0);
            df[ks] = load_frag<T, VEC>(d, c, in ? p.D : 0);
            const Pack<T, 8> x = __builtin_bit_cast(Pack<T, 8>, df[ks]);
            const Pack<T, 8> y = __builtin_bit_cast(Pack<T, 8>, load_frag<T, VEC>((const T*)p.o + at, c, in ? p.D : 0));
#pragma unroll
            for (int e = 0; e < 8; ++e) delta = fmaf((float)x.e[e], (float)y.e[e], delta);
            if (p.rest) {
                const Pack<T, 8> z = __builtin_bit_cast(Pack<T, 8>, load_frag<T, VEC>((const T*)p.rest + at, c, in ? p.D : 0));
#pragma unroll
                for (int e = 0; e < 8; ++e) delta = fmaf((float)x.e[e], (float)z.e[e], delta);
            }
        }
        delta = M::col_sum(delta);
    }
    constexpr bool kScaled = std::is_same_v<T, f16>;
    GradScale gs;
    // +inf: the row sees no key, and has no gradient whatever dout and q hold
    float lse = in ? p.lse[bh * p.M + r] : -kNegInf;  // past the end: probabilities 0
    const bool none = lse == -kNegInf;
    if constexpr (kScaled) lse -= gs.e;  // probabilities, and with them the score gradients, times 2^e
    if (in && slot == 0 && wk == 0 && split == 0) p.delta[bh * p.M + r] = -delta;
    if (!p.out) return;

    Acc acc[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) acc[db] = M::fill(0.f);
    Keys keys(p, b, j, split, mem, start_mem);
    auto use = [&](int64_t tile, auto part) __attribute__((always_inline)) {
        const unsigned char *const lk = keys.keys(tile), *const lv = keys.values(tile);
#pragma unroll
        for (int n0 = 0; n0 < KW; n0 += NP * S) {  // NP score tiles make whole products
            Acc ds[NP];
#pragma unroll
            for (int h = 0; h < NP; ++h) {
                const int row = wk * KW + n0 + h * S;
                Acc s, dp = M::fill(-delta);  // the product's own sum: dp - delta
                if constexpr (part.value) s = start_scores<M>(keys.start(tile) + row, lane);
                else s = M::fill(0.f);
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
                    if (M::step_in(ks, p.D)) s = M::mma(M::template frag<W>(lk, row, ks, lane), qf[ks], s);
#pragma unroll
                for (int ks = 0; ks < KS; ++ks)
                    if (M::step_in(ks, p.D)) dp = M::mma(M::template frag<W>(lv, row, ks, lane), df[ks], dp);
#pragma unroll
                for (int e = 0; e < 4 * M::Q; ++e) ds[h][e] = __builtin_amdgcn_exp2f(fmaf(s[e], p.c, -lse)) * dp[e];
            }
            if constexpr (kScaled) {
                const float top = GradScale::top<M>(ds);
                if (GradScale::passed(top)) {
                    const int was = gs.e;
                    const float f = gs.lower<M>(top);
                    lse -= gs.e - was;
#pragma unroll
                    for (int h = 0; h < NP; ++h) ds[h] *= f;
#pragma unroll
                    for (int db = 0; db < DB; ++db) acc[db] *= f;
                }
            }
#pragma unroll
            for (int kk = 0; kk < NP * S / M::K; ++kk) {
                const Frag8<T> sf = M::pack(ds, kk);
#pragma unroll
                for (int db = 0; db < DB; ++db)
                    acc[db] = M::mma(M::template frag_t<W>(lk, wk * KW + n0 + kk * M::K, db, lane), sf, acc[db]);
            }
        }
    };
    keys.walk(p, [&](int64_t t) { use(t, std::false_type()); }, [&](int64_t t) { use(t, std::true_type()); });
    if constexpr (kScaled) {
        const float f = gs.undo();
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[db] *= f;
    }
    if (none) {
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[db] = M::fill(0.f);
    }

    if constexpr (WK > 1) {  // add the waves of equal rows, in order
        constexpr int DA = DB * S;
        float* const jo = (float*)mem;  // [WK][ROWS][DA]
        const int at = wm * S + li;
        __syncthreads();
#pragma unroll
        for (int db = 0; db < DB; ++db)
#pragma unroll
            for (int q = 0; q < M::Q; ++q)
                *(f32x4*)(jo + (wk * ROWS + at) * DA + db * S + M::row4(q, lane)) = M::quad(acc[db], q);
        __syncthreads();
        if (wk != 0) return;
#pragma unroll
        for (int w = 1; w < WK; ++w)
#pragma unroll
            for (int db = 0; db < DB; ++db)
#pragma unroll
                for (int q = 0; q < M::Q; ++q) {
                    const f32x4 v = *(const f32x4*)(jo + (w * ROWS + at) * DA + db * S + M::row4(q, lane));
#pragma unroll
                    for (int e = 0; e < 4; ++e) acc[db][4 * q + e] += v[e];
                }
    }
    if (!in) return;
    const int dp = (p.D + 3) & ~3;
    float* const po = p.part + (((int64_t)split * p.B * p.KH + bh) * p.M + r) * dp;
    T* const o = (T*)p.out + (int64_t)b * p.Nq * p.H * p.D + row_at(p, r, (int64_t)p.H * p.D, p.D, j);
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int q = 0; q < M::Q; ++q) {
            const int c = db * S + M::row4(q, lane);
            if (p.splits == 1) store4<T>(o, c, p.D, M::quad(acc[db], q) * p.scale);
            else if (c < p.D) *(f32x4*)(po + c) = M::quad(acc[db], q);
        }
}

// 128 keys of one key head per workgroup, 32 per wave; rows in tiles of
// kTileRows, two of them in LDS: one is read while the next arrives.
constexpr int kTileRows = 64;

template <typename T, int DP, bool VEC>
__global__ __launch_bounds__(256, (kResidentBwd<T, DP>)) void k_cross_bwd_kv(CrossArgs p) {
    constexpr int S = 32;
    typedef Shape<T, S> M;
    typedef typename M::Acc Acc;
    constexpr int W = DP, KS = W / M::K, DB = DP / S, TQ = kTileRows, KEYS = 4 * S;
    typedef Stage<T, TQ, W, VEC> St;
    __shared__ __attribute__((aligned(16))) unsigned char mem[2][2][St::kBytes];  // [buffer][q, dout]
    __shared__ __attribute__((aligned(16))) float ll[2][TQ], lde[2][TQ];

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = M::col(lane), slot = M::slot(lane);
    const uint32_t key_tiles = (uint32_t)cdiv(p.Nk, KEYS);
    const HeadTile ht = head_tile(blockIdx.x, gridDim.x, key_tiles * p.splits);
    const int bh = ht.bh, b = bh / p.KH, j = bh - b * p.KH, split = (int)(ht.tile / key_tiles);
    const int64_t n0 = (int64_t)(ht.tile - split * key_tiles) * KEYS, n = n0 + wave * S + li;  // this lane's key
    const int64_t len = seen_length(p, b);
    const uint32_t tiles = ((uint32_t)p.M + TQ - 1) / TQ, per = (tiles + p.splits - 1) / p.splits;
    const int64_t t0 = split * per, t1 = n0 < len ? lesser(tiles, split * per + per) : t0;
    const bool seen = n < len && (!p.mask || p.mask[b * p.mask_b + n * p.mask_n]);

    Frag8<T> kf[KS], vf[KS];
    {
        const T* const k = (const T*)p.k + b * p.kb + j * p.kh + (seen ? n * p.kn : 0);
        const T* const v = (const T*)p.v + b * p.vb + j * p.vh + (seen ? n * p.vn : 0);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            kf[ks] = load_frag<T, VEC>(k, ks * M::K + slot * 8, seen ? p.D : 0);
            vf[ks] = load_frag<T, VEC>(v, ks * M::K + slot * 8, seen ? p.D : 0);
        }
    }

    const T* const qbase = (const T*)p.q + b * p.qb + (int64_t)j * p.G * p.qh;
    const T* const dbase = (const T*)p.dout + b * p.gb + (int64_t)j * p.G * p.gh;
    St sq, sd;
    // A tile's rows are whole queries where G divides it: their offsets from the
    // tile's first are then the same for every tile.
    const bool whole = TQ % p.G == 0;
    uint32_t at_q[St::kCount], at_d[St::kCount];
    auto offsets = [&](const RowTile& rt) {
#pragma unroll
        for (int i = 0; i < St::kCount; ++i) {
            at_q[i] = row_tile_at(p, rt, St::row(i), p.qn, p.qh, sizeof(T));
            at_d[i] = row_tile_at(p, rt, St::row(i), p.gn, p.gh, sizeof(T));
        }
    };
    offsets({0, 0});
    auto fetch = [&](int64_t tile) {
        const RowTile rt = row_tile(p, tile * TQ);
        if (!whole) offsets(rt);
        const int rows = (int)lesser<int64_t>(p.M - tile * TQ, TQ);
        const Buffer rq = open_buffer(qbase + rt.n0 * p.qn), rd = open_buffer(dbase + rt.n0 * p.gn);
#pragma unroll
        for (int i = 0; i < St::kCount; ++i) {
            const bool in = St::row(i) < rows;
            sq.load(i, rq, in ? at_q[i] : kOOB, p.D, mem[tile & 1][0]);
            sd.load(i, rd, in ? at_d[i] : kOOB, p.D, mem[tile & 1][1]);
        }
        // Past the end zeros, as for the rows themselves: a probability of 1
        // then meets a gradient of 0.
        if (wave < 2) {
            const uint32_t at = lane < rows ? lane * 4 : kOOB;
            if (wave == 0) load_word_to_lds(open_buffer(p.lse + bh * p.M + tile * TQ).q, at, ll[tile & 1]);
            else load_word_to_lds(open_buffer(p.delta + bh * p.M + tile * TQ).q, at, lde[tile & 1]);
        }
    };
    auto arrive = [&](int64_t tile) {
        sq.store(mem[tile & 1][0]);
        sd.store(mem[tile & 1][1]);
        landed();
    };
    Acc dk[DB], dv[DB];
#pragma unroll
    for (int db = 0; db < DB; ++db) dk[db] = dv[db] = M::fill(0.f);
    constexpr bool kScaled = std::is_same_v<T, f16>;
    GradScale gs;
    float w = seen ? __builtin_ldexpf(1.f, gs.e) : 0.f;  // 2^e; unseen: nothing that lowers it
    auto use = [&](int64_t tile) __attribute__((always_inline)) {
        __syncthreads();
        if (tile + 1 < t1) fetch(tile + 1);
        const unsigned char *const lq = mem[tile & 1][0], *const ld = mem[tile & 1][1];
        const float *const l_tile = ll[tile & 1], *const d_tile = lde[tile & 1];
#pragma unroll
        for (int row = 0; row < TQ; row += S) {
            // A lane's scores are all of one key: those of a key that is not
            // seen stay in its own columns, which are stored as zeros.
            Acc s = M::fill(0.f), ds[1], &dp = ds[0];
#pragma unroll
            for (int q = 0; q < M::Q; ++q) {
                const f32x4 d4 = *(const f32x4*)(d_tile + row + M::row4(q, lane));
#pragma unroll
                for (int e = 0; e < 4; ++e) dp[4 * q + e] = d4[e];  // -delta: the product's own sum is dp - delta
            }
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                if (M::step_in(ks, p.D)) s = M::mma(M::template frag<W>(lq, row, ks, lane), kf[ks], s);
#pragma unroll
            for (int ks = 0; ks < KS; ++ks)
                if (M::step_in(ks, p.D)) dp = M::mma(M::template frag<W>(ld, row, ks, lane), vf[ks], dp);
#pragma unroll
            for (int q = 0; q < M::Q; ++q) {
                const f32x4 l4 = *(const f32x4*)(l_tile + row + M::row4(q, lane));
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[4 * q + e] = __builtin_amdgcn_exp2f(fmaf(s[4 * q + e], p.c, -l4[e]));
                    dp[4 * q + e] *= kScaled ? s[4 * q + e] * w : s[4 * q + e];
                    if constexpr (kScaled) s[4 * q + e] *= p.up;
                }
            }
            if constexpr (kScaled) {
                const float top = GradScale::top<M>(ds);
                if (GradScale::passed(top)) {
                    const float f = gs.lower<M>(top);
                    w *= f;
                    dp *= f;
#pragma unroll
                    for (int db = 0; db < DB; ++db) dk[db] *= f;
                }
            }
#pragma unroll
            for (int kk = 0; kk < S / M::K; ++kk) {
                const Frag8<T> pf = M::pack(&s, kk), sf = M::pack(&dp, kk);
#pragma unroll
                for (int db = 0; db < DB; ++db) {
                    dv[db] = M::mma(M::template frag_t<W>(ld, row + kk * M::K, db, lane), pf, dv[db]);
                    dk[db] = M::mma(M::template frag_t<W>(lq, row + kk * M::K, db, lane), sf, dk[db]);
                }
            }
        }
        if (tile + 1 < t1) arrive(tile + 1);
    };
    if (t0 < t1) {
        fetch(t0);
        arrive(t0);
        for (int64_t tile = t0; tile < t1; ++tile) use(tile);
    }
    if (n >= p.Nk) return;
    const float undo = kScaled ? gs.undo() : 1.f;
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    const int dp4 = (p.D + 3) & ~3;
    const int64_t all = (int64_t)p.B * p.KH * p.Nk * dp4, at = (((int64_t)b * p.Nk + n) * p.KH + j) * p.D;
    float* const po = p.part + 2 * split * all + (bh * p.Nk + n) * dp4;
#pragma unroll
    for (int db = 0; db < DB; ++db)
#pragma unroll
        for (int q = 0; q < M::Q; ++q) {
            const int c = db * S + M::row4(q, lane);
            const f32x4 gk = seen ? M::quad(dk[db], q) * undo : zero, gv = seen ? M::quad(dv[db], q) * p.down : zero;
            if (p.splits == 1) {
                store4<T>((T*)p.dk + at, c, p.D, gk * p.scale);
                store4<T>((T*)p.dv + at, c, p.D, gv);
            } else if (c < p.D) {
                *(f32x4*)(po + c) = gk;
                *(f32x4*)(po + all + c) = gv;
            }
        }
}

// The splits of dq added in order
template <typename T, int G>
__global__ __launch_bounds__(256) void k_cross_sum_q(CrossArgs p) {
    const JoinChunk<G> j;
    const uint32_t nd = (p.D + 3) / 4, rows = (uint32_t)(p.B * p.KH * p.M);
    const bool in = j.e < rows * nd;
    const f32x4 acc = join_groups<G>(split_sum<G>(p.part + (in ? (int64_t)j.e * 4 : 0), (int64_t)rows * nd * 4, p.splits, j.g), j);
    if (j.g != 0 || !in) return;
    const uint32_t at = j.e / nd, bh = at / (uint32_t)p.M, r = at - bh * (uint32_t)p.M, b = bh / p.KH, head = bh - b * p.KH;
    store4<T>((T*)p.out + b * p.Nq * p.H * p.D + row_at(p, r, (int64_t)p.H * p.D, p.D, head), (int)(j.e - at * nd) * 4, p.D,
              acc * p.scale);
}

// The splits of dk and dv
template <typename T, int G>
__global__ __launch_bounds__(256) void k_cross_sum_kv(CrossArgs p) {
    const JoinChunk<G> j;
    const uint32_t nd = (p.D + 3) / 4, rows = (uint32_t)(p.B * p.KH * p.Nk), all = rows * nd;
    const bool in = j.e < 2 * all, is_v = in && j.e >= all;
    const f32x4 acc = join_groups<G>(split_sum<G>(p.part + (in ? (int64_t)j.e * 4 : 0), 2 * (int64_t)all * 4, p.splits, j.g), j);
    if (j.g != 0 || !in) return;
    const uint32_t e = is_v ? j.e - all : j.e, at = e / nd, bh = at / (uint32_t)p.Nk, n = at - bh * (uint32_t)p.Nk;
    const uint32_t b = bh / p.KH, head = bh - b * p.KH;
    T* const to = (T*)(is_v ? p.dv : p.dk) + ((b * p.Nk + n) * p.KH + head) * p.D;
    store4<T>(to, (int)(e - at * nd) * 4, p.D, is_v ? acc : acc * p.scale);
}

template <typename T, int WM, int S>
static void launch_cross_bwd_q(const CrossArgs& p, hipStream_t st) {
    const unsigned grid = (unsigned)(cdiv(p.M, WM * S) * p.B * p.KH * p.splits);
    if (!p.vec) {
        if (p.D <= 32) k_cross_bwd_q<T, 32, WM, S, false><<<grid, 256, 0, st>>>(p);
        else k_cross_bwd_q<T, 128, WM, S, false><<<grid, 256, 0, st>>>(p);
    } else if (p.D <= 32) k_cross_bwd_q<T, 32, WM, S, true><<<grid, 256, 0, st>>>(p);
    else if (p.D <= 64) k_cross_bwd_q<T, 64, WM, S, true><<<grid, 256, 0, st>>>(p);
    else k_cross_bwd_q<T, 128, WM, S, true><<<grid, 256, 0, st>>>(p);
}

template <typename T>
void cross_bwd_q(const CrossArgs& p, int wave_rows, hipStream_t st) {
    if (wave_rows == 4) launch_cross_bwd_q<T, 4, 32>(p, st);
    else if (wave_rows == 2) launch_cross_bwd_q<T, 2, 32>(p, st);
    else launch_cross_bwd_q<T, 1, 16>(p, st);
    if (p.splits > 1 && p.out) {
        const int64_t n = (int64_t)p.B * p.KH * p.M * ((p.D + 3) / 4);
        if (p.splits <= kOneGroup) k_cross_sum_q<T, 1><<<(unsigned)cdiv(n, 256), 256, 0, st>>>(p);
        else k_cross_sum_q<T, kJoinGroups><<<(unsigned)cdiv(n, 256 / kJoinGroups), 256, 0, st>>>(p);
    }
}

template <typename T>
void cross_bwd_kv(const CrossArgs& p, hipStream_t st) {
    const unsigned grid = (unsigned)(cdiv(p.Nk, kCrossKvKeys) * p.B * p.KH * p.splits);
    if (!p.vec) {
        if (p.D <= 32) k_cross_bwd_kv<T, 32, false><<<grid, 256, 0, st>>>(p);
        else k_cross_bwd_kv<T, 128, false><<<grid, 256, 0, st>>>(p);
    } else if (p.D <= 32) k_cross_bwd_kv<T, 32, true><<<grid, 256, 0, st>>>(p);
    else if (p.D <= 64) k_cross_bwd_kv<T, 64, true><<<grid, 256, 0, st>>>(p);
    else k_cross_bwd_kv<T, 128, true><<<grid, 256, 0, st>>>(p);
    if (p.splits > 1) {
        const int64_t n = 2 * (int64_t)p.B * p.KH * p.Nk * ((p.D + 3) / 4);
        if (p.splits <= kOneGroup) k_cross_sum_kv<T, 1><<<(unsigned)cdiv(n, 256), 256, 0, st>>>(p);
        else k_cross_sum_kv<T, kJoinGroups><<<(unsigned)cdiv(n, 256 / kJoinGroups), 256, 0, st>>>(p);
    }
}

}  // namespace svtad
