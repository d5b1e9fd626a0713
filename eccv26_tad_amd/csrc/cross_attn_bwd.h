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
// score matrix in memory. p and ds are rounded to T as operands of the second
// products; all sums are float32.
#pragma once

#include "cross_attn_fwd.h"

namespace svtad {

template <typename T, int DP, int WM, int R, bool VEC>
__global__ __launch_bounds__(256) void k_cross_bwd_q(CrossArgs p) {
    constexpr int W = DP < 32 ? 32 : DP, KS = W / 32, DB = DP / 16;
    constexpr int WK = 4 / WM, TK = kTileKeys<WM>, KW = TK / WK, NB = KW / 16, ROWS = WM * R * 16;
    typedef LdsTile<T, W> Tile;
    typedef KeyTiles<T, TK, W, VEC> Keys;
    constexpr size_t kJoin = WK > 1 ? (size_t)WK * ROWS * DP * 4 : 0;
    __shared__ __attribute__((aligned(16))) unsigned char mem[Keys::kBytes > kJoin ? Keys::kBytes : kJoin];
    __shared__ __attribute__((aligned(16))) uint8_t seen_mem[Keys::kBuffers * TK];

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, wm = wave % WM, wk = wave / WM;
    const int g = lane >> 4, li = lane & 15;
    const uint32_t row_tiles = ((uint32_t)p.M + ROWS - 1) / ROWS;
    const HeadTile ht = head_tile(blockIdx.x, gridDim.x, row_tiles * p.splits);
    const int bh = ht.bh, b = bh / p.KH, j = bh - b * p.KH, split = (int)(ht.tile / row_tiles);
    const int64_t r0 = (int64_t)(ht.tile - split * row_tiles) * ROWS;
    Frag8<T> qf[R][KS], df[R][KS];
    float lse[R], delta[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int64_t r = r0 + (wm * R + i) * 16 + li;
        const bool in = r < p.M;
        const T* const q = (const T*)p.q + b * p.qb + (in ? row_at(p, r, p.qn, p.qh, j) : 0);
        const T* const o = (const T*)p.o + b * p.ob + (in ? row_at(p, r, p.on, p.oh, j) : 0);
        const T* const d = (const T*)p.dout + b * p.gb + (in ? row_at(p, r, p.gn, p.gh, j) : 0);
        float s = 0.f;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            const int c = ks * 32 + g * 8;
            qf[i][ks] = load_frag<T, VEC>(q, c, in ? p.D : 0);
            df[i][ks] = load_frag<T, VEC>(d, c, in ? p.D : 0);
            const Pack<T, 8> x = __builtin_bit_cast(Pack<T, 8>, df[i][ks]);
            const Pack<T, 8> y = __builtin_bit_cast(Pack<T, 8>, load_frag<T, VEC>(o, c, in ? p.D : 0));
#pragma unroll
            for (int e = 0; e < 8; ++e) s = fmaf((float)x.e[e], (float)y.e[e], s);
        }
        delta[i] = across_groups_sum(s);
        lse[i] = in ? p.lse[bh * p.M + r] : -kNegInf;
        if (in && g == 0 && wk == 0 && split == 0) p.delta[bh * p.M + r] = -delta[i];
    }
    if (!p.out) return;

    f32x4 acc[DB][R];
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int db = 0; db < DB; ++db) acc[db][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    Keys keys(p, b, j, split, mem, seen_mem);
    auto use = [&](int64_t tile, auto part) __attribute__((always_inline)) {
        const unsigned char *const lk = keys.keys(tile), *const lv = keys.values(tile);
        const int left = keys.left(tile) - wk * KW - 4 * g;
#pragma unroll
        for (int kg = 0; kg < NB / 2; ++kg) {
            f32x4 ds[2][R];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = wk * KW + kg * 32 + h * 16;
                f32x4 s[R], dp[R];
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    s[i] = f32x4{0.f, 0.f, 0.f, 0.f};
                    dp[i] = f32x4{-delta[i], -delta[i], -delta[i], -delta[i]};  // the product's own sum: dp - delta
                }
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const Frag8<T> a = Tile::frag(lk, row, ks, lane);
                    const Frag8<T> v = Tile::frag(lv, row, ks, lane);
#pragma unroll
                    for (int i = 0; i < R; ++i) {
                        s[i] = mma<T>(a, qf[i][ks], s[i]);
                        dp[i] = mma<T>(v, df[i][ks], dp[i]);
                    }
                }
                if constexpr (part.value) {  // an unseen key was staged as zeros: its score is 0, not -inf
                    const uint32_t w = keys.mask ? *(const uint32_t*)(keys.seen(tile) + row + 4 * g) : 0x01010101u;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const bool in = kg * 32 + h * 16 + e < left && ((w >> (8 * e)) & 0xff);
#pragma unroll
                        for (int i = 0; i < R; ++i) s[i][e] = in ? s[i][e] : kNegInf;
                    }
                }
#pragma unroll
                for (int i = 0; i < R; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) ds[h][i][e] = __builtin_amdgcn_exp2f(fmaf(s[i][e], p.c, -lse[i])) * dp[i][e];
            }
            Frag8<T> sf[R];
#pragma unroll
            for (int i = 0; i < R; ++i) sf[i] = pack_frag<T>(ds[0][i], ds[1][i]);
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                const Frag8<T> a = Tile::frag_t(lk, wk * KW + kg * 32, db, lane);
#pragma unroll
                for (int i = 0; i < R; ++i) acc[db][i] = mma<T>(a, sf[i], acc[db][i]);
            }
        }
    };
    keys.walk(p, [&](int64_t t) { use(t, std::false_type()); }, [&](int64_t t) { use(t, std::true_type()); });

    if constexpr (WK > 1) {  // add the waves of equal rows, in order
        float* const jo = (float*)mem;  // [WK][ROWS][DP]
        __syncthreads();
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int db = 0; db < DB; ++db)
                *(f32x4*)(jo + (wk * ROWS + (wm * R + i) * 16 + li) * DP + db * 16 + 4 * g) = acc[db][i];
        __syncthreads();
        if (wk != 0) return;
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int w = 1; w < WK; ++w)
#pragma unroll
                for (int db = 0; db < DB; ++db)
                    acc[db][i] += *(const f32x4*)(jo + (w * ROWS + (wm * R + i) * 16 + li) * DP + db * 16 + 4 * g);
    }
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int64_t r = r0 + (wm * R + i) * 16 + li;
        if (r >= p.M) continue;
        if (p.splits > 1) {
            const int dp = (p.D + 3) & ~3;
            float* const po = p.part + (((int64_t)split * p.B * p.KH + bh) * p.M + r) * dp;
#pragma unroll
            for (int db = 0; db < DB; ++db)
                if (db * 16 + 4 * g < p.D) *(f32x4*)(po + db * 16 + 4 * g) = acc[db][i];
            continue;
        }
        T* const o = (T*)p.out + (int64_t)b * p.Nq * p.H * p.D + row_at(p, r, (int64_t)p.H * p.D, p.D, j);
#pragma unroll
        for (int db = 0; db < DB; ++db) store4<T>(o, db * 16 + 4 * g, p.D, acc[db][i] * p.scale);
    }
}

// 128 keys (R 2) or 64 (R 1) of one key head per workgroup, 16 R per wave;
// rows in tiles of kTileRows.
constexpr int kTileRows = 64;

template <typename T, int DP, int R, bool VEC>
__global__ __launch_bounds__(256) void k_cross_bwd_kv(CrossArgs p) {
    constexpr int W = DP < 32 ? 32 : DP, KS = W / 32, DB = DP / 16, TQ = kTileRows, KEYS = 64 * R;
    typedef LdsTile<T, W> Tile;
    typedef Stage<T, TQ, W, VEC> S;
    // two tiles of rows: one is read while the next arrives
    __shared__ __attribute__((aligned(16))) unsigned char mem[2][2][S::kBytes];  // [buffer][q, dout]
    __shared__ __attribute__((aligned(16))) float ll[2][TQ], lde[2][TQ];

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, g = lane >> 4, li = lane & 15;
    const uint32_t key_tiles = (uint32_t)cdiv(p.Nk, KEYS);
    const HeadTile ht = head_tile(blockIdx.x, gridDim.x, key_tiles * p.splits);
    const int bh = ht.bh, b = bh / p.KH, j = bh - b * p.KH, split = (int)(ht.tile / key_tiles);
    const int64_t n0 = (int64_t)(ht.tile - split * key_tiles) * KEYS;
    const int64_t len = seen_length(p, b);
    const uint32_t tiles = ((uint32_t)p.M + TQ - 1) / TQ, per = (tiles + p.splits - 1) / p.splits;
    const int64_t t0 = split * per, t1 = n0 < len ? lesser(tiles, split * per + per) : t0;

    const uint8_t* const mbase = p.mask ? p.mask + b * p.mask_b : nullptr;
    Frag8<T> kf[R][KS], vf[R][KS];
    bool seen[R];
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int64_t n = n0 + (wave * R + i) * 16 + li;
        seen[i] = n < len && (!mbase || mbase[n * p.mask_n]);
        const T* const k = (const T*)p.k + b * p.kb + j * p.kh + (seen[i] ? n * p.kn : 0);
        const T* const v = (const T*)p.v + b * p.vb + j * p.vh + (seen[i] ? n * p.vn : 0);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            kf[i][ks] = load_frag<T, VEC>(k, ks * 32 + g * 8, seen[i] ? p.D : 0);
            vf[i][ks] = load_frag<T, VEC>(v, ks * 32 + g * 8, seen[i] ? p.D : 0);
        }
    }

    const T* const qbase = (const T*)p.q + b * p.qb + (int64_t)j * p.G * p.qh;
    const T* const dbase = (const T*)p.dout + b * p.gb + (int64_t)j * p.G * p.gh;
    S sq, sd;
    auto fetch = [&](int64_t tile) {
        const RowTile rt = row_tile(p, tile * TQ);
        const int n = (int)lesser<int64_t>(p.M - tile * TQ, TQ);
        const Buffer rq = open_buffer(qbase + rt.n0 * p.qn), rd = open_buffer(dbase + rt.n0 * p.gn);
#pragma unroll
        for (int i = 0; i < S::kCount; ++i) {
            const int r = S::row(i);
            sq.load(i, rq, r < n ? row_tile_at(p, rt, r, p.qn, p.qh, sizeof(T)) : kOOB, p.D, mem[tile & 1][0]);
            sd.load(i, rd, r < n ? row_tile_at(p, rt, r, p.gn, p.gh, sizeof(T)) : kOOB, p.D, mem[tile & 1][1]);
        }
        // Past the end zeros, as for the rows themselves: a probability of 1
        // then meets a gradient of 0.
        if (wave < 2) {
            const uint32_t at = lane < n ? lane * 4 : kOOB;
            if (wave == 0) load_word_to_lds(open_buffer(p.lse + bh * p.M + tile * TQ).q, at, ll[tile & 1]);
            else load_word_to_lds(open_buffer(p.delta + bh * p.M + tile * TQ).q, at, lde[tile & 1]);
        }
    };
    auto arrive = [&](int64_t tile) {
        sq.store(mem[tile & 1][0]);
        sd.store(mem[tile & 1][1]);
        landed();
    };
    f32x4 dk[DB][R], dv[DB][R];
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
        for (int db = 0; db < DB; ++db) dk[db][i] = dv[db][i] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto use = [&](int64_t tile) __attribute__((always_inline)) {
        __syncthreads();
        if (tile + 1 < t1) fetch(tile + 1);
        const unsigned char *const lq = mem[tile & 1][0], *const ld = mem[tile & 1][1];
        const float *const l_tile = ll[tile & 1], *const d_tile = lde[tile & 1];
#pragma unroll
        for (int rg = 0; rg < TQ / 32; ++rg) {
            f32x4 pr[2][R], ds[2][R];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                const int row = rg * 32 + h * 16;
                f32x4 s[R], dp[R];
                const f32x4 l4 = *(const f32x4*)(l_tile + row + 4 * g), d4 = *(const f32x4*)(d_tile + row + 4 * g);
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    s[i] = f32x4{0.f, 0.f, 0.f, 0.f};
                    dp[i] = d4;  // -delta: the product's own sum is dp - delta
                }
#pragma unroll
                for (int ks = 0; ks < KS; ++ks) {
                    const Frag8<T> a = Tile::frag(lq, row, ks, lane);
                    const Frag8<T> d = Tile::frag(ld, row, ks, lane);
#pragma unroll
                    for (int i = 0; i < R; ++i) {
                        s[i] = mma<T>(a, kf[i][ks], s[i]);
                        dp[i] = mma<T>(d, vf[i][ks], dp[i]);
                    }
                }
                // A lane's scores are all of one key: those of a key that is
                // not seen stay in its own columns, which are stored as zeros.
#pragma unroll
                for (int i = 0; i < R; ++i)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        pr[h][i][e] = __builtin_amdgcn_exp2f(fmaf(s[i][e], p.c, -l4[e]));
                        ds[h][i][e] = pr[h][i][e] * dp[i][e];
                    }
            }
            Frag8<T> pf[R], sf[R];
#pragma unroll
            for (int i = 0; i < R; ++i) {
                pf[i] = pack_frag<T>(pr[0][i], pr[1][i]);
                sf[i] = pack_frag<T>(ds[0][i], ds[1][i]);
            }
#pragma unroll
            for (int db = 0; db < DB; ++db) {
                const Frag8<T> d = Tile::frag_t(ld, rg * 32, db, lane);
                const Frag8<T> a = Tile::frag_t(lq, rg * 32, db, lane);
#pragma unroll
                for (int i = 0; i < R; ++i) {
                    dv[db][i] = mma<T>(d, pf[i], dv[db][i]);
                    dk[db][i] = mma<T>(a, sf[i], dk[db][i]);
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
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int i = 0; i < R; ++i) {
        const int64_t n = n0 + (wave * R + i) * 16 + li;
        if (n >= p.Nk) continue;
        if (p.splits > 1) {
            const int dp = (p.D + 3) & ~3;
            const int64_t all = (int64_t)p.B * p.KH * p.Nk * dp;
            float* const po = p.part + 2 * split * all + (bh * p.Nk + n) * dp;
#pragma unroll
            for (int db = 0; db < DB; ++db)
                if (db * 16 + 4 * g < p.D) {
                    *(f32x4*)(po + db * 16 + 4 * g) = seen[i] ? dk[db][i] : zero;
                    *(f32x4*)(po + all + db * 16 + 4 * g) = seen[i] ? dv[db][i] : zero;
                }
            continue;
        }
        const int64_t at = (((int64_t)b * p.Nk + n) * p.KH + j) * p.D;
#pragma unroll
        for (int db = 0; db < DB; ++db) {
            store4<T>((T*)p.dk + at, db * 16 + 4 * g, p.D, seen[i] ? dk[db][i] * p.scale : zero);
            store4<T>((T*)p.dv + at, db * 16 + 4 * g, p.D, seen[i] ? dv[db][i] : zero);
        }
    }
}

// The splits of dq added in order, one thread per 4 values
template <typename T>
__global__ __launch_bounds__(256) void k_cross_sum_q(CrossArgs p) {
    const int dp = (p.D + 3) & ~3, nd = dp / 4;
    const int64_t rows = (int64_t)p.B * p.KH * p.M, e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (e >= rows * nd) return;
    const int64_t at = e / nd;
    const int c = (int)(e - at * nd) * 4;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < p.splits; ++s) acc += *(const f32x4*)(p.part + (s * rows + at) * dp + c);
    const int64_t bh = at / p.M, r = at - bh * p.M, b = bh / p.KH;
    const int j = (int)(bh - b * p.KH);
    store4<T>((T*)p.out + b * p.Nq * p.H * p.D + row_at(p, r, (int64_t)p.H * p.D, p.D, j), c, p.D, acc * p.scale);
}

// The splits of dk and dv
template <typename T>
__global__ __launch_bounds__(256) void k_cross_sum_kv(CrossArgs p) {
    const int dp = (p.D + 3) & ~3, nd = dp / 4;
    const int64_t rows = (int64_t)p.B * p.KH * p.Nk, all = rows * dp;
    int64_t e = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (e >= 2 * rows * nd) return;
    const bool is_v = e >= rows * nd;
    if (is_v) e -= rows * nd;
    const int64_t at = e / nd;
    const int c = (int)(e - at * nd) * 4;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int s = 0; s < p.splits; ++s) acc += *(const f32x4*)(p.part + (2 * s + is_v) * all + at * dp + c);
    const int64_t bh = at / p.Nk, n = at - bh * p.Nk, b = bh / p.KH;
    const int j = (int)(bh - b * p.KH);
    T* const to = (T*)(is_v ? p.dv : p.dk) + ((b * p.Nk + n) * p.KH + j) * p.D;
    store4<T>(to, c, p.D, is_v ? acc : acc * p.scale);
}

template <typename T, int WM, int R>
static void launch_cross_bwd_q(const CrossArgs& p, hipStream_t st) {
    const unsigned grid = (unsigned)(cdiv(p.M, WM * R * 16) * p.B * p.KH * p.splits);
    if (!p.vec) {
        if (p.D <= 32) k_cross_bwd_q<T, 32, WM, R, false><<<grid, 256, 0, st>>>(p);
        else k_cross_bwd_q<T, 128, WM, R, false><<<grid, 256, 0, st>>>(p);
    } else if (p.D <= 16) k_cross_bwd_q<T, 16, WM, R, true><<<grid, 256, 0, st>>>(p);
    else if (p.D <= 32) k_cross_bwd_q<T, 32, WM, R, true><<<grid, 256, 0, st>>>(p);
    else if (p.D <= 64) k_cross_bwd_q<T, 64, WM, R, true><<<grid, 256, 0, st>>>(p);
    else k_cross_bwd_q<T, 128, WM, R, true><<<grid, 256, 0, st>>>(p);
}

template <typename T>
void cross_bwd_q(const CrossArgs& p, int wave_rows, hipStream_t st) {
    if (wave_rows == 4) launch_cross_bwd_q<T, 4, 2>(p, st);
    else if (wave_rows == 2) launch_cross_bwd_q<T, 2, 2>(p, st);
    else launch_cross_bwd_q<T, 1, 1>(p, st);
    if (p.splits > 1 && p.out) {
        const int64_t n = (int64_t)p.B * p.KH * p.M * ((p.D + 3) / 4);
        k_cross_sum_q<T><<<(unsigned)cdiv(n, 256), 256, 0, st>>>(p);
    }
}

template <typename T>
void cross_bwd_kv(const CrossArgs& p, hipStream_t st) {
    const unsigned grid = (unsigned)(cdiv(p.Nk, cross_kv_keys(p.D)) * p.B * p.KH * p.splits);
    if (!p.vec) {
        if (p.D <= 32) k_cross_bwd_kv<T, 32, 2, false><<<grid, 256, 0, st>>>(p);
        else if (p.D <= 64) k_cross_bwd_kv<T, 64, 2, false><<<grid, 256, 0, st>>>(p);
        else k_cross_bwd_kv<T, 128, 1, false><<<grid, 256, 0, st>>>(p);
    } else if (p.D <= 16) k_cross_bwd_kv<T, 16, 2, true><<<grid, 256, 0, st>>>(p);
    else if (p.D <= 32) k_cross_bwd_kv<T, 32, 2, true><<<grid, 256, 0, st>>>(p);
    else if (p.D <= 64) k_cross_bwd_kv<T, 64, 2, true><<<grid, 256, 0, st>>>(p);
    else k_cross_bwd_kv<T, 128, 1, true><<<grid, 256, 0, st>>>(p);
    if (p.splits > 1) {
        const int64_t n = 2 * (int64_t)p.B * p.KH * p.Nk * ((p.D + 3) / 4);
        k_cross_sum_kv<T><<<(unsigned)cdiv(n, 256), 256, 0, st>>>(p);
    }
}

}  // namespace svtad
