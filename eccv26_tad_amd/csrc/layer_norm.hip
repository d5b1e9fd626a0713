// Layer norm over the last axis, forward and backward, for rows of any width
// up to kMaxWidth in float16, bfloat16 or float32 (gfx950).
//
//   y  = (x - mean) rstd w + b,  rstd = 1 / sqrt(var + eps)
//   dx = rstd (g - mean(g) - xhat mean(g xhat)),  g = dy w,  xhat = (x - mean) rstd
//   dw = sum over rows of dy xhat,  db = sum over rows of dy
//
// A row stays in registers between its sums and its store, so memory sees it
// once; the kernels are bound by its bytes (49154 x 1024 in bfloat16: forward 33
// us, 6.0 TB/s, backward 56 us, 5.4 TB/s; a copy reaches 5.2 to 5.6). A group of G
// lanes holds a row, K vectors of 16 bytes per lane (lane g's vector j starts at
// (j G + g) V): G is the power of two up to 64 that covers the width with one
// vector, so that the short rows of per-head norms share a wave, and beyond a
// wave's 3 or 4 vectors per lane a whole workgroup takes a row. Sums and
// statistics are float32.
#include <algorithm>

#include "sv_internal.h"
#include "sv_vec.h"

namespace svtad {

constexpr int kMaxWidth = 8192;

struct LnArgs {
    const void* x;
    const void* dy;
    const void* w;      // NULL: 1
    const void* b;      // NULL: 0
    void* y;            // forward: y; backward: dx (NULL: not wanted)
    float* stats;       // [rows][2] mean, rstd; forward: NULL = not kept
    float* part;        // backward: [workgroups][2][c] sums of dy xhat and dy (NULL: not wanted)
    int64_t rows;
    int c, lanes;       // width; lanes of a row's group
    uint32_t n1, n2;    // the rows' axes [., n1, n2]; n1 = n2 = 1: one stride s0
    int64_t s0, s1, s2;     // x's strides in elements
    int64_t t0, t1, t2;     // dy's
    float eps;
    bool p32;           // w and b are float32
};

__device__ __forceinline__ int64_t row_offset(int64_t r, uint32_t n1, uint32_t n2, int64_t s0, int64_t s1, int64_t s2) {
    if (n1 == 1 && n2 == 1) return r * s0;
    const uint32_t q = (uint32_t)r / n2, i2 = (uint32_t)r - q * n2, i0 = q / n1, i1 = q - i0 * n1;
    return i0 * s0 + i1 * s1 + i2 * s2;
}

// Elements c0 .. c0 + V - 1 of a row as float32, 0 past its end (TAIL: the
// width is no multiple of V).
template <typename T, bool TAIL>
__device__ __forceinline__ void load_vec(float (&f)[kVec<T>], const T* row, int c0, int c) {
    constexpr int V = kVec<T>;
    if (c0 + V <= c) {
        const Pack<T, V> v = *(const Pack<T, V>*)(row + c0);
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = (float)v.e[e];
    } else {
#pragma unroll
        for (int e = 0; e < V; ++e) f[e] = TAIL && c0 + e < c ? (float)row[c0 + e] : 0.f;
    }
}

template <typename T, bool TAIL>
__device__ __forceinline__ void store_vec(T* row, const float (&f)[kVec<T>], int c0, int c) {
    constexpr int V = kVec<T>;
    if (c0 + V <= c) {
        Pack<T, V> v;
#pragma unroll
        for (int e = 0; e < V; ++e) v.e[e] = (T)f[e];
        *(Pack<T, V>*)(row + c0) = v;
    } else if (TAIL) {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (c0 + e < c) row[c0 + e] = (T)f[e];
    }
}

// V parameters as float32, `none` where there are none
template <typename T, bool TAIL>
__device__ __forceinline__ void load_params(float (&f)[kVec<T>], const void* p, bool p32, int c0, int c, float none) {
    constexpr int V = kVec<T>;
#pragma unroll
    for (int e = 0; e < V; ++e) f[e] = none;
    if (!p || c0 >= c) return;
    if (p32) {
#pragma unroll
        for (int e = 0; e < V; ++e)
            if (!TAIL || c0 + e < c) f[e] = ((const float*)p)[c0 + e];
    } else {
        load_vec<T, TAIL>(f, (const T*)p, c0, c);
    }
}

// Sums over a row's lanes; WG: the workgroup's 4 waves hold one row and meet in
// red. The next sum goes through another red, the one after through this again: by
// then all have passed that one's barrier.
template <bool WG>
__device__ __forceinline__ float row_sum(float v, int lanes, float* red) {
    v = group_sum(v, lanes);
    if constexpr (WG) {
        if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
        __syncthreads();
        v = (red[0] + red[1]) + (red[2] + red[3]);
    }
    return v;
}

template <typename T, int K, bool WG, bool TAIL>
__global__ __launch_bounds__(256) void k_layer_norm(LnArgs p) {
    constexpr int V = kVec<T>;
    __shared__ float red[2][4];
    const int G = WG ? 256 : p.lanes, g = threadIdx.x & (G - 1), per = 256 / G, c = p.c;
    float w[K][V], b[K][V];
#pragma unroll
    for (int j = 0; j < K; ++j) {
        load_params<T, TAIL>(w[j], p.w, p.p32, (j * G + g) * V, c, 1.f);
        load_params<T, TAIL>(b[j], p.b, p.p32, (j * G + g) * V, c, 0.f);
    }
    const float ic = 1.f / c;
    for (int64_t r0 = (int64_t)blockIdx.x * per; r0 < p.rows; r0 += (int64_t)gridDim.x * per) {
        const int64_t r = r0 + threadIdx.x / G;
        const bool in = r < p.rows;  // of one row for all lanes of a group
        const T* const x = (const T*)p.x + (in ? row_offset(r, p.n1, p.n2, p.s0, p.s1, p.s2) : 0);
        float f[K][V], s = 0.f;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            load_vec<T, TAIL>(f[j], x, in ? (j * G + g) * V : c, c);
#pragma unroll
            for (int e = 0; e < V; ++e) s += f[j][e];
        }
        const float mean = row_sum<WG>(s, min(G, 64), red[0]) * ic;
        s = 0.f;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const int c0 = (j * G + g) * V;
#pragma unroll
            for (int e = 0; e < V; ++e) {
                f[j][e] -= mean;
                if (TAIL ? c0 + e < c : c0 < c) s += f[j][e] * f[j][e];
            }
        }
        const float rstd = rsqrtf(row_sum<WG>(s, min(G, 64), red[1]) * ic + p.eps);
        if (!in) continue;
        T* const y = (T*)p.y + r * c;
#pragma unroll
        for (int j = 0; j < K; ++j) {
#pragma unroll
            for (int e = 0; e < V; ++e) f[j][e] = f[j][e] * rstd * w[j][e] + b[j][e];
            store_vec<T, TAIL>(y, f[j], (j * G + g) * V, c);
        }
        if (p.stats && g == 0) {
            p.stats[r * 2] = mean;
            p.stats[r * 2 + 1] = rstd;
        }
    }
}

// A row's vectors of x and dy as they lie in memory, and its statistics
template <typename T, int K, bool TAIL>
struct LnRow {
    static constexpr int V = kVec<T>;
    Pack<T, V> x[K], d[K];
    float mean, rstd;
    bool in;

    __device__ __forceinline__ void load(const LnArgs& p, int64_t r, int G, int g) {
        in = r < p.rows;
        const T* const x0 = (const T*)p.x + (in ? row_offset(r, p.n1, p.n2, p.s0, p.s1, p.s2) : 0);
        const T* const d0 = (const T*)p.dy + (in ? row_offset(r, p.n1, p.n2, p.t0, p.t1, p.t2) : 0);
        const int c = in ? p.c : 0;
        mean = in ? p.stats[r * 2] : 0.f, rstd = in ? p.stats[r * 2 + 1] : 0.f;
#pragma unroll
        for (int j = 0; j < K; ++j) {
            const int c0 = (j * G + g) * V;
            if (c0 + V <= c) {
                x[j] = *(const Pack<T, V>*)(x0 + c0);
                d[j] = *(const Pack<T, V>*)(d0 + c0);
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    x[j].e[e] = TAIL && c0 + e < c ? x0[c0 + e] : (T)0.f;
                    d[j].e[e] = TAIL && c0 + e < c ? d0[c0 + e] : (T)0.f;  // 0 past the row's end, as the sums need it
                }
            }
        }
    }
};

// dx, and the workgroup's partial sums of dy xhat and dy in p.part. The next
// row's loads are in flight while a row's sums are exchanged.
template <typename T, int K, bool WG, bool TAIL>
__global__ __launch_bounds__(256) void k_layer_norm_bwd(LnArgs p) {
    constexpr int V = kVec<T>, W = 64 * K * V;  // the widest row of a wave's group
    __shared__ float red[2][2][4];  // [row's parity]
    const int G = WG ? 256 : p.lanes, g = threadIdx.x & (G - 1), per = 256 / G, c = p.c;
    float w[K][V], sw[K][V], sb[K][V];
#pragma unroll
    for (int j = 0; j < K; ++j) {
        load_params<T, TAIL>(w[j], p.w, p.p32, (j * G + g) * V, c, 1.f);
#pragma unroll
        for (int e = 0; e < V; ++e) sw[j][e] = sb[j][e] = 0.f;
    }
    const float ic = 1.f / c;
    int odd = 0;
    const int64_t step = (int64_t)gridDim.x * per;
    LnRow<T, K, TAIL> next;
    next.load(p, (int64_t)blockIdx.x * per + threadIdx.x / G, G, g);
    for (int64_t r0 = (int64_t)blockIdx.x * per; r0 < p.rows; r0 += step) {
        const int64_t r = r0 + threadIdx.x / G;
        const LnRow<T, K, TAIL> row = next;
        if (r0 + step < p.rows) next.load(p, r + step, G, g);
        float xh[K][V], d[K][V], s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int j = 0; j < K; ++j) {
#pragma unroll
            for (int e = 0; e < V; ++e) {
                xh[j][e] = ((float)row.x[j].e[e] - row.mean) * row.rstd;
                const float t = (float)row.d[j].e[e];
                sw[j][e] += t * xh[j][e];
                sb[j][e] += t;
                d[j][e] = t * w[j][e];
                s1 += d[j][e];
                s2 += d[j][e] * xh[j][e];
            }
        }
        if (!p.y) continue;
        s1 = group_sum(s1, min(G, 64)), s2 = group_sum(s2, min(G, 64));
        if constexpr (WG) {  // both through one barrier
            if ((threadIdx.x & 63) == 0) red[odd][0][threadIdx.x >> 6] = s1, red[odd][1][threadIdx.x >> 6] = s2;
            __syncthreads();
            s1 = (red[odd][0][0] + red[odd][0][1]) + (red[odd][0][2] + red[odd][0][3]);
            s2 = (red[odd][1][0] + red[odd][1][1]) + (red[odd][1][2] + red[odd][1][3]);
            odd ^= 1;
        }
        s1 *= ic, s2 *= ic;
        if (!row.in) continue;
        T* const dx = (T*)p.y + r * c;
#pragma unroll
        for (int j = 0; j < K; ++j) {
#pragma unroll
            for (int e = 0; e < V; ++e) d[j][e] = row.rstd * (d[j][e] - s1 - xh[j][e] * s2);
            store_vec<T, TAIL>(dx, d[j], (j * G + g) * V, c);
        }
    }
    if (!p.part) return;
    float* const part = p.part + (int64_t)blockIdx.x * 2 * c;
    if constexpr (WG) {  // every channel has one thread
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                const int ch = (j * G + g) * V + e;
                if (ch < c) {
                    part[ch] = sw[j][e];
                    part[c + ch] = sb[j][e];
                }
            }
    } else {
        // the groups of a wave by lane exchange, then the waves in order
        __shared__ float sums[4][2][W];
#pragma unroll
        for (int j = 0; j < K; ++j)
#pragma unroll
            for (int e = 0; e < V; ++e) {
                for (int m = G; m < 64; m <<= 1) {
                    sw[j][e] += __shfl_xor(sw[j][e], m, 64);
                    sb[j][e] += __shfl_xor(sb[j][e], m, 64);
                }
                if ((threadIdx.x & 63) < G) {
                    sums[threadIdx.x >> 6][0][(j * G + g) * V + e] = sw[j][e];
                    sums[threadIdx.x >> 6][1][(j * G + g) * V + e] = sb[j][e];
                }
            }
        __syncthreads();
        for (int e = threadIdx.x; e < 2 * c; e += 256) {
            const int which = e >= c, ch = e - which * c;
            part[e] = (sums[0][which][ch] + sums[1][which][ch]) + (sums[2][which][ch] + sums[3][which][ch]);
        }
    }
}

// dw, db: the partial sums of all workgroups added in a fixed order (32 thread
// groups take consecutive shares of them, then the groups), one rounding. A
// workgroup owns 32 sums, 8 lanes of 4 each.
template <typename P>
__global__ __launch_bounds__(256) void k_layer_norm_sum(const float* __restrict__ part, int groups, int c,
                                                        P* __restrict__ dw, P* __restrict__ db) {
    __shared__ float red[32][33];
    const int lane = threadIdx.x & 7, g = threadIdx.x >> 3;
    const int e = blockIdx.x * 32 + lane * 4;
    const int per = (groups + 31) / 32, g0 = min(groups, g * per), n = min(groups, g0 + per) - g0;
    float s[4] = {0.f, 0.f, 0.f, 0.f};
    if (e + 4 <= 2 * c) {
        add_strided(s, part + (int64_t)g0 * 2 * c + e, 2 * c, n);
    } else {
        for (int q = g0; q < g0 + n; ++q)
            for (int k = 0; k < 4; ++k) s[k] += e + k < 2 * c ? part[(int64_t)q * 2 * c + e + k] : 0.f;
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) red[g][lane * 4 + k] = s[k];
    __syncthreads();
    const int o = blockIdx.x * 32 + threadIdx.x;
    if (threadIdx.x >= 32 || o >= 2 * c) return;
    float v = 0.f;
#pragma unroll
    for (int q = 0; q < 32; ++q) v += red[q][threadIdx.x];
    P* const to = o < c ? dw : db;
    if (to) to[o < c ? o : o - c] = (P)v;
}

// ---------------------------------------------------------------------------

// Lanes of a row's group and vectors per lane: the smallest power of two of
// lanes that takes the row at one vector each, at most a wave; then up to 4
// vectors per lane (3 in the forward); then a workgroup per row (0 lanes). A wave
// per row against a workgroup, forward and backward: 49154 x 1024 in bfloat16 32 +
// 58 us against 51 + 150, 20000 x 1536 23 + 37 against 25 + 58, 20000 x 2048 33 + 55
// against 28 + 61, 20000 x 1024 in float32 28 + 44 against 26 + 48.
struct LnShape {
    int lanes, k;
    bool tail;
};

static LnShape ln_shape(int c, int dtype, bool bwd) {
    const int v = dtype == SVTAD_F32 ? 4 : 8, vecs = (int)cdiv(c, v);
    LnShape s{1, 1, c % v != 0};
    while (s.lanes < vecs && s.lanes < 64) s.lanes *= 2;
    if (vecs > 64) s.k = (int)cdiv(vecs, 64);
    if (s.k > (bwd ? 4 : 3)) s.lanes = 0, s.k = vecs <= 512 ? 2 : vecs <= 1024 ? 4 : 8;
    return s;
}

// Workgroups of the backward: as many as the 256 compute units hold at two
// each, and no more than the rows need (49154 x 1024 in bfloat16: 58 us with 512, 88
// with 256, 66 with 1024, whose partial sums cost more); one each for rows so wide
// that partial sums weigh more still (5000 x 8192 in bfloat16 65 us against 78 with
// 512, 10000 x 4096 63 against 54).
static int ln_bwd_groups(int64_t rows, int c, const LnShape& s) {
    const int per = s.lanes ? 256 / s.lanes : 1;
    return (int)std::max<int64_t>(1, std::min<int64_t>(cdiv(rows, per), c > 4096 ? 256 : 512));
}

template <typename T, int K, bool WG>
static void launch_ln(const LnArgs& a, bool bwd, bool tail, int grid, hipStream_t st) {
    if (bwd) {
        if (tail) k_layer_norm_bwd<T, K, WG, true><<<grid, 256, 0, st>>>(a);
        else k_layer_norm_bwd<T, K, WG, false><<<grid, 256, 0, st>>>(a);
    } else if constexpr (WG || K < 4) {
        if (tail) k_layer_norm<T, K, WG, true><<<grid, 256, 0, st>>>(a);
        else k_layer_norm<T, K, WG, false><<<grid, 256, 0, st>>>(a);
    }
}

template <typename T>
static void launch_ln_type(const LnArgs& a, bool bwd, const LnShape& s, int grid, hipStream_t st) {
    if (!s.lanes) {
        if constexpr (sizeof(T) == 4) {
            if (s.k == 8) return launch_ln<T, 8, true>(a, bwd, s.tail, grid, st);
        }
        if (s.k == 2) return launch_ln<T, 2, true>(a, bwd, s.tail, grid, st);
        return launch_ln<T, 4, true>(a, bwd, s.tail, grid, st);
    }
    switch (s.k) {
        case 1: return launch_ln<T, 1, false>(a, bwd, s.tail, grid, st);
        case 2: return launch_ln<T, 2, false>(a, bwd, s.tail, grid, st);
        case 3: return launch_ln<T, 3, false>(a, bwd, s.tail, grid, st);
        default: return launch_ln<T, 4, false>(a, bwd, s.tail, grid, st);
    }
}

static int ln_check(const svtad_norm_args* p, int dtype) {
    if (!p) return set_error(SVTAD_ERR_INVALID, "layer_norm: args is NULL");
    if (dtype != SVTAD_F32 && dtype != SVTAD_F16 && dtype != SVTAD_BF16)
        return set_error(SVTAD_ERR_INVALID, "layer_norm: dtype must be float32, float16 or bfloat16");
    if (p->d0 < 0 || p->d1 < 0 || p->d2 < 0) return set_error(SVTAD_ERR_INVALID, "layer_norm: negative row count");
    if (p->c < 1 || p->c > kMaxWidth)
        return set_error(SVTAD_ERR_UNSUPPORTED, "layer_norm: the width must be 1 to 8192");
    if (p->d1 > UINT32_MAX || p->d2 > UINT32_MAX ||
        ((p->d1 != 1 || p->d2 != 1) && (double)p->d0 * (double)p->d1 * (double)p->d2 > (double)UINT32_MAX))
        return set_error(SVTAD_ERR_UNSUPPORTED, "layer_norm: 2^32 rows or more need one row stride");
    if (p->d0 * p->d1 * p->d2 > ((int64_t)1 << 40))
        return set_error(SVTAD_ERR_UNSUPPORTED, "layer_norm: too many rows");
    return SVTAD_OK;
}

static LnArgs ln_args(const svtad_norm_args* p, const LnShape& s) {
    LnArgs a{};
    a.x = p->x, a.w = p->w, a.b = p->b;
    a.stats = p->stats;
    a.rows = p->d0 * p->d1 * p->d2;
    a.c = p->c, a.lanes = s.lanes;
    a.n1 = (uint32_t)p->d1, a.n2 = (uint32_t)p->d2;
    a.s0 = p->s0, a.s1 = p->s1, a.s2 = p->s2;
    a.t0 = p->t0, a.t1 = p->t1, a.t2 = p->t2;
    a.eps = p->eps;
    a.p32 = p->params_f32 != 0;
    return a;
}

static void ln_launch(const LnArgs& a, bool bwd, const LnShape& s, int dtype, int grid, hipStream_t st) {
    if (dtype == SVTAD_F32) launch_ln_type<float>(a, bwd, s, grid, st);
    else if (dtype == SVTAD_F16) launch_ln_type<f16>(a, bwd, s, grid, st);
    else launch_ln_type<bf16>(a, bwd, s, grid, st);
}

}  // namespace svtad

using namespace svtad;

extern "C" int svtad_norm(const svtad_norm_args* p, void* y, int dtype, void* stream) {
    const int st = ln_check(p, dtype);
    if (st) return st;
    const LnShape s = ln_shape(p->c, dtype, false);
    LnArgs a = ln_args(p, s);
    if (a.rows == 0) return SVTAD_OK;
    if (!p->x || !y) return set_error(SVTAD_ERR_INVALID, "layer_norm: NULL pointer");
    a.y = y;
    const int64_t per = s.lanes ? 256 / s.lanes : 1;
    ln_launch(a, false, s, dtype, (int)std::min<int64_t>(cdiv(a.rows, per), 4096), (hipStream_t)stream);
    return launch_status();
}

extern "C" size_t svtad_norm_bwd_workspace_bytes(int64_t rows, int c, int dtype) {
    if (rows < 1 || c < 1 || c > kMaxWidth) return 0;
    return (size_t)ln_bwd_groups(rows, c, ln_shape(c, dtype, true)) * 2 * (size_t)c * sizeof(float);
}

extern "C" int svtad_norm_bwd(const svtad_norm_args* p, const void* dy, void* dx, void* dw, void* db, void* workspace,
                              size_t workspace_bytes, int dtype, void* stream) {
    const int st = ln_check(p, dtype);
    if (st) return st;
    const LnShape s = ln_shape(p->c, dtype, true);
    LnArgs a = ln_args(p, s);
    const bool sums = dw || db;
    hipStream_t hs = (hipStream_t)stream;
    int grid = 0;
    if (a.rows > 0) {
        if (!p->x || !dy || !p->stats) return set_error(SVTAD_ERR_INVALID, "layer_norm_bwd: NULL pointer");
        grid = ln_bwd_groups(a.rows, a.c, s);
        if (sums && (!workspace || workspace_bytes < svtad_norm_bwd_workspace_bytes(a.rows, a.c, dtype)))
            return set_error(SVTAD_ERR_WORKSPACE, "layer_norm_bwd: workspace too small");
        a.dy = dy, a.y = dx, a.part = sums ? (float*)workspace : nullptr;
        if (dx || sums) ln_launch(a, true, s, dtype, grid, hs);
    }
    if (sums) {  // no row: zeros
        const int blocks = (int)cdiv(2 * a.c, 32);
        const float* part = (const float*)workspace;
        if (a.p32 || dtype == SVTAD_F32) k_layer_norm_sum<float><<<blocks, 256, 0, hs>>>(part, grid, a.c, (float*)dw, (float*)db);
        else if (dtype == SVTAD_F16) k_layer_norm_sum<f16><<<blocks, 256, 0, hs>>>(part, grid, a.c, (f16*)dw, (f16*)db);
        else k_layer_norm_sum<bf16><<<blocks, 256, 0, hs>>>(part, grid, a.c, (bf16*)dw, (bf16*)db);
    }
    return launch_status();
}
