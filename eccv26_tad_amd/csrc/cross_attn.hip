// C ABI of cross attention: checks, the split of the work, dispatch by type.
#include "cross_attn.h"

#include <algorithm>
#include <cmath>

namespace svtad {

constexpr int kMaxHeadDim = 128;

// Workgroups of one launch: with 256 threads each, the runtime takes a grid of 2^32
// threads and more modulo 2^32, without an error.
constexpr int64_t kMaxGrid = (1 << 24) - 1;

// Splits of an axis of `tiles` tiles for `groups` workgroups of `rows` results:
// as many as fill one, two, three or four workgroups per compute unit, or none,
// whichever is estimated to take least. The estimate is in times of one tile on a
// compute unit of its own: for two products 0.87 us in 16 bits at a head dimension
// of 64, 7 times as much in float32. Two and more workgroups share a unit and take 0.75 of it each,
// unless one fills it (float32, wide heads). Partial results cost a launch (4.4 us)
// and their writing, reading and adding (0.026 us for 128 rows of 64). Measured in
// bfloat16 at 64, 1000 rows, forward, split against whole: 48 groups over 1500
// keys 17.5 us in four against 25.9, 192 over 500 keys 23.8 in two against 12.3, 192
// over 20000 keys 176 in four against 202 in two and 277. One query over 8 x 31361
// keys of 4 heads: 47.3 us in 16, 53.5 in 8, 55.1 in 24. Heads of 33 to 64 whose rows
// are not read in whole vectors run in the 128-wide kernel, which the estimate does
// not tell from the 64-wide one.
static int splits(const svtad_cross_args& a, int dtype, int64_t groups, int64_t tiles, int rows, double products) {
    const bool alone = dtype == SVTAD_F32 || a.head_dim > 64;
    const double tile = products / 2. * (dtype == SVTAD_F32 ? 7 : 1) * (0.5 + a.head_dim / 128.);
    const double launch = 5 / tile, part = 0.03 * rows * a.head_dim / (128 * 64) / tile;
    int best = 1;
    double least = (double)tiles * (double)cdiv(groups, 256);
    for (int rounds = 1; rounds <= 4 && groups > 0; ++rounds) {
        const int64_t most = std::min<int64_t>({256 * rounds / groups, tiles, (int64_t)kMaxSplits});
        if (most < 2) continue;
        const int64_t each = cdiv(tiles, most), s = cdiv(tiles, each);  // no more splits than these tiles each need
        const double time = (double)each * rounds * (rounds == 1 || alone ? 1 : 0.75) + launch + part * (double)(groups * s);
        if (time < least) best = (int)s, least = time;
    }
    return best;
}

// How a kernel over row tiles (forward, dq) is cut: waves along the rows, and
// splits of the keys. Rows are not padded to more than twice their number where
// fewer waves can hold them (bfloat16, 8 samples of 16 heads over 8192 keys: 48 us
// by 64 rows a workgroup against 75 by 16 at 17 rows, 74 against 57 by 128 at 65;
// float32, one row: 98 us by 16 against 157 by 64 and 312 by 128).
struct RowPlan {
    int wave_rows, splits;
};

static int row_tile(int64_t m) { return m <= 16 ? 16 : m <= 64 ? 64 : 128; }

static RowPlan row_plan(const svtad_cross_args& a, int dtype) {
    const int64_t m = a.nq * (a.heads / a.kv_heads);
    const int rows = row_tile(m);
    RowPlan r{rows == 128 ? 4 : rows == 64 ? 2 : 1, 1};
    r.splits = splits(a, dtype, cdiv(m, rows) * a.batch * a.kv_heads, cdiv(a.nk, r.wave_rows == 1 ? 128 : 64), rows, 2);
    return r;
}

// Splits of the rows in the kernel over key tiles.
static int key_plan(const svtad_cross_args& a, int dtype) {
    const int64_t m = a.nq * (a.heads / a.kv_heads);
    return splits(a, dtype, cdiv(a.nk, kCrossKvKeys) * a.batch * a.kv_heads, cdiv(m, 64), kCrossKvKeys, 3.4);  // four, and what they share
}

static size_t align256(size_t n) { return (n + 255) & ~(size_t)255; }
static int64_t all_rows(const svtad_cross_args& a) { return a.batch * a.heads * a.nq; }
static int64_t pad4(int d) { return (d + 3) & ~3; }

static size_t fwd_bytes(const svtad_cross_args& a, int dtype) {
    const int s = row_plan(a, dtype).splits;
    return s > 1 ? (size_t)s * all_rows(a) * (pad4(a.head_dim) + 2) * 4 : 0;
}

static size_t bwd_bytes(const svtad_cross_args& a, int dtype) {
    const int sq = row_plan(a, dtype).splits, sk = key_plan(a, dtype);
    const size_t pq = sq > 1 ? (size_t)sq * all_rows(a) * pad4(a.head_dim) * 4 : 0;
    const size_t pk = sk > 1 ? (size_t)sk * 2 * a.batch * a.kv_heads * a.nk * pad4(a.head_dim) * 4 : 0;
    return align256((size_t)all_rows(a) * 4) + std::max(pq, pk);
}

// The strides of a tensor [batch, tokens, heads, .] as the kernels take them: that of
// an axis with one place, which may be any number, as 0.
struct Strides {
    int64_t b, n, h;
};
static Strides strides(const int64_t* s, int64_t batch, int64_t tokens, int heads) {
    return {batch > 1 ? s[0] : 0, tokens > 1 ? s[1] : 0, heads > 1 ? s[2] : 0};
}
static Strides q_strides(const svtad_cross_args& a, const int64_t* s) { return strides(s, a.batch, a.nq, a.heads); }
static Strides k_strides(const svtad_cross_args& a, const int64_t* s) { return strides(s, a.batch, a.nk, a.kv_heads); }

// Offsets within a tile of 128 tokens, over the heads of one key head, are 32
// bits in the kernels.
static bool near_strides(const Strides& s, int group, int dtype) {
    const double size = dtype == SVTAD_F32 ? 4 : 2;
    return s.n >= 0 && s.h >= 0 && ((double)s.n * 128 + (double)s.h * group + 128) * size < 2147483648.0;
}

static int cross_check(const svtad_cross_args* a, int dtype, bool bwd) {
    if (!a) return set_error(SVTAD_ERR_INVALID, "cross_attention: args is NULL");
    if (dtype != SVTAD_F32 && dtype != SVTAD_F16 && dtype != SVTAD_BF16)
        return set_error(SVTAD_ERR_INVALID, "cross_attention: dtype must be float32, float16 or bfloat16");
    if (a->batch < 0 || a->nq < 0 || a->nk < 0) return set_error(SVTAD_ERR_INVALID, "cross_attention: negative size");
    if (a->heads < 1 || a->kv_heads < 1 || a->heads % a->kv_heads)
        return set_error(SVTAD_ERR_INVALID, "cross_attention: the query heads must be a multiple of the key heads");
    if (a->head_dim < 1 || a->head_dim > kMaxHeadDim)
        return set_error(SVTAD_ERR_UNSUPPORTED, "cross_attention: the head dimension must be 1 to 128");
    if (!(a->scale > 0.f) || !std::isfinite(a->scale))
        return set_error(SVTAD_ERR_INVALID, "cross_attention: scale must be positive and finite");
    const double m = (double)a->nq * (a->heads / a->kv_heads), bk = (double)a->batch * a->kv_heads;
    if ((m / 16 + 1) * bk * kMaxSplits > INT32_MAX || ((double)a->nk / 64 + 1) * bk * kMaxSplits > INT32_MAX ||
        bk * std::max(m, (double)a->nk) > (double)INT32_MAX || std::ceil(m / row_tile((int64_t)m)) * bk > kMaxGrid ||
        (bwd && std::ceil((double)a->nk / kCrossKvKeys) * bk > kMaxGrid))
        return set_error(SVTAD_ERR_UNSUPPORTED, "cross_attention: too many rows or keys for one launch");
    const int g = a->heads / a->kv_heads;
    if (!near_strides(q_strides(*a, a->q_stride), g, dtype) || !near_strides(k_strides(*a, a->k_stride), 1, dtype) ||
        !near_strides(k_strides(*a, a->v_stride), 1, dtype))
        return set_error(SVTAD_ERR_UNSUPPORTED, "cross_attention: 128 tokens must lie within 2 GiB");
    return SVTAD_OK;
}

// Whether rows are read 16 bytes at a time: every start at 16 bytes and every
// stride a multiple of 8 elements.
static bool whole_vectors(const void* p, const Strides& s) {
    return (uintptr_t)p % 16 == 0 && s.b % 8 == 0 && s.n % 8 == 0 && s.h % 8 == 0;
}

static CrossArgs cross_args(const svtad_cross_args& a, int dtype) {
    CrossArgs p{};
    p.q = a.q, p.k = a.k, p.v = a.v;
    const Strides q = q_strides(a, a.q_stride), k = k_strides(a, a.k_stride), v = k_strides(a, a.v_stride);
    p.qb = q.b, p.qn = q.n, p.qh = q.h;
    p.kb = k.b, p.kn = k.n, p.kh = k.h;
    p.vb = v.b, p.vn = v.n, p.vh = v.h;
    p.lengths = a.lengths;
    p.mask = a.mask, p.mask_b = a.mask_stride[0], p.mask_n = a.mask_stride[1];
    p.B = (int)a.batch, p.H = a.heads, p.KH = a.kv_heads, p.G = a.heads / a.kv_heads, p.D = a.head_dim;
    p.Nq = a.nq, p.Nk = a.nk, p.M = a.nq * p.G;
    p.scale = a.scale;
    p.c = (float)((double)a.scale * 1.4426950408889634);
    p.inv_g = 1.f / p.G;
    p.vec = a.head_dim % 8 == 0 && whole_vectors(a.q, q) && whole_vectors(a.k, k) && whole_vectors(a.v, v);
    p.up = p.down = 1.f;
    if (dtype == SVTAD_F16)
        for (int64_t n = 2; n <= a.nk && n <= 8192; n *= 2) p.up *= 2.f, p.down *= 0.5f;
    p.splits = 1;
    return p;
}

}  // namespace svtad

using namespace svtad;

extern "C" size_t svtad_cross_attention_workspace_bytes(const svtad_cross_args* a, int dtype) {
    return cross_check(a, dtype, false) ? 0 : fwd_bytes(*a, dtype);
}

extern "C" size_t svtad_cross_attention_bwd_workspace_bytes(const svtad_cross_args* a, int dtype) {
    return cross_check(a, dtype, true) ? 0 : bwd_bytes(*a, dtype);
}

extern "C" int svtad_cross_attention(const svtad_cross_args* a, void* out, float* lse, void* rest, void* workspace,
                                     size_t workspace_bytes, int dtype, void* stream) {
    const int st = cross_check(a, dtype, false);
    if (st) return st;
    if (all_rows(*a) == 0) return SVTAD_OK;
    if (!a->q || !out || (a->nk > 0 && (!a->k || !a->v))) return set_error(SVTAD_ERR_INVALID, "cross_attention: NULL pointer");
    const size_t need = fwd_bytes(*a, dtype);
    if (need && (!workspace || workspace_bytes < need))
        return set_error(SVTAD_ERR_WORKSPACE, "cross_attention: workspace too small");
    const RowPlan plan = row_plan(*a, dtype);
    CrossArgs p = cross_args(*a, dtype);
    p.out = out, p.lse = lse, p.rest = dtype == SVTAD_F32 ? nullptr : rest;
    p.splits = plan.splits, p.part = (float*)workspace;
    if (dtype == SVTAD_F16) cross_fwd<f16>(p, plan.wave_rows, (hipStream_t)stream);
    else if (dtype == SVTAD_BF16) cross_fwd<bf16>(p, plan.wave_rows, (hipStream_t)stream);
    else cross_fwd<float>(p, plan.wave_rows, (hipStream_t)stream);
    return launch_status();
}

template <typename T>
static void cross_bwd(CrossArgs p, const svtad_cross_args& a, int dtype, hipStream_t st) {
    const RowPlan plan = row_plan(a, dtype);
    float* const part = p.part;
    if (p.M > 0) {
        p.splits = p.out ? plan.splits : 1;
        cross_bwd_q<T>(p, plan.wave_rows, st);
    }
    if (p.dk && a.nk > 0) {
        p.splits = key_plan(a, dtype), p.part = part;
        cross_bwd_kv<T>(p, st);
    }
}

extern "C" int svtad_cross_attention_bwd(const svtad_cross_args* a, const void* out, const void* rest, const float* lse,
                                         const void* dout, const int64_t* dout_stride, void* dq, void* dk, void* dv, void* workspace,
                                         size_t workspace_bytes, int dtype, void* stream) {
    const int st = cross_check(a, dtype, true);
    if (st) return st;
    if (!dk != !dv) return set_error(SVTAD_ERR_INVALID, "cross_attention_bwd: dk and dv come together");
    if ((!dq && !dk) || a->batch == 0) return SVTAD_OK;
    // without queries dk and dv are written all the same, by a kernel that holds k and v
    if ((a->nq > 0 && (!a->q || !out || !lse || !dout || !dout_stride)) ||
        (a->nk > 0 && (a->nq > 0 || dk) && (!a->k || !a->v)))
        return set_error(SVTAD_ERR_INVALID, "cross_attention_bwd: NULL pointer");
    const size_t need = bwd_bytes(*a, dtype);
    if (need && (!workspace || workspace_bytes < need))
        return set_error(SVTAD_ERR_WORKSPACE, "cross_attention_bwd: workspace too small");
    CrossArgs p = cross_args(*a, dtype);
    p.rest = dtype == SVTAD_F32 ? nullptr : const_cast<void*>(rest);
    p.o = out, p.on = (int64_t)a->heads * a->head_dim, p.oh = a->head_dim, p.ob = a->nq * p.on;
    p.dout = dout;
    const Strides g = dout_stride ? q_strides(*a, dout_stride) : Strides{0, 0, 0};
    if (!near_strides(g, p.G, dtype))
        return set_error(SVTAD_ERR_UNSUPPORTED, "cross_attention_bwd: 128 tokens of dout must lie within 2 GiB");
    p.vec = p.vec && (uintptr_t)out % 16 == 0 && (uintptr_t)p.rest % 16 == 0 && whole_vectors(dout, g);
    p.gb = g.b, p.gn = g.n, p.gh = g.h;
    p.out = dq, p.dk = dk, p.dv = dv;
    p.lse = const_cast<float*>(lse);
    p.delta = (float*)workspace;
    p.part = (float*)((char*)workspace + align256((size_t)all_rows(*a) * 4));
    hipStream_t hs = (hipStream_t)stream;
    if (dtype == SVTAD_F16) cross_bwd<f16>(p, *a, dtype, hs);
    else if (dtype == SVTAD_BF16) cross_bwd<bf16>(p, *a, dtype, hs);
    else cross_bwd<float>(p, *a, dtype, hs);
    return launch_status();
}
