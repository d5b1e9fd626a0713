// The norm over all gradients of a model, and the gradients scaled down to a
// limit (gfx950).
//
//   n = (sum over tensors and elements of g^2)^(1/2)   or   max |g|
//   out = g scale min(1, limit / (n |scale| + 1e-6))
//
// Two passes over many tensors, each launch over up to kTensors of them, consecutive
// and of one pair of types, whose addresses travel in the kernel's arguments: no table in memory, no copy, and
// a captured graph replays it. The elements of a launch's tensors, laid end to
// end, are cut into one equal range per workgroup, which finds its first
// tensor by bisection and walks on from there, so that a model's many small
// tensors cost no workgroup of their own.
//
// Squares are summed in float64: float32 gradients neither overflow nor lose
// small addends, at a rate the vector units outrun memory at (bound by its
// bytes). Every workgroup leaves one partial sum; the scaling pass adds them
// in one fixed order in each of its workgroups, without a launch between (8 KB for
// each launch of the norm's pass: lists of many launches read them many times). Both
// are bound by memory (326 M elements of bfloat16 into float32: the norm 132 us, 4.9
// TB/s, the scaling 428 us, 4.6 TB/s).
#include <algorithm>
#include <cstdlib>
#include <type_traits>

#include "sv_internal.h"
#include "sv_vec.h"

namespace svtad {

constexpr int kTensors = 160;  // of a launch: 24 bytes each of the 4 KB of kernel arguments
constexpr int kMaxGroups = 1024;
constexpr double kClipEps = 1e-6;

struct ClipList {
    const void* g[kTensors];
    void* out[kTensors];
    int64_t end[kTensors];  // elements of the tensors up to and with this one
    int count, g_type, out_type;
};
static_assert(sizeof(ClipList) + 64 <= 4096, "kernel arguments");

struct ClipScale {
    const double* part;
    float* norm;         // written by one workgroup of one launch (NULL: not by this one)
    int parts;
    float limit, scale;  // limit < 0: no clipping
    bool inf;
};

// The list in LDS, one entry per thread: kernel arguments lie in host memory, and
// a search through them there waits for one far load after another (81 M elements
// of 160 tensors in bfloat16: 52 us against 50).
struct ClipTable {
    const void* g[kTensors];
    void* out[kTensors];
    int64_t end[kTensors];
    int first[4];

    // Fills it; the first tensor whose end is past element e
    __device__ __forceinline__ int open(const ClipList& t, int64_t e) {
        const int i = threadIdx.x;
        bool past = false;
        if (i < t.count) {
            g[i] = t.g[i], out[i] = t.out[i], end[i] = t.end[i];
            past = t.end[i] > e;
        }
        const uint64_t m = __ballot(i < t.count && !past);
        if ((i & 63) == 0) first[i >> 6] = __popcll(m);
        __syncthreads();
        return first[0] + first[1] + first[2] + first[3];
    }
};

template <bool INF>
__device__ __forceinline__ double clip_join(double a, double b) {
    if constexpr (INF) return (b > a || b != b) ? b : a;  // a NaN stays
    else return a + b;
}

// Over the workgroup's 256 threads, in a fixed order, in every thread
template <bool INF>
__device__ __forceinline__ double clip_reduce(double v) {
    __shared__ double red[4];
#pragma unroll
    for (int m = 1; m < 64; m <<= 1) v = clip_join<INF>(v, __shfl_xor(v, m, 64));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = v;
    __syncthreads();
    return clip_join<INF>(clip_join<INF>(red[0], red[1]), clip_join<INF>(red[2], red[3]));
}

// n elements of a workgroup, V at a time: vectors(offset, count) for count vectors,
// 256 V elements apart, from where `lines` (elements of S bytes, the wider of what
// is read and written) reaches a cache line on, one(offset) for the others. A
// tensor inside a bucket starts anywhere; a wave that stores parts of lines alone
// costs a third more.
template <int S, int V, int UNROLL, typename F, typename G>
__device__ __forceinline__ void clip_walk(const void* lines, int64_t n, F vectors, G one) {
    int64_t head = ((128 - ((uintptr_t)lines & 127)) & 127) / S;
    head = head < n ? head : n;
    const int64_t end = head + (n - head) / V * V;
    if ((int64_t)threadIdx.x < head) one((int64_t)threadIdx.x);
    int64_t at = head + threadIdx.x * V;
    for (; at + (UNROLL - 1) * 256 * V < end; at += UNROLL * 256 * V) vectors(at, std::integral_constant<int, UNROLL>());
    for (; at < end; at += 256 * V) vectors(at, std::integral_constant<int, 1>());
    if (end + threadIdx.x < n) one(end + threadIdx.x);
}

template <typename T, bool INF>
__global__ __launch_bounds__(256) void k_grad_norm(ClipList t, double* part) {
    constexpr int V = kVec<T>;
    const int64_t total = t.end[t.count - 1];
    const int64_t per = cdiv(cdiv(total, gridDim.x), 64) * 64;
    int64_t e = (int64_t)blockIdx.x * per;
    const int64_t e1 = min<int64_t>(total, e + per);
    double acc[4] = {0.0, 0.0, 0.0, 0.0};
    auto add = [&](T v, int k) {
        const double d = (double)(float)v;
        acc[k] = INF ? clip_join<true>(acc[k], fabs(d)) : fma(d, d, acc[k]);
    };
    __shared__ ClipTable tab;
    for (int i = tab.open(t, e); e < e1; ++i) {
        const int64_t first = i ? tab.end[i - 1] : 0, stop = min<int64_t>(e1, tab.end[i]);
        const T* const g = (const T*)tab.g[i] + (e - first);
        clip_walk<(int)sizeof(T), V, 4>(g, stop - e,
            [&](int64_t at, auto unroll) {
                Pack<T, V> v[unroll.value];
#pragma unroll
                for (int u = 0; u < unroll.value; ++u) v[u] = load_once<Pack<T, V>>(g + at + u * 256 * V);
#pragma unroll
                for (int u = 0; u < unroll.value; ++u)
#pragma unroll
                    for (int k = 0; k < V; ++k) add(v[u].e[k], k & 3);
            },
            [&](int64_t at) { add(g[at], 0); });
        e = stop;
    }
    const double sum = clip_reduce<INF>(clip_join<INF>(clip_join<INF>(acc[0], acc[1]), clip_join<INF>(acc[2], acc[3])));
    if (threadIdx.x == 0) part[blockIdx.x] = sum;
}

// The norm of all partial sums (before scale), in every thread
__device__ __forceinline__ double clip_norm(const ClipScale& s) {
    double a = 0.0;
    if (s.inf) {
        for (int i = threadIdx.x; i < s.parts; i += 256) a = clip_join<true>(a, s.part[i]);
        return clip_reduce<true>(a);
    }
    for (int i = threadIdx.x; i < s.parts; i += 256) a += s.part[i];
    return sqrt(clip_reduce<false>(a));
}

__global__ __launch_bounds__(256) void k_grad_norm_out(ClipScale s) {
    const double n = clip_norm(s) * fabs((double)s.scale);
    if (threadIdx.x == 0) *s.norm = (float)n;
}

// Ranges in the opposite order: what the norm's pass read last is in the cache
// still.
template <typename T, typename O>
__global__ __launch_bounds__(256) void k_grad_scale(ClipList t, ClipScale s) {
    // as many elements as the wider of the two types has in 16 bytes, so that a
    // wave's stores are whole lines (twice 16 bytes per lane: 207 us against 150)
    constexpr int V = 16 / (sizeof(T) > sizeof(O) ? (int)sizeof(T) : (int)sizeof(O));
    constexpr int kBytesInFlight = 64;  // of loads, per thread
    const double n = clip_norm(s) * fabs((double)s.scale);
    if (s.norm && blockIdx.x == 0 && threadIdx.x == 0) *s.norm = (float)n;
    double c = s.limit < 0.f ? 1.0 : (double)s.limit / (n + kClipEps);
    c = (c > 1.0 ? 1.0 : c) * (double)s.scale;
    const float f = (float)c;
    // in place and under the limit: every element keeps its value
    if (f == 1.f && sizeof(T) == sizeof(O) && t.g[0] == t.out[0]) return;
    const int64_t total = t.end[t.count - 1];
    const int64_t per = cdiv(cdiv(total, gridDim.x), 64) * 64;
    int64_t e = (int64_t)(gridDim.x - 1 - blockIdx.x) * per;
    const int64_t e1 = min<int64_t>(total, e + per);
    __shared__ ClipTable tab;
    for (int i = tab.open(t, e); e < e1; ++i) {
        const int64_t first = i ? tab.end[i - 1] : 0, stop = min<int64_t>(e1, tab.end[i]);
        const T* const g = (const T*)tab.g[i] + (e - first);
        O* const o = (O*)tab.out[i] + (e - first);
        clip_walk<16 / V, V, kBytesInFlight / (V * (int)sizeof(T))>(
            sizeof(T) > sizeof(O) ? (const void*)g : o, stop - e,
            [&](int64_t at, auto unroll) {
                Pack<T, V> v[unroll.value];
#pragma unroll
                for (int u = 0; u < unroll.value; ++u) v[u] = load_once<Pack<T, V>>(g + at + u * 256 * V);
#pragma unroll
                for (int u = 0; u < unroll.value; ++u) {
                    Pack<O, V> w;
#pragma unroll
                    for (int k = 0; k < V; ++k) w.e[k] = (O)((float)v[u].e[k] * f);
                    store_once(o + at + u * 256 * V, w);
                }
            },
            [&](int64_t at) { o[at] = (O)((float)g[at] * f); });
        e = stop;
    }
}

// Workgroups for `total` elements: one for every 16 KB or so, at most four per
// compute unit in the norm's pass (each leaves a partial sum), eight in the other
// (25 tensors of 16 K in bfloat16 8.0 us, 8.6 with one for 64 KB; 25 of 256 K 15.9,
// 17.1 with half as many in the scaling pass).
static int clip_groups(int64_t total, int most = kMaxGroups) {
    return (int)std::max<int64_t>(1, std::min<int64_t>(cdiv(total, 4096), most));
}

static int64_t type_size(int dtype) { return dtype == SVTAD_F16 || dtype == SVTAD_BF16 ? 2 : 4; }

static bool share(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes) {
    return (uintptr_t)a < (uintptr_t)b + b_bytes && (uintptr_t)b < (uintptr_t)a + a_bytes;
}

// How the memory of a list's tensors is shared. Workgroups of a launch run in no
// order, so what one of them writes no other may read or write.
enum class Shared {
    kNo,
    kRepeats,  // tensors written in place alone: in launches of their own each mention scales
    kBad,      // an output and something else
    kUnknown,  // no host memory to find out
};

// Tensors in the order of their addresses, outputs beside them or in place, are
// seen to be apart in one walk; others are sorted.
static Shared shared(const svtad_grad* t, int64_t count) {
    enum { READ, OUT, IN_PLACE };
    struct Span {
        uintptr_t lo, hi;
        int kind;
    };
    uintptr_t g_lo = UINTPTR_MAX, g_hi = 0, o_lo = UINTPTR_MAX, o_hi = 0;
    bool ordered = true;
    for (int64_t i = 0; i < count; ++i) {
        if (t[i].count <= 0) continue;
        const uintptr_t g = (uintptr_t)t[i].g, o = (uintptr_t)t[i].out;
        ordered = ordered && g >= g_hi;
        g_lo = std::min(g_lo, g), g_hi = std::max<uintptr_t>(g_hi, g + t[i].count * type_size(t[i].g_type));
        if (o == g && t[i].g_type == t[i].out_type) continue;
        ordered = ordered && o >= o_hi;
        o_lo = std::min(o_lo, o), o_hi = std::max<uintptr_t>(o_hi, o + t[i].count * type_size(t[i].out_type));
    }
    if (ordered && (o_lo >= g_hi || g_lo >= o_hi)) return Shared::kNo;
    Span* const spans = (Span*)malloc((size_t)count * 2 * sizeof(Span));
    if (!spans) return Shared::kUnknown;
    int64_t n = 0;
    for (int64_t i = 0; i < count; ++i) {
        if (t[i].count <= 0) continue;
        const uintptr_t g = (uintptr_t)t[i].g, o = (uintptr_t)t[i].out;
        const bool in_place = o == g && t[i].g_type == t[i].out_type;
        spans[n++] = {g, g + t[i].count * type_size(t[i].g_type), in_place ? IN_PLACE : READ};
        if (!in_place) spans[n++] = {o, o + t[i].count * type_size(t[i].out_type), OUT};
    }
    std::sort(spans, spans + n, [](const Span& a, const Span& b) { return a.lo < b.lo; });
    Shared found = Shared::kNo;
    uintptr_t hi[3] = {0, 0, 0};  // where those so far end, by kind
    for (int64_t i = 0; i < n && found != Shared::kBad; ++i) {
        const Span& s = spans[i];
        for (int kind : {READ, OUT, IN_PLACE}) {
            if (s.lo >= hi[kind] || (s.kind == READ && kind == READ)) continue;
            if (s.kind != IN_PLACE || kind != IN_PLACE) found = Shared::kBad;
            else if (found == Shared::kNo) found = Shared::kRepeats;
        }
        hi[s.kind] = std::max(hi[s.kind], s.hi);
    }
    free(spans);
    return found;
}

struct ClipPlan {  // the launches of a list of tensors of any length
    const svtad_grad* t;
    int64_t count;
    bool once = false;  // no memory twice in a launch: one that writes it

    // The tensors from `at` on that one launch takes: one pair of types, none
    // empty. Returns the next tensor's number.
    int64_t take(int64_t at, ClipList& l) const {
        l.count = 0;
        int64_t total = 0;
        for (; at < count && l.count < kTensors; ++at) {
            const svtad_grad& q = t[at];
            if (q.count == 0) continue;
            if (l.count == 0) l.g_type = q.g_type, l.out_type = q.out_type;
            else if (l.g_type != q.g_type || l.out_type != q.out_type || (l.g[0] == l.out[0]) != (q.g == q.out)) break;
            if (once) {
                const int64_t size = type_size(q.g_type);
                int i = 0;
                while (i < l.count && !share(q.g, q.count * size, l.g[i], (l.end[i] - (i ? l.end[i - 1] : 0)) * size)) ++i;
                if (i < l.count) break;
            }
            l.g[l.count] = q.g, l.out[l.count] = q.out;
            total += q.count;
            l.end[l.count++] = total;
        }
        return at;
    }

    int64_t parts() const {
        ClipList l;
        int64_t n = 0;
        for (int64_t at = 0; at < count;) {
            at = take(at, l);
            if (l.count) n += clip_groups(l.end[l.count - 1]);
        }
        return n;
    }
};

template <typename T>
static void launch_norm(const ClipList& l, bool inf, int grid, double* part, hipStream_t st) {
    if (inf) k_grad_norm<T, true><<<grid, 256, 0, st>>>(l, part);
    else k_grad_norm<T, false><<<grid, 256, 0, st>>>(l, part);
}

template <typename T>
static void launch_scale(const ClipList& l, const ClipScale& s, int grid, hipStream_t st) {
    if (l.out_type == SVTAD_F32) k_grad_scale<T, float><<<grid, 256, 0, st>>>(l, s);
    else if (l.out_type == SVTAD_F16) k_grad_scale<T, f16><<<grid, 256, 0, st>>>(l, s);
    else k_grad_scale<T, bf16><<<grid, 256, 0, st>>>(l, s);
}

static int clip_check(const svtad_grad* t, int64_t count, bool with_out) {
    if (count < 0 || (count > 0 && !t)) return set_error(SVTAD_ERR_INVALID, "grad_clip: bad tensor list");
    auto ok = [](int d) { return d == SVTAD_F32 || d == SVTAD_F16 || d == SVTAD_BF16; };
    for (int64_t i = 0; i < count; ++i) {
        if (!ok(t[i].g_type) || (with_out && !ok(t[i].out_type)))
            return set_error(SVTAD_ERR_INVALID, "grad_clip: tensors must be float32, float16 or bfloat16");
        if (t[i].count < 0) return set_error(SVTAD_ERR_INVALID, "grad_clip: negative element count");
        if (t[i].count > 0 && (!t[i].g || (with_out && !t[i].out))) return set_error(SVTAD_ERR_INVALID, "grad_clip: NULL pointer");
    }
    return SVTAD_OK;
}

}  // namespace svtad

using namespace svtad;

extern "C" size_t svtad_grad_clip_workspace_bytes(const svtad_grad* tensors, int64_t count) {
    if (!tensors || count < 1) return 0;
    return (size_t)ClipPlan{tensors, count}.parts() * sizeof(double);
}

extern "C" int svtad_grad_clip(const svtad_grad* tensors, int64_t count, int norm_type, float max_norm, float scale,
                         int write, float* norm, void* workspace, size_t workspace_bytes, void* stream) {
    const int st = clip_check(tensors, count, write != 0);
    if (st) return st;
    if (norm_type != SVTAD_NORM_2 && norm_type != SVTAD_NORM_INF)
        return set_error(SVTAD_ERR_INVALID, "grad_clip: norm_type must be the 2-norm or the maximum");
    if (!norm) return set_error(SVTAD_ERR_INVALID, "grad_clip: NULL pointer");
    const Shared memory = write ? shared(tensors, count) : Shared::kNo;
    if (memory == Shared::kBad) return set_error(SVTAD_ERR_INVALID, "grad_clip: an output shares memory with another tensor");
    if (memory == Shared::kUnknown) return set_error(SVTAD_ERR_UNSUPPORTED, "grad_clip: out of host memory");
    const ClipPlan plan{tensors, count};
    const int64_t parts = plan.parts();
    if (parts > INT32_MAX) return set_error(SVTAD_ERR_UNSUPPORTED, "grad_clip: too many tensors");
    if (parts > 0 && (!workspace || workspace_bytes < (size_t)parts * sizeof(double)))
        return set_error(SVTAD_ERR_WORKSPACE, "grad_clip: workspace too small");
    hipStream_t hs = (hipStream_t)stream;
    double* const part = (double*)workspace;
    const bool inf = norm_type == SVTAD_NORM_INF;
    ClipList l;
    int64_t done = 0, starts[64];  // where launches begin; the 64th stands for all that follow
    int n_starts = 0;
    for (int64_t at = 0; at < count;) {
        if (n_starts < 64) starts[n_starts++] = at;
        at = plan.take(at, l);
        if (!l.count) continue;
        const int grid = clip_groups(l.end[l.count - 1]);
        if (l.g_type == SVTAD_F32) launch_norm<float>(l, inf, grid, part + done, hs);
        else if (l.g_type == SVTAD_F16) launch_norm<f16>(l, inf, grid, part + done, hs);
        else launch_norm<bf16>(l, inf, grid, part + done, hs);
        done += grid;
    }
    ClipScale s{part, norm, (int)parts, max_norm, scale, inf};
    if (!write || parts == 0) {
        k_grad_norm_out<<<1, 256, 0, hs>>>(s);
        return launch_status();
    }
    // the last launch's tensors first: the cache holds them still
    for (int i = n_starts - 1; i >= 0; --i) {
        const ClipPlan part{tensors, i + 1 < n_starts ? starts[i + 1] : count, memory == Shared::kRepeats};
        for (int64_t at = starts[i]; at < part.count;) {
            at = part.take(at, l);
            if (!l.count) continue;
            const int grid = clip_groups(l.end[l.count - 1], 2 * kMaxGroups);
            if (l.g_type == SVTAD_F32) launch_scale<float>(l, s, grid, hs);
            else if (l.g_type == SVTAD_F16) launch_scale<f16>(l, s, grid, hs);
            else launch_scale<bf16>(l, s, grid, hs);
            s.norm = nullptr;
        }
    }
    return launch_status();
}
