// The extension's transformer operators: layer norm, cross attention, gradient
// clipping. Checks, outputs and workspaces through the caching allocator, and
// the current stream of the input's device.
#include <torch/csrc/autograd/functions/basic_ops.h>

#include <tuple>
#include <vector>

#include "torch_ext.h"

namespace {

// Also that no tangent of forward-mode differentiation comes with it, which these
// functions would drop in silence.
void check_float(const at::Tensor& t, const char* name) {
    check_gpu(t, name);
    TORCH_CHECK_NOT_IMPLEMENTED(!t._fw_grad(0).defined(), "opentad_sparse_ops: forward-mode differentiation is not supported (",
                                name, " has a tangent)");
    const auto st = t.scalar_type();
    TORCH_CHECK(st == at::kFloat || st == at::kHalf || st == at::kBFloat16, "opentad_sparse_ops: ", name,
                " must be float32, float16 or bfloat16, got ", st);
}

at::Tensor workspace(size_t bytes, const at::Tensor& like) {
    return bytes ? at::empty({(int64_t)bytes}, like.options().dtype(at::kByte)) : at::Tensor();
}

void* ptr(const at::Tensor& t) { return t.defined() ? t.data_ptr() : nullptr; }
void* ptr(const c10::optional<at::Tensor>& t) { return t.has_value() ? ptr(*t) : nullptr; }

int64_t row_count(const at::Tensor& t) { return t.size(-1) == 0 ? 0 : t.numel() / t.size(-1); }

// The rows of t [..., c] as at most three axes with strides, c's stride 1; a
// tensor whose axes do not collapse that far, or whose last axis is strided, is
// copied.
struct Rows {
    at::Tensor t;
    int64_t d[3], s[3];
};

Rows rows_of(const at::Tensor& t_in) {
    Rows r{t_in, {1, 1, 1}, {0, 0, 0}};
    for (int pass = 0; pass < 2; ++pass) {
        const at::Tensor& t = r.t;
        std::vector<int64_t> d, s;  // innermost first
        if (t.size(-1) <= 1 || t.stride(-1) == 1) {
            for (int64_t i = t.dim() - 2; i >= 0; --i) {
                if (t.size(i) == 1) continue;
                if (!d.empty() && t.stride(i) == d.back() * s.back()) d.back() *= t.size(i);
                else d.push_back(t.size(i)), s.push_back(t.stride(i));
            }
            const int64_t rows = row_count(t);
            if (d.size() <= 1 || (d.size() <= 3 && rows < ((int64_t)1 << 32))) {
                // one axis goes first, its neighbours with size 1
                for (size_t i = 0; i < d.size(); ++i) {
                    const size_t at = d.size() == 1 ? 0 : 2 - i;
                    r.d[at] = d[i], r.s[at] = s[i];
                }
                return r;
            }
        }
        r.t = t.contiguous();
    }
    TORCH_CHECK(false, "opentad_sparse_ops: rows of ", t_in.sizes(), " cannot be walked");
}

struct NormCall {
    svtad_norm_args a{};
    Rows x;
    at::Tensor w, b;
};

NormCall norm_call(const at::Tensor& x, const c10::optional<at::Tensor>& w, const c10::optional<at::Tensor>& b, double eps,
                   const char* who) {
    check_float(x, "x");
    TORCH_CHECK(x.dim() >= 1, "opentad_sparse_ops.", who, ": x needs an axis");
    const int64_t c = x.size(-1);
    TORCH_CHECK(c >= 1 && c <= 8192, "opentad_sparse_ops.", who, ": the width must be 1 to 8192, got ", c);
    TORCH_CHECK(eps >= 0, "opentad_sparse_ops.", who, ": eps must not be negative");
    NormCall n;
    bool f32 = false, first = true;
    for (const auto* p : {&w, &b}) {
        if (!p->has_value() || !(*p)->defined()) continue;
        const at::Tensor& t = **p;
        check_float(t, "weight and bias");
        TORCH_CHECK(t.device() == x.device(), "opentad_sparse_ops.", who, ": weight and bias must be on x's device");
        TORCH_CHECK(t.dim() == 1 && t.size(0) == c, "opentad_sparse_ops.", who, ": weight and bias must have ", c, " elements");
        const bool is32 = t.scalar_type() == at::kFloat;
        TORCH_CHECK(is32 || t.scalar_type() == x.scalar_type(), "opentad_sparse_ops.", who,
                    ": weight and bias must be float32 or have x's dtype");
        TORCH_CHECK(first || is32 == f32, "opentad_sparse_ops.", who, ": weight and bias must have one dtype");
        f32 = is32, first = false;
        (p == &w ? n.w : n.b) = t.contiguous();
    }
    n.x = rows_of(x);
    n.a.x = n.x.t.data_ptr();
    n.a.w = ptr(n.w), n.a.b = ptr(n.b);
    n.a.d0 = n.x.d[0], n.a.d1 = n.x.d[1], n.a.d2 = n.x.d[2];
    n.a.s0 = n.x.s[0], n.a.s1 = n.x.s[1], n.a.s2 = n.x.s[2];
    n.a.c = (int)c, n.a.params_f32 = f32, n.a.eps = (float)eps;
    return n;
}

}  // namespace

// layer_norm(x [..., c], weight, bias, eps, stats) -> (y, stats [rows, 2] float32 or empty)
std::tuple<at::Tensor, at::Tensor> op_layer_norm(const at::Tensor& x, const c10::optional<at::Tensor>& w,
                                                 const c10::optional<at::Tensor>& b, double eps, bool want_stats) {
    NormCall n = norm_call(x, w, b, eps, "layer_norm");
    c10::DeviceGuard g(x.device());
    at::Tensor y = at::empty(x.sizes(), x.options());
    at::Tensor stats = at::empty({want_stats ? row_count(x) : 0, 2}, x.options().dtype(at::kFloat));
    n.a.stats = want_stats ? stats.data_ptr<float>() : nullptr;
    check_status(svtad_norm(&n.a, y.data_ptr(), dtype_code(x), stream_of(x)), "layer_norm");
    return {y, stats};
}

// layer_norm_bwd(dy, x, stats, weight, params_f32, need_x, need_w, need_b) -> (dx, dw, db), undefined where not needed
std::tuple<at::Tensor, at::Tensor, at::Tensor> op_layer_norm_bwd(const at::Tensor& dy, const at::Tensor& x,
                                                                 const at::Tensor& stats, const c10::optional<at::Tensor>& w,
                                                                 bool params_f32, bool need_x, bool need_w, bool need_b) {
    NormCall n = norm_call(x, w, c10::nullopt, 0.0, "layer_norm_bwd");
    check_float(dy, "dy");
    const int64_t rows = row_count(x), c = x.size(-1);
    TORCH_CHECK(dy.sizes() == x.sizes() && dy.scalar_type() == x.scalar_type() && dy.device() == x.device(),
                "opentad_sparse_ops.layer_norm_bwd: dy must be like x");
    TORCH_CHECK(stats.is_contiguous() && stats.scalar_type() == at::kFloat && stats.numel() == 2 * rows &&
                    stats.device() == x.device(),
                "opentad_sparse_ops.layer_norm_bwd: stats must be the forward's");
    TORCH_CHECK(!n.w.defined() || (n.w.scalar_type() == at::kFloat) == params_f32 || x.scalar_type() == at::kFloat,
                "opentad_sparse_ops.layer_norm_bwd: params_f32 does not match the weight");
    c10::DeviceGuard g(x.device());
    // dy's rows along x's axes: the same split, or both dense
    Rows d = rows_of(dy);
    if (d.d[0] != n.x.d[0] || d.d[1] != n.x.d[1] || d.d[2] != n.x.d[2]) {
        auto flat = [rows](const Rows& r) { return r.d[1] == 1 && r.d[2] == 1 && r.d[0] == rows; };
        if (!flat(d)) d = rows_of(dy.contiguous());
        if (!flat(n.x)) {  // dy has one stride: the same rows along x's axes
            const int64_t s = d.s[0];
            for (int i = 0; i < 3; ++i) d.d[i] = n.x.d[i];
            d.s[2] = s, d.s[1] = s * d.d[2], d.s[0] = s * d.d[2] * d.d[1];
        }
    }
    n.a.t0 = d.s[0], n.a.t1 = d.s[1], n.a.t2 = d.s[2];
    n.a.stats = stats.data_ptr<float>();
    n.a.params_f32 = params_f32;
    at::Tensor dx, dw, db;
    const auto param = x.options().dtype(params_f32 ? at::kFloat : x.scalar_type());
    if (need_x) dx = at::empty(x.sizes(), x.options());
    if (need_w) dw = at::empty({c}, param);
    if (need_b) db = at::empty({c}, param);
    const size_t bytes = need_w || need_b ? svtad_norm_bwd_workspace_bytes(rows, (int)c, dtype_code(x)) : 0;
    at::Tensor ws = workspace(bytes, x);
    check_status(svtad_norm_bwd(&n.a, d.t.data_ptr(), ptr(dx), ptr(dw), ptr(db), ptr(ws), bytes, dtype_code(x), stream_of(x)),
                 "layer_norm_bwd");
    return {dx, dw, db};
}

namespace {

struct CrossCall {
    svtad_cross_args a{};
    at::Tensor q, k, v;
};

// t [batch, tokens, heads, head_dim] as the kernels read it: a strided last axis,
// or 128 tokens that lie further apart than 2 GiB, are copied (an axis with one place
// may have any stride)
at::Tensor readable(const at::Tensor& t, int64_t group) {
    const double n = t.size(1) > 1 ? t.stride(1) : 0, h = t.size(2) > 1 ? t.stride(2) : 0;
    const double apart = (n * 128 + h * group + 128) * t.element_size();
    return (t.size(-1) <= 1 || t.stride(-1) == 1) && apart < 2147483648.0 ? t : t.contiguous();
}

CrossCall cross_call(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const c10::optional<at::Tensor>& lengths,
                     const c10::optional<at::Tensor>& mask, double scale, const char* who) {
    check_float(q, "q");
    check_float(k, "k");
    check_float(v, "v");
    TORCH_CHECK(q.dim() == 4 && k.dim() == 4, "opentad_sparse_ops.", who, ": q and k must be [batch, tokens, heads, head_dim]");
    TORCH_CHECK(k.sizes() == v.sizes(), "opentad_sparse_ops.", who, ": k and v must have one shape, got ", k.sizes(), " and ",
                v.sizes());
    TORCH_CHECK(q.size(0) == k.size(0) && q.size(3) == k.size(3), "opentad_sparse_ops.", who,
                ": q and k must have one batch and one head dimension, got ", q.sizes(), " and ", k.sizes());
    TORCH_CHECK(q.scalar_type() == k.scalar_type() && q.scalar_type() == v.scalar_type(), "opentad_sparse_ops.", who,
                ": q, k and v must have one dtype");
    TORCH_CHECK(q.device() == k.device() && q.device() == v.device(), "opentad_sparse_ops.", who,
                ": q, k and v must be on one device");
    TORCH_CHECK(q.size(0) <= INT32_MAX && q.size(2) <= INT32_MAX && k.size(2) <= INT32_MAX, "opentad_sparse_ops.", who,
                ": batch or head count too large");
    CrossCall c;
    const int64_t group = k.size(2) > 0 ? q.size(2) / k.size(2) : 1;
    c.q = readable(q, group), c.k = readable(k, 1), c.v = readable(v, 1);
    for (int i = 0; i < 3; ++i) {
        c.a.q_stride[i] = c.q.stride(i);
        c.a.k_stride[i] = c.k.stride(i);
        c.a.v_stride[i] = c.v.stride(i);
    }
    c.a.q = c.q.data_ptr(), c.a.k = c.k.data_ptr(), c.a.v = c.v.data_ptr();
    c.a.batch = q.size(0), c.a.nq = q.size(1), c.a.nk = k.size(1);
    c.a.heads = (int)q.size(2), c.a.kv_heads = (int)k.size(2);
    TORCH_CHECK(q.size(3) >= 1 && q.size(3) <= 128, "opentad_sparse_ops.", who, ": the head dimension must be 1 to 128, got ",
                q.size(3));
    c.a.head_dim = (int)q.size(3);
    c.a.scale = (float)scale;
    if (lengths.has_value() && lengths->defined()) {
        TORCH_CHECK(lengths->is_cuda() && lengths->device() == q.device() && lengths->scalar_type() == at::kInt &&
                        lengths->dim() == 1 && lengths->size(0) == q.size(0) && lengths->is_contiguous(),
                    "opentad_sparse_ops.", who, ": key_lengths must be contiguous int32 [batch] on q's device");
        c.a.lengths = lengths->data_ptr<int32_t>();
    }
    if (mask.has_value() && mask->defined()) {
        TORCH_CHECK(mask->is_cuda() && mask->device() == q.device() && mask->scalar_type() == at::kBool && mask->dim() == 2 &&
                        mask->size(0) == q.size(0) && mask->size(1) == k.size(1),
                    "opentad_sparse_ops.", who, ": key_mask must be bool [batch, keys] on q's device");
        c.a.mask = (const uint8_t*)mask->data_ptr();
        c.a.mask_stride[0] = mask->stride(0), c.a.mask_stride[1] = mask->stride(1);
    }
    return c;
}

}  // namespace

// cross_attention(q, k, v, key_lengths, key_mask, scale, train) -> (out, lse, rest): for the backward one float32
// per row and what the output's rounding took, or empty
std::tuple<at::Tensor, at::Tensor, at::Tensor> op_cross_attention(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                                                  const c10::optional<at::Tensor>& lengths,
                                                                  const c10::optional<at::Tensor>& mask, double scale,
                                                                  bool train) {
    CrossCall c = cross_call(q, k, v, lengths, mask, scale, "cross_attention");
    c10::DeviceGuard g(q.device());
    const int dt = dtype_code(q);
    at::Tensor out = at::empty(q.sizes(), q.options().memory_format(at::MemoryFormat::Contiguous)), lse, rest;
    if (train) lse = at::empty({q.size(0), q.size(2), q.size(1)}, q.options().dtype(at::kFloat));
    if (train && q.scalar_type() != at::kFloat) rest = at::empty_like(out);
    const size_t bytes = svtad_cross_attention_workspace_bytes(&c.a, dt);
    at::Tensor ws = workspace(bytes, q);
    check_status(svtad_cross_attention(&c.a, out.data_ptr(), (float*)ptr(lse), ptr(rest), ptr(ws), bytes, dt, stream_of(q)),
                 "cross_attention");
    return {out, lse, rest};
}

// cross_attention_bwd(dout, q, k, v, out, lse, rest (or None), key_lengths, key_mask, scale, need_q, need_kv) -> (dq, dk, dv)
std::tuple<at::Tensor, at::Tensor, at::Tensor> op_cross_attention_bwd(
    const at::Tensor& dout_in, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v, const at::Tensor& out,
    const at::Tensor& lse, const c10::optional<at::Tensor>& rest, const c10::optional<at::Tensor>& lengths,
    const c10::optional<at::Tensor>& mask, double scale, bool need_q, bool need_kv) {
    CrossCall c = cross_call(q, k, v, lengths, mask, scale, "cross_attention_bwd");
    check_float(dout_in, "dout");
    const bool has_rest = rest.has_value() && rest->defined();
    for (const at::Tensor* t : {&dout_in, &out, has_rest ? &*rest : &out})
        TORCH_CHECK(t->sizes() == q.sizes() && t->scalar_type() == q.scalar_type() && t->device() == q.device(),
                    "opentad_sparse_ops.cross_attention_bwd: dout, out and rest must be like q");
    TORCH_CHECK(out.is_contiguous() && (!has_rest || rest->is_contiguous()) && lse.is_contiguous() &&
                    lse.scalar_type() == at::kFloat && lse.numel() == q.size(0) * q.size(1) * q.size(2) &&
                    lse.device() == q.device(),
                "opentad_sparse_ops.cross_attention_bwd: out, lse and rest must be the forward's");
    c10::DeviceGuard g(q.device());
    const int dt = dtype_code(q);
    const at::Tensor dout = readable(dout_in, q.size(2) / k.size(2));
    const int64_t ds[3] = {dout.stride(0), dout.stride(1), dout.stride(2)};
    const auto dense = [](const at::Tensor& t) { return at::empty(t.sizes(), t.options()); };
    at::Tensor dq, dk, dv;
    if (need_q) dq = dense(q);
    if (need_kv) dk = dense(k), dv = dense(v);
    const size_t bytes = svtad_cross_attention_bwd_workspace_bytes(&c.a, dt);
    at::Tensor ws = workspace(bytes, q);
    check_status(svtad_cross_attention_bwd(&c.a, out.data_ptr(), ptr(rest), lse.data_ptr<float>(), dout.data_ptr(), ds,
                                           ptr(dq), ptr(dk), ptr(dv), ptr(ws), bytes, dt, stream_of(q)),
                 "cross_attention_bwd");
    return {dq, dk, dv};
}

// grad_clip(grads, outs (None: in place), write, max_norm (negative: no limit), scale, inf) -> norm, a float32
// scalar; without write the norm alone. Tensors whose elements do not fill one span of memory go by way of a copy.
at::Tensor op_grad_clip(const std::vector<at::Tensor>& grads, const c10::optional<std::vector<at::Tensor>>& outs, bool write,
                        double max_norm, double scale, bool inf) {
    TORCH_CHECK(!grads.empty(), "opentad_sparse_ops.grad_clip: no tensors");
    const bool apart = write && outs.has_value();
    TORCH_CHECK(!apart || outs->size() == grads.size(), "opentad_sparse_ops.grad_clip: ", grads.size(), " gradients and ",
                apart ? outs->size() : 0, " outputs");
    at::NoGradGuard no_grad;
    c10::DeviceGuard g(grads[0].device());
    std::vector<svtad_grad> list(grads.size());
    std::vector<at::Tensor> copies;
    std::vector<size_t> copied;
    for (size_t i = 0; i < grads.size(); ++i) {
        at::Tensor t = grads[i];
        check_float(t, "gradients");
        TORCH_CHECK(t.device() == grads[0].device(), "opentad_sparse_ops.grad_clip: gradients must be on one device");
        if (!t.is_non_overlapping_and_dense()) {
            // one copy for all mentions of a tensor, which is scaled once for each
            const auto is_t = [&t](const at::Tensor& u) {
                return u.data_ptr() == t.data_ptr() && u.scalar_type() == t.scalar_type() && u.sizes() == t.sizes() &&
                       u.strides() == t.strides();
            };
            size_t same = 0;
            while (same < copied.size() && !is_t(grads[copied[same]])) ++same;
            if (same < copied.size()) t = copies[same];
            else {
                t = t.contiguous();
                copies.push_back(t);
                if (!apart) copied.push_back(i);
            }
        }
        list[i].g = t.data_ptr(), list[i].count = t.numel(), list[i].g_type = dtype_code(t);
        if (!write) continue;
        const at::Tensor& o = apart ? (*outs)[i] : t;
        if (apart) {
            check_float(o, "outputs");
            TORCH_CHECK(o.device() == t.device() && o.sizes() == t.sizes() &&
                            ((o.is_contiguous() && t.is_contiguous()) || o.strides() == t.strides()),
                        "opentad_sparse_ops.grad_clip: an output must have its gradient's device, shape and strides");
            TORCH_CHECK(t.numel() == 0 || o.data_ptr() != t.data_ptr() || o.scalar_type() == t.scalar_type(),
                        "opentad_sparse_ops.grad_clip: in place an output must have its gradient's dtype");
        }
        list[i].out = o.data_ptr(), list[i].out_type = dtype_code(o);
        if (!o.is_inference()) o.unsafeGetTensorImpl()->bump_version();
    }
    at::Tensor norm = at::empty({}, grads[0].options().dtype(at::kFloat));
    const size_t bytes = svtad_grad_clip_workspace_bytes(list.data(), (int64_t)list.size());
    at::Tensor ws = workspace(bytes, grads[0]);
    check_status(svtad_grad_clip(list.data(), (int64_t)list.size(), inf ? SVTAD_NORM_INF : SVTAD_NORM_2, (float)max_norm,
                                 (float)scale, write, norm.data_ptr<float>(), ptr(ws), bytes, stream_of(grads[0])),
                 "grad_clip");
    if (write) {
        size_t at = 0;
        for (size_t i : copied) grads[i].copy_(copies[at++]);
    }
    return norm;
}

namespace {

// The autograd nodes. They are written here and not in Python because a small
// layer's backward is host time: the engine's thread then needs no interpreter
// (64 x 32 rows of layer norm, forward and backward: 68 us, 91 with a Python node).

using torch::autograd::AutogradContext;
using torch::autograd::variable_list;

// Gradients of a node that is differentiable once: a second derivative raises.
// The gradients hang on all they were made `from`, so that no path to those is
// left out in silence.
variable_list once(variable_list grads, const variable_list& from, const char* who) {
    if (!at::GradMode::is_enabled()) return grads;
    variable_list given;
    for (const auto& g : grads)
        if (g.defined()) given.push_back(g.detach().requires_grad_(true));
    if (given.empty()) return grads;
    for (const auto& t : from)
        if (t.defined()) given.push_back(t);
    auto error = std::make_shared<torch::autograd::DelayedError>(
        std::string("trying to differentiate ") + who + " twice", (int64_t)given.size());
    given = (*error)(std::move(given));
    size_t at = 0;
    for (auto& g : grads)
        if (g.defined()) g = given[at++];
    return grads;
}

// Whether input `i` of the forward needs a gradient: tensors are numbered
// without the absent ones.
struct Needs {
    AutogradContext* ctx;
    size_t at = 0;
    bool next(bool present) { return present && ctx->needs_input_grad(at++); }
};

struct LayerNormNode : torch::autograd::Function<LayerNormNode> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& x, const c10::optional<at::Tensor>& w,
                              const c10::optional<at::Tensor>& b, double eps) {
        at::Tensor y, stats;
        std::tie(y, stats) = op_layer_norm(x, w, b, eps, true);
        const bool has_w = w.has_value() && w->defined(), has_b = b.has_value() && b->defined();
        ctx->save_for_backward({x, stats, has_w ? *w : at::Tensor()});
        ctx->saved_data["has_w"] = has_w;
        ctx->saved_data["has_b"] = has_b;
        ctx->saved_data["f32"] = (has_w && w->scalar_type() == at::kFloat) || (has_b && b->scalar_type() == at::kFloat);
        return y;
    }
    static variable_list backward(AutogradContext* ctx, variable_list dy) {
        const auto saved = ctx->get_saved_variables();
        const bool has_w = ctx->saved_data["has_w"].toBool(), has_b = ctx->saved_data["has_b"].toBool();
        Needs needs{ctx};
        const bool need_x = needs.next(true), need_w = needs.next(has_w), need_b = needs.next(has_b);
        at::Tensor dx, dw, db;
        if (dy[0].defined()) {
            at::NoGradGuard guard;
            std::tie(dx, dw, db) = op_layer_norm_bwd(dy[0], saved[0], saved[1], has_w ? c10::make_optional(saved[2]) : c10::nullopt,
                                                     ctx->saved_data["f32"].toBool(), need_x, need_w, need_b);
        }
        variable_list g = once({dx, dw, db}, {dy[0], saved[0], saved[2]}, "layer_norm");
        g.emplace_back();
        return g;
    }
};

struct CrossAttentionNode : torch::autograd::Function<CrossAttentionNode> {
    static at::Tensor forward(AutogradContext* ctx, const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                              const c10::optional<at::Tensor>& lengths, const c10::optional<at::Tensor>& mask, double scale) {
        at::Tensor out, lse, rest;
        std::tie(out, lse, rest) = op_cross_attention(q, k, v, lengths, mask, scale, true);
        ctx->save_for_backward({q, k, v, out, lse, rest, lengths.value_or(at::Tensor()), mask.value_or(at::Tensor())});
        ctx->saved_data["scale"] = scale;
        return out;
    }
    static variable_list backward(AutogradContext* ctx, variable_list dout) {
        const auto s = ctx->get_saved_variables();
        const bool need_q = ctx->needs_input_grad(0), need_k = ctx->needs_input_grad(1), need_v = ctx->needs_input_grad(2);
        at::Tensor dq, dk, dv;
        if (dout[0].defined()) {
            at::NoGradGuard guard;
            const auto given = [](const at::Tensor& t) { return t.defined() ? c10::make_optional(t) : c10::nullopt; };
            std::tie(dq, dk, dv) = op_cross_attention_bwd(dout[0], s[0], s[1], s[2], s[3], s[4], given(s[5]), given(s[6]),
                                                          given(s[7]),
                                                          ctx->saved_data["scale"].toDouble(), need_q, need_k || need_v);
        }
        variable_list g = once({dq, need_k ? dk : at::Tensor(), need_v ? dv : at::Tensor()},
                               {dout[0], s[0], s[1], s[2]}, "cross_attention");
        g.resize(6);
        return g;
    }
};

}  // namespace

// layer_norm and cross_attention as differentiable functions. A tangent is refused
// here: within the node's forward, forward mode is off and none is seen.
at::Tensor op_layer_norm_grad(const at::Tensor& x, const c10::optional<at::Tensor>& w, const c10::optional<at::Tensor>& b,
                              double eps) {
    check_float(x, "x");
    for (const auto* p : {&w, &b})
        if (p->has_value() && (*p)->defined()) check_float(**p, "weight and bias");
    return LayerNormNode::apply(x, w, b, eps);
}
at::Tensor op_cross_attention_grad(const at::Tensor& q, const at::Tensor& k, const at::Tensor& v,
                                   const c10::optional<at::Tensor>& lengths, const c10::optional<at::Tensor>& mask,
                                   double scale) {
    check_float(q, "q");
    check_float(k, "k");
    check_float(v, "v");
    return CrossAttentionNode::apply(q, k, v, lengths, mask, scale);
}

void bind_operators(pybind11::module& m) {
    m.def("layer_norm", &op_layer_norm, "Layer norm over the last axis (y, stats)", py::arg("x"), py::arg("weight"),
          py::arg("bias"), py::arg("eps"), py::arg("stats"));
    m.def("layer_norm_grad", &op_layer_norm_grad, "layer_norm as a differentiable function", py::arg("x"), py::arg("weight"),
          py::arg("bias"), py::arg("eps"));
    m.def("layer_norm_bwd", &op_layer_norm_bwd, "Its gradients (dx, dw, db)", py::arg("dy"), py::arg("x"), py::arg("stats"),
          py::arg("weight"), py::arg("params_f32"), py::arg("need_x"), py::arg("need_w"), py::arg("need_b"));
    m.def("cross_attention", &op_cross_attention, "Attention of queries to the keys of another sequence (out, lse, rest)",
          py::arg("q"), py::arg("k"), py::arg("v"), py::arg("key_lengths"), py::arg("key_mask"), py::arg("scale"),
          py::arg("train"));
    m.def("cross_attention_grad", &op_cross_attention_grad, "cross_attention as a differentiable function", py::arg("q"),
          py::arg("k"), py::arg("v"), py::arg("key_lengths"), py::arg("key_mask"), py::arg("scale"));
    m.def("cross_attention_bwd", &op_cross_attention_bwd, "Its gradients (dq, dk, dv)", py::arg("dout"), py::arg("q"),
          py::arg("k"), py::arg("v"), py::arg("out"), py::arg("lse"), py::arg("rest"), py::arg("key_lengths"), py::arg("key_mask"),
          py::arg("scale"), py::arg("need_q"), py::arg("need_kv"));
    m.def("grad_clip", &op_grad_clip, "The norm over all gradients, and the gradients scaled down to a limit",
          py::arg("grads"), py::arg("outs"), py::arg("write"), py::arg("max_norm"), py::arg("scale"), py::arg("inf"));
}
