"""The CrossAttention module against the same layers in float64, its serving
form, the operators' differentiability, and the example that runs them together."""
from __future__ import annotations

import math

import pytest
import torch
import torch.nn.functional as F

pytestmark = pytest.mark.gpu


def _reference(m, x, context, lengths=None):
    """The module's computation in float64 from its parameters; returns the
    output, the leaves and their names."""
    P = {n: p.detach().double().requires_grad_(True) for n, p in m.named_parameters()}
    X, C = x.detach().double().requires_grad_(True), context.detach().double().requires_grad_(True)
    norm = lambda t, n: F.layer_norm(t, (t.shape[-1],), P[f"{n}.weight"], P[f"{n}.bias"], m.norm.eps)  # noqa: E731
    lin = lambda t, n: F.linear(t, P[f"{n}.weight"], P[f"{n}.bias"])  # noqa: E731
    B, Nq, E = X.shape
    Nk, D, G = C.shape[1], m.head_dim, m.num_heads // m.kv_heads
    q = norm(lin(norm(X, "norm"), "q").view(B, Nq, m.num_heads, D), "q_norm").transpose(1, 2)
    kv = lin(norm(C, "context_norm"), "kv").view(B, Nk, 2, m.kv_heads, D)
    k = norm(kv[:, :, 0], "k_norm").repeat_interleave(G, 2).transpose(1, 2)
    v = kv[:, :, 1].repeat_interleave(G, 2).transpose(1, 2)
    s = q @ k.transpose(2, 3).contiguous() / math.sqrt(D)
    if lengths is not None:
        s = s.masked_fill((torch.arange(Nk, device=x.device) >= lengths[:, None])[:, None, None], -math.inf)
    att = (torch.softmax(s, -1) @ v.contiguous()).transpose(1, 2).reshape(B, Nq, E)
    return X + lin(att, "proj"), [X, C, *P.values()], ["x", "context", *P]


def _rel(a, b):
    return float((a.detach().double() - b).norm() / b.norm().clamp_min(1e-30))


@pytest.mark.parametrize("heads,kv_heads,context_dims", [(6, 6, None), (6, 2, 100), (3, 1, 384)])
@pytest.mark.parametrize("ragged", [False, True])
def test_float32(dev, heads, kv_heads, context_dims, ragged):
    import eccv26_tad_amd as sv

    torch.manual_seed(1)
    m = sv.CrossAttention(384, heads, context_dims, kv_heads).to(dev)
    x = torch.randn(3, 17, 384, device=dev, requires_grad=True)
    c = torch.randn(3, 90, context_dims or 384, device=dev, requires_grad=True)
    lengths = torch.tensor([90, 1, 40], device=dev) if ragged else None
    y = m(x, c, key_lengths=lengths)
    Y, leaves, names = _reference(m, x, c, lengths)
    g = torch.randn_like(y)
    got = torch.autograd.grad(y, [x, c, *m.parameters()], g)
    want = torch.autograd.grad(Y, leaves, g.double())
    assert _rel(y, Y.detach()) <= 1e-5
    for n, a, b in zip(names, got, want):
        # the key norm's bias moves every score of a query alike: zero but for rounding
        if n == "k_norm.bias":
            assert float(a.norm()) <= 1e-3 * float(g.norm())
        else:
            assert _rel(a, b) <= 1e-4, n


def test_autocast(dev):
    """float32 parameters under autocast(bfloat16), as the training loop runs: a
    float32 residual stream, gradients in float32, bfloat16's accuracy (six
    roundings in a row, 2^-8 each)."""
    import eccv26_tad_amd as sv

    torch.manual_seed(2)
    m = sv.CrossAttention(384, 6, kv_heads=2).to(dev)
    x, c = torch.randn(2, 40, 384, device=dev, requires_grad=True), torch.randn(2, 700, 384, device=dev)
    lengths = torch.tensor([700, 300], dtype=torch.int32, device=dev)
    with torch.autocast("cuda", dtype=torch.bfloat16):
        y = m(x, c, key_lengths=lengths)
    assert y.dtype == torch.float32
    Y, leaves, names = _reference(m, x, c, lengths)
    g = torch.randn_like(y)
    got = torch.autograd.grad(y, [x, *m.parameters()], g)
    want = torch.autograd.grad(Y, [leaves[0], *leaves[2:]], g.double())
    assert _rel(y, Y.detach()) <= 6 * 2.0 ** -8
    for n, a, b in zip([names[0], *names[2:]], got, want):
        assert a.dtype == torch.float32
        if n not in ("k_norm.bias",):
            assert _rel(a, b) <= 12 * 2.0 ** -8, n


@pytest.mark.parametrize("dtype", [torch.float16, torch.float32])
def test_serving_tokens_one_by_one(dev, dtype):
    """Queries one at a time over keys and values that are projected once agree
    with all queries together."""
    import eccv26_tad_amd as sv

    torch.manual_seed(3)
    m = sv.CrossAttention(384, 6, kv_heads=2).to(dev, dtype)
    x, c = torch.randn(1, 9, 384, device=dev).to(dtype), torch.randn(1, 1500, 384, device=dev).to(dtype)
    with torch.no_grad():
        kv = m.project_context(c)
        one = torch.cat([m(x[:, i : i + 1], kv=kv) for i in range(9)], 1)
        assert _rel(one, m(x, c).double()) <= (2.0 ** -9 if dtype == torch.float16 else 1e-5)


def test_arguments(dev):
    import eccv26_tad_amd as sv

    m = sv.CrossAttention(64, 2).to(dev)
    x = torch.randn(1, 2, 64, device=dev)
    with pytest.raises(ValueError, match="either"):
        m(x)
    with pytest.raises(ValueError, match="either"):
        m(x, x, kv=m.project_context(x))


def test_differentiable_once(dev):
    import eccv26_tad_amd as sv

    x = torch.randn(5, 64, device=dev, requires_grad=True)
    (g,) = torch.autograd.grad(sv.layer_norm(x).square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="layer_norm twice"):
        torch.autograd.grad(g.sum(), x)
    q = torch.randn(1, 3, 2, 16, device=dev, requires_grad=True)
    k = torch.randn(1, 7, 2, 16, device=dev)
    (g,) = torch.autograd.grad(sv.cross_attention(q, k, k).square().sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="cross_attention twice"):
        torch.autograd.grad(g.sum(), q)


def test_changed_inputs_are_noticed(dev):
    """An input changed in place between the passes, or clipped gradients that a
    graph still holds, raise as everywhere in autograd."""
    import eccv26_tad_amd as sv

    x = torch.randn(5, 64, device=dev)
    w = torch.ones(64, device=dev, requires_grad=True)
    y = sv.layer_norm(x, w)
    x.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.sum().backward()
    g = torch.randn(64, device=dev)
    y = (w * g).sum()
    sv.clip_grads([g], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace"):
        y.backward()


def test_graph_replays(dev):
    """Layer norm and cross attention recorded once, forward and backward, replayed
    on new inputs: the eager call's bits each time."""
    import eccv26_tad_amd as sv

    q = torch.randn(2, 20, 4, 32, device=dev, dtype=torch.bfloat16)
    k, v = (torch.randn(2, 900, 2, 32, device=dev, dtype=torch.bfloat16) for _ in range(2))
    w = torch.ones(32, device=dev)
    dout = torch.randn_like(q)
    n = torch.tensor([900, 500], dtype=torch.int32, device=dev)

    def step():
        ls = [t.detach().requires_grad_(True) for t in (q, k, v, w)]
        out = sv.cross_attention(sv.layer_norm(ls[0], ls[3]), ls[1], ls[2], key_lengths=n)
        return (out.detach(), *torch.autograd.grad(out, ls, dout))

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        for _ in range(2):
            step()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = step()
    for i in range(3):
        q.normal_()
        k.normal_()
        want = step()
        torch.cuda.synchronize()
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(captured, want)), i


def test_example(dev):
    import importlib.util
    import os

    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "cross_attention_decoder.py")
    spec = importlib.util.spec_from_file_location("cross_attention_decoder", path)
    mod = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(mod)
    losses, norms, together, served = mod.main(steps=8)
    assert losses[-1] < losses[0] and all(math.isfinite(v) for v in losses + norms)
    assert served.shape == together.shape == (1, mod.QUERIES, 2)
    # two bfloat16 layers of equal inputs whose keys are summed in another order
    assert float((served - together).abs().max()) <= 2.0 ** -6


def test_second_derivative_is_never_partial(dev):
    """A second derivative that has another path to the input raises as well."""
    import eccv26_tad_amd as sv

    x = torch.randn(5, 64, device=dev, requires_grad=True)
    w = torch.rand(64, device=dev, requires_grad=True)
    (g,) = torch.autograd.grad((sv.layer_norm(x, w) * x).sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="layer_norm twice"):
        torch.autograd.grad(g.sum(), w)
    q, k = (torch.randn(1, 5, 2, 16, device=dev, requires_grad=True) for _ in range(2))
    (g,) = torch.autograd.grad((sv.cross_attention(q, k, k) * q).sum(), q, create_graph=True)
    with pytest.raises(RuntimeError, match="cross_attention twice"):
        torch.autograd.grad(g.sum(), k)


def test_forward_mode_raises(dev):
    """A tangent is not carried by these operators: it raises, with gradients on or
    off, in the operator, in its backward and in the clipping of gradients."""
    import torch.autograd.forward_ad as fw

    import eccv26_tad_amd as sv

    x, w = torch.randn(5, 64, device=dev), torch.rand(64, device=dev)
    q, k = torch.randn(1, 5, 2, 16, device=dev), torch.randn(1, 7, 2, 16, device=dev)
    with fw.dual_level():
        dual = lambda t: fw.make_dual(t, torch.ones_like(t))  # noqa: E731
        calls = [lambda: sv.layer_norm(dual(x), w), lambda: sv.layer_norm(x, dual(w)), lambda: sv.layer_norm(x, w, dual(w)),
                 lambda: sv.layer_norm(dual(x.clone().requires_grad_(True)), w),
                 lambda: sv.cross_attention(dual(q), k, k), lambda: sv.cross_attention(q, dual(k), k),
                 lambda: sv.cross_attention(q, k, dual(k)), lambda: sv.cross_attention(dual(q), k.clone().requires_grad_(True), k),
                 lambda: sv.clip_grads([x.clone(), dual(x)], 1.0), lambda: sv.grad_norm([dual(x)])]
        for i, call in enumerate(calls):
            for context in (torch.enable_grad, torch.no_grad):
                with context(), pytest.raises((RuntimeError, NotImplementedError)):
                    call()
                    pytest.fail(f"call {i} dropped a tangent")
        y = sv.layer_norm(x.clone().requires_grad_(True), w)
        with pytest.raises((RuntimeError, NotImplementedError)):
            y.backward(dual(torch.ones_like(y)))
            pytest.fail("the norm's backward dropped a tangent")
        out = sv.cross_attention(q.clone().requires_grad_(True), k, k)
        with pytest.raises((RuntimeError, NotImplementedError)):
            out.backward(dual(torch.ones_like(out)))
            pytest.fail("the attention's backward dropped a tangent")
        # without a tangent all is as outside
        assert torch.equal(sv.layer_norm(x, w), sv.layer_norm(x.clone().requires_grad_(True), w))


NORMS = ["norm", "context_norm", "q_norm", "k_norm"]


@pytest.mark.parametrize("autocast", [False, True])
@pytest.mark.parametrize("which", NORMS)
def test_norms_are_called_where_a_call_does_more(dev, which, autocast):
    """Hooks on a norm run, a replaced forward or another layer in its place is
    taken; otherwise the kernels compute the same."""
    import eccv26_tad_amd as sv

    torch.manual_seed(4)
    m = sv.CrossAttention(64, 2, context_dims=48, kv_heads=1).to(dev)
    x, c = torch.randn(2, 5, 64, device=dev), torch.randn(2, 30, 48, device=dev)

    def run():
        with torch.autocast("cuda", dtype=torch.bfloat16, enabled=autocast):
            return m(x, c)

    tol = 12 * 2.0 ** -8 if autocast else 1e-5
    want, layer, calls = run(), getattr(m, which), []
    handle = layer.register_forward_hook(lambda mod, a, out: calls.append(which))
    assert _rel(run(), want.double()) <= tol and calls == [which]
    handle.remove()
    handle = layer.register_forward_pre_hook(lambda mod, a: (2 * a[0],))
    twice = run()
    handle.remove()
    layer.forward = lambda t: torch.nn.LayerNorm.forward(layer, 2 * t)
    assert torch.equal(run(), twice)
    del layer.forward
    handle = torch.nn.modules.module.register_module_forward_hook(lambda mod, a, out: calls.append(mod))
    run()
    handle.remove()
    assert layer in calls
    assert torch.equal(run(), want)
    setattr(m, which, torch.nn.Identity())
    assert run().shape == want.shape
    # without a norm before them the other layers see what it was given
    seen = []
    setattr(m, which, torch.nn.LayerNorm(layer.normalized_shape, elementwise_affine=False, device=dev))
    getattr(m, which).register_forward_hook(lambda mod, a, out: seen.append(a[0]) or a[0])
    hooked = run()
    setattr(m, which, torch.nn.Identity())
    assert len(seen) == 1 and torch.equal(run(), hooked)


def test_hooked_norm_gradients(dev):
    import eccv26_tad_amd as sv

    torch.manual_seed(5)
    m = sv.CrossAttention(64, 2).to(dev)
    x = torch.randn(1, 5, 64, device=dev)
    g = torch.randn(1, 5, 64, device=dev)
    want = torch.autograd.grad(m(x, x), list(m.parameters()), g)
    for n in NORMS:
        getattr(m, n).register_forward_hook(lambda mod, a, out: None)
    got = torch.autograd.grad(m(x, x), list(m.parameters()), g)
    for (n, _), a, b in zip(m.named_parameters(), got, want):
        assert n == "k_norm.bias" or _rel(a, b.double()) <= 1e-4, n
