"""Layer norm forward and backward against float64, at the widths where the
kernels change shape (one lane group, a wave, a workgroup per row), with odd
widths, strided rows and the parameters' types; the refusals."""
from __future__ import annotations

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
# One rounding of a float32 evaluation: the unit roundoff of the type; float32
# itself: sums of up to 8192 terms in a tree, a square root and four products.
TOL = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 2e-6}
# Sums over rows: float32 in a chain of at most rows / workgroups terms and a tree.
SUM_TOL = 1e-5
EPS = 1e-5


def _rel(got, exact):
    return float((got.detach().double() - exact).norm() / exact.norm().clamp_min(1e-30))


def _exact(x, w, b, dy):
    X = x.double().requires_grad_(True)
    W, B = (None if p is None else p.double().requires_grad_(True) for p in (w, b))
    var, mean = torch.var_mean(X, -1, correction=0, keepdim=True)
    y = (X - mean) / (var + EPS).sqrt()
    y = y if W is None else y * W
    y = y if B is None else y + B
    leaves = [t for t in (X, W, B) if t is not None]
    return y.detach(), dict(zip([n for n, t in (("x", X), ("w", W), ("b", B)) if t is not None],
                                torch.autograd.grad(y, leaves, dy.double())))


def _check(x, w, b, dy):
    import eccv26_tad_amd as sv

    xs, ws, bs = (None if t is None else t.detach().requires_grad_(True) for t in (x, w, b))
    y = sv.layer_norm(xs, ws, bs, EPS)
    assert y.shape == x.shape and y.dtype == x.dtype and y.is_contiguous()
    with torch.no_grad():
        assert torch.equal(sv.layer_norm(x, w, b, EPS), y)
    leaves = {n: t for n, t in (("x", xs), ("w", ws), ("b", bs)) if t is not None}
    got = dict(zip(leaves, torch.autograd.grad(y, list(leaves.values()), dy)))
    Y, want = _exact(x, w, b, dy)
    assert _rel(y, Y) <= TOL[x.dtype]
    for n, t in got.items():
        assert t.dtype == leaves[n].dtype and t.shape == leaves[n].shape
        # dx sums two float32 means that cancel part of dy w: twice the tolerance
        tol = 2 * TOL[x.dtype] if n == "x" else SUM_TOL + (TOL[t.dtype] if t.dtype != torch.float32 else 0)
        assert _rel(t, want[n]) <= tol, n
    return got


def _inputs(dev, shape, T, P, seed=0):
    g = torch.Generator(device=dev).manual_seed(seed + shape[-1])
    r = lambda *s: torch.randn(*s, generator=g, device=dev)  # noqa: E731
    c = shape[-1]
    return (1 + 2 * r(*shape)).to(T), (1 + 0.3 * r(c)).to(P), (0.3 * r(c)).to(P), r(*shape).to(T)


@pytest.mark.parametrize("dtype,param", [("f16", "f16"), ("f16", "f32"), ("bf16", "bf16"), ("bf16", "f32"), ("f32", "f32")])
@pytest.mark.parametrize("c", [3, 7, 16, 29, 32, 64, 100, 257, 384, 512, 768, 1024, 1025, 1536, 2048, 2049, 4096, 4100, 8191, 8192])
@pytest.mark.parametrize("rows", [1, 3, 67])
def test_widths(dev, c, rows, dtype, param):
    _check(*_inputs(dev, (rows, c), DTYPES[dtype], DTYPES[param]))


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,c", [(8192, 24), (8193, 32), (40001, 16), (5000, 384), (4099, 768), (2051, 1000), (1025, 4096)])
def test_many_rows(dev, rows, c, dtype):
    _check(*_inputs(dev, (rows, c), DTYPES[dtype], torch.float32))


def test_one_channel(dev):
    """A width of 1: the deviation is 0, the output the bias and dx exactly 0."""
    import eccv26_tad_amd as sv

    x, w, b, dy = _inputs(dev, (9, 1), torch.float32, torch.float32)
    xs = x.requires_grad_(True)
    y = sv.layer_norm(xs, w, b)
    assert torch.equal(y, b.expand(9, 1))
    (dx,) = torch.autograd.grad(y, xs, dy)
    assert not dx.any()


def test_two_channels(dev):
    """A width of 2: xhat is +-1 but for eps, so that dx is what eps leaves of
    equal terms, rstd (g - mean g) and rstd xhat mean(g xhat): float32 holds it
    to the size of those."""
    import eccv26_tad_amd as sv

    x, w, b, dy = _inputs(dev, (67, 2), torch.float32, torch.float32)
    xs = x.clone().requires_grad_(True)
    y = sv.layer_norm(xs, w, b, EPS)
    (dx,) = torch.autograd.grad(y, xs, dy)
    Y, want = _exact(x, w, b, dy)
    g = dy.double() * w.double()
    term = (g - g.mean(-1, keepdim=True)) / (x.double().var(-1, correction=0, keepdim=True) + EPS).sqrt()
    assert _rel(y, Y) <= TOL[torch.float32]
    assert float((dx.double() - want["x"]).norm()) <= 2 * TOL[torch.float32] * float(term.norm())


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("c", [16, 29, 64])
def test_strided_rows(dev, dtype, c):
    """The queries of a joint projection [B, N, 3, H, c], in place and permuted,
    a slice of tokens, every second channel, a broadcast input."""
    T = DTYPES[dtype]
    x, w, b, _ = _inputs(dev, (2, 37, 3, 4, c), T, torch.float32)
    dy = torch.randn(2, 37, 4, c, device=dev, generator=torch.Generator(device=dev).manual_seed(1)).to(T)
    _check(x[:, :, 1], w, b, dy)
    _check(x[:, :, 1].transpose(1, 2), w, b, dy.transpose(1, 2))
    _check(x[:, 5:, 0, 0], w, b, dy[:, 5:, 0])
    _check(x.transpose(0, 1)[:, :, 2], w, b, dy.transpose(0, 1))  # x's axes do not collapse, dy's neither
    _check(x[..., ::2], *_inputs(dev, (1, (c + 1) // 2), T, torch.float32)[1:3], x[..., 1::2] if c % 2 == 0 else x[..., ::2])
    _check(x[:, :1, 0].expand(2, 37, 4, c), w, b, dy)
    _check(x[:, :, 0], w, b, dy[:1, :1, :1].expand(2, 37, 4, c))


@pytest.mark.parametrize("offset", [1, 3])
@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_unaligned_start(dev, dtype, offset):
    T = DTYPES[dtype]
    flat, w, b, dy = _inputs(dev, (1, 5 * 384 + offset), T, torch.float32)
    _check(flat[0, offset:].view(5, 384), w[:384], b[:384], dy[0, offset:].view(5, 384))


@pytest.mark.parametrize("which", ["none", "weight", "bias"])
def test_missing_parameters(dev, which):
    x, w, b, dy = _inputs(dev, (50, 100), torch.bfloat16, torch.float32)
    _check(x, w if which == "weight" else None, b if which == "bias" else None, dy)


def test_only_what_is_needed(dev):
    """A frozen input or frozen parameters leave the other gradients as they are."""
    import eccv26_tad_amd as sv

    x, w, b, dy = _inputs(dev, (100, 384), torch.bfloat16, torch.float32)
    full = _check(x, w, b, dy)
    xs = x.clone().requires_grad_(True)
    assert torch.equal(torch.autograd.grad(sv.layer_norm(xs, w, b, EPS), xs, dy)[0], full["x"])
    ws, bs = w.clone().requires_grad_(True), b.clone().requires_grad_(True)
    gw, gb = torch.autograd.grad(sv.layer_norm(x, ws, bs, EPS), (ws, bs), dy)
    assert torch.equal(gw, full["w"]) and torch.equal(gb, full["b"])


def test_parameters_of_a_third_type_are_widened(dev):
    import eccv26_tad_amd as sv

    x, w, b, _ = _inputs(dev, (10, 64), torch.float16, torch.bfloat16)
    assert torch.equal(sv.layer_norm(x, w, b), sv.layer_norm(x, w.float(), b.float()))
    assert torch.equal(sv.layer_norm(x, w, b.float()), sv.layer_norm(x, w.float(), b.float()))


def test_no_rows(dev):
    import eccv26_tad_amd as sv

    x = torch.empty(0, 64, device=dev, requires_grad=True)
    w = torch.ones(64, device=dev, requires_grad=True)
    y = sv.layer_norm(x, w)
    dx, dw = torch.autograd.grad(y, (x, w), torch.empty(0, 64, device=dev))
    assert y.shape == dx.shape == (0, 64) and torch.equal(dw, torch.zeros_like(w))


def test_rows_do_not_mix(dev):
    """NaN and infinities stay in their rows, the parameter sums show them."""
    import eccv26_tad_amd as sv

    x, w, b, dy = _inputs(dev, (64, 40), torch.float32, torch.float32)
    clean = sv.layer_norm(x, w, b)
    x[5, 3], x[9, 0] = float("nan"), float("inf")
    y = sv.layer_norm(x, w, b)
    keep = torch.ones(64, dtype=torch.bool, device=dev)
    keep[[5, 9]] = False
    assert torch.equal(y[keep], clean[keep]) and not y[~keep].isfinite().any()


def test_against_differences(dev):
    """The directional derivative of <dy, y> by central differences, in
    float32: h = 1e-2 leaves a truncation error of order h^2 and a rounding
    error of order 1e-7 / h relative to |dy| |y|."""
    import eccv26_tad_amd as sv

    x, w, b, dy = _inputs(dev, (33, 100), torch.float32, torch.float32)
    xs, ws, bs = (t.clone().requires_grad_(True) for t in (x, w, b))
    grads = torch.autograd.grad(sv.layer_norm(xs, ws, bs, EPS), (xs, ws, bs), dy)
    f = lambda *a: (sv.layer_norm(*a, EPS).double() * dy.double()).sum()  # noqa: E731
    h = 1e-2
    for i, t in enumerate((x, w, b)):
        d = torch.randn(t.shape, device=dev, generator=torch.Generator(device=dev).manual_seed(7 + i))
        at = lambda s: f(*(p + s * d if p is t else p for p in (x, w, b)))  # noqa: E731
        numeric = float((at(h) - at(-h)) / (2 * h))
        analytic = float((grads[i].double() * d.double()).sum())
        assert abs(numeric - analytic) <= 1e-3 * float(grads[i].norm() * d.norm())


def test_repeats_and_other_streams(dev):
    import eccv26_tad_amd as sv

    x, w, b, dy = _inputs(dev, (20000, 256), torch.bfloat16, torch.float32)
    first = _check(x, w, b, dy)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        xs, ws, bs = (t.clone().requires_grad_(True) for t in (x, w, b))
        again = torch.autograd.grad(sv.layer_norm(xs, ws, bs, EPS), (xs, ws, bs), dy)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(p, q) for p, q in zip(first.values(), again))


def test_offsets_past_32_bits(dev):
    """Rows whose elements start beyond 2^32 bytes and 2^31 elements."""
    import eccv26_tad_amd as sv

    rows, c = (1 << 21) + 70, 1024
    x = torch.zeros(rows, c, dtype=torch.float16, device=dev)
    tail = torch.randn(70, c, device=dev, generator=torch.Generator(device=dev).manual_seed(3)).half()
    x[-70:] = tail
    assert torch.equal(sv.layer_norm(x)[-70:], sv.layer_norm(tail))


def test_refusals(dev):
    import eccv26_tad_amd as sv

    x = torch.randn(4, 64, device=dev)
    w = torch.ones(64, device=dev)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        sv.layer_norm(x.cpu())
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        sv.layer_norm(x.double())
    with pytest.raises(RuntimeError, match="64 elements"):
        sv.layer_norm(x, w[:63])
    with pytest.raises(RuntimeError, match="1 to 8192"):
        sv.layer_norm(torch.zeros(2, 8193, device=dev))
    with pytest.raises(RuntimeError, match="eps"):
        sv.layer_norm(x, w, eps=-1.0)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        sv.layer_norm(x, w.cpu())


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("rows,c", [(1600, 1280), (1600, 2056), (1100, 5000), (900, 8192)])
def test_several_wide_rows_per_workgroup(dev, rows, c, dtype):
    """The rows of a workgroup follow one another in the backward; twice the same bits."""
    import eccv26_tad_amd as sv

    x = torch.randn(rows, c, device=dev).to(DTYPES[dtype]).requires_grad_(True)
    w, b = torch.rand(c, device=dev).requires_grad_(True), torch.randn(c, device=dev).requires_grad_(True)
    dy = torch.randn(rows, c, device=dev).to(DTYPES[dtype])
    y = sv.layer_norm(x, w, b, 1e-6)
    got = torch.autograd.grad(y, (x, w, b), dy)
    again = torch.autograd.grad(sv.layer_norm(x, w, b, 1e-6), (x, w, b), dy)
    X, W, B = (t.detach().double().requires_grad_(True) for t in (x, w, b))
    Y = torch.nn.functional.layer_norm(X, (c,), W, B, 1e-6)
    want = torch.autograd.grad(Y, (X, W, B), dy.double())
    u = {"f16": 2.0 ** -11, "bf16": 2.0 ** -8, "f32": 2e-6}[dtype]  # y and dx are rounded once; dw and db are float32 sums
    for a, e, tol in ((y, Y, u), (got[0], want[0], u), (got[1], want[1], 1e-5), (got[2], want[2], 1e-5)):
        assert float((a.double() - e).norm() / e.norm()) <= tol
    assert all(torch.equal(a, e) for a, e in zip(got, again))
