"""Gradient norm and clipping over many tensors against float64."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
# The norm is summed in float64 and rounded once to float32; the factor is
# rounded once to float32, each product once to the output's type.
NORM_TOL = 2.0 ** -23
U = {torch.float16: 2.0 ** -10, torch.bfloat16: 2.0 ** -7, torch.float32: 2.0 ** -22}
SIZES = [(1,), (7,), (300, 5), (128, 256), (0, 4), (4097,), (9, 33, 65), (1,), (70001,)]


def _grads(dev, T, sizes=SIZES, seed=0, gain=1.0):
    g = torch.Generator(device=dev).manual_seed(seed)
    return [(gain * torch.randn(*s, generator=g, device=dev)).to(T) for s in sizes]


def _norm(grads, norm_type=2.0):
    flat = torch.cat([g.double().flatten() for g in grads])
    return float(flat.norm() if norm_type == 2.0 else flat.abs().max())


def _check(out, grads, factor):
    for o, g in zip(out, grads):
        want = g.double() * factor
        tiny = torch.finfo(o.dtype).smallest_normal
        assert bool(((o.double() - want).abs() <= U[o.dtype] * want.abs() + tiny * 2.0 ** -9).all())


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("limit", [1.0, 1e6])
def test_in_place(dev, dtype, norm_type, limit):
    import eccv26_tad_amd as sv

    grads = _grads(dev, DTYPES[dtype])
    before = [g.clone() for g in grads]
    n = _norm(before, norm_type)
    got = sv.clip_grads(grads, limit, norm_type)
    assert got.shape == () and got.dtype == torch.float32 and abs(float(got) - n) <= NORM_TOL * n
    if limit > n:
        assert all(torch.equal(a, b) for a, b in zip(grads, before))
    else:
        _check(grads, before, limit / (n + 1e-6))
    assert abs(float(sv.grad_norm(before, norm_type)) - n) <= NORM_TOL * n


@pytest.mark.parametrize("src,dst", [("f16", "f32"), ("bf16", "f32"), ("f32", "bf16"), ("f16", "f16"), ("f32", "f32"), ("bf16", "f16")])
@pytest.mark.parametrize("limit", [0.5, 1e6])
@pytest.mark.parametrize("scale", [1.0, 2.0 ** -5, -0.25])
def test_into_other_buffers(dev, src, dst, limit, scale):
    import eccv26_tad_amd as sv

    grads = _grads(dev, DTYPES[src])
    before = [g.clone() for g in grads]
    out = [torch.full_like(g, 7, dtype=DTYPES[dst]) for g in grads]
    n = _norm(before) * abs(scale)
    got = sv.clip_grads(grads, limit, out=out, scale=scale)
    assert abs(float(got) - n) <= NORM_TOL * n
    assert all(torch.equal(a, b) for a, b in zip(grads, before))
    _check(out, before, scale * min(1.0, limit / (n + 1e-6)))


def test_many_tensors_of_all_types(dev):
    """More tensors than one launch takes, types mixed, views of one bucket at
    every alignment."""
    import eccv26_tad_amd as sv

    g = torch.Generator(device=dev).manual_seed(2)
    sizes = [int(x) for x in torch.randint(0, 400, (700,), generator=torch.Generator().manual_seed(1))]
    grads = []
    for T in DTYPES.values():
        grads += list(torch.randn(sum(sizes), generator=g, device=dev).to(T).split(sizes))
    order = torch.randperm(len(grads), generator=torch.Generator().manual_seed(3)).tolist()
    grads = [grads[i] for i in order]
    before = [t.clone() for t in grads]
    n = _norm(before)
    assert abs(float(sv.clip_grads(grads, 3.0)) - n) <= NORM_TOL * n
    _check(grads, before, 3.0 / (n + 1e-6))


def test_layouts(dev):
    """Transposed (dense) tensors in place; a strided view as well, its
    neighbours untouched."""
    import eccv26_tad_amd as sv

    base = _grads(dev, torch.float32, [(40, 60), (50, 80)])
    keep = [b.clone() for b in base]
    grads = [base[0].t(), base[1][:, ::2]]
    n = _norm(grads)
    assert abs(float(sv.grad_norm(grads)) - n) <= NORM_TOL * n
    sv.clip_grads(grads, 1.0)
    f = 1.0 / (n + 1e-6)
    _check([base[0]], [keep[0]], f)
    _check([base[1][:, ::2]], [keep[1][:, ::2]], f)
    assert torch.equal(base[1][:, 1::2], keep[1][:, 1::2])


def test_range(dev):
    """float32 gradients whose squares overflow or vanish in float32."""
    import eccv26_tad_amd as sv

    for gain in (1e30, 1e-30):
        grads = _grads(dev, torch.float32, [(1000,), (33,)], gain=gain)
        n = _norm(grads)
        assert abs(float(sv.grad_norm(grads)) - n) <= NORM_TOL * n
    big = _grads(dev, torch.float32, [(1000,)], gain=1e30)
    out = [torch.empty_like(g) for g in big]
    sv.clip_grads(big, 1.0, out=out)
    assert abs(_norm(out) - 1.0) <= 1e-6


@pytest.mark.parametrize("norm_type", [2.0, math.inf])
@pytest.mark.parametrize("at", [0, 5000])
def test_not_finite(dev, norm_type, at):
    import eccv26_tad_amd as sv

    for bad in (math.nan, math.inf, -math.inf):
        grads = _grads(dev, torch.float32, [(6000,), (77,)])
        grads[0][at] = bad
        ref = [torch.nn.Parameter(torch.zeros_like(g)) for g in grads]
        for p, g in zip(ref, grads):
            p.grad = g.clone()
        want = torch.nn.utils.clip_grad_norm_(ref, 1.0, norm_type, foreach=False)
        norm = sv.clip_grads(grads, 1.0, norm_type)
        assert torch.equal(norm.isnan(), want.isnan()) and torch.equal(norm.isinf(), want.isinf())
        for p, g in zip(ref, grads):
            assert torch.equal(g.isnan(), p.grad.isnan()) and torch.equal(g.nan_to_num(), p.grad.nan_to_num())


def test_parameters(dev):
    import eccv26_tad_amd as sv

    params = [torch.nn.Parameter(torch.zeros(s, device=dev)) for s in ((20, 30), (7,), (3,))]
    for p, g in zip(params[:2], _grads(dev, torch.float32, [(20, 30), (7,)])):
        p.grad = g
    before = [p.grad.clone() for p in params[:2]]
    n = _norm(before)
    got = sv.clip_grad_norm_(params, 1.0)
    assert abs(float(got) - n) <= NORM_TOL * n and params[2].grad is None
    _check([p.grad for p in params[:2]], before, 1.0 / (n + 1e-6))
    one = params[0]
    n1 = _norm([one.grad])
    assert abs(float(sv.clip_grad_norm_(one, 0.1)) - n1) <= NORM_TOL * n1
    one.grad[0, 0] = math.nan
    kept = one.grad.clone()
    with pytest.raises(RuntimeError, match="non-finite"):
        sv.clip_grad_norm_(params, 1.0, error_if_nonfinite=True)
    assert torch.equal(one.grad.nan_to_num(), kept.nan_to_num())
    assert float(sv.clip_grad_norm_([params[2]], 1.0)) == 0.0


def test_zero_gradients(dev):
    import eccv26_tad_amd as sv

    grads = [torch.zeros(100, device=dev), torch.zeros(0, device=dev)]
    assert float(sv.clip_grads(grads, 1.0)) == 0.0 and not grads[0].any()
    assert float(sv.grad_norm([torch.zeros(0, device=dev)])) == 0.0
    assert float(sv.clip_grads([torch.zeros(0, device=dev)], 1.0)) == 0.0


def test_offsets_past_32_bits(dev):
    import eccv26_tad_amd as sv

    n = (1 << 31) + 1001
    g = torch.zeros(n, dtype=torch.bfloat16, device=dev)
    g[-1000:] = 2.0
    g[5] = 3.0
    norm = math.sqrt(4000 + 9)
    assert abs(float(sv.clip_grads([g], norm / 2)) - norm) <= NORM_TOL * norm
    assert float(g[-1]) == 1.0 and float(g[5]) == 1.5 and int(torch.count_nonzero(g)) == 1001


def test_repeats_and_graph_replays(dev):
    """Equal bits on every call, and from a captured graph on every replay."""
    import eccv26_tad_amd as sv

    grads = _grads(dev, torch.float32, 20 * SIZES)
    out = [torch.empty_like(g) for g in grads]
    norm = sv.clip_grads(grads, 1.0, out=out)
    want = [o.clone() for o in out]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        assert torch.equal(sv.clip_grads(grads, 1.0, out=out), norm)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        captured = sv.clip_grads(grads, 1.0, out=out)
    for _ in range(3):
        for o in out:
            o.fill_(5)
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(captured, norm) and all(torch.equal(a, b) for a, b in zip(out, want))


def test_refusals(dev):
    import eccv26_tad_amd as sv

    g = [torch.ones(4, device=dev)]
    with pytest.raises(ValueError, match="max_norm"):
        sv.clip_grads(g, -1.0)
    with pytest.raises(ValueError, match="max_norm"):
        sv.clip_grads(g, math.nan)
    with pytest.raises(ValueError, match="norm_type"):
        sv.clip_grads(g, 1.0, norm_type=1.0)
    with pytest.raises(RuntimeError, match="GPU tensor"):
        sv.clip_grads([torch.ones(4)], 1.0)
    with pytest.raises(RuntimeError, match="float32, float16 or bfloat16"):
        sv.clip_grads([torch.ones(4, device=dev, dtype=torch.float64)], 1.0)
    with pytest.raises(RuntimeError, match="outputs"):
        sv.clip_grads(g, 1.0, out=2 * g)
    with pytest.raises(RuntimeError, match="shape"):
        sv.clip_grads(g, 1.0, out=[torch.ones(5, device=dev)])
    with pytest.raises(RuntimeError, match="no tensors"):
        sv.grad_norm([])


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_gradients_listed_more_than_once(dev, dtype):
    """A shared parameter's gradient counts and is scaled once per mention, one
    tensor after the other, and so are views that share some elements."""
    import eccv26_tad_amd as sv

    T = DTYPES[dtype]
    big, small, strided = _grads(dev, T, [(700, 999), (5,), (60, 80)])
    lists = [big, small, big, strided[:, ::2], small, strided[:, ::2], big]
    before = [g.clone() for g in lists]
    n = _norm(before)
    keep = strided.clone()
    got = sv.clip_grads(lists, n / 2)
    assert abs(float(got) - n) <= NORM_TOL * n
    c = n / 2 / (n + 1e-6)
    # each of the m products is rounded: m roundings of a value that only shrinks
    for g, m, was in ((big, 3, before[0]), (small, 2, before[1]), (strided[:, ::2], 2, before[3])):
        want = was.double() * c ** m
        assert bool(((g.double() - want).abs() <= m * (U[T] * want.abs() + torch.finfo(T).smallest_normal * 2.0 ** -9)).all())
    assert torch.equal(strided[:, 1::2], keep[:, 1::2])
    flat = _grads(dev, T, [(300000,)])[0]
    a, b, was = flat[:200000], flat[100000:], flat.clone()
    n = _norm([a, b])
    sv.clip_grads([a, b], n / 4)
    c = n / 4 / (n + 1e-6)
    want = was.double() * c
    want[100000:200000] *= c
    assert bool(((flat.double() - want).abs() <= 2 * (U[T] * want.abs() + torch.finfo(T).smallest_normal * 2.0 ** -9)).all())


def test_a_shared_parameter_as_torch(dev):
    import eccv26_tad_amd as sv

    p, q = (torch.nn.Parameter(torch.zeros(300, 500, device=dev)) for _ in range(2))
    p.grad, = _grads(dev, torch.float32, [(300, 500)])
    q.grad = p.grad.clone()
    want = torch.nn.utils.clip_grad_norm_([p, p], 1.0, foreach=False)
    got = sv.clip_grad_norm_([q, q], 1.0)
    assert abs(float(got) - float(want)) <= 1e-5 * float(want)
    assert float((q.grad - p.grad).norm()) <= 1e-5 * float(p.grad.norm())


def test_outputs_that_share_memory_are_refused(dev):
    import eccv26_tad_amd as sv

    grads = _grads(dev, torch.float32, [(100,), (100,)])
    buf = torch.full((300,), 7.0, device=dev)
    for out in ([buf[:100], buf[50:150]], [buf[:100], buf[:100]], [buf[:100], grads[0]], [grads[0], grads[0]]):
        with pytest.raises(RuntimeError, match="shares memory"):
            sv.clip_grads(grads, 1.0, out=out)
    assert bool((buf == 7.0).all())
    sv.clip_grads([grads[0], grads[0]], 1.0, out=[buf[:100], buf[100:200]])  # read twice, written once each
    assert torch.equal(buf[:100], buf[100:200]) and bool((buf[200:] == 7.0).all())
