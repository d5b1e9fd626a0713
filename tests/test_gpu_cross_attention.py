"""Cross attention forward and backward against float64, around the kernels'
tile edges (16, 64 and 128 rows, 64 and 128 keys, splits), every head layout,
lengths, masks and rows without a key; the refusals."""
from __future__ import annotations

import math

import pytest
import torch

pytestmark = pytest.mark.gpu

DTYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "f32": torch.float32}
# Unit roundoff of the operand type. 16-bit types: probabilities (or score
# gradients) are rounded once as operands and the result once: 2 u; float32:
# scores are sums of up to 128 products whose rounding the exponential passes
# on, 1e-5 covers |s| up to about 50.
U = {torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float32: 5e-6}


def _exact(q, k, v, dout, lengths, mask, scale):
    """Results in float64, and what the rounding of the output to its type may
    move the gradients by per unit of roundoff: delta = sum dout out enters dq
    as delta * mean key and dk as delta * p * q."""
    q, k, v, dout = (t.double() for t in (q, k, v, dout))
    (B, Nq, H, D), KH = q.shape, k.shape[2]
    Nk = k.shape[1]
    seen = torch.ones(B, Nk, dtype=torch.bool, device=q.device)
    if lengths is not None:
        seen &= torch.arange(Nk, device=q.device) < lengths[:, None]
    if mask is not None:
        seen &= mask
    k, v = (torch.where(seen[:, :, None, None], t, 0.0) for t in (k, v))  # unseen places may hold anything
    K, V = (t.repeat_interleave(H // KH, 2).permute(0, 2, 1, 3) for t in (k, v))
    Q, DO = q.permute(0, 2, 1, 3), dout.permute(0, 2, 1, 3)
    s = (Q @ K.transpose(2, 3).contiguous() * scale).masked_fill(~seen[:, None, None], -math.inf)
    p = torch.where(seen.any(1)[:, None, None, None], torch.softmax(s, -1), 0.0).nan_to_num(0.0)
    out = p @ V
    dp = DO @ V.transpose(2, 3).contiguous()
    ds = p * (dp - (p * dp).sum(-1, keepdim=True)) * scale
    pt, dst = p.transpose(2, 3).contiguous(), ds.transpose(2, 3).contiguous()
    grp = lambda t: t.view(B, KH, H // KH, Nk, D).sum(2).permute(0, 2, 1, 3)  # noqa: E731
    row = lambda t: t.permute(0, 2, 1, 3)  # noqa: E731
    moved = (DO.abs() * out.abs()).sum(-1, keepdim=True) * scale
    return ((row(out), row(ds @ K), grp(dst @ Q), grp(pt @ DO)),
            (None, row(moved * (p @ K).abs()), grp(pt @ (moved * Q.abs())), None))


def _near(got, want, moved, tol, name):
    allow = tol * want.norm() + (0 if moved is None else tol * moved.norm())
    off = (got.double() - want).norm()
    assert got.isfinite().all() and float(off) <= float(allow) + 1e-30, (name, float(off), float(allow))


def _check(q, k, v, dout, lengths=None, mask=None, scale=None, grads=True):
    import eccv26_tad_amd as sv

    ls = [t.detach().requires_grad_(True) for t in (q, k, v)]
    out = sv.cross_attention(*ls, key_lengths=lengths, key_mask=mask, scale=scale)
    assert out.shape == q.shape and out.dtype == q.dtype and out.is_contiguous()
    with torch.no_grad():
        assert torch.equal(sv.cross_attention(q, k, v, key_lengths=lengths, key_mask=mask, scale=scale), out)
    got = (out.detach(), *torch.autograd.grad(out, ls, dout))
    want, moved = _exact(q, k, v, dout, lengths, mask, q.shape[-1] ** -0.5 if scale is None else scale)
    u = U[q.dtype]
    for n, g, w, m, tol in zip(("out", "dq", "dk", "dv"), got, want, moved, (2 * u, 3 * u, 3 * u, 3 * u)):
        assert g.shape == w.shape and g.dtype == q.dtype
        _near(g, w, m, tol, n)
    return got


def _inputs(dev, B, Nq, Nk, H, KH, D, T, seed=0):
    g = torch.Generator(device=dev).manual_seed(1000 * seed + Nq + 7 * Nk + D)
    r = lambda *s: torch.randn(*s, generator=g, device=dev).to(T)  # noqa: E731
    return r(B, Nq, H, D), r(B, Nk, KH, D), r(B, Nk, KH, D), r(B, Nq, H, D)


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("Nq,Nk", [(1, 1), (1, 2), (1, 197), (2, 64), (15, 63), (16, 65), (17, 127), (33, 128), (64, 129),
                                   (65, 300), (127, 31), (128, 700), (129, 1), (200, 33), (300, 257)])
def test_lengths(dev, Nq, Nk, dtype):
    _check(*_inputs(dev, 2, Nq, Nk, 4, 4, 32, DTYPES[dtype]))


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("D", [1, 3, 8, 9, 16, 17, 24, 31, 32, 40, 63, 64, 65, 80, 100, 127, 128])
@pytest.mark.parametrize("Nq,Nk", [(3, 150), (70, 90), (150, 70)])
def test_head_dims(dev, D, Nq, Nk, dtype):
    _check(*_inputs(dev, 2, Nq, Nk, 2, 2, D, DTYPES[dtype]))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
@pytest.mark.parametrize("H,KH", [(1, 1), (3, 1), (6, 2), (12, 12), (16, 4), (64, 1)])
@pytest.mark.parametrize("Nq,Nk", [(1, 300), (5, 77), (90, 50)])
def test_shared_heads(dev, H, KH, Nq, Nk, dtype):
    _check(*_inputs(dev, 2, Nq, Nk, H, KH, 32, DTYPES[dtype]))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("Nq,Nk", [(1, 5000), (40, 3001), (2000, 20), (1500, 130)])
def test_split_axes(dev, Nq, Nk, dtype):
    """Few rows split the keys, few keys split the rows."""
    _check(*_inputs(dev, 1, Nq, Nk, 2, 2, 64, DTYPES[dtype]))


@pytest.mark.parametrize("dtype", ["f16", "bf16"])
def test_probabilities_below_the_types_normal_range(dev, dtype):
    """Among 20000 keys a probability is 5e-5, below float16's normal values."""
    _check(*_inputs(dev, 1, 70, 20000, 2, 2, 32, DTYPES[dtype]))


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("Nq,Nk", [(1, 700), (20, 200), (150, 130)])
@pytest.mark.parametrize("kind", ["lengths", "mask", "both"])
def test_unseen_keys(dev, Nq, Nk, kind, dtype):
    """Ragged lengths (0, 1, past the end, negative) and masks (none of a
    sample, one key, whole tiles), with NaN, infinities and the type's lowest
    value in the unseen places."""
    T = DTYPES[dtype]
    q, k, v, dout = _inputs(dev, 6, Nq, Nk, 4, 2, 32, T)
    lengths = mask = None
    if kind != "mask":
        lengths = torch.tensor([0, 1, Nk, Nk + 9, -3, Nk // 2 + 1], dtype=torch.int32, device=dev)
    if kind != "lengths":
        mask = torch.rand(6, Nk, device=dev, generator=torch.Generator(device=dev).manual_seed(5)) < 0.5
        mask[0], mask[1] = False, False
        mask[1, Nk - 1] = True
        mask[2, : Nk // 2 + 3] = False
    seen = torch.ones(6, Nk, dtype=torch.bool, device=dev) if mask is None else mask.clone()
    if lengths is not None:
        seen &= torch.arange(Nk, device=dev) < lengths[:, None]
    want = _check(q, k, v, dout, lengths, mask)
    for j, bad in enumerate((math.nan, math.inf, -math.inf, torch.finfo(T).min)):
        k2, v2 = (torch.where(seen[:, :, None, None], t, torch.full_like(t, bad)) for t in (k, v))
        got = _check(q, k2, v2, dout, lengths, mask)
        assert all(torch.equal(a, b) for a, b in zip(got, want)), bad
    none = ~seen.any(1)
    assert none.any() and not want[0][none].any() and not want[1][none].any()
    assert not want[2][~seen].any() and not want[3][~seen].any()


def test_lengths_in_64_bits(dev):
    import eccv26_tad_amd as sv

    q, k, v, _ = _inputs(dev, 3, 4, 50, 2, 2, 16, torch.float16)
    n = torch.tensor([10, 50, 1 << 40], device=dev)
    assert torch.equal(sv.cross_attention(q, k, v, key_lengths=n),
                       sv.cross_attention(q, k, v, key_lengths=torch.tensor([10, 50, 50], dtype=torch.int32, device=dev)))


@pytest.mark.parametrize("Nq,Nk", [(0, 5), (5, 0), (0, 0)])
def test_no_tokens(dev, Nq, Nk):
    out, dq, dk, dv = _check_empty(dev, Nq, Nk)
    assert out.shape == dq.shape == (2, Nq, 4, 32) and dk.shape == dv.shape == (2, Nk, 4, 32)
    assert not any(t.any() for t in (out, dq, dk, dv))


def _check_empty(dev, Nq, Nk):
    import eccv26_tad_amd as sv

    q, k, v, dout = _inputs(dev, 2, Nq, Nk, 4, 4, 32, torch.float16)
    ls = [t.requires_grad_(True) for t in (q, k, v)]
    out = sv.cross_attention(*ls)
    return (out.detach(), *torch.autograd.grad(out, ls, dout))


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("D", [32, 37])
def test_strides(dev, D, dtype):
    """Joint projections, head-major and token-major orders, a strided last
    axis, an unaligned start, one context shared by all samples."""
    T, B, Nq, Nk, H = DTYPES[dtype], 3, 70, 90, 4
    q, k, v, dout = _inputs(dev, B, Nq, Nk, H, H, D, T)
    kv = torch.stack([k, v], 2)
    want = _check(q, kv[:, :, 0], kv[:, :, 1], dout)
    head = lambda t: t.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3)  # noqa: E731
    token = lambda t: t.permute(1, 0, 2, 3).contiguous().permute(1, 0, 2, 3)  # noqa: E731
    last = lambda t: t.permute(3, 0, 1, 2).contiguous().permute(1, 2, 3, 0)  # noqa: E731

    def shifted(t):
        flat = torch.empty(t.numel() + 1, dtype=t.dtype, device=t.device)
        return flat[1:].view(t.shape).copy_(t)

    for lay in (head, token, last, shifted):
        got = _check(lay(q), lay(k), lay(v), lay(dout))
        assert all(torch.equal(a, b) for a, b in zip(got, want)), lay
    _check(q, k[:1].expand(B, Nk, H, D), v[:1].expand(B, Nk, H, D), dout)
    _check(q[:, :, :1].expand(B, Nq, H, D), k, v, dout[:1, :1, :1, :1].expand(B, Nq, H, D))


def test_gradients_of_a_shared_context(dev):
    """One context for all samples: its gradient is the sum over them."""
    import eccv26_tad_amd as sv

    q, k, v, dout = _inputs(dev, 4, 20, 90, 4, 2, 32, torch.float32)
    k1, v1 = (t[:1].clone().requires_grad_(True) for t in (k, v))
    gk, gv = torch.autograd.grad(sv.cross_attention(q, k1.expand_as(k), v1.expand_as(v)), (k1, v1), dout)
    want, _ = _exact(q, k1.detach().expand_as(k), v1.detach().expand_as(v), dout, None, None, 32 ** -0.5)
    assert float((gk.double() - want[2].sum(0, keepdim=True)).norm()) <= 4 * U[torch.float32] * float(want[2].norm())
    assert float((gv.double() - want[3].sum(0, keepdim=True)).norm()) <= 4 * U[torch.float32] * float(want[3].norm())


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
def test_steep_scores(dev, dtype):
    """Scores far apart (up to a few hundred): the running maximum moves, and
    no power overflows."""
    q, k, v, dout = _inputs(dev, 2, 40, 500, 2, 2, 32, DTYPES[dtype])
    k = (k.float() * torch.linspace(0.1, 8, 500, device=dev)[None, :, None, None]).to(k.dtype)
    import eccv26_tad_amd as sv

    out = sv.cross_attention(q, k, v, scale=2.0)
    want, _ = _exact(q, k, v, dout, None, None, 2.0)
    # the scores' own rounding in float32: |s| 2^-24 sqrt(D), |s| up to 400
    _near(out, want[0], None, 2 * U[q.dtype] + 1e-3, "out")


def test_scale(dev):
    _check(*_inputs(dev, 1, 30, 60, 2, 2, 32, torch.float32), scale=0.5)


def test_only_what_is_needed(dev):
    import eccv26_tad_amd as sv

    q, k, v, dout = _inputs(dev, 2, 50, 200, 4, 2, 32, torch.bfloat16)
    full = _check(q, k, v, dout)
    for i, name in enumerate(("q", "k", "v")):
        ls = [t.clone().requires_grad_(j == i) for j, t in enumerate((q, k, v))]
        (g,) = torch.autograd.grad(sv.cross_attention(*ls), ls[i], dout)
        assert torch.equal(g, full[1 + i]), name


def test_against_differences(dev):
    """The directional derivative of <dout, out> by central differences in
    float32: h = 1e-2 leaves a truncation error of order h^2 and a rounding
    error of order 1e-6 / h."""
    import eccv26_tad_amd as sv

    q, k, v, dout = _inputs(dev, 2, 20, 70, 4, 2, 24, torch.float32)
    n = torch.tensor([70, 33], dtype=torch.int32, device=dev)
    ls = [t.clone().requires_grad_(True) for t in (q, k, v)]
    grads = torch.autograd.grad(sv.cross_attention(*ls, key_lengths=n), ls, dout)
    f = lambda *a: (sv.cross_attention(*a, key_lengths=n).double() * dout.double()).sum()  # noqa: E731
    h = 1e-2
    for i, t in enumerate((q, k, v)):
        d = torch.randn(t.shape, device=dev, generator=torch.Generator(device=dev).manual_seed(11 + i))
        at = lambda s: f(*(p + s * d if p is t else p for p in (q, k, v)))  # noqa: E731
        numeric = float((at(h) - at(-h)) / (2 * h))
        analytic = float((grads[i].double() * d.double()).sum())
        assert abs(numeric - analytic) <= 1e-3 * float(grads[i].norm() * d.norm())


def test_repeats_and_other_streams(dev):
    import eccv26_tad_amd as sv

    q, k, v, dout = _inputs(dev, 2, 40, 3000, 4, 2, 32, torch.bfloat16)
    first = _check(q, k, v, dout)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        ls = [t.clone().requires_grad_(True) for t in (q, k, v)]
        out = sv.cross_attention(*ls)
        again = (out.detach(), *torch.autograd.grad(out, ls, dout))
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, again))


def test_long_cache(dev):
    """Keys and values whose bytes pass 2^32 in one sample."""
    import eccv26_tad_amd as sv

    Nk, KH, D = (1 << 24) + 5000, 2, 64
    g = torch.Generator(device=dev).manual_seed(1)
    q = torch.randn(1, 1, 4, D, generator=g, device=dev).half()
    k = torch.zeros(1, Nk, KH, D, dtype=torch.float16, device=dev)
    v = torch.zeros(1, Nk, KH, D, dtype=torch.float16, device=dev)
    tail = 300  # the last keys alone have scores above 0, far above
    k[:, -tail:] = q[:, :, ::2] * 4 + torch.randn(1, tail, KH, D, generator=g, device=dev).half()
    v[:, -tail:] = torch.randn(1, tail, KH, D, generator=g, device=dev).half()
    out = sv.cross_attention(q, k, v, scale=1.0)
    want, _ = _exact(q, k[:, -tail:], v[:, -tail:], q, None, None, 1.0)
    _near(out[:, :, ::2], want[0][:, :, ::2], None, 2 * U[torch.float16] + 1e-3, "out")


def test_refusals(dev):
    import eccv26_tad_amd as sv

    q, k, v, _ = _inputs(dev, 2, 4, 6, 4, 2, 32, torch.float16)
    no = lambda match, *a, **kw: pytest.raises((RuntimeError, ValueError), match=match)  # noqa: E731
    with no("GPU tensor"):
        sv.cross_attention(q.cpu(), k, v)
    with no("one dtype"):
        sv.cross_attention(q, k.float(), v)
    with no("float32, float16 or bfloat16"):
        sv.cross_attention(q.double(), k.double(), v.double())
    with no("one shape"):
        sv.cross_attention(q, k, v[:, :5])
    with no("one batch"):
        sv.cross_attention(q[:1], k, v)
    with no("multiple of the key heads"):
        sv.cross_attention(q[:, :, :3], k, v)
    with no("tokens, heads"):
        sv.cross_attention(q[0], k[0], v[0])
    big = torch.zeros(1, 2, 1, 129, device=dev)
    with no("1 to 128"):
        sv.cross_attention(big, big, big)
    for bad in (0.0, -1.0, math.inf, math.nan):
        with no("scale"):
            sv.cross_attention(q, k, v, scale=bad)
    with no("key_lengths"):
        sv.cross_attention(q, k, v, key_lengths=torch.ones(3, dtype=torch.int32, device=dev))
    with no("key_lengths"):
        sv.cross_attention(q, k, v, key_lengths=torch.ones(2, dtype=torch.int32))
    with no("key_mask"):
        sv.cross_attention(q, k, v, key_mask=torch.ones(2, 5, dtype=torch.bool, device=dev))
    with no("key_mask"):
        sv.cross_attention(q, k, v, key_mask=torch.ones(2, 6, device=dev))


def _check_gradients(dev, q, k, v, dout, rows=False):
    """Gradients in float16 against float64. Beside the relative roundings of
    `_check` stands the result's own below the type's normal range: half of
    2^-24, its spacing there. With `rows` every query's dq is held to its own
    size."""
    import eccv26_tad_amd as sv

    ls = [t.detach().requires_grad_(True) for t in (q, k, v)]
    got = torch.autograd.grad(sv.cross_attention(*ls), ls, dout)
    want, moved = _exact(q, k, v, dout, None, None, q.shape[-1] ** -0.5)
    u = U[q.dtype]
    for name, g, w, m in zip(("dq", "dk", "dv"), got, want[1:], moved[1:]):
        assert float(w.abs().max()) < 6e4 and g.isfinite().all(), name
        dims = (2, 3) if rows and name == "dq" else (0, 1, 2, 3)
        size = lambda t: torch.linalg.vector_norm(t, dim=dims)  # noqa: E731
        count = w[0, 0].numel() if rows and name == "dq" else w.numel()
        allow = 3 * u * (size(w) + (0 if m is None else size(m))) + 2.0 ** -25 * math.sqrt(count)
        off = size(g.double() - w)
        assert bool((off <= allow).all()), (name, float((off / allow).max()))


@pytest.mark.parametrize("gain", [1.0, 1e-2, 1e-3])
@pytest.mark.parametrize("Nq,Nk", [(70, 20000), (2000, 8192), (1, 31361), (3000, 100)])
def test_small_float16_gradients(dev, Nq, Nk, gain):
    """A score gradient among n keys is near 1 / n of dout, below float16's normal
    values where dout is not."""
    q, k, v, dout = _inputs(dev, 1, Nq, Nk, 2, 2, 32, torch.float32, seed=1)
    _check_gradients(dev, q.half(), k.half(), v.half(), (gain * dout).half())


@pytest.mark.parametrize("Nq,Nk", [(5, 3), (40, 150)])
def test_large_float16_gradients(dev, Nq, Nk):
    """Score gradients past float16's largest value, whose sums are within it."""
    q, k, v, dout = _inputs(dev, 1, Nq, Nk, 2, 2, 128, torch.float32, seed=1)
    # few keys, or scores so steep that few keys count: probabilities of order 1
    q = q * (1 if Nk < 10 else 3)
    _check_gradients(dev, q.half(), k.half(), (10 * v).half(), (1600 * dout / math.sqrt(Nq / 5)).half())


def test_float16_gradients_of_many_sizes(dev):
    """Queries whose gradients lie 4^9 apart, side by side in a tile, some zero;
    and keys that are seen by large ones first or last."""
    q, k, v, dout = _inputs(dev, 1, 300, 700, 2, 2, 32, torch.float32, seed=2)
    size = 4.0 ** -(torch.arange(300, device=dev) % 10)
    size[::17] = 0
    for order in (size, size.sort().values, size.sort(descending=True).values):
        _check_gradients(dev, q.half(), k.half(), v.half(), (100 * dout * order[None, :, None, None]).half(), rows=True)


@pytest.mark.parametrize("dtype", ["bf16", "f32"])
@pytest.mark.parametrize("masked", [False, True])
@pytest.mark.parametrize("Nq,Nk", [(1, 9), (3, 20000), (20, 200), (70, 300)])
def test_nan_of_a_query_or_a_seen_key_is_kept(dev, Nq, Nk, masked, dtype):
    """It reaches the results of its query, or of its sample and key head, and no others."""
    import eccv26_tad_amd as sv

    q, k, v, _ = _inputs(dev, 2, Nq, Nk, 4, 2, 32, DTYPES[dtype])
    mask = None
    if masked:
        mask = torch.zeros(2, Nk, dtype=torch.bool, device=dev)
        mask[:, Nk - 2 :] = True
    want = sv.cross_attention(q, k, v, key_mask=mask)
    bad = q.clone()
    bad[0, Nq - 1, 1] = math.nan
    got = sv.cross_attention(bad, k, v, key_mask=mask)
    hit = torch.zeros_like(q, dtype=torch.bool)
    hit[0, Nq - 1, 1] = True
    assert bool(got[hit].isnan().all()) and torch.equal(got[~hit], want[~hit])
    bad = k.clone()
    bad[1, Nk - 2, 0, 3] = math.nan
    if masked:
        mask[:, Nk - 1] = False  # one key alone is seen
        want = sv.cross_attention(q, k, v, key_mask=mask)
    got = sv.cross_attention(q, bad, v, key_mask=mask)
    hit = torch.zeros_like(q, dtype=torch.bool)
    hit[1, :, :2] = True
    assert bool(got[hit].isnan().all()) and torch.equal(got[~hit], want[~hit])


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("Nq,Nk", [(1, 700), (20, 200), (150, 130), (3, 20000), (2000, 90)])
@pytest.mark.parametrize("kind", ["lengths", "mask", "both"])
def test_queries_without_keys_may_hold_anything(dev, Nq, Nk, kind, dtype):
    """Queries and upstream gradients of a sample whose keys are all hidden, by a
    length or by the mask: zeros, whatever they hold, and the other samples' bits
    stay."""
    T = DTYPES[dtype]
    q, k, v, dout = _inputs(dev, 3, Nq, Nk, 4, 2, 32, T)
    lengths = torch.tensor([Nk, 0, Nk - 1], dtype=torch.int32, device=dev) if kind == "lengths" else None
    mask = None
    if kind != "lengths":
        mask = torch.rand(3, Nk, device=dev, generator=torch.Generator(device=dev).manual_seed(6)) < 0.5
        mask[:, 0] = True
        mask[1] = False
        if kind == "both":  # only the keys past the length are seen
            lengths = torch.tensor([Nk, Nk // 2, Nk - 1], dtype=torch.int32, device=dev)
            mask[1, Nk // 2 :] = True
    want = _check(q, k, v, dout, lengths, mask)
    for bad_q, bad_g in ((math.nan, 1.0), (math.inf, 1.0), (1.0, math.nan), (1.0, -math.inf), (-math.inf, math.inf)):
        import eccv26_tad_amd as sv

        q2, g2 = q.clone(), dout.clone()
        q2[1], g2[1] = q2[1] * bad_q, g2[1] * bad_g
        ls = [t.detach().requires_grad_(True) for t in (q2, k, v)]
        out = sv.cross_attention(*ls, key_lengths=lengths, key_mask=mask)
        got = (out.detach(), *torch.autograd.grad(out, ls, g2))
        for name, a, b in zip(("out", "dq", "dk", "dv"), got, want):
            assert not a[1].any() and torch.equal(a, b), (name, bad_q, bad_g)


def test_stride_of_an_axis_of_one(dev):
    """What stride an axis with one place has is no matter."""
    import eccv26_tad_amd as sv

    q, k, v, _ = _inputs(dev, 1, 1, 1, 1, 1, 32, torch.float16)
    far = lambda t: t.as_strided(t.shape, (1 << 40, 1 << 40, 1 << 40, 1))  # noqa: E731
    assert torch.equal(sv.cross_attention(far(q), far(k), far(v)), sv.cross_attention(q, k, v))
    q, k, v, dout = _inputs(dev, 1, 1, 90, 4, 2, 32, torch.bfloat16)
    one = q.as_strided(q.shape, (0, 1 << 30, 32, 1))
    want = _check(q, k, v, dout)
    assert all(torch.equal(a, b) for a, b in zip(_check(one, k, v, dout.as_strided(q.shape, (0, 1 << 30, 32, 1))), want))


@pytest.mark.parametrize("dtype", ["f16", "f32"])
def test_masks_of_any_strides(dev, dtype):
    """One mask for all samples, every other place of a wider one, and the
    transpose of [keys, samples]."""
    q, k, v, dout = _inputs(dev, 3, 20, 150, 2, 2, 32, DTYPES[dtype])
    wide = torch.rand(3, 300, device=dev, generator=torch.Generator(device=dev).manual_seed(3)) < 0.6
    turned = wide[:, :150].t().contiguous().t()
    for mask in (wide[:1, :150].expand(3, 150), wide[:, ::2], turned, wide[:, :1].expand(3, 150)):
        got, want = (_check(q, k, v, dout, None, m) for m in (mask, mask.contiguous()))
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.parametrize("dtype", ["f16", "bf16", "f32"])
@pytest.mark.parametrize("Nq,Nk", [(1, 5000), (20, 5000), (200, 5000)])
def test_probabilities_far_below_the_largest(dev, Nq, Nk, dtype):
    """One key in 64 takes nearly all of the weight and has no value, as the first
    token of a sequence often does: the result is the others', which at 7e-7 of the
    largest are below float16's normal values, all alike. Their rounding has the
    sums' full relative size: 2 u as elsewhere."""
    import eccv26_tad_amd as sv

    T = DTYPES[dtype]
    q = torch.zeros(2, Nq, 2, 32, device=dev)
    q[..., 0] = 1
    k = torch.zeros(2, Nk, 2, 32, device=dev)
    k[..., 0] = -14.1953125  # exp of it is 11.48 2^-24; exact in all types
    v = 100 * torch.rand(2, Nk, 2, 32, device=dev, generator=torch.Generator(device=dev).manual_seed(4))
    if T is torch.bfloat16:
        k[..., 0] = -14.1875
    k[:, ::64], v[:, ::64] = 0, 0
    q, k, v = q.to(T), k.to(T), v.to(T)
    want, _ = _exact(q, k, v, q, None, None, 1.0)
    _near(sv.cross_attention(q, k, v, scale=1.0), want[0], None, 2 * U[T], "out")
