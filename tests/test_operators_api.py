"""CPU checks of the transformer operators: the C ABI rejects bad arguments on
the host, before any launch, and the Python functions refuse CPU tensors."""
import ctypes
import os

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
LIB = os.path.join(ROOT, "eccv26_tad_amd", "libsvtad_sparse.so")

I64, P, I, F = ctypes.c_int64, ctypes.c_void_p, ctypes.c_int, ctypes.c_float
OK, INVALID, WORKSPACE, UNSUPPORTED = 0, -1, -2, -3
F32, F16, F64 = 0, 1, 3


class NormArgs(ctypes.Structure):
    _fields_ = [("x", P), ("w", P), ("b", P), ("stats", P), ("d0", I64), ("d1", I64), ("d2", I64), ("s0", I64), ("s1", I64),
                ("s2", I64), ("t0", I64), ("t1", I64), ("t2", I64), ("c", I), ("params_f32", I), ("eps", F)]


class CrossArgs(ctypes.Structure):
    _fields_ = [("q", P), ("k", P), ("v", P), ("lengths", P), ("mask", P), ("q_stride", I64 * 3), ("k_stride", I64 * 3),
                ("v_stride", I64 * 3), ("mask_stride", I64 * 2), ("batch", I64), ("nq", I64), ("nk", I64), ("heads", I),
                ("kv_heads", I), ("head_dim", I), ("scale", F)]


class Grad(ctypes.Structure):
    _fields_ = [("g", P), ("out", P), ("count", I64), ("g_type", I), ("out_type", I)]


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(LIB):
        pytest.fail("libsvtad_sparse.so not built (run python eccv26_tad_amd/build.py)")
    L = ctypes.CDLL(LIB)
    L.svtad_last_error.restype = ctypes.c_char_p
    for n in ("svtad_norm_bwd_workspace_bytes", "svtad_cross_attention_workspace_bytes",
              "svtad_cross_attention_bwd_workspace_bytes", "svtad_grad_clip_workspace_bytes"):
        getattr(L, n).restype = ctypes.c_size_t
    return L


def _norm(**kw):
    a = NormArgs(d0=4, d1=1, d2=1, s0=64, t0=64, c=64, eps=1e-5)
    for k, v in kw.items():
        setattr(a, k, v)
    return ctypes.byref(a)


def test_norm(lib):
    call = lambda dt=F32, y=None, **kw: lib.svtad_norm(_norm(**kw), y, dt, None)  # noqa: E731
    assert call(dt=F64) == INVALID and b"dtype" in lib.svtad_last_error()
    assert call(c=0) == UNSUPPORTED and call(c=8193) == UNSUPPORTED and b"8192" in lib.svtad_last_error()
    assert call(d0=-1) == INVALID and call() == INVALID and b"NULL" in lib.svtad_last_error()
    assert call(d0=1 << 20, d1=1 << 10, d2=1 << 10) == UNSUPPORTED
    assert call(d0=0) == OK
    assert lib.svtad_norm(None, None, F32, None) == INVALID
    bwd = lambda size=0, ws=None, **kw: lib.svtad_norm_bwd(  # noqa: E731
        _norm(x=16, stats=16, **kw), P(16), None, P(16), None, ws, ctypes.c_size_t(size), F32, None)
    assert bwd() == WORKSPACE and bwd(size=8, ws=P(16)) == WORKSPACE
    assert lib.svtad_norm_bwd(_norm(), None, None, None, None, None, ctypes.c_size_t(0), F32, None) == INVALID
    assert lib.svtad_norm_bwd_workspace_bytes(I64(1 << 20), 1024, F16) == 512 * 2 * 1024 * 4
    assert lib.svtad_norm_bwd_workspace_bytes(I64(3), 64, F32) == 2 * 64 * 4
    assert lib.svtad_norm_bwd_workspace_bytes(I64(0), 64, F32) == 0


def _cross(**kw):
    a = CrossArgs(batch=2, nq=10, nk=20, heads=4, kv_heads=2, head_dim=32, scale=0.1)
    a.q_stride[:] = [10 * 128, 128, 32]
    a.k_stride[:] = a.v_stride[:] = [20 * 64, 64, 32]
    for k, v in kw.items():
        if k.endswith("stride"):
            getattr(a, k)[:] = v
        else:
            setattr(a, k, v)
    return ctypes.byref(a)


def test_cross_attention(lib):
    Z = ctypes.c_size_t(0)
    call = lambda dt=F16, **kw: lib.svtad_cross_attention(_cross(**kw), None, None, None, None, Z, dt, None)  # noqa: E731
    assert call(dt=F64) == INVALID and b"dtype" in lib.svtad_last_error()
    assert call(heads=3) == INVALID and b"multiple" in lib.svtad_last_error()
    assert call(kv_heads=0) == INVALID and call(nq=-1) == INVALID
    assert call(head_dim=129) == UNSUPPORTED and call(head_dim=0) == UNSUPPORTED
    for bad in (0.0, -1.0, float("nan"), float("inf")):
        assert call(scale=bad) == INVALID and b"scale" in lib.svtad_last_error()
    assert call(k_stride=[0, 1 << 24, 32]) == UNSUPPORTED and b"2 GiB" in lib.svtad_last_error()
    assert call(q_stride=[0, -128, 32]) == UNSUPPORTED
    assert call(batch=1 << 30) == UNSUPPORTED and b"too many" in lib.svtad_last_error()
    assert call() == INVALID and b"NULL" in lib.svtad_last_error()
    assert call(nq=0) == OK and call(batch=0) == OK
    assert lib.svtad_cross_attention(None, None, None, None, None, Z, F16, None) == INVALID
    few = _cross(q=16, k=16, v=16, nq=1, nk=8192)
    need = lib.svtad_cross_attention_workspace_bytes(few, F16)
    assert need > 0
    assert lib.svtad_cross_attention(few, P(16), None, None, P(16), ctypes.c_size_t(need - 1), F16, None) == WORKSPACE
    bwd = lambda dk=None, dv=None, **kw: lib.svtad_cross_attention_bwd(  # noqa: E731
        _cross(**kw), None, None, None, None, None, None, dk, dv, None, Z, F16, None)
    assert bwd(dk=P(16)) == INVALID and b"together" in lib.svtad_last_error()
    assert bwd() == OK and bwd(dk=P(16), dv=P(16)) == INVALID


def test_grad_clip(lib):
    norm = (ctypes.c_float * 1)()

    def call(tensors, kind=0, write=1, out=norm, ws=None, size=0):
        arr = (Grad * len(tensors))(*tensors)
        return lib.svtad_grad_clip(arr, I64(len(tensors)), kind, F(1.0), F(1.0), write, out, ws, ctypes.c_size_t(size), None)

    one = Grad(16, 16, 10, F32, F32)
    assert call([Grad(16, 16, 10, F64, F32)]) == INVALID and call([Grad(16, 16, 10, F32, 7)]) == INVALID
    assert call([Grad(16, 16, -1, F32, F32)]) == INVALID and call([Grad(None, 16, 1, F32, F32)]) == INVALID
    assert call([Grad(16, None, 1, F32, F32)]) == INVALID
    assert call([one], kind=2) == INVALID and b"norm_type" in lib.svtad_last_error()
    assert call([one], out=None) == INVALID and call([one]) == WORKSPACE
    assert lib.svtad_grad_clip(None, I64(1), 0, F(1.0), F(1.0), 1, norm, None, ctypes.c_size_t(0), None) == INVALID
    arr = (Grad * 300)(*[Grad(16, 16, 1000, F32, F32)] * 300)
    assert lib.svtad_grad_clip_workspace_bytes(arr, I64(300)) % 8 == 0
    assert 0 < lib.svtad_grad_clip_workspace_bytes(arr, I64(300)) <= 2 * 1024 * 8
    assert lib.svtad_grad_clip_workspace_bytes((Grad * 1)(Grad(None, None, 0, F32, F32)), I64(1)) == 0


def test_python_functions_off_the_gpu():
    import torch

    import eccv26_tad_amd as sv

    x = torch.randn(2, 3, 2, 16)
    for call in (lambda: sv.layer_norm(x), lambda: sv.cross_attention(x, x, x), lambda: sv.clip_grads([x], 1.0),
                 lambda: sv.grad_norm([x])):
        with pytest.raises(RuntimeError, match="GPU tensor"):
            call()
    with pytest.raises(ValueError, match="max_norm"):
        sv.clip_grads([x], -1.0)
    with pytest.raises(ValueError, match="norm_type"):
        sv.clip_grads([x], 1.0, norm_type=3)
    with pytest.raises(RuntimeError, match="no tensors"):
        sv.grad_norm([])
    p = torch.nn.Parameter(x)
    assert float(sv.clip_grad_norm_([p], 1.0)) == 0.0
    for bad in (dict(embed_dims=100, num_heads=3), dict(embed_dims=96, num_heads=4, kv_heads=3),
                dict(embed_dims=1024, num_heads=4)):
        with pytest.raises(ValueError):
            sv.CrossAttention(**bad)


def test_module_parameters():
    import eccv26_tad_amd as sv

    m = sv.CrossAttention(96, 6, context_dims=40, kv_heads=2)
    shapes = {n: tuple(p.shape) for n, p in m.named_parameters()}
    assert shapes == {
        "norm.weight": (96,), "norm.bias": (96,), "context_norm.weight": (40,), "context_norm.bias": (40,),
        "q_norm.weight": (16,), "q_norm.bias": (16,), "k_norm.weight": (16,), "k_norm.bias": (16,),
        "q.weight": (96, 96), "q.bias": (96,), "kv.weight": (64, 40), "kv.bias": (64,), "proj.weight": (96, 96),
        "proj.bias": (96,)}


def test_cross_attention_bwd_without_queries(lib):
    """dk and dv of no queries are zeros, which the kernel that holds k and v
    writes: both have to be there, as with queries."""
    Z = ctypes.c_size_t(0)
    bwd = lambda **kw: lib.svtad_cross_attention_bwd(  # noqa: E731
        _cross(nq=0, **kw), None, None, None, None, None, None, P(16), P(16), None, Z, F16, None)
    for given in (dict(), dict(k=16), dict(v=16)):
        assert bwd(**given) == INVALID and b"NULL" in lib.svtad_last_error()
    assert bwd(batch=0) == OK


def test_grad_clip_shared_memory(lib):
    """An output that shares memory with another tensor is refused; gradients in
    place may share it with one another."""

    def call(*tensors, write=1):
        arr, norm = (Grad * len(tensors))(*tensors), (ctypes.c_float * 1)()
        return lib.svtad_grad_clip(arr, I64(len(tensors)), 0, F(1.0), F(1.0), write, norm, None, ctypes.c_size_t(0), None)

    A, B, C = 4096, 8192, 16384  # 1000 float32 elements from each on do not meet
    at = lambda g, out=None, n=1000, to=F32: Grad(g, g if out is None else out, n, F32, to)  # noqa: E731
    for good in ((at(A), at(A)), (at(B), at(A, n=1025), at(C)), (at(A, C), at(A, B)), (at(B, C), at(A)),
                 (at(A, C), at(B, C + 4000))):
        assert call(*good) == WORKSPACE
    for bad in ((at(A, C), at(B, C)), (at(A, B), at(B, C)), (at(B, C), at(A, B)), (at(A), at(A, C)), (at(A, C), at(C)),
                (at(A, A + 4),), (at(A, B), at(C, B + 3996)), (at(A, A, to=F16),)):
        assert call(*bad) == INVALID and b"shares memory" in lib.svtad_last_error()
        assert call(*bad, write=0) == WORKSPACE


def test_cross_attention_stride_of_an_axis_of_one(lib):
    Z = ctypes.c_size_t(0)
    call = lambda **kw: lib.svtad_cross_attention(_cross(**kw), None, None, None, None, Z, F16, None)  # noqa: E731
    far = 1 << 40
    for given in (dict(nq=1, q_stride=[128, far, 32]), dict(nq=1, q_stride=[128, -far, 32]),
                  dict(nk=1, k_stride=[64, far, 32], v_stride=[64, far, 32]),
                  dict(heads=1, kv_heads=1, q_stride=[320, 32, far], k_stride=[640, 32, far], v_stride=[640, 32, -far])):
        assert call(**given) == INVALID and b"NULL" in lib.svtad_last_error()
    assert call(nq=2, q_stride=[128, far, 32]) == UNSUPPORTED


def test_cross_attention_grids_within_the_runtimes(lib):
    """2^24 workgroups of 256 threads are 2^32 threads, of which the runtime would
    start none: a call that needs so many is refused."""
    Z = ctypes.c_size_t(0)
    call = lambda **kw: lib.svtad_cross_attention(_cross(**kw), None, None, None, None, Z, F16, None)  # noqa: E731
    bwd = lambda **kw: lib.svtad_cross_attention_bwd(  # noqa: E731
        _cross(**kw), None, None, None, None, None, None, P(16), P(16), None, Z, F16, None)
    one = dict(heads=1, kv_heads=1, head_dim=8, q_stride=[8, 8, 8], k_stride=[8, 8, 8], v_stride=[8, 8, 8])
    for sizes in (dict(batch=1 << 24, nq=1, nk=1), dict(batch=1 << 24, nq=16, nk=1), dict(batch=1 << 23, nq=129, nk=1),
                  dict(batch=1 << 22, nq=400, nk=10)):
        assert call(**one, **sizes) == UNSUPPORTED and b"too many" in lib.svtad_last_error()
        assert bwd(**one, **sizes) == UNSUPPORTED
    for sizes in (dict(batch=(1 << 24) - 1, nq=16, nk=1), dict(batch=(1 << 23) - 1, nq=17, nk=1)):
        assert call(**one, **sizes) == INVALID and b"NULL" in lib.svtad_last_error()
        assert bwd(**one, **sizes) == INVALID
    keys = dict(batch=1 << 23, nq=1, nk=129)  # the keys' kernel alone
    assert call(**one, **keys) == INVALID and bwd(**one, **keys) == UNSUPPORTED
