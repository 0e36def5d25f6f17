"""Host side of the training-step operators (rms_norm, grad_norm / clip_grad_norm_, GraphAdam(max_norm)): what they refuse, and
the argument checks of their C entry points.  Nothing is launched."""
import contextlib
import ctypes as C

import numpy as np
import pytest
import torch

from ggsplat import _lib
from ggsplat import adam as A
from ggsplat import stylenet as SN


def _rc(fn, *args):
    rc = fn(*args)
    return rc, _lib.lib().ggs_last_error().decode()


def test_rms_norm_refusals():
    x = torch.zeros(2, 4, 3)
    for bad, exc in [(dict(x=torch.zeros(4)), ValueError), (dict(x=torch.zeros(2, 0, 3)), ValueError),
                     (dict(x=torch.zeros(2, 4, 3, dtype=torch.int32)), TypeError),
                     (dict(residual=torch.zeros(2, 4, 4)), ValueError), (dict(residual=torch.zeros(2, 4, 3).half()), ValueError),
                     (dict(weight=torch.zeros(3)), ValueError), (dict(weight=torch.zeros(4).half()), ValueError),
                     (dict(weight=torch.zeros(4, 1)), ValueError), (dict(eps=0.0), ValueError), (dict(eps=-1.0), ValueError),
                     (dict(eps=float("nan")), ValueError), (dict(eps=float("inf")), ValueError)]:
        with pytest.raises(exc, match="rms_norm"):
            SN.rms_norm(**{"x": x, **bad})
    with pytest.raises(RuntimeError, match="CUDA"):
        SN.rms_norm(x)
    with pytest.raises(ValueError, match="norm"):
        SN.StyleUNetLite(size=32, channels={k: 4 for k in SN.CHANNELS}, norm="batch")


def test_rms_norm_native_is_the_formula():
    x = torch.tensor([[3.0, 4.0], [0.0, 0.0]], dtype=torch.float64)
    r = torch.tensor([[0.0, 0.0], [1.0, -1.0]], dtype=torch.float64)
    y, h = SN.rms_norm(x, torch.tensor([1.0, 2.0]), residual=r, eps=1e-300, impl="native")
    s = 12.5 ** 0.5
    assert torch.equal(h, x + r) and torch.allclose(y, torch.tensor([[3 / s, 8 / s], [1.0, -2.0]], dtype=torch.float64))
    assert torch.equal(SN.rms_norm(torch.zeros(1, 5), impl="native"), torch.zeros(1, 5))


@pytest.fixture
def norm_on_the_host(monkeypatch):
    """rms_norm's C call computed on the host (float, channels-first), for what happens around it."""
    class Lib:
        @staticmethod
        def ggs_rms_norm_forward(code, outer, c, inner, x, r, w, w32, eps, y, h, q, stream):
            view = lambda at, *n: None if at is None else np.ctypeslib.as_array((C.c_float * int(np.prod(n))).from_address(at)).reshape(n)    # noqa: E731
            assert code == 0 and all(type(n) is int for n in (outer, c, inner))
            s = view(x, outer, c, inner) + (0 if r is None else view(r, outer, c, inner))
            inv = 1 / np.sqrt((s * s).mean(1, keepdims=True) + eps)
            view(y, outer, c, inner)[:] = s * inv * (1 if w is None else view(w, c, 1))
            if h is not None:
                view(h, outer, c, inner)[:] = s
            if q is not None:
                view(q, outer, 1, inner)[:] = inv
            return 0
    monkeypatch.setattr(SN, "lib", lambda: Lib)
    monkeypatch.setattr(SN, "on_device", lambda dev: contextlib.nullcontext())
    monkeypatch.setattr(SN, "stream_ptr", lambda dev: None)
    monkeypatch.setattr(torch.Tensor, "is_cuda", property(lambda t: True))


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_rms_norm_in_a_trace_is_a_call(norm_on_the_host):
    x, r, w = torch.randn(3, 5, 2), torch.randn(3, 5, 2), torch.rand(5)
    with torch.no_grad():
        one = torch.jit.trace(lambda t: SN.rms_norm(t) + 1, (x,))                # (traced twice and compared)
    two = torch.jit.trace(lambda a, b, c: SN.rms_norm(a, c, residual=b), (x, r, w))
    for shape in ((3, 5, 2), (0, 5, 2), (1, 5, 7), (4, 9, 1)):                   # other sizes than the traced ones
        x, r, w = torch.randn(shape), torch.randn(shape), torch.rand(shape[1])
        assert torch.allclose(one(x), SN.rms_norm(x, impl="native") + 1, rtol=1e-5, atol=1e-6)
        for a, b in zip(two(x, r, w), SN.rms_norm(x, w, residual=r, impl="native")):
            assert torch.allclose(a, b, rtol=1e-5, atol=1e-6)
    t = torch.randn(2, 4, 3).transpose(0, 1)
    assert torch.allclose(one(t), SN.rms_norm(t, impl="native") + 1, rtol=1e-5, atol=1e-6)
    for bad in ((x, r[:1], w), (x, r, w[:2]), (x, r.double(), w), (x[0, 0], r[0, 0], w)):      # checked in every run
        with pytest.raises(Exception, match="rms_norm"):
            two(*bad)


def test_rms_norm_refuses_forward_mode(norm_on_the_host):
    from torch.autograd import forward_ad as fw
    x, t = torch.randn(3, 5), torch.randn(3, 5)
    with fw.dual_level():
        for args in ((fw.make_dual(x, t),), (x, fw.make_dual(t[0], t[0])), (x, None, fw.make_dual(x, t))):
            with torch.no_grad(), pytest.raises(NotImplementedError):
                SN.rms_norm(*args)
        assert torch.allclose(SN.rms_norm(x), SN.rms_norm(x, impl="native"), rtol=1e-5, atol=1e-6)      # no tangent: as ever
        assert fw.unpack_dual(SN.rms_norm(fw.make_dual(x, t), impl="native")).tangent is not None


def test_norm_of_the_network_adds_only_its_gains():
    ch = {k: 4 for k in SN.CHANNELS}
    a, b = (SN.StyleUNetLite(size=32, style_dim=8, out_ch=3, channels=ch, norm=n, impl="native") for n in (None, "rms"))
    extra = set(b.state_dict()) - set(a.state_dict())
    assert extra == {"gains.0"} and set(a.state_dict()) < set(b.state_dict())


def test_gradient_list_refusals():
    for fn in (A.grad_norm, lambda g: A.clip_grad_norm_(g, 1.0)):
        with pytest.raises(RuntimeError, match="GPU only"):
            fn([torch.zeros(3)])
        with pytest.raises(TypeError, match="tensors"):
            fn([3.0])
        assert float(fn([])) == 0.0 and float(fn([None])) == 0.0
    for bad in (-1.0, float("nan"), -float("inf")):
        with pytest.raises(ValueError, match="max_norm"):
            A.clip_grad_norm_([], bad)
    assert float(A.clip_grad_norm_([], float("inf"))) == 0.0


def test_norm_of_nothing_is_float32():
    keep = torch.get_default_dtype()
    try:
        torch.set_default_dtype(torch.float64)
        for n in (A.grad_norm([]), A.clip_grad_norm_([None], 1.0)):
            assert n.dtype is torch.float32 and n.shape == () and float(n) == 0.0
    finally:
        torch.set_default_dtype(keep)


def test_gradient_norms_are_not_traced():
    for fn in (A.grad_norm, lambda g: A.clip_grad_norm_(g, 1.0)):
        with pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(lambda g: fn([]) + g, (torch.zeros(3),), check_trace=False)


def test_span_of_layouts():
    t = torch.zeros(4, 6, 5)
    assert A._span(t) == (120, True, False) and A._span(t.permute(2, 0, 1)) == (120, True, False)
    assert A._span(t[:, ::2]) == (3 * 30 + 2 * 10 + 4 + 1, False, False)
    assert A._span(torch.zeros(1).expand(7))[2] and A._span(torch.zeros(8).as_strided((3, 3), (2, 1)))[2]
    assert A._span(torch.zeros(3, 1, 2).to(memory_format=torch.contiguous_format)) == (6, True, False)
    assert A._span(torch.zeros(5)[2:3]) == (1, True, False)


def test_c_entry_points_check_before_any_launch():
    L = _lib.lib()
    one = C.c_void_p(256)                                          # never dereferenced
    sizes, ptrs = (C.c_size_t * 1)(4), (C.c_void_p * 1)(256)
    odd, null = (C.c_void_p * 1)(258), (C.c_void_p * 1)(None)
    bad_type, f32 = (C.c_int * 1)(2), (C.c_int * 1)(0)
    assert L.ggs_grad_norm_workspace_bytes(0) == 0 and L.ggs_grad_norm_workspace_bytes(128) * 2 == L.ggs_grad_norm_workspace_bytes(129)
    assert _rc(L.ggs_grad_norm, -1, sizes, ptrs, f32, one, one, 1 << 20, None)[0] == -1
    assert _rc(L.ggs_grad_norm, 1, None, ptrs, f32, one, one, 1 << 20, None)[0] == -1
    assert "dtype" in _rc(L.ggs_grad_norm, 1, sizes, ptrs, bad_type, one, one, 1 << 20, None)[1]
    assert "NULL tensor" in _rc(L.ggs_grad_norm, 1, sizes, null, f32, one, one, 1 << 20, None)[1]
    assert "aligned" in _rc(L.ggs_grad_norm, 1, sizes, odd, f32, one, one, 1 << 20, None)[1]
    assert "NULL norm" in _rc(L.ggs_grad_norm, 1, sizes, ptrs, f32, None, one, 1 << 20, None)[1]
    rc, msg = _rc(L.ggs_grad_norm, 1, sizes, ptrs, f32, one, one, 0, None)
    assert rc == -3 and "workspace" in msg
    assert "workspace" in _rc(L.ggs_grad_norm, 1, sizes, ptrs, f32, one, None, 1 << 20, None)[1]
    huge = (C.c_size_t * 1)(1 << 41)
    assert _rc(L.ggs_grad_norm, 1, huge, ptrs, f32, one, one, 1 << 20, None)[0] == -3
    for m in (-1.0, float("nan")):
        assert "max_norm" in _rc(L.ggs_grad_clip, 1, sizes, ptrs, f32, m, one, one, 1 << 20, None)[1]
        assert "max_norm" in _rc(L.ggs_adam_clip_step, 1, sizes, *[ptrs] * 6, 0.9, 0.999, 1e-15, m, 1, None, one, one, 1 << 20, None)[1]
    assert "aligned" in _rc(L.ggs_adam_clip_step, 1, sizes, (C.c_void_p * 1)(260), *[ptrs] * 5, 0.9, 0.999, 1e-15, 1.0, 1, None, one, one, 1 << 20, None)[1]
    assert "NULL" in _rc(L.ggs_adam_clip_step, 1, sizes, *[ptrs] * 5, None, 0.9, 0.999, 1e-15, 1.0, 1, None, one, one, 1 << 20, None)[1]

    fwd = lambda *a: _rc(L.ggs_rms_norm_forward, *a)               # noqa: E731
    assert "dtype" in fwd(7, 1, 4, 1, one, None, None, 0, 1e-8, one, None, None, None)[1]
    assert "channels" in fwd(0, 1, 0, 1, one, None, None, 0, 1e-8, one, None, None, None)[1]
    assert "eps" in fwd(0, 1, 4, 1, one, None, None, 0, 0.0, one, None, None, None)[1]
    assert "NULL" in fwd(0, 1, 4, 1, None, None, None, 0, 1e-8, one, None, None, None)[1]
    assert "channels" in fwd(0, 1, (1 << 22) + 1, 1, one, None, None, 0, 1e-8, one, None, None, None)[1]
    assert fwd(0, 1 << 40, 1 << 20, 1 << 40, one, None, None, 0, 1e-8, one, None, None, None)[0] == -3
    assert fwd(0, 0, 4, 1, None, None, None, 0, 1e-8, None, None, None, None)[0] == 0          # nothing to do
    assert L.ggs_rms_norm_workspace_bytes(0, 0, 4, 1) == 0
    nb = L.ggs_rms_norm_workspace_bytes(0, 1000, 64, 7)
    assert nb > 0 and L.ggs_rms_norm_workspace_bytes(2, 1000, 64, 7) > 0
    bwd = lambda *a: _rc(L.ggs_rms_norm_backward, *a)              # noqa: E731
    assert "workspace" in bwd(0, 1000, 64, 7, one, None, one, 0, one, one, None, one, one, one, nb - 1, None)[1]
    assert "NULL" in bwd(0, 1000, 64, 7, one, None, one, 0, None, one, None, one, None, None, 0, None)[1]
    two = lambda *a: _rc(L.ggs_rms_norm_double_backward, *a)       # noqa: E731
    nb = L.ggs_rms_norm_double_workspace_bytes(0, 1000, 64, 7)
    assert nb >= 4 * 7000 and L.ggs_rms_norm_double_workspace_bytes(2, 1000, 64, 7) == 2 * nb
    assert "workspace" in two(0, 1000, 64, 7, one, None, one, 0, one, one, one, None, one, one, one, one, nb - 1, None)[1]
    assert "NULL" in two(0, 1000, 64, 7, one, None, one, 0, one, None, one, None, one, one, one, one, nb, None)[1]


def test_which_maps_the_one_pass_kernels_take():
    """Their workspace is a row of partials a workgroup (8192 / waves at most), that of the two-pass kernels at most 64 rows: a map
    whose elements or whose float q lie beyond 32-bit byte offsets goes to the latter."""
    L = _lib.lib()
    rows = lambda code, c, inner: L.ggs_rms_norm_workspace_bytes(code, 1, c, inner) // (4 * c)                # noqa: E731
    for code in (1, 3):                                                          # 16 bits: 2 bytes an element, 4 a q
        assert rows(code, 1, 2 ** 30 - 1) == 8192 and rows(code, 1, 2 ** 30) == 64 and rows(code, 1, 2 ** 31 - 1) == 64
        assert rows(code, 2, 2 ** 30 - 1) == 8192 and rows(code, 2, 2 ** 30) == 64
    assert rows(0, 1, 2 ** 30 - 1) == 8192 and rows(0, 1, 2 ** 30) == 64


def test_training_setup_clips_only_with_the_gpu_optimiser():
    from types import SimpleNamespace
    from ggsplat.inner_step import DEFAULT_OPT
    from ggsplat.mesh_gaussian_model import MeshGaussianModel
    m = MeshGaussianModel(sh_degree=0)
    m._xyz = torch.zeros(3, 3, requires_grad=True)
    m.spatial_lr_scale = 1.0
    m.mesh = SimpleNamespace(v=torch.zeros(3, 3, requires_grad=True))
    opt = SimpleNamespace(**{**vars(DEFAULT_OPT), "max_grad_norm": 1.0})
    with pytest.raises(ValueError, match="max_grad_norm"):
        m.training_setup(opt, is_ff=False)
