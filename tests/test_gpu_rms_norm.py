"""ggsplat.stylenet.rms_norm on the GPU against its formula in 64 bits: every element type, rows / channels-first / channels-last,
odd sizes, residual and weight present or not, forward and backward; memory it may not touch; streams, graphs, large offsets.

Tolerances.  u = half a step of the element type, a = half a step of the accumulation type (2^-24, 2^-53 for double), C channels,
P pixels.  The sum of C squares and the handful of operations around it are off by at most (C + 16) a relative to the magnitudes
that enter (and half of that after the square root); every output is rounded once more, by u.  dweight adds P such products: its
rounding errors are of either sign, 4 sqrt(P) a covers 4 standard deviations of their sum.  The 64-bit reference itself is off by
as much where the type is double: factor 2."""
import pytest
import torch

from ggsplat import _lib
from ggsplat import stylenet as SN

pytestmark = pytest.mark.gpu
EPS = 1e-8
HALF = {torch.float32: 2.0 ** -24, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8, torch.float64: 2.0 ** -53}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134, torch.float64: 0.0}   # half a subnormal step


def reference(x, w, r, gy, gh, eps=EPS):
    """(y, h, dx, dw) and the magnitudes their errors are relative to, in double."""
    d = lambda t: None if t is None else t.detach().double().movedim(1, -1)     # noqa: E731
    x, r, gy, gh = d(x), d(r), d(gy), d(gh)
    w = torch.ones(x.shape[-1], dtype=torch.float64, device=x.device) if w is None else w.detach().double()
    h = x if r is None else x + r
    s = (h.square().mean(-1, keepdim=True) + eps).sqrt()
    n = h / s
    out = {"y": n * w, "h": h}
    size = {"y": (n * w).abs(), "h": h.abs()}
    if gy is not None:
        g = gy * w
        out["dx"] = (g - n * (g * n).mean(-1, keepdim=True)) / s
        size["dx"] = (g.abs() + n.abs() * (g * n).abs().mean(-1, keepdim=True)) / s
        if gh is not None:
            out["dx"] = out["dx"] + gh
            size["dx"] = size["dx"] + gh.abs()
        back = lambda t: t.reshape(-1, t.shape[-1]).sum(0)                      # noqa: E731
        out["dw"], size["dw"] = back(gy * n), back((gy * n).abs())
    front = lambda k, t: t if k == "dw" else t.movedim(-1, 1)                   # noqa: E731
    return {k: front(k, v) for k, v in out.items()}, {k: front(k, v) for k, v in size.items()}


def held(name, got, ref, size, C, P, dtype):
    a = HALF[torch.float64] * 2 if dtype is torch.float64 else HALF[torch.float32]
    acc = (C + 16 + (4 * P ** 0.5 if name == "dw" else 0)) * a
    u = HALF[got.dtype] * (2 if dtype is torch.float64 else 1)
    off = (got.double() - ref).abs()
    allowed = u * ref.abs() * (1 + acc) + acc * size + TINY[got.dtype]
    worst = float((off - allowed).max()) if off.numel() else 0.0
    assert worst <= 0.0, f"{name}: {float(off.max()):.3g} off, {worst:.3g} over what is allowed"


def tensors(shape, dtype, weight, residual, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    rnd = lambda *s: torch.randn(*s, device="cuda", generator=g)                # noqa: E731
    x = (rnd(*shape) * (rnd(1, shape[1], *[1] * (len(shape) - 2)) * 0.5).exp()).to(dtype)
    w = None if weight is None else (1 + 0.3 * rnd(shape[1])).to(dtype if weight == "same" else torch.float32)
    r, gh = (rnd(*shape).to(dtype), rnd(*shape).to(dtype)) if residual else (None, None)
    return x, w, r, rnd(*shape).to(dtype), gh


def passes(x, w, r, gy, gh, eps=EPS):
    leaves = [t.detach().requires_grad_() for t in (x, w, r) if t is not None]
    it = iter(leaves)
    xl, wl, rl = next(it), next(it) if w is not None else None, next(it) if r is not None else None
    out = SN.rms_norm(xl, wl, residual=rl, eps=eps)
    outs, into = (out, (gy, gh)) if r is not None else ((out,), (gy,))
    grads = dict(zip([n for n, t in (("dx", x), ("dw", w), ("dr", r)) if t is not None], torch.autograd.grad(outs, leaves, into)))
    return {"y": outs[0].detach(), **({"h": outs[1].detach()} if r is not None else {}), **grads}


def check(shape, dtype, weight, residual, change=lambda t: t, seed=0):
    x, w, r, gy, gh = tensors(shape, dtype, weight, residual, seed)
    x, r, gy, gh = (None if t is None else change(t) for t in (x, r, gy, gh))
    ref, size = reference(x, w, r, gy, gh)
    got = passes(x, w, r, gy, gh)
    P = max(1, x.numel() // shape[1])
    for k, v in got.items():
        key = "dx" if k == "dr" else k
        assert v.shape == ref[key].shape and v.dtype == (w.dtype if k == "dw" else dtype)
        held(k, v, ref[key], size[key], shape[1], P, dtype)
    quiet = SN.rms_norm(x, w, residual=r, eps=EPS)                               # without autograd: the same bits
    quiet = quiet if residual else (quiet,)
    assert torch.equal(quiet[0], got["y"]) and (not residual or torch.equal(quiet[1], got["h"]))
    return got


SHAPES = [(1, 1), (1, 512), (3, 7), (1000, 51), (37, 300), (5, 2050), (2, 10001), (3, 16390), (300, 4096), (70000, 8),
          (1, 512, 8, 8), (2, 3, 1, 1), (3, 100, 37, 53), (1, 1, 5, 7), (2, 33, 1, 129), (1, 1030, 3, 5), (2, 1025, 65, 1), (4, 16, 64, 64),
          (2, 5, 9), (1, 8, 2, 3, 5), (2, 257, 20, 9), (1, 32, 3, 700), (5, 64, 4, 4), (1, 600, 31, 33)]


@pytest.mark.parametrize("residual", [False, True], ids=["plain", "residual"])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16, torch.float64], ids=str)
@pytest.mark.parametrize("shape", SHAPES, ids=str)
def test_against_64_bits(shape, dtype, residual):
    check(shape, dtype, [None, "same", "float32"][(sum(shape) + residual) % 3], residual)


# What the sizes above do not reach of the map kernels: 64 floats of a channel a workgroup (at least 32768 pixels), loads past the
# caches (128 MiB and more), several tiles a workgroup of several waves (its share of dweight, and the two LDS buffers by turns),
# one pixel a vector with more than one channel, the border between two forms.
@pytest.mark.parametrize("shape,dtype", [
    ((2, 128, 256, 256), torch.float32), ((1, 256, 181, 182), torch.float32), ((1, 30, 181, 182), torch.float32),
    ((3, 250, 96, 116), torch.float32), ((4, 100, 90, 91), torch.bfloat16), ((2, 512, 128, 128), torch.bfloat16), ((1, 300, 330, 331), torch.float16), ((1, 200, 590, 591), torch.bfloat16),
    ((1, 32, 1024, 1024), torch.float16), ((2, 520, 180, 180), torch.bfloat16), ((1, 1000, 257, 255), torch.bfloat16), ((9, 600, 61, 64), torch.float32)], ids=str)
@pytest.mark.parametrize("residual", [False, True], ids=["plain", "residual"])
def test_large_maps(shape, dtype, residual):
    check(shape, dtype, "float32", residual, seed=3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("C", [5, 300, 600, 1024])
@pytest.mark.parametrize("pixels", [(3, 2, 1), (2, 1, 7), (2, 3, 1), (400, 1, 3)], ids=str)
def test_maps_narrower_than_a_vector(pixels, C, dtype):
    check((pixels[0], C, pixels[1], pixels[2]), dtype, ["same", "float32", None][C % 3], C != 300, seed=4)


@pytest.mark.parametrize("weight", [None, "same", "float32"], ids=str)
@pytest.mark.parametrize("shape", [(129, 770), (2, 40, 30, 31)], ids=str)
def test_weights(shape, weight):
    for dtype in (torch.float32, torch.float16, torch.bfloat16, torch.float64):
        check(shape, dtype, weight, True, seed=3)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float64], ids=str)
def test_layouts(dtype):
    last = lambda t: t.contiguous(memory_format=torch.channels_last)             # noqa: E731
    got = check((2, 48, 19, 23), dtype, "float32", True, last)
    for k in ("y", "h", "dx"):
        assert got[k].is_contiguous(memory_format=torch.channels_last), k
    turned = lambda t: t.transpose(1, 2).contiguous().transpose(1, 2)            # noqa: E731
    assert check((3, 65, 77), dtype, "same", True, turned)["y"].stride(1) == 1
    check((3, 64, 17, 9), dtype, "same", True, lambda t: t.transpose(2, 3).contiguous().transpose(2, 3))      # another order of pixels
    check((4, 30, 8, 8), dtype, None, False, lambda t: torch.stack([t, t], -1)[..., 0])                        # strided
    for lead in (1, 2, 3):                                                       # off every 16-byte border
        def shift(t):
            flat = torch.zeros(t.numel() + lead, dtype=t.dtype, device=t.device)
            flat[lead:] = t.reshape(-1)
            return flat[lead:].view(t.shape)
        check((3, 40, 6, 10), dtype, "same", True, shift)
        check((50, 128), dtype, "same", True, shift)


def test_mixed_layouts_and_broadcast_gradients():
    x, w, r, gy, gh = tensors((2, 24, 6, 5), torch.float32, "same", True)
    last = lambda t: t.contiguous(memory_format=torch.channels_last)             # noqa: E731
    ref = passes(x, w, r, gy, gh)
    for mix in ((last(x), r, gy, gh), (x, last(r), gy, last(gh)), (last(x), last(r), gy, gh)):
        got = passes(mix[0], w, mix[1], mix[2], mix[3])
        for k in ("y", "h"):
            assert torch.allclose(got[k], ref[k], rtol=1e-6, atol=1e-7), k
    one = torch.ones((), device="cuda")
    got = passes(x, w, r, one.expand(x.shape), one.expand(x.shape))
    ref64, size = reference(x, w, r, one.expand(x.shape), one.expand(x.shape))
    for k in ("dx", "dw", "dr"):
        held(k, got[k], ref64["dx" if k == "dr" else k], size["dx" if k == "dr" else k], 24, 60, torch.float32)


def test_gradients_against_differences():
    g = torch.Generator().manual_seed(4)
    for shape in ((3, 5), (2, 6, 3, 2), (2, 70, 2, 1)):
        x, r = (torch.randn(*shape, generator=g, dtype=torch.float64).cuda().requires_grad_() for _ in range(2))
        w = torch.randn(shape[1], generator=g, dtype=torch.float64).cuda().requires_grad_()
        assert torch.autograd.gradcheck(lambda a, b, c: SN.rms_norm(a, b, residual=c, eps=1e-3), (x, w, r))
        assert torch.autograd.gradcheck(lambda a: SN.rms_norm(a, eps=1e-3), (x,))


def test_second_derivatives_against_differences():
    g = torch.Generator().manual_seed(8)
    for shape in ((3, 5), (2, 6, 3, 2), (2, 70, 2, 1), (300, 2, 3)):
        x, r, gy, gh = (torch.randn(*shape, generator=g, dtype=torch.float64).cuda().requires_grad_() for _ in range(4))
        w = torch.randn(shape[1], generator=g, dtype=torch.float64).cuda().requires_grad_()
        fast = dict(fast_mode=True) if x.numel() > 100 else {}
        assert torch.autograd.gradgradcheck(lambda a, b, c: SN.rms_norm(a, b, residual=c, eps=1e-2), (x, w, r), (gy, gh), **fast)
        assert torch.autograd.gradgradcheck(lambda a, b: SN.rms_norm(a, b, eps=1e-2), (x, w), (gy,), **fast)
        assert torch.autograd.gradgradcheck(lambda a: SN.rms_norm(a, eps=1e-2), (x,), (gy,), **fast)
        last = x.detach().movedim(1, -1).contiguous().movedim(-1, 1).requires_grad_()
        assert torch.autograd.gradgradcheck(lambda a, b: SN.rms_norm(a, b, eps=1e-2), (last, w), (gy,), **fast)


def test_second_derivatives_of_strided_inputs():
    """Inputs that the call has to bring into another order first: the second derivatives reach the tensors themselves."""
    g = torch.Generator().manual_seed(11)
    wide = torch.randn(2, 6, 3, 4, generator=g, dtype=torch.float64).cuda()
    x, r = wide[..., ::2].detach().requires_grad_(), wide.flip(0)[..., 1::2].detach().requires_grad_()
    w = torch.randn(12, generator=g, dtype=torch.float64).cuda()[::2].detach().requires_grad_()
    gy = torch.randn(2, 6, 3, 2, generator=g, dtype=torch.float64).cuda().requires_grad_()
    assert not x.is_contiguous() and not w.is_contiguous()
    last = wide[..., :2].movedim(1, -1).contiguous().movedim(-1, 1).requires_grad_()
    assert torch.autograd.gradgradcheck(lambda a, b: SN.rms_norm(a, b, eps=1e-2), (x, w), (gy,))
    assert torch.autograd.gradgradcheck(lambda a, b, c: SN.rms_norm(a, b, residual=c, eps=1e-2), (x, w, r), (gy, gy.detach().clone().requires_grad_()))
    assert torch.autograd.gradgradcheck(lambda a, b, c: SN.rms_norm(a, b, residual=c, eps=1e-2), (last, w, r), (gy, gy.detach().clone().requires_grad_()))
    h, hr = wide[..., ::2].half().float().detach(), wide.flip(0)[..., 1::2].float().half().float().detach()
    got = []
    for impl, cast in (("hip", torch.Tensor.half), ("native", torch.Tensor.double)):              # 16 bits keep both summands
        a, b = (cast(t) for t in (h, hr))
        a, b = (torch.stack([t, t], -1)[..., 0].requires_grad_() for t in (a, b))
        y, _ = SN.rms_norm(a, residual=b, eps=1e-2, impl=impl)
        (gx,) = torch.autograd.grad((y.double() * gy).sum(), a, create_graph=True)
        got.append(torch.autograd.grad((gx.double() * gy.flip(0)).sum(), (a, b)))
    for p, q in zip(*got):
        assert float((p.double() - q).norm() / q.norm()) <= 4 * HALF[torch.float16]


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16], ids=str)
@pytest.mark.parametrize("shape", [(40, 51), (2, 65, 9, 7), (3, 1030, 2, 2)], ids=str)
def test_second_derivatives(shape, dtype):
    """A gradient penalty's gradients against the same through the plain form in double.  Every value passes two normalisations:
    off by at most 2 (C + 16) a of the largest magnitudes that enter and u once (16 bits: dx and dw, whose squares the penalty sums,
    are rounded on the way, u each); compared in norm, where independent roundings do not add up."""
    x, w, r, gy, gh = tensors(shape, dtype, "float32", True, seed=9)
    got = []
    for impl, cast in (("hip", lambda t: t), ("native", lambda t: t.double())):
        leaves = [cast(t).detach().requires_grad_() for t in (x, w, r, gy, gh)]
        y, h = SN.rms_norm(leaves[0], leaves[1], residual=leaves[2], impl=impl)
        gx, gw = torch.autograd.grad((y, h), leaves[:2], (leaves[3], leaves[4]), create_graph=True)
        if impl == "native":                                                    # the cotangents the other side works with
            gx, gw = gx + (first[0].double() - gx).detach(), gw + (first[1].double() - gw).detach()
        else:
            first = (gx.detach(), gw.detach())
        got.append(torch.autograd.grad((gx.double().square().sum() + gw.double().square().sum()) / 2, leaves))
    for name, a, b in zip(("x", "w", "r", "gy", "gh"), *got):
        assert a.shape == b.shape
        off = float((a.double() - b).norm() / b.norm())
        assert off <= 2 * HALF[dtype] + 2 * (shape[1] + 16) * HALF[torch.float32], (name, off)


def test_third_derivatives_are_refused():
    x = torch.randn(4, 6, device="cuda", requires_grad=True)
    (g,) = torch.autograd.grad(SN.rms_norm(x).sin().sum(), x, create_graph=True)
    torch.autograd.grad(g.square().sum(), x, retain_graph=True)
    with pytest.raises(RuntimeError, match="not differentiable again"):
        torch.autograd.grad(g.square().sum(), x, create_graph=True)


def test_which_gradients_are_asked_for():
    x, w, r, gy, gh = tensors((2, 12, 5, 5), torch.float32, "same", True)
    full = passes(x, w, r, gy, gh)
    for ask in ((0,), (1,), (2,), (0, 1), (1, 2)):
        t = [v.detach().requires_grad_(i in ask) for i, v in enumerate((x, w, r))]
        y, h = SN.rms_norm(t[0], t[1], residual=t[2], eps=EPS)
        got = torch.autograd.grad((y, h), [t[i] for i in ask], (gy, gh))
        for i, v in zip(ask, got):
            assert torch.equal(v, full[("dx", "dw", "dr")[i]])
    t = [v.detach().requires_grad_() for v in (x, w, r)]
    y, h = SN.rms_norm(t[0], t[1], residual=t[2], eps=EPS)
    dx, dw, dr = torch.autograd.grad(h, t, gh, allow_unused=True, retain_graph=True)              # only the sum is used
    assert torch.equal(dx, gh) and torch.equal(dr, gh) and dw is None
    dx, dw = torch.autograd.grad(y, t[:2], gy)                                                    # only the norm is used
    ref, size = reference(x, w, r, gy, None)
    held("dx", dx, ref["dx"], size["dx"], 12, 50, torch.float32)
    a = x.detach().requires_grad_()                                                               # x is its own residual
    y, h = SN.rms_norm(a, w, residual=a, eps=EPS)
    (ga,) = torch.autograd.grad((y, h), a, (gy, gh))
    ref, size = reference(x, w, x, gy, gh)
    held("dx", ga, 2 * ref["dx"], 2 * size["dx"], 12, 50, torch.float32)


def test_empty_zero_and_not_finite():
    for shape in ((0, 5), (3, 5, 0), (0, 5, 2, 2)):
        x = torch.zeros(shape, device="cuda", requires_grad=True)
        w = torch.ones(5, device="cuda", requires_grad=True)
        y, h = SN.rms_norm(x, w, residual=torch.zeros(shape, device="cuda"))
        assert y.shape == h.shape == x.shape
        (y.sum() + h.sum()).backward()
        assert torch.equal(w.grad, torch.zeros(5, device="cuda")) and x.grad.shape == x.shape
    z = torch.zeros(2, 6, 3, 3, device="cuda")
    got = passes(z, None, z, z + 1, z)
    assert torch.equal(got["y"], z) and torch.isfinite(got["dx"]).all()
    for dtype in HALF:                                                           # an eps that a float does not hold
        assert not SN.rms_norm(z.to(dtype), eps=1e-60).any()
    for shape in ((40, 70), (2, 70, 9, 9), (1, 1100, 3, 3), (9, 9000)):
        x, w, r, gy, gh = tensors(shape, torch.float32, "same", True)
        clean = passes(x, w, r, gy, gh)
        xb = x.movedim(1, -1).reshape(-1, shape[1]).clone()
        xb[2, 3], xb[5, 1] = float("nan"), float("inf")
        xb = xb.reshape(x.movedim(1, -1).shape).movedim(-1, 1).contiguous()
        got = passes(xb, w, r, gy, gh)
        for k in ("y", "dx"):                                                    # a bad value stays in its pixel
            a, b = (t[k].movedim(1, -1).reshape(-1, shape[1]) for t in (got, clean))
            keep = torch.ones(len(a), dtype=torch.bool, device="cuda")
            keep[2] = keep[5] = False
            assert torch.equal(a[keep], b[keep]) and torch.isnan(a[2]).all() and torch.isnan(a[5, 1])


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("outer,C,inner", [(3, 51, 1), (7, 515, 1), (2, 9001, 1), (2, 33, 67), (1, 1030, 5), (3, 64, 16), (1, 500, 130)])
def test_writes_nothing_else(outer, C, inner, dtype):
    """Outputs as windows of larger buffers (at an odd element): what lies in front of and behind them stays as it was."""
    L, n, pad, code = _lib.lib(), outer * C * inner, 1031, SN._RMS_TYPES[dtype]
    g = torch.Generator(device="cuda").manual_seed(1)
    x, r, gy, gh = (torch.randn(n, device="cuda", generator=g).to(dtype) for _ in range(4))
    w = torch.ones(C, device="cuda")

    def window(count, dt):
        buf = torch.full((count + 2 * pad,), 7.0, device="cuda", dtype=dt)
        return buf, buf[pad:pad + count]
    bufs = {k: window(c, t) for k, c, t in (("y", n, dtype), ("h", n, dtype), ("q", outer * inner, torch.float32), ("dx", n, dtype),
                                            ("dw", C, torch.float32))}
    nb = L.ggs_rms_norm_workspace_bytes(code, outer, C, inner)
    wsb, ws = window(nb // 4, torch.float32)
    s = torch.cuda.current_stream().cuda_stream
    p = {k: v[1].data_ptr() for k, v in bufs.items()}
    assert L.ggs_rms_norm_forward(code, outer, C, inner, x.data_ptr(), r.data_ptr(), w.data_ptr(), 1, EPS, p["y"], p["h"], p["q"], s) == 0
    assert L.ggs_rms_norm_backward(code, outer, C, inner, x.data_ptr(), r.data_ptr(), w.data_ptr(), 1, p["q"], gy.data_ptr(), gh.data_ptr(),
                                   p["dx"], p["dw"], ws.data_ptr(), nb, s) == 0
    for k, (buf, inside) in [*bufs.items(), ("workspace", (wsb, ws))]:
        assert (buf[:pad] == 7).all() and (buf[len(buf) - pad:] == 7).all(), k
        if k != "workspace":
            assert not (inside == 7).all(), k
    shape = (outer, C, inner)
    ref, size = reference(x.view(shape), w, r.view(shape), gy.view(shape), gh.view(shape))
    for k in ("y", "h", "dx"):
        held(k, bufs[k][1].view(shape), ref[k], size[k], C, outer * inner, dtype)
    held("dw", bufs["dw"][1], ref["dw"], size["dw"], C, outer * inner, dtype)


def test_same_bits_on_streams_and_in_graphs():
    cases = [tensors(s, t, "float32", True, seed=i) for i, (s, t) in enumerate(
        [((500, 51), torch.float32), ((2, 96, 40, 40), torch.bfloat16), ((1, 512, 16, 16), torch.float32), ((64, 2048), torch.float16)])]
    eager = [passes(*c) for c in cases]
    streams = [torch.cuda.Stream() for _ in cases]
    torch.cuda.synchronize()
    got = []
    for c, s in zip(cases, streams):                                             # four calls at once, a stream each
        with torch.cuda.stream(s):
            got.append(passes(*c))
    torch.cuda.synchronize()
    for a, b in zip(eager, got):
        assert all(torch.equal(a[k], b[k]) for k in a)
    static = [[None if t is None else t.clone() for t in c] for c in cases]
    torch.cuda.current_stream().synchronize()
    graph = torch.cuda.CUDAGraph()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        [passes(*c) for c in static]
    torch.cuda.current_stream().wait_stream(side)
    with torch.cuda.graph(graph):
        out = [passes(*c) for c in static]
    for turn in range(4):
        for c, s in zip(cases, static):
            for a, b in zip(c, s):
                if a is not None:
                    b.copy_(a * (1 + turn))
        graph.replay()
        want = [passes(*[None if t is None else t * (1 + turn) for t in c]) for c in cases]
        torch.cuda.synchronize()
        for a, b in zip(want, out):
            assert all(torch.equal(a[k], b[k]) for k in a), turn


def test_offsets_beyond_32_bits():
    """More than 2^31 elements: the last pixels / rows, and one in the middle, against the formula."""
    for shape in ((1, 3, 2 ** 30 // 1024, 701), (2 ** 21 + 3, 1025)):
        n = 1
        for s in shape:
            n *= s
        assert n > 2 ** 31
        x = torch.empty(shape, device="cuda", dtype=torch.float16)
        x.view(-1)[:2 ** 30].normal_(generator=torch.Generator(device="cuda").manual_seed(2))
        rest = x.view(-1)[2 ** 30:]
        rest.copy_(x.view(-1)[:2 ** 30].repeat(-(-rest.numel() // 2 ** 30))[:rest.numel()])
        x.requires_grad_()
        y = SN.rms_norm(x)
        gy = x.detach().flip(0) if len(shape) == 2 else x.detach()
        (dx,) = torch.autograd.grad(y, x, gy)
        last = lambda t: (t[-9:] if len(shape) == 2 else t[:, :, -1, -9:]).detach()              # noqa: E731
        first = lambda t: (t[:9] if len(shape) == 2 else t[:, :, 0, :9]).detach()                # noqa: E731
        mid = lambda t: (t[2 ** 20:2 ** 20 + 9] if len(shape) == 2 else t[:, :, 2 ** 19, :9]).detach()      # noqa: E731
        for part in (first, mid, last):
            ref, size = reference(part(x), None, None, part(gy), None)
            held("y", part(y), ref["y"], size["y"], shape[1], 9, torch.float16)
            held("dx", part(dx), ref["dx"], size["dx"], shape[1], 9, torch.float16)
        del x, y, dx, gy, rest
        torch.cuda.empty_cache()


def test_one_channel_with_more_pixels_than_its_q_has_32_bit_offsets_for():
    """2^30 pixels and some, one channel in 16 bits: under 2^32 bytes of map, over 2^32 bytes of q."""
    shape, n = (1, 1, 2 ** 15, 2 ** 15 + 8), 2 ** 15 * (2 ** 15 + 8)
    x = torch.empty(shape, device="cuda", dtype=torch.float16)
    flat = x.view(-1)
    flat[:2 ** 28].normal_(generator=torch.Generator(device="cuda").manual_seed(4))
    flat[2 ** 28:] = flat[:2 ** 28].flip(0).repeat(n // 2 ** 28 + 1)[:n - 2 ** 28]                # other values 2^30 pixels on
    w = torch.full((1,), 1.5, device="cuda", requires_grad=True)
    x.requires_grad_()
    y = SN.rms_norm(x, w, eps=1.0)
    dx, dw = torch.autograd.grad(y, (x, w), x.detach())
    rows = lambda t, k: t.detach()[:, :, k:k + 1]                                 # noqa: E731
    for k in (0, 1, 2 ** 14, 2 ** 15 - 9, 2 ** 15 - 8, 2 ** 15 - 7, 2 ** 15 - 1):         # (pixel 2^30 lies in row 2^15 - 8)
        ref, size = reference(rows(x, k), w, None, rows(x, k), None, eps=1.0)
        for name, v in (("y", y), ("dx", dx)):
            held(name, rows(v, k), ref[name], size[name], 1, 9, torch.float16)
    want = 0.0
    for part in flat.detach().split(2 ** 26):
        d = part.double()
        want += float((d * d / (d * d + 1).sqrt()).sum())
    # (every term is positive: a thread adds up to 2^30 / 2^14 + 1 = 65537 of them one after the other, half a float step each)
    assert abs(float(dw) - want) <= want * 65600 * 2.0 ** -24, (float(dw), want)


@pytest.mark.parametrize("shape,dtype", [((2 ** 29 + 5, 1), torch.float16), ((2 ** 25 + 3, 1, 3), torch.float16), ((2 ** 23 + 3, 1), torch.float64),
                                         ((2 ** 23 + 3, 1, 2), torch.float64)], ids=str)
def test_more_work_than_one_launch_takes(shape, dtype):
    """2^31 threads and some: rows and maps behind the first launch, and dweight over all of them."""
    x = torch.empty(shape, device="cuda", dtype=dtype)
    x.view(-1)[:2 ** 16].normal_(generator=torch.Generator(device="cuda").manual_seed(2))
    n = x.numel()
    x.view(-1)[2 ** 16:] = x.view(-1)[:2 ** 16].repeat(n // 2 ** 16 + 1)[:n - 2 ** 16]
    w = torch.full((1,), 1.5, device="cuda", dtype=torch.float64 if dtype is torch.float64 else torch.float32, requires_grad=True)
    x.requires_grad_()
    y = SN.rms_norm(x, w, eps=1.0)
    dx, dw = torch.autograd.grad(y, (x, w), x.detach())
    for part in (slice(0, 9), slice(shape[0] // 2, shape[0] // 2 + 9), slice(shape[0] - 9, shape[0])):
        ref, size = reference(x[part], w, None, x[part], None, eps=1.0)
        for k, v in (("y", y), ("dx", dx)):
            held(k, v[part].detach(), ref[k], size[k], 1, 9, dtype)
    want = 0.0
    for part in x.detach().view(-1).split(2 ** 26):
        d = part.double()
        want += float((d * d / (d * d + 1).sqrt()).sum())
    # (every term is positive: a thread adds up to 2^29 / 2^16 = 8192 of them one after the other, half a float step each)
    assert abs(float(dw) - want) <= want * 8200 * 2.0 ** -24, (float(dw), want)


def test_gradients_of_two_leaves_do_not_share_memory():
    x, w, r, gy, gh = tensors((2, 12, 5, 5), torch.float32, "same", True)
    x.requires_grad_()
    r.requires_grad_()
    y, h = SN.rms_norm(x, w, residual=r)
    torch.autograd.backward((y, h), (gy, gh))
    assert torch.equal(x.grad, r.grad) and x.grad.data_ptr() != r.grad.data_ptr()


@pytest.mark.filterwarnings("ignore::torch.jit.TracerWarning")
def test_traced_calls():
    """torch.jit.trace of calls with and without a gradient: run on tensors of other sizes, layouts and values, and differentiated."""
    x, w, r, gy, gh = tensors((2, 12, 5, 5), torch.float32, "same", True)
    with torch.no_grad():
        one = torch.jit.trace(lambda t: SN.rms_norm(t), (x,))
    two = torch.jit.trace(lambda a, b, c: SN.rms_norm(a, c, residual=b, eps=EPS), (x.requires_grad_(), r, w))
    for shape in ((2, 12, 5, 5), (1, 12, 3, 70), (5, 40, 1, 1), (0, 12, 5, 5)):
        x, w, r, gy, gh = tensors(shape, torch.float32, "same", True, seed=1)
        assert torch.equal(one(x), SN.rms_norm(x))
        xl = x.to(memory_format=torch.channels_last)
        ref, size = reference(xl, None, None, None, None)
        held("y", one(xl), ref["y"], size["y"], shape[1], 1, torch.float32)
        want = passes(x, w, r, gy, gh)
        leaves = [t.detach().requires_grad_() for t in (x, r, w)]
        y, h = two(*leaves)
        dx, dr, dw = torch.autograd.grad((y, h), leaves, (gy, gh))
        for k, v in (("y", y), ("h", h), ("dx", dx), ("dr", dr), ("dw", dw)):
            assert torch.equal(v, want[k]), k


@pytest.mark.parametrize("weight_f32", [0, 1])
@pytest.mark.parametrize("code,dtype", [(0, torch.float32), (1, torch.float16), (2, torch.float64), (3, torch.bfloat16)])
def test_no_pixels_give_a_dweight_of_zeros(code, dtype, weight_f32):
    """The C entry points: with no pixel there is nothing to read and no workspace, and dw is a sum of nothing."""
    L, C = _lib.lib(), 301
    s = torch.cuda.current_stream().cuda_stream
    for outer, inner in ((0, 1), (0, 7), (3, 0)):
        assert L.ggs_rms_norm_workspace_bytes(code, outer, C, inner) == L.ggs_rms_norm_double_workspace_bytes(code, outer, C, inner) == 0
        for double in (False, True):
            buf = torch.full((C + 64,), 7.0, device="cuda", dtype=torch.float32 if weight_f32 else dtype)
            dw = buf[32:32 + C].data_ptr()
            if double:
                rc = L.ggs_rms_norm_double_backward(code, outer, C, inner, None, None, None, weight_f32, None, None, None, None, None, None, dw, None, 0, s)
            else:
                rc = L.ggs_rms_norm_backward(code, outer, C, inner, None, None, None, weight_f32, None, None, None, None, dw, None, 0, s)
            assert rc == 0 and not buf[32:32 + C].any() and (buf[:32] == 7).all() and (buf[32 + C:] == 7).all()
