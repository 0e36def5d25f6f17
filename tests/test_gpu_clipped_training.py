"""rms_norm, gradient clipping and the clipped update in the framework's own paths: StyleUNetLite(norm="rms") against its plain
PyTorch twin, the captured appearance iteration with that network and GraphAdam(max_norm), the captured registration iteration of a
model whose training_setup asks for clipping."""
import copy
from types import SimpleNamespace

import pytest
import torch

from ggsplat import adam as A
from ggsplat import stylenet as SN
from test_gpu_graph_step import H, W, _scene

pytestmark = pytest.mark.gpu


def _rel(a, b):
    return float((a.double() - b.double()).abs().sum() / (b.double().abs().sum() + 1e-30))


def test_network_with_norm_against_its_native_twin():
    """In double every value and parameter gradient agrees to the 1e-6 of the other operators' fp32 gain constants."""
    ch = {k: min(v, 24) for k, v in SN.CHANNELS.items()}
    torch.manual_seed(5)
    hip = SN.StyleUNetLite(size=64, out_ch=7, style_dim=32, channels=ch, norm="rms").cuda().double()
    nat = SN.StyleUNetLite(size=64, out_ch=7, style_dim=32, channels=ch, norm="rms", impl="native").cuda().double()
    with torch.no_grad():
        for g in hip.gains:
            g.uniform_(0.5, 1.5)
    nat.load_state_dict(copy.deepcopy(hip.state_dict()))
    g = torch.Generator().manual_seed(6)
    cond, style = torch.randn(2, 4, 64, 64, generator=g).cuda().double(), torch.randn(2, 32, generator=g).cuda().double()
    w = torch.randn(2, 7, 64, 64, generator=g).cuda().double()
    outs = []
    for net in (hip, nat):
        out = net(cond, style)
        (out * w).sum().backward()
        outs.append((out.detach(), {n: p.grad for n, p in net.named_parameters() if p.grad is not None}))
    assert _rel(outs[0][0], outs[1][0]) <= 1e-6
    assert set(outs[0][1]) == set(outs[1][1]) and any(n.startswith("gains") for n in outs[0][1])
    for n in outs[0][1]:
        assert _rel(outs[0][1][n], outs[1][1][n]) <= 1e-6, n


def test_network_with_norm_in_half_precision(monkeypatch):
    """The 16-bit network, forward and backward: every rms_norm call that it makes against its definition in 64 bits, and the gains'
    gradients.  (The convolutions, not this library's, are computed in float and rounded.)"""
    from test_gpu_rms_norm import held, reference
    for name in ("conv2d", "conv_transpose2d"):
        def wide(x, w, b=None, fn=getattr(SN.F, name), **kw):
            return fn(x.float(), w.float(), None if b is None else b.float(), **kw).to(x.dtype)
        monkeypatch.setattr(SN.F, name, wide)
    calls, plain = [], SN.rms_norm

    def recorded(x, weight=None, residual=None, **kw):
        out = plain(x, weight, residual=residual, **kw)
        y = out if residual is None else out[0]
        call = {"in": [None if t is None else t.detach() for t in (x, weight, residual)], "y": y.detach()}
        if y.requires_grad:
            y.register_hook(lambda g: call.__setitem__("gy", g.detach()))
        calls.append(call)
        return out
    monkeypatch.setattr(SN, "rms_norm", recorded)
    torch.manual_seed(5)
    net = SN.StyleUNetLite(size=64, out_ch=7, style_dim=32, channels={k: min(v, 24) for k, v in SN.CHANNELS.items()}, norm="rms").cuda().half()
    with torch.no_grad():
        for p in net.gains:
            p.uniform_(0.5, 1.5)
    g = torch.Generator().manual_seed(6)
    cond, style = torch.randn(2, 4, 64, 64, generator=g).cuda().half(), torch.randn(2, 32, generator=g).cuda().half()
    out = net(cond, style)
    (out.float() * torch.randn(2, 7, 64, 64, generator=g).cuda()).sum().backward()
    assert out.dtype is torch.float16 and torch.isfinite(out).all() and len(calls) == 1 + len(net.gains)
    for call, gain in zip(calls, [None, *net.gains]):
        x, w, r = call["in"]
        assert x.dtype is torch.float16 and (r is None) == (gain is None)
        gy = call.get("gy", torch.zeros_like(x))
        ref, size = reference(x, w, r, gy, None, eps=1e-8)
        held("y", call["y"], ref["y"], size["y"], x.shape[1], 1, torch.float16)
        if gain is not None:
            assert "gy" in call and gy.any()
            held("dw", gain.grad, ref["dw"], size["dw"], x.shape[1], x.numel() // x.shape[1], torch.float16)


def test_captured_appearance_iteration_with_norm_and_clipping():
    """Replays of the captured iteration (network with rms_norm, clipped update) against the same iteration run eagerly."""
    from ggsplat.inner_step import DEFAULT_OPT, GraphedAppearanceStep, appearance_step
    from ggsplat.mesh_gaussian_model import MeshGaussianModel
    opt = SimpleNamespace(**{**vars(DEFAULT_OPT), "threshold_xyz": 0.05, "threshold_scale": 0.02})
    v, f, params, cams, gts, masks = _scene(seed=6)
    P = f.shape[0]
    bg = torch.zeros(3, device="cuda")
    g = torch.Generator().manual_seed(21)
    uv, vis = torch.rand(P, 2, generator=g).cuda(), (torch.rand(P, generator=g) > 0.3).cuda()
    cond = torch.randn(1, 4, 64, 64, generator=g).cuda()
    torch.manual_seed(22)
    unet = SN.StyleUNetLite(size=64, in_ch=4, out_ch=6, style_dim=32, channels={k: min(c, 16) for k, c in SN.CHANNELS.items()}, norm="rms")
    net_g = SN.TexelOffsets(unet, uv, 1, vis, cond).cuda()
    net_e = copy.deepcopy(net_g)
    sides = []
    for net in (net_e, net_g):
        m = MeshGaussianModel.from_tensors(v, f, params, sh_degree=0, device="cuda")
        groups = [{"params": list(net.parameters()), "lr": 1e-3, "name": "net"}, {"params": [m._opacity], "lr": 1e-2, "name": "opacity"}]
        sides.append((m, A.GraphAdam(groups, lr=0.0, eps=1e-15, max_norm=1e-5)))
    (me, oe), (mg, og) = sides
    step = GraphedAppearanceStep(mg, net_g, W, H, bg, og, opt=opt)
    for ci in (0, 2, 4):
        ref = appearance_step(me, net_e, cams[ci], gts[ci], masks[ci], bg, optimizer=oe, opt=opt, fused_loss=True)
        out = step(cams[ci], gts[ci], masks[ci])
        for k in ("img", "ssim", "loss"):
            r = float(ref[k].detach())
            assert abs(float(out[k]) - r) <= 2e-4 * max(1.0, abs(r)), (ci, k, float(out[k]), r)
        n, e = float(og.last_grad_norm), float(oe.last_grad_norm)
        assert n > 1e-5 and abs(n - e) <= 1e-2 * e, (ci, n, e)                   # clipped; convolution gradients differ in their order of sums
    assert step.recaptures == 0 and og.step_count == 3 and oe.step_count == 3
    assert all(torch.isfinite(p).all() for p in net_g.parameters())


@pytest.mark.parametrize("slack", [1.0, 0.002])
def test_captured_registration_iteration_with_clipping(slack):
    """slack 0.002: the first replay overflows its binning capacity, the guard voids the clipped update with the rest of the step,
    and the step is captured again."""
    from ggsplat import inner_step as IS
    from ggsplat import rasterizer as R
    from ggsplat.mesh_gaussian_model import MeshGaussianModel
    v, f, params, cams, gts, masks = _scene(seed=6)
    bg = torch.zeros(3, device="cuda")
    limit = 1e-4
    opt = SimpleNamespace(**{**vars(IS.DEFAULT_OPT), "max_grad_norm": limit})
    models = []
    for _ in range(2):
        m = MeshGaussianModel.from_tensors(v, f, params, sh_degree=0, device="cuda")
        m.training_setup(opt, is_ff=True)
        assert isinstance(m.optimizer, A.GraphAdam) and m.optimizer.max_norm == limit
        models.append(m)
    eager, graphed = models
    R._cap_hint.clear()
    step = IS.GraphedRegistrationStep(graphed, W, H, bg, opt=opt, first_frame_template=True, capacity_slack=slack)
    for ci in (0, 1, 3, 0):
        IS.registration_step(eager, cams[ci], gts[ci], masks[ci], bg, opt=opt, first_frame_template=True, fused_loss=True)
        step(cams[ci], gts[ci], masks[ci])
        a, b = float(eager.optimizer.last_grad_norm), float(graphed.optimizer.last_grad_norm)
        assert a > limit and abs(a - b) <= 1e-3 * a, (ci, a, b)
    assert graphed.optimizer.step_count == eager.optimizer.step_count == 4
    assert step.recaptures == (0 if slack == 1.0 else 1)
    for n in ("_xyz", "_features_dc", "_opacity", "_scaling", "_rotation"):
        a, b = getattr(eager, n).detach(), getattr(graphed, n).detach()
        assert float((a - b).abs().mean()) <= 2e-4 * float(a.abs().mean()) + 1e-6, n


def test_pipelined_and_replica_iterations_with_clipping():
    """Two captured copies of one clipped iteration replayed alternately, and two models replayed side by side on streams of their
    own: the same trajectories as the plain captured iteration."""
    from ggsplat import inner_step as IS
    from ggsplat.mesh_gaussian_model import MeshGaussianModel
    v, f, params, cams, gts, masks = _scene(seed=6)
    bg = torch.zeros(3, device="cuda")
    opt = SimpleNamespace(**{**vars(IS.DEFAULT_OPT), "max_grad_norm": 1e-4})

    def model():
        m = MeshGaussianModel.from_tensors(v, f, params, sh_degree=0, device="cuda")
        m.training_setup(opt, is_ff=True)
        return m
    plain, piped, r0, r1 = (model() for _ in range(4))
    one = IS.GraphedRegistrationStep(plain, W, H, bg, opt=opt)
    two = IS.PipelinedRegistrationStep(piped, W, H, bg, opt=opt)
    many = IS.ReplicaRegistrationSteps([r0, r1], W, H, bg, opt=opt)
    norms = []
    for ci in (0, 1, 3, 0, 2):
        one(cams[ci], gts[ci], masks[ci])
        norms.append(float(plain.optimizer.last_grad_norm))
        two(cams[ci], gts[ci], masks[ci])
        many([cams[ci]] * 2, [gts[ci]] * 2, [masks[ci]] * 2)
        for r in (r0, r1):
            assert abs(float(r.optimizer.last_grad_norm) - norms[-1]) <= 1e-3 * norms[-1]
    two.flush()
    assert abs(float(piped.optimizer.last_grad_norm) - norms[-1]) <= 1e-3 * norms[-1]
    for m in (piped, r0, r1):
        assert m.optimizer.step_count == 5
        for n in ("_xyz", "_features_dc", "_opacity", "_scaling", "_rotation"):
            a, b = getattr(plain, n).detach(), getattr(m, n).detach()
            assert float((a - b).abs().mean()) <= 2e-4 * float(a.abs().mean()) + 1e-6, n
