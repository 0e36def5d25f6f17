"""ggsplat.adam.grad_norm / clip_grad_norm_ and GraphAdam(max_norm) on the GPU against 64 bits.

Tolerances: squares are added in double and the root is rounded to float once, so the norm is within half a float step
(2^-24 relative, and 1e-12 for the double sums); the factor is rounded to float (2^-24) and the scaled gradient once to its own
type (u: half a step).  The update: every one of its <= 8 float operations a quantity passes is off by half a step of the
magnitudes that enter."""
import copy
import math

import pytest
import torch

from ggsplat import _lib
from ggsplat import adam as A

pytestmark = pytest.mark.gpu
U32 = 2.0 ** -24
HALF = {torch.float32: U32, torch.float16: 2.0 ** -11, torch.bfloat16: 2.0 ** -8}
TINY = {torch.float32: 2.0 ** -149, torch.float16: 2.0 ** -25, torch.bfloat16: 2.0 ** -134}


def norm64(gs):
    return math.sqrt(sum(float(g.detach().double().square().sum()) for g in gs))


def same_norm(got, gs):
    ref = norm64(gs)
    assert got.shape == () and got.dtype == torch.float32 and got.device.type == "cuda"
    assert abs(float(got) - ref) <= ref * (U32 + 1e-12) + 2.0 ** -149, (float(got), ref)


def grads(sizes, dtypes=(torch.float32,), seed=0, scale=1.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [(torch.randn(s, device="cuda", generator=g) * scale * (1 + i % 5)).to(dtypes[i % len(dtypes)]) for i, s in enumerate(sizes)]


LISTS = {"one": [1], "odd": [1, 2, 3, 5, 7, 9, 4095, 4096, 4097], "empty_among": [0, 17, 0, 1000, 0], "only_empty": [0, 0],
         "gaussians": [(1002, 3), (2000, 3), (2000, 1, 3), (2000, 15, 3), (2000, 1), (2000, 3), (2000, 4)],
         "many": [(k * 37) % 300 + 1 for k in range(300)], "exactly_128": [64] * 128, "129": [65] * 129,
         "uneven": [3_000_001, 5, 900_000, 1], "matrix": [(513, 2049)], "wide": [20_000_000]}


@pytest.mark.parametrize("kind", ["float32", "bfloat16", "float16", "mixed"])
@pytest.mark.parametrize("name", LISTS)
def test_norm_and_clipping(name, kind):
    types = (torch.float32, torch.bfloat16, torch.float16) if kind == "mixed" else (getattr(torch, kind),)
    for seed, scale in ((1, 1.0), (2, 1e-3)):
        gs = grads(LISTS[name], types, seed, scale)
        total = A.grad_norm(gs)
        same_norm(total, gs)
        ref = norm64(gs)
        for max_norm in (ref * 0.25, ref * 1.001 + 1e-5, 0.0, float("inf")):
            work = [g.clone() for g in gs]
            got = A.clip_grad_norm_(work, max_norm)
            assert torch.equal(got, total)
            c = min(1.0, max_norm / (ref + 1e-6))
            for a, b in zip(work, gs):
                want = b.double() * c
                off = (a.double() - want).abs() - want.abs() * (HALF[b.dtype] + 1.01 * (U32 + 1e-12) * 2) - TINY[b.dtype]
                assert not off.numel() or float(off.max()) <= 0.0
                if c == 1.0:
                    assert torch.equal(a, b)


def test_views_of_a_bucket_and_other_layouts():
    g = torch.Generator(device="cuda").manual_seed(3)
    for dtype in HALF:
        for lead in range(9):                                                    # every offset from a 16-byte border
            sizes = [1, 3, 8, 1021, 2, 16, 5000]
            flat = torch.randn(lead + sum(sizes) + 64, device="cuda", generator=g).to(dtype)
            keep, at, views = flat.clone(), lead, []
            for s in sizes:
                views.append(flat[at:at + s])
                at += s
            same_norm(A.grad_norm(views), views)
            A.clip_grad_norm_(views, 0.5 * norm64(views))
            assert torch.equal(flat[:lead], keep[:lead]) and torch.equal(flat[at:], keep[at:])     # nothing beside the views
            assert not torch.equal(flat[lead:at], keep[lead:at])
    x = torch.randn(6, 10, 8, 9, device="cuda", generator=g)
    for view in (x.permute(3, 1, 0, 2), x.to(memory_format=torch.channels_last), x[:, ::2], x[..., 1:7], x.transpose(0, 2)[1:]):
        v = view.clone() if view.is_contiguous() else view
        base = x.clone()
        ref = v.double().clone()
        n = norm64([v])
        same_norm(A.grad_norm(v), [v])
        A.clip_grad_norm_([v], 0.5 * n)
        assert torch.allclose(v.double(), ref * (0.5 * n / (n + 1e-6)), rtol=4 * U32, atol=1e-30)
        if v._is_view() and v.data_ptr() >= x.data_ptr() and v.numel() < x.numel():
            touched = torch.zeros_like(x, dtype=torch.bool)
            mark = touched[:, ::2] if v.shape == x[:, ::2].shape else touched[..., 1:7] if v.shape == x[..., 1:7].shape else touched.transpose(0, 2)[1:]
            mark.fill_(True)
            assert torch.equal(x[~touched], base[~touched])
    e = torch.ones(1, device="cuda").expand(50)
    same_norm(A.grad_norm([e]), [e])


def test_refusals():
    a, b = torch.ones(64, device="cuda"), torch.ones(64, device="cuda")
    for bad in ([a, a], [a, b, a[10:20]], [a.view(8, 8)[:, :4], a.view(8, 8)[:, 4:]]):
        with pytest.raises(ValueError, match="overlap"):
            A.clip_grad_norm_(bad, 1.0)
    with pytest.raises(ValueError, match="share memory"):
        A.clip_grad_norm_([torch.ones(1, device="cuda").expand(5)], 1.0)
    for bad, exc in ((torch.ones(3, device="cuda", dtype=torch.float64), TypeError), (torch.ones(3, device="cuda", dtype=torch.int32), TypeError),
                     (torch.nn.Parameter(torch.ones(3, device="cuda")), ValueError), (torch.ones(3), RuntimeError),
                     (torch.ones(3, device="cuda").to_sparse(), TypeError)):
        for fn in (A.grad_norm, lambda g: A.clip_grad_norm_(g, 1.0)):
            with pytest.raises(exc):
                fn([bad])
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            A.clip_grad_norm_([a], bad)
        with pytest.raises(ValueError, match="max_norm"):
            A.GraphAdam([torch.nn.Parameter(a.clone())], max_norm=bad)
    assert torch.equal(a, torch.ones_like(a)) and torch.equal(b, torch.ones_like(b))


def test_not_finite():
    g = torch.tensor([1.0, float("inf"), -2.0], device="cuda")
    n = A.clip_grad_norm_([g], 1.0)
    assert math.isinf(float(n)) and torch.equal(g.isnan(), torch.tensor([False, True, False], device="cuda")) and g[0] == 0 and g[2] == 0
    g = torch.tensor([1.0, float("nan")], device="cuda").bfloat16()
    other = torch.ones(5, device="cuda")
    assert math.isnan(float(A.clip_grad_norm_([g, other], 1.0))) and g.isnan().all() and other.isnan().all()
    for bad in (float("inf"), float("nan")):
        g = torch.tensor([1.0, bad], device="cuda")
        keep = g.clone()
        with pytest.raises(RuntimeError, match="not clipped"):
            A.clip_grad_norm_([g], 1.0, error_if_nonfinite=True)
        assert torch.equal(g[:1], keep[:1]) and not math.isfinite(float(g[1]))
    g = torch.tensor([3.0, 4.0], device="cuda")
    assert float(A.clip_grad_norm_([g], 1.0, error_if_nonfinite=True)) == 5.0
    big = torch.full((1000,), 3e30, device="cuda")                                # squares beyond float's range
    same_norm(A.clip_grad_norm_([big], 1.0), [torch.full((1000,), 3e30, device="cuda")])
    assert torch.allclose(big, torch.full_like(big, 1000 ** -0.5), rtol=1e-6)
    small = torch.full((1000,), 1e-30, device="cuda")
    same_norm(A.grad_norm([small]), [small])


def test_same_bits_on_streams_and_in_graphs():
    sets = [grads(LISTS["gaussians"], seed=5), grads([70000, 33], (torch.bfloat16,), 6), grads(LISTS["many"], seed=7)]
    want = []
    for s in sets:
        w = [g.clone() for g in s]
        want.append((A.clip_grad_norm_(w, 1.0), w))
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in sets], []
    for s, st in zip(sets, streams):
        with torch.cuda.stream(st):
            w = [g.clone() for g in s]
            got.append((A.clip_grad_norm_(w, 1.0), w))
    torch.cuda.synchronize()
    for a, b in zip(want, got):
        assert torch.equal(a[0], b[0]) and all(torch.equal(x, y) for x, y in zip(a[1], b[1]))
    static = [[g.clone() for g in s] for s in sets]
    graphs, norms = [], []
    for s in static:                                                             # a graph each, replayed side by side
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            A.grad_norm(s)
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norms.append((A.grad_norm(s), A.clip_grad_norm_(s, 1.0)))
            with pytest.raises(RuntimeError, match="captured"):
                A.clip_grad_norm_(s, 1.0, error_if_nonfinite=True)
        graphs.append(graph)
    for turn in range(4):
        for s, st in zip(sets, static):
            for a, b in zip(s, st):
                b.copy_(a * (turn + 1))
        torch.cuda.synchronize()
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for s, st, (n0, n1) in zip(sets, static, norms):
            w = [g * (turn + 1) for g in s]
            n = A.clip_grad_norm_(w, 1.0)
            assert torch.equal(n, n0) and torch.equal(n, n1) and all(torch.equal(x, y) for x, y in zip(w, st)), turn


def test_more_than_2_31_elements():
    n = 2 ** 31 + 11
    g = torch.full((n,), 0.5, device="cuda", dtype=torch.bfloat16)
    g[-1], g[2 ** 31] = 4096.0, -4096.0
    ref = math.sqrt(0.25 * (n - 2) + 2 * 4096.0 ** 2)
    assert abs(float(A.grad_norm([g])) - ref) <= ref * (U32 + 1e-9)
    A.clip_grad_norm_([g], ref / 2)
    assert g[-1] == 2048.0 and g[2 ** 31] == -2048.0 and g[0] == 0.25 and bool((g[2 ** 31 + 1:-1] == 0.25).all())


# ---- GraphAdam(max_norm) ----------------------------------------------------------------------------------------------------
def params(sizes, seed=0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return [torch.nn.Parameter(torch.randn(s, device="cuda", generator=g)) for s in sizes]


def adam64(p, m, v, g, k, lr, b1=0.9, b2=0.999, eps=1e-15):
    m = m + (1 - b1) * (g - m)
    v = b2 * v + (1 - b2) * g * g
    step = lr / (1 - b1 ** k) * m / ((v / (1 - b2 ** k)).sqrt() + eps)
    return p - step, m, v, step


SIZES = {"one": [1], "gaussians": LISTS["gaussians"], "odd": [1, 2, 3, 5, 7, 1025, 70001], "48": [33] * 48, "64": [33] * 64, "65": [7] * 65, "many": [(k * 53) % 700 + 1 for k in range(140)],
         "empty_among": [0, 5, 0, 300], "large": [5_000_001, 12]}


@pytest.mark.parametrize("name", SIZES)
def test_clipped_update(name):
    ps = params(SIZES[name])
    lrs = [1e-3 * (1 + i % 3) for i in range(len(ps))]
    opt = A.GraphAdam([{"params": [p], "lr": lr} for p, lr in zip(ps, lrs)], max_norm=1.0)
    for k, scale in ((1, 3.0), (2, 1e-4), (3, 50.0)):                             # over, under, over the limit
        gs = grads(SIZES[name], seed=k, scale=scale)
        before = [(p.detach().double(), opt.state[p]["exp_avg"].double(), opt.state[p]["exp_avg_sq"].double()) for p in ps]
        for p, g in zip(ps, gs):
            p.grad = g.clone()
        opt.step()
        same_norm(opt.last_grad_norm, gs)
        c = min(1.0, 1.0 / (norm64(gs) + 1e-6))
        for p, g, lr, (p0, m0, v0) in zip(ps, gs, lrs, before):
            assert torch.equal(p.grad, g)                                        # the gradients stay as they were
            if not p.numel():
                continue
            want, m, v, step = adam64(p0, m0, v0, g.double() * c, k, lr)
            gm = (g.double() * c).abs()
            em = 8 * U32 * (m0.abs() + gm)
            ev = 8 * U32 * (v0 + gm * gm * 1e-3)
            assert float(((opt.state[p]["exp_avg"].double() - m).abs() - em).max()) <= 1e-44
            assert float(((opt.state[p]["exp_avg_sq"].double() - v).abs() - ev - 2.0 ** -149).max()) <= 0
            ep = U32 * want.abs() * 1.01 + lr / (1 - 0.9 ** k) * em / ((v / (1 - 0.999 ** k)).sqrt() + 1e-15) + step.abs() * (16 * U32 + 0.5 * ev / (v + 1e-300))
            tiny = v < 1e-36                                                     # squares that a float holds with few bits or none
            assert float((((p.detach().double() - want).abs() - ep) * ~tiny).max()) <= 0
    assert opt.step_count == 3


def test_without_a_limit_the_update_keeps_its_bits():
    for sizes in (SIZES["gaussians"], SIZES["many"]):
        a = params(sizes)
        b = [torch.nn.Parameter(p.detach().clone()) for p in a]
        oa, ob = A.GraphAdam(a, lr=1e-3), A.GraphAdam(b, lr=1e-3, max_norm=float("inf"))
        for k in range(3):
            for p, q, g in zip(a, b, grads(sizes, seed=k)):
                p.grad, q.grad = g, g
            oa.step()
            ob.step()
        for p, q in zip(a, b):
            assert torch.equal(p, q) and all(torch.equal(oa.state[p][k], ob.state[q][k]) for k in ("exp_avg", "exp_avg_sq", "state"))


def test_against_clipping_first():
    """The clipped update = clip_grad_norm_ on the gradients, then the plain update: the same factor on the same gradients."""
    a = params(SIZES["gaussians"])
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    oa, ob = A.GraphAdam(a, lr=1e-3), A.GraphAdam(b, lr=1e-3, max_norm=0.7)
    for k in range(3):
        for p, q, g in zip(a, b, grads(SIZES["gaussians"], seed=k)):
            p.grad, q.grad = g.clone(), g.clone()
        n = A.clip_grad_norm_([p.grad for p in a], 0.7)
        oa.step()
        ob.step()
        assert torch.equal(n, ob.last_grad_norm)
    for p, q in zip(a, b):
        assert torch.equal(p, q) and torch.equal(oa.state[p]["exp_avg_sq"], ob.state[q]["exp_avg_sq"])


def test_guard_missing_gradients_and_checkpoints():
    ps = params([700, 50, 9])
    opt = A.GraphAdam(ps, lr=1e-2, max_norm=0.5)
    guard = torch.ones(1, dtype=torch.int64, device="cuda")
    for p, g in zip(ps, grads([700, 50, 9])):
        p.grad = g
    keep = [p.detach().clone() for p in ps]
    opt.step(guard=guard)                                                        # void
    assert all(torch.equal(p, k) for p, k in zip(ps, keep)) and opt.step_count == 0 and float(opt.last_grad_norm) == 0.0
    guard.zero_()
    opt.step(guard=guard)
    assert opt.step_count == 1 and not torch.equal(ps[0], keep[0])
    ps[1].grad = None                                                            # not part of this step, nor of its norm
    k1 = ps[1].detach().clone()
    opt.step()
    same_norm(opt.last_grad_norm, [ps[0].grad, ps[2].grad])
    assert torch.equal(ps[1], k1)
    states = [int(opt.state[p]["state"][:8].view(torch.int64)) for p in ps]
    assert states == [2, 1, 2]
    twin_p = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    twin = A.GraphAdam(twin_p, lr=1e-2, max_norm=0.5)
    twin.load_state_dict(opt.state_dict())
    for p, q in zip(ps, twin_p):
        p.grad = torch.ones_like(p)
        q.grad = torch.ones_like(q)
    opt.step()
    twin.step()
    for p, q in zip(ps, twin_p):
        assert torch.allclose(p, q, rtol=1e-6, atol=1e-7)
    for p in ps:
        p.grad = None
    opt.step()                                                                   # nothing to do: a norm of zero
    assert float(opt.last_grad_norm) == 0.0
    opt.max_norm = -1.0
    ps[0].grad = torch.ones_like(ps[0])
    with pytest.raises(ValueError, match="max_norm"):
        opt.step()
    assert copy.deepcopy(opt).max_norm == -1.0


def test_tick_false_leaves_the_states():
    ps = params([3000, 5])
    opt = A.GraphAdam(ps, lr=1e-3, max_norm=1.0)
    twin_p = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    twin = A.GraphAdam(twin_p, lr=1e-3, max_norm=1.0)
    L = _lib.lib()
    import ctypes as C
    for k in range(3):
        for p, q, g in zip(ps, twin_p, grads([3000, 5], seed=k)):
            p.grad, q.grad = g, g
        opt.step()
        st = twin.tick_states()
        assert L.ggs_adam_tick_multi(2, (C.c_void_p * 2)(*st), 0.9, 0.999, None, torch.cuda.current_stream().cuda_stream) == 0
        twin.step(tick=False)
    assert twin.step_count == 3 and all(torch.equal(p, q) for p, q in zip(ps, twin_p))


def test_captured_clipped_step():
    ps = params(SIZES["gaussians"])
    qs = [torch.nn.Parameter(p.detach().clone()) for p in ps]
    opt, ref = A.GraphAdam(ps, lr=1e-3, max_norm=1.0), A.GraphAdam(qs, lr=1e-3, max_norm=1.0)
    static = grads(SIZES["gaussians"])
    guard = torch.ones(1, dtype=torch.int64, device="cuda")
    for p, g in zip(ps, static):
        p.grad = g
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        opt.step(guard=guard)                                                    # void: only warms up
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step(guard=guard)
    guard.zero_()
    for k in range(5):
        new = grads(SIZES["gaussians"], seed=k, scale=10.0 ** (k - 3))
        for s, n, q in zip(static, new, qs):
            s.copy_(n)
            q.grad = n
        graph.replay()
        ref.step()
        torch.cuda.synchronize()
        assert torch.equal(opt.last_grad_norm, ref.last_grad_norm)
        assert all(torch.equal(p, q) for p, q in zip(ps, qs)), k
    assert opt.step_count == 5


def test_writes_in_place_are_seen_by_autograd():
    x = torch.ones(8, device="cuda", requires_grad=True)
    g = torch.full((8,), 2.0, device="cuda")
    y = (x * g).sum()                                                            # saves g
    A.clip_grad_norm_([g], 0.1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    p = torch.nn.Parameter(torch.ones(8, device="cuda"))
    opt = A.GraphAdam([p], lr=1e-2, max_norm=1.0)
    y = (p * p).sum()
    p.grad = torch.ones_like(p)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


@pytest.mark.parametrize("max_norm", [None, 1.0], ids=str)
def test_every_step_is_seen_by_autograd_and_by_cached_bindings(max_norm):
    """With and without clipping: a tensor saved before the step, and the mesh binding that a model keeps between its getters."""
    from types import SimpleNamespace
    from ggsplat.inner_step import DEFAULT_OPT
    from ggsplat.mesh_gaussian_model import MeshGaussianModel
    from test_gpu_graph_step import _scene
    p = torch.nn.Parameter(torch.ones(8, device="cuda"))
    unused = torch.nn.Parameter(torch.ones(8, device="cuda"))
    opt = A.GraphAdam([p, unused], lr=1e-2, max_norm=max_norm)
    y, z = (p * p).sum(), (unused * unused).sum()
    p.grad = torch.ones_like(p)
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()
    z.backward()                                                                 # had no gradient, was not written
    v, f, params, _, _, _ = _scene(seed=6)
    m = MeshGaussianModel.from_tensors(v, f, params, sh_degree=0, device="cuda")
    m.training_setup(SimpleNamespace(**{**vars(DEFAULT_OPT), "max_grad_norm": max_norm}), is_ff=True)
    for q, get in ((m._xyz, lambda: m.get_xyz), (m._scaling, lambda: m.get_scaling), (m._rotation, lambda: m.get_rotation)):
        before = get().detach().clone()
        q.grad = torch.randn(q.shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(1))
        m.optimizer.step()
        m.optimizer.zero_grad()
        got = get().detach().clone()
        m.update_face_coor()
        assert torch.equal(got, get()) and not torch.equal(got, before)


@pytest.mark.parametrize("lean", [True, False])
def test_a_replayed_step_is_seen_by_cached_bindings(lean):
    from ggsplat.inner_step import DEFAULT_OPT, GraphedRegistrationStep
    from ggsplat.mesh_gaussian_model import MeshGaussianModel
    from test_gpu_graph_step import H, W, _scene
    v, f, params, cams, gts, masks = _scene(seed=6)
    m = MeshGaussianModel.from_tensors(v, f, params, sh_degree=0, device="cuda")
    m.training_setup(DEFAULT_OPT, is_ff=True)
    step = GraphedRegistrationStep(m, W, H, torch.zeros(3, device="cuda"), opt=DEFAULT_OPT, lean=lean)
    for ci in (0, 1, 3):                                                         # the capture, then replays alone
        before = m.get_xyz.detach().clone()
        step(cams[ci], gts[ci], masks[ci])
        got = m.get_xyz.detach().clone()
        m.update_face_coor()
        assert torch.equal(got, m.get_xyz) and not torch.equal(got, before), ci
    y = (m._xyz * m._xyz).sum()
    step(cams[0], gts[0], masks[0])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.backward()


def test_a_void_step_without_gradients_keeps_the_norm():
    p = torch.nn.Parameter(torch.zeros(2, device="cuda"))
    opt = A.GraphAdam([p], lr=1e-2, max_norm=1.0)
    p.grad = torch.tensor([3.0, 4.0], device="cuda")
    opt.step()
    guard = torch.ones(1, dtype=torch.int64, device="cuda")
    for void in (p.grad, None):
        p.grad = void
        opt.step(guard=guard)
        assert float(opt.last_grad_norm) == 5.0
    guard.zero_()
    opt.step(guard=guard)
    assert float(opt.last_grad_norm) == 0.0


def test_gradients_that_were_computed_with_a_graph():
    p, q = (torch.nn.Parameter(torch.linspace(0.5, 2.0, n, device="cuda")) for n in (7, 30))
    with pytest.warns(UserWarning, match="create_graph"):
        ((p ** 3).sum() + (q ** 4).sum()).backward(create_graph=True)
    gs = [p.grad, q.grad]
    assert all(g.requires_grad for g in gs)
    keep = [g.detach().clone() for g in gs]
    total = A.grad_norm(gs)
    same_norm(total, keep)
    assert not total.requires_grad
    assert torch.equal(A.clip_grad_norm_(gs, 1.0), total)
    A.clip_grad_norm_(keep, 1.0)
    assert all(torch.equal(g, k) for g, k in zip(gs, keep))
    opt = A.GraphAdam([p, q], lr=1e-2, max_norm=0.5)
    opt.step()
    same_norm(opt.last_grad_norm, keep)
    p.grad = q.grad = None


def test_traces_and_forward_mode_are_refused():
    from torch.autograd import forward_ad as fw
    g = torch.tensor([3.0, 4.0], device="cuda")
    for fn in (A.grad_norm, lambda t: A.clip_grad_norm_(t, 1.0)):
        with pytest.raises(RuntimeError, match="trace"):
            torch.jit.trace(fn, (g,), check_trace=False)
        with fw.dual_level(), pytest.raises(NotImplementedError, match="forward-mode"):
            fn([g, fw.make_dual(g, g)])
    assert torch.equal(g, torch.tensor([3.0, 4.0], device="cuda"))
    with fw.dual_level():
        assert float(A.grad_norm([g])) == 5.0                                    # a level that is open, no tangent


def test_interleaved_views_are_refused_by_name_and_their_base_is_taken():
    m = torch.arange(64.0, device="cuda").view(8, 8)
    keep = m.clone()
    views = [m[:, :4], m[:, 4:]]
    with pytest.raises(ValueError, match="interleave"):
        A.clip_grad_norm_(views, 1.0)
    assert torch.equal(m, keep)
    same_norm(A.grad_norm(views), [keep])                                        # reading them is fine
    same_norm(A.clip_grad_norm_(m, 1.0), [keep])
    A.clip_grad_norm_([keep[:4], keep[4:]], 1.0)                                 # as are views that lie one behind the other
    assert torch.equal(m, keep)


def test_a_parameter_listed_twice_is_refused():
    p, q = (torch.nn.Parameter(torch.ones(n, device="cuda")) for n in (5000, 3))
    for groups in ([p, q, p], [{"params": [p]}, {"params": [q, p]}], [p, q, torch.nn.Parameter(p.detach())]):
        opt = A.GraphAdam(groups, lr=1e-2, max_norm=1.0)
        for g in opt.param_groups:
            for t in g["params"]:
                t.grad = torch.ones_like(t)
        with pytest.raises(ValueError, match="listed twice"):
            opt.step()
        assert torch.equal(p, torch.ones_like(p)) and opt.step_count == 0
