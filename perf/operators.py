"""Workloads of the training-step operators: root-mean-square norm over channels with a residual, the global gradient norm with
clipping, and the Adam update whose gradients are clipped by that norm.

With `own` false every operator runs in its plain form, in elementary torch operations; with `own` true through ggsplat."""
import os
import sys

import numpy as np
import torch

own = False

EPS = 1e-8                    # added to the mean square, as StyledConv's demodulation adds it
BETAS, ADAM_EPS = (0.9, 0.999), 1e-15
LIMIT = 0.1                   # max_norm of the clipping cases
CHANNELS = {4: 512, 8: 512, 16: 512, 32: 512, 64: 512, 128: 256, 256: 128, 512: 64, 1024: 32, 2048: 16}
TYPES = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def listed():
    return [
        # a style vector on its way into the mapping layers: one row, no gain
        norm("style_b1", (1, 512), "float32"),
        # feature rows of 100k Gaussians (3 position + 48 colour channels, an odd row length), training
        norm("gaussian_rows_train", (100000, 51), "float32", weight="float32", train=True),
        # long rows in 16 bits, training with 32-bit gains
        norm("long_rows_train", (4096, 4096), "bfloat16", weight="float32", residual=True, train=True),
        # the 64 x 64 block of the texture network (512 channels) for one view, training
        norm("block64_train", (1, 512, 64, 64), "float32", weight="float32", residual=True, train=True),
        # its 256 x 256 block for two views, training
        norm("block256_train", (2, 128, 256, 256), "float32", weight="float32", residual=True, train=True),
        # its 1024 x 1024 block, 16 bits, forward only (rendering a trained network)
        norm("block1024_serve", (1, 32, 1024, 1024), "float16", weight="same", residual=True),
        # a cropped texture: plane size and channel count odd, so no row of pixels starts on a 16-byte border
        norm("crop_train", (3, 100, 37, 53), "float16", weight="same", residual=True, train=True),
        # gradients of 100k Gaussians with SH degree 3 and their mesh, over the limit: every gradient is scaled
        grads("clip_gaussians", "clip", "gaussians", 100000, "float32", clipped=True),
        # gradients of the texture network in 16 bits, over the limit
        grads("clip_network_bf16", "clip", "network", 512, "bfloat16", clipped=True),
        # the same network in 32 bits, under the limit: the common step, nothing is scaled
        grads("clip_network_under", "clip", "network", 512, "float32", clipped=False),
        # the update of a small scene: latency
        grads("adam_small", "adam", "gaussians", 600, "float32", clipped=True),
        # the update of the texture network
        grads("adam_network", "adam", "network", 512, "float32", clipped=True),
    ]


def norm(name, shape, dtype, weight="none", residual=False, train=False):
    case = {"name": name, "op": "norm", "dtype": dtype, "weight": weight, "residual": residual, "train": train,
            "batch": shape[0], "channels": shape[1], "height": 0, "width": 0}
    if len(shape) == 4:
        case["height"], case["width"] = shape[2], shape[3]
    return case


def grads(name, op, model, size, dtype, clipped):
    return {"name": name, "op": op, "model": model, "size": size, "dtype": dtype, "clipped": clipped}


def draw(rng):
    span = lambda lo, hi: int(round(lo * (hi / lo) ** rng.random()))  # noqa: E731
    kind = rng.choice(["rows", "planes", "planes", "clip", "adam"])
    if kind == "rows":
        channels = span(8, 8192)
        case = norm("", (span(1, 2 ** 24 // channels), channels), "")
    elif kind == "planes":
        channels, batch = span(8, 1024), rng.randint(1, 4)
        most = 2 ** 24 // (channels * batch)
        height = span(1, max(1, min(2048, int(most ** 0.5 * 2))))
        case = norm("", (batch, channels, height, span(1, max(1, min(2048, most // height)))), "")
    else:
        case = grads("", kind, rng.choice(["gaussians", "network"]), 0, "float32", rng.random() < 0.6)
        case["size"] = span(100, 300000) if case["model"] == "gaussians" else rng.choice([32, 64, 128, 256, 512])
        if kind == "clip":
            case["dtype"] = rng.choice(sorted(TYPES))
    if case["op"] == "norm":
        case["dtype"], case["weight"] = rng.choice(sorted(TYPES)), rng.choice(["none", "same", "float32"])
        case["residual"], case["train"] = rng.random() < 0.5, rng.random() < 0.6
    del case["name"]
    return case


def shapes(case):
    """The parameter tensors of a mesh-bound Gaussian model with `size` Gaussians, or of the texture network of that size."""
    n = case["size"]
    if case["model"] == "gaussians":
        return [(n // 2 + 2, 3), (n, 3), (n, 1, 3), (n, 15, 3), (n, 1), (n, 3), (n, 4)]
    style, res, cin, got = 512, n // 2, CHANNELS[n // 2], []
    got += [(style, style), (style,), (style, style), (style,), (cin, 4, 3, 3), (cin,), (cin, cin, 3, 3), (cin,)]
    levels = []
    while res > 8:
        levels.append(res)
        res //= 2
        got += [(CHANNELS[res], cin, 3, 3), (CHANNELS[res],)]
        cin = CHANNELS[res]
    for res in reversed(levels):
        c = CHANNELS[res]
        got += [(1, c, cin, 3, 3), (cin, style), (cin,), (c,), (c, 2 * c, 3, 3), (c,), (1, c, c, 3, 3), (c, style), (c,), (c,), (204, c, 1, 1), (204,)]
        cin = c
    return got


def counts(case):
    return [int(np.prod(s)) for s in shapes(case)]


def slots(case):
    """Where each tensor lies in a flat buffer: back to back for gradients (as the all-reduce bucket has them), on 16-byte
    borders for what the optimiser updates."""
    unit, at, got = 4 if case["op"] == "adam" else 1, 0, []
    for n in counts(case):
        got.append((at, n))
        at += -(-n // unit) * unit
    return got, at


def split(flat, case):
    return [flat[o:o + n].view(s) for (o, n), s in zip(slots(case)[0], shapes(case))]


def inputs(case, seed):
    """Every input of a case from its seed, as a dict of tensors."""
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    normal = lambda *s: torch.randn(*s, device="cuda", generator=g)  # noqa: E731
    t = TYPES[case["dtype"]]
    if case["op"] == "norm":
        shape = (case["batch"], case["channels"]) + ((case["height"], case["width"]) if case["height"] else ())
        per = (1, case["channels"]) + (1,) * (len(shape) - 2)
        got = {"x": (normal(*shape) * normal(*per).mul_(0.5).exp_()).to(t)}
        if case["weight"] != "none":
            got["w"] = (1 + 0.2 * normal(case["channels"])).to(t if case["weight"] == "same" else torch.float32)
        if case["residual"]:
            got["r"] = normal(*shape).to(t)
        if case["train"]:
            got["gy"] = normal(*shape).to(t)
            if case["residual"]:
                got["gh"] = normal(*shape).to(t)
        return got
    at, total = slots(case)
    std = (4.0 if case["clipped"] else 0.2) * LIMIT / sum(counts(case)) ** 0.5
    flat = torch.zeros(total, device="cuda")
    for (o, n), s in zip(at, normal(len(at)).mul_(0.5).exp_().mul_(std).tolist()):
        flat[o:o + n] = normal(n) * s
    got = {"g": flat.to(t)}
    if case["op"] == "adam":
        got["p"] = normal(total) * 0.05
        got["m"] = normal(total) * std
        got["v"] = (normal(total) * std).square_()
        for k in ("p", "m", "v"):
            keep = torch.zeros(total, device="cuda")
            for o, n in at:
                keep[o:o + n] = 1
            got[k] *= keep
    return got


def steps_before(case):
    return 40


def prepare(case, seed):
    state = dict(inputs(case, seed), case=case, step=steps_before(case))
    if case["op"] == "norm":
        if case["train"]:
            state["leaves"] = [state[k].requires_grad_(own) for k in ("x", "w", "r") if k in state]
        return state
    state["grads"] = split(state["g"], case)
    if case["op"] == "adam":
        for k in ("p", "m", "v"):
            state[k + "s"] = split(state[k], case)
        state["lrs"] = [1e-4 * (1 + i % 3) for i in range(len(state["ps"]))]
        if own:
            package()
            from ggsplat.adam import GraphAdam
            ps = [torch.nn.Parameter(p) for p in state["ps"]]
            opt = GraphAdam([{"params": [p], "lr": lr} for p, lr in zip(ps, state["lrs"])], betas=BETAS, eps=ADAM_EPS, max_norm=LIMIT)
            sd = opt.state_dict()
            sd["state"] = {i: {"step": steps_before(case), "exp_avg": m, "exp_avg_sq": v} for i, (m, v) in enumerate(zip(state["ms"], state["vs"]))}
            opt.load_state_dict(sd)
            for p, g, m, v in zip(ps, state["grads"], state["ms"], state["vs"]):
                p.grad = g
                opt.state[p]["exp_avg"], opt.state[p]["exp_avg_sq"] = m, v      # the moments in flat buffers too
            state["opt"] = opt
    return state


def package():
    at = os.path.join(os.getcwd(), "gaussian-garments_amd")
    if at not in sys.path:
        sys.path.insert(0, at)


def run(state):
    case = state["case"]
    if not own:
        return {"norm": plain_norm, "clip": plain_clip, "adam": plain_adam}[case["op"]](state)
    package()
    if case["op"] == "norm":
        from ggsplat.stylenet import rms_norm
        out = rms_norm(state["x"], state.get("w"), residual=state.get("r"), eps=EPS)
        if not case["train"]:
            return out
        outs, into = (out, (state["gy"], state["gh"])) if case["residual"] else ((out,), (state["gy"],))
        return outs, torch.autograd.grad(outs, state["leaves"], into)
    if case["op"] == "clip":
        from ggsplat.adam import clip_grad_norm_
        total = clip_grad_norm_(state["grads"], LIMIT)
        return total, state["g"]
    state["opt"].step()
    return state["opt"].last_grad_norm, state["p"], state["m"], state["v"]


def plain_norm(state):
    t = state["x"].dtype
    h = state["x"].float()
    if "r" in state:
        h = h + state["r"].float()
    inv = torch.rsqrt((h * h).mean(1, keepdim=True) + EPS)
    n = h * inv
    per = (1, -1) + (1,) * (h.dim() - 2)
    w = state["w"].float().view(per) if "w" in state else None
    y = (n * w if w is not None else n).to(t)
    outs = (y, h.to(t)) if "r" in state else (y,)
    if not state["case"]["train"]:
        return outs if "r" in state else y
    gy = state["gy"].float()
    g = gy * w if w is not None else gy
    gx = inv * (g - n * (g * n).mean(1, keepdim=True))
    if "gh" in state:
        gx = gx + state["gh"].float()
    gx = gx.to(t)
    back = [gx]
    if w is not None:
        back.append((gy * n).sum([0] + list(range(2, h.dim()))).to(state["w"].dtype))
    if "r" in state:
        back.append(gx)
    return outs, tuple(back)


def total_norm(gs):
    return torch.stack([g.float().square().sum() for g in gs]).sum().sqrt()


def plain_clip(state):
    total = total_norm(state["grads"])
    scale = (LIMIT / (total + 1e-6)).clamp(max=1.0)
    _ = [g.copy_(g.float() * scale) for g in state["grads"]]
    return total, state["g"]


def plain_adam(state):
    state["step"] += 1
    b1, b2 = BETAS
    c1, c2 = 1 - b1 ** state["step"], (1 - b2 ** state["step"]) ** 0.5
    total = total_norm(state["grads"])
    scale = (LIMIT / (total + 1e-6)).clamp(max=1.0)
    _ = [plain_update(p, g * scale, m, v, b1, b2, lr / c1, c2) for p, g, m, v, lr in
         zip(state["ps"], state["grads"], state["ms"], state["vs"], state["lrs"])]
    return total, state["p"], state["m"], state["v"]


def plain_update(p, g, m, v, b1, b2, rate, c2):
    m.add_((g - m) * (1 - b1))
    v.mul_(b2).add_(g * g * (1 - b2))
    p.sub_(rate * m / (v.sqrt() / c2 + ADAM_EPS))


def work(case):
    size = {"float32": 4, "float16": 2, "bfloat16": 2}[case["dtype"]]
    if case["op"] == "norm":
        n = case["batch"] * case["channels"] * max(1, case["height"]) * max(1, case["width"])
        tensors = 2 + 2 * case["residual"] + case["train"] * (2 + case["residual"])     # x y | r h | gy gx | gh
        w = 0 if case["weight"] == "none" else case["channels"] * (4 if case["weight"] == "float32" else size)
        return {"bytes": n * size * tensors + w * (1 + case["train"]), "flops": n * (4 + case["residual"] + case["train"] * (9 + case["residual"]))}
    n = sum(counts(case))
    if case["op"] == "clip":
        return {"bytes": n * size * (2 if case["clipped"] else 1) + 4, "flops": n * (3 if case["clipped"] else 2)}
    return {"bytes": n * 28 + 4, "flops": n * 15}


def exact(case, seed):
    """The operators' definitions in 64 bits: y = w h / sqrt(mean h^2 + eps) and its gradients by the quotient rule; the length of
    the gradients as one vector; the update's recurrences."""
    d = {k: v.double() for k, v in inputs(case, seed).items()}
    if case["op"] == "norm":
        h = d["x"] + d["r"] if case["residual"] else d["x"]
        c = case["channels"]
        h = h.movedim(1, -1)
        size = (h.pow(2).sum(-1, keepdim=True) / c + EPS).sqrt()
        w = d.get("w", torch.ones((), dtype=torch.float64, device=h.device))
        y = (w * h / size).movedim(-1, 1)
        outs = (y, h.movedim(-1, 1)) if case["residual"] else (y,)
        if not case["train"]:
            return outs if case["residual"] else y
        gy = d["gy"].movedim(1, -1)
        along = (gy * w * h).sum(-1, keepdim=True)
        gx = gy * w / size - h * along / (c * size ** 3)
        if case["residual"]:
            gx = gx + d["gh"].movedim(1, -1)
        gx = gx.movedim(-1, 1)
        back = [gx]
        if case["weight"] != "none":
            back.append((gy * h / size).reshape(-1, c).sum(0))
        return outs, tuple(back + ([gx] if case["residual"] else []))
    g = d["g"]
    total = torch.linalg.vector_norm(g)
    g = g * min(1.0, LIMIT / (total.item() + 1e-6))
    if case["op"] == "clip":
        return total, g
    b1, b2 = BETAS
    k = steps_before(case) + 1
    m = b1 * d["m"] + (1 - b1) * g
    v = b2 * d["v"] + (1 - b2) * g ** 2
    rate = torch.zeros_like(g)
    for i, (o, n) in enumerate(slots(case)[0]):
        rate[o:o + n] = 1e-4 * (1 + i % 3)
    p = d["p"] - rate * (m / (1 - b1 ** k)) / ((v / (1 - b2 ** k)).sqrt() + ADAM_EPS)
    return total, p, m, v
