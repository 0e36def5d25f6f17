"""GraphAdam -- the optimiser of the inner loops on the graph-capturable kernels of libggsplat.so.

Stands where the reference builds ``torch.optim.Adam(l, lr=0.0, eps=1e-15)`` (scene/mesh_gaussian_model.py:375,
gaussian_model.py:165, avatar_net.py:50): same `param_groups` shape ({"params", "lr", "name"}), same update
(single-tensor Adam without amsgrad / weight decay), `step()` / `zero_grad()`.  Differences, all so that a whole
optimisation step can be replayed as one hipGraph:
  * step count, bias corrections and the learning rates live in device memory (`push_lr()` uploads the host-side
    `param_groups[i]["lr"]` after a schedule update -- a 4-byte-per-group async copy, no re-capture);
  * moments are allocated up front (nothing is allocated or zero-filled inside a captured step);
  * `step(guard=...)`: a device int64/uint64 word that voids the whole step when non-zero -- the binning-overflow
    flag of the forward of the same step (ggsplat.rasterizer.last_header()[1:2]);
  * `max_norm=...`: the update reads the gradients scaled by min(1, max_norm / (N + 1e-6)), N the norm of all gradients of the
    step as one vector -- torch.nn.utils.clip_grad_norm_ without its pass that rewrites them and without a host sync.

`grad_norm` / `clip_grad_norm_` are the same norm and scaling on any list of gradients (of another optimiser, of a bucket that
was just all-reduced); they take GRADIENTS, like ggsplat.dist.all_reduce_grads, not parameters.
"""
from __future__ import annotations

import ctypes as C
import math
from typing import Dict, Iterable, List, Optional

import torch
from torch.autograd import forward_ad
from torch.autograd.graph import increment_version

from ._lib import check, lib, on_device, ptr, stream_ptr


def _checked_max_norm(max_norm) -> float:
    m = float(max_norm)
    if not m >= 0.0:                       # NaN too
        raise ValueError(f"ggsplat: max_norm must be a number that is not negative, got {max_norm}")
    return m


def _span(t: torch.Tensor):
    """(elements from the first to the last one, whether they fill that span without gaps, whether some of them share memory)."""
    span, dense, shared = 1, True, False
    for stride, size in sorted(zip(t.stride(), t.size())):
        if size > 1:
            shared = shared or stride < span
            dense = dense and stride == span
            span += stride * (size - 1)
    return span, dense, shared


_GRAD_CODES = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 3}              # GGS_DTYPE_*
_GRAD_SIZE = {0: 4, 1: 2, 3: 2}


class _GradList:
    """The gradients of one call as the C ABI takes them: sizes, addresses, types.  The order of a tensor's elements is of no
    matter to the norm, so any dense layout is read in place; a strided one is read (and written back) through a copy."""

    def __init__(self, grads, in_place: bool):
        if torch.jit.is_tracing():                 # the trace would hold the allocation of the norm and not what fills it
            raise RuntimeError("ggsplat: gradient norms cannot be recorded by torch.jit.trace")
        self.device, self.copies, self.keep = None, [], []
        dual = forward_ad._current_level >= 0
        index, numel, ptrs, types, ends = None, [], [], [], []
        for g in ([grads] if isinstance(grads, torch.Tensor) else grads):
            if g is None:
                continue
            if not isinstance(g, torch.Tensor):
                raise TypeError(f"ggsplat: gradients are tensors, got {type(g).__name__}")
            at = g.get_device()
            if at < 0:
                raise RuntimeError("ggsplat: gradient norms run on the GPU only (no CPU path in the product)")
            if g.requires_grad and g.is_leaf:      # (gradients of backward(create_graph=True) require grad, but are no leaves)
                raise ValueError("ggsplat: pass the gradients ([p.grad for p in params]), not the parameters")
            if dual and forward_ad.unpack_dual(g).tangent is not None:
                raise NotImplementedError("ggsplat: gradient norms have no forward-mode derivative")
            if g.layout is not torch.strided:
                raise TypeError("ggsplat: sparse gradients are not supported")
            if at != index:
                if index is not None:
                    raise ValueError("ggsplat: the gradients are on different devices")
                index, self.device = at, g.device
            code = _GRAD_CODES.get(g.dtype)
            if code is None:
                raise TypeError(f"ggsplat: gradients are float32, float16 or bfloat16, got {g.dtype}")
            n = g.numel()
            if n == 0:
                continue
            span = n
            if not g.is_contiguous():
                span, dense, shared = _span(g)
                if in_place and shared:
                    raise ValueError("ggsplat: a gradient's elements share memory (an expanded tensor?): make it contiguous first")
                if in_place:
                    ends.append((g.data_ptr(), g.data_ptr() + span * _GRAD_SIZE[code]))
                if not dense:
                    c = g.contiguous()
                    self.copies.append((g, c))
                    g = c
            elif in_place:
                ends.append((g.data_ptr(), g.data_ptr() + n * _GRAD_SIZE[code]))
            self.keep.append(g)
            numel.append(n)
            ptrs.append(g.data_ptr())
            types.append(code)
        if in_place and len(ends) > 1:
            ends.sort()
            last = 0
            for lo, hi in ends:
                if lo < last:
                    raise ValueError("ggsplat: the memory of two gradients overlaps, from first to last element (the same one listed "
                                     "twice, or strided views that interleave: clip the tensor that they are views of)")
                last = hi
        self.n = n = len(numel)
        self.numel, self.ptrs, self.types = (C.c_size_t * n)(*numel), (C.c_void_p * n)(*ptrs), (C.c_int * n)(*types)

    def buffers(self):
        """(the norm, workspace bytes, workspace): new for every call, so that calls on several streams and captured graphs
        never share them."""
        nb = int(lib().ggs_grad_norm_workspace_bytes(self.n))
        return (torch.empty((), dtype=torch.float32, device=self.device), nb,
                torch.empty(nb, dtype=torch.uint8, device=self.device) if nb else None)


@torch.no_grad()
def grad_norm(grads) -> torch.Tensor:
    """The length of `grads` (a tensor, or tensors of float32 / float16 / bfloat16 in any mixture; None entries are skipped) as
    ONE vector: sqrt(sum of all squares), a 0-dim float32 tensor on their device (0 on the default device for no gradients at
    all).  Asynchronous on the current stream, capturable; sums in double, the same bits on every run.  Not differentiable."""
    gl = _GradList(grads, False)
    if gl.device is None:
        return torch.zeros((), dtype=torch.float32)
    with on_device(gl.device):
        norm, nb, ws = gl.buffers()
        check(lib().ggs_grad_norm(gl.n, gl.numel, gl.ptrs, gl.types, norm.data_ptr(), ptr(ws), nb, stream_ptr(gl.device)),
              "ggs_grad_norm")
    return norm


@torch.no_grad()
def clip_grad_norm_(grads, max_norm: float, error_if_nonfinite: bool = False) -> torch.Tensor:
    """Scales every gradient in place by min(1, max_norm / (N + 1e-6)) and returns N = grad_norm(grads), as
    torch.nn.utils.clip_grad_norm_ does for the gradients of its parameters (norm_type 2).  A NaN norm makes every gradient NaN,
    an infinite one zero (NaN where it was infinite); `error_if_nonfinite` raises instead and leaves the gradients as they were,
    which needs the norm on the host: a synchronisation, refused inside a capture.  No two gradients may overlap in memory,
    first to last element: strided views that interleave (columns of one matrix) are refused too, clip what they are views of.
    Gradients that were computed with create_graph=True are scaled as plain values."""
    max_norm = _checked_max_norm(max_norm)
    gl = _GradList(grads, True)
    if gl.device is None:
        return torch.zeros((), dtype=torch.float32)
    if error_if_nonfinite:
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("ggsplat: error_if_nonfinite needs the norm on the host and cannot be captured")
        total = float(grad_norm(gl.keep))
        if not math.isfinite(total):
            raise RuntimeError(f"ggsplat: the gradient norm is {total}: the gradients were not clipped")
    with on_device(gl.device):
        norm, nb, ws = gl.buffers()
        check(lib().ggs_grad_clip(gl.n, gl.numel, gl.ptrs, gl.types, max_norm, norm.data_ptr(), ptr(ws), nb,
                                  stream_ptr(gl.device)), "ggs_grad_clip")
        for g, c in gl.copies:
            g.copy_(c)
    increment_version(gl.keep)                     # written in place, as autograd's checks of saved tensors see it
    return norm


class _LrStaging:
    """Pinned staging rows of GraphAdam.push_lr, used round robin, each with the event of its last upload: with iterations in
    flight (PipelinedRegistrationStep has no per-iteration host sync) the next push must not rewrite a row whose copy has not
    run yet.  A deep copy of the optimiser (tests clone whole models) gets fresh rows: events are not copyable."""
    ROWS = 4

    def __init__(self, n_groups: int):
        self.n = n_groups
        self.rows = torch.zeros(self.ROWS, n_groups, dtype=torch.float32).pin_memory()
        self.events = [None] * self.ROWS
        self.slot = 0

    def __deepcopy__(self, memo):
        return _LrStaging(self.n)

    def next_row(self) -> torch.Tensor:
        k = self.slot
        self.slot = (k + 1) % self.ROWS
        if self.events[k] is not None:
            self.events[k].synchronize()          # the copy that last read this row (four pushes ago) has run
        self._k = k
        return self.rows[k]

    def uploaded(self, dev) -> None:
        ev = self.events[self._k] = self.events[self._k] or torch.cuda.Event()
        ev.record(torch.cuda.current_stream(dev))


class GraphAdam:
    def __init__(self, params: Iterable, lr: float = 0.0, betas=(0.9, 0.999), eps: float = 1e-15,
                 max_norm: Optional[float] = None):
        """max_norm: clip the gradients of every step() by their global norm (None: no clipping).  A plain attribute that
        step() reads: a captured step keeps the value it was captured with.  `last_grad_norm` (0-dim, on the device) is the
        norm of the last step that was not void, before clipping."""
        groups = list(params)
        if groups and not isinstance(groups[0], dict):
            groups = [{"params": groups}]
        self.param_groups: List[Dict] = []
        for g in groups:
            g = dict(g)
            g["params"] = list(g["params"])
            g.setdefault("lr", lr)
            self.param_groups.append(g)
        self.betas, self.eps = (float(betas[0]), float(betas[1])), float(eps)
        first = self.param_groups[0]["params"][0]
        if first.device.type != "cuda":
            raise RuntimeError("ggsplat GraphAdam runs on the GPU only (no CPU path in the product)")
        dev = self.device = first.device
        self.max_norm = None if max_norm is None else _checked_max_norm(max_norm)
        self.last_grad_norm = torch.zeros((), dtype=torch.float32, device=dev)
        L = lib()
        self._state_bytes = int(L.ggs_adam_state_bytes())
        self._lr_dev = torch.zeros(len(self.param_groups), dtype=torch.float32, device=dev)
        self._lr_host = _LrStaging(len(self.param_groups))
        self.state: Dict[torch.Tensor, Dict[str, torch.Tensor]] = {}
        for g in self.param_groups:
            for p in g["params"]:
                if p.dtype != torch.float32 or not p.is_contiguous():
                    raise ValueError("GraphAdam: parameters must be contiguous float32 tensors")
                self.state[p] = {"exp_avg": torch.zeros_like(p), "exp_avg_sq": torch.zeros_like(p),
                                 # step count + bias corrections of THIS parameter (torch counts steps per parameter)
                                 "state": torch.zeros(self._state_bytes, dtype=torch.uint8, device=dev)}
        self.push_lr()

    # ---- learning rates ---------------------------------------------------------------------------------
    def push_lr(self) -> None:
        """Upload param_groups[i]["lr"] to the device (call after changing a learning rate, outside a capture).  Asynchronous:
        the values take effect for the work queued AFTER this call on the current stream."""
        row = self._lr_host.next_row()
        for i, g in enumerate(self.param_groups):
            row[i] = float(g["lr"])
        self._lr_dev.copy_(row, non_blocking=True)
        self._lr_host.uploaded(self.device)

    @property
    def step_count(self) -> int:
        """Steps taken by the most-stepped parameter."""
        return max((int(st["state"][:8].view(torch.int64).item()) for st in self.state.values()), default=0)

    # ---- checkpoints (the reference's capture() / restore() store optimizer.state_dict(), scene/gaussian_model.py:63-90) --
    def state_dict(self) -> Dict:
        """torch.optim.Optimizer.state_dict() layout: parameters numbered in group order, per-parameter state {step, exp_avg,
        exp_avg_sq}, param_groups with "params" = those numbers."""
        idx, state, groups = 0, {}, []
        for g in self.param_groups:
            ids = []
            for p in g["params"]:
                st = self.state[p]
                state[idx] = {"step": st["state"][:8].view(torch.int64)[0].to(torch.float32).clone(),
                              "exp_avg": st["exp_avg"].clone(), "exp_avg_sq": st["exp_avg_sq"].clone()}
                ids.append(idx)
                idx += 1
            # the keys torch.optim.Adam keeps per group, with the values this optimiser implements: a torch.optim.Adam built
            # over the same parameters can load_state_dict() this dictionary and continue (its loader REPLACES the groups)
            groups.append({"weight_decay": 0, "amsgrad": False, "maximize": False, "foreach": None, "capturable": False,
                           "differentiable": False, "fused": None, "decoupled_weight_decay": False,
                           **{k: v for k, v in g.items() if k != "params"}, "betas": self.betas, "eps": self.eps, "params": ids})
        return {"state": state, "param_groups": groups}

    def load_state_dict(self, sd: Dict) -> None:
        """Accepts its own state_dict() and torch.optim.Adam's (same layout; amsgrad / weight decay / maximize are refused:
        this optimiser does not implement them).  The bias corrections are rebuilt from the step count with Python pow, while
        the kernel keeps running products: a restored optimiser continues within one ulp of the original per step."""
        for gs in sd["param_groups"]:
            if gs.get("amsgrad") or gs.get("maximize") or gs.get("weight_decay"):
                raise ValueError("GraphAdam.load_state_dict: amsgrad / maximize / weight_decay are not implemented")
        flat = [p for g in self.param_groups for p in g["params"]]
        for i, st in sd["state"].items():
            p = flat[int(i)]
            mine = self.state[p]
            mine["exp_avg"].copy_(st["exp_avg"])
            mine["exp_avg_sq"].copy_(st["exp_avg_sq"])
            # the device-side AdamState {i64 step, f32 1 - b1^t, f32 sqrt(1 - b2^t), f64 b1^t, f64 b2^t} (csrc/ggs_adam.hip)
            n = int(float(st["step"]))
            b1, b2 = self.betas
            import struct
            raw = struct.pack("<qffdd", n, 1.0 - b1 ** n, (1.0 - b2 ** n) ** 0.5, b1 ** n, b2 ** n)
            mine["state"][:32].copy_(torch.frombuffer(bytearray(raw), dtype=torch.uint8))
        for g, gs in zip(self.param_groups, sd["param_groups"]):
            g["lr"] = gs["lr"]
        self.push_lr()

    # ---- torch.optim.Optimizer surface ------------------------------------------------------------------
    def zero_grad(self, set_to_none: bool = True) -> None:
        for g in self.param_groups:
            for p in g["params"]:
                if p.grad is not None:
                    if set_to_none:
                        p.grad = None
                    else:
                        p.grad.zero_()

    def tick_states(self, params=None) -> List[int]:
        """Device addresses of the states step() would advance if every parameter of `params` (default: all) had a gradient --
        for a caller that advances them itself (ggs_registration_aux_tail) and then calls step(tick=False)."""
        ps = [p for g in self.param_groups for p in g["params"]] if params is None else list(params)
        return [self.state[p]["state"].data_ptr() for p in ps if p.numel()]

    @torch.no_grad()
    def step(self, guard: Optional[torch.Tensor] = None, tick: bool = True) -> None:
        """tick=False: the step counts / bias corrections of the tensors that have a gradient were advanced already."""
        L = lib()
        stream = stream_ptr(self.device)
        if guard is not None and (guard.element_size() != 8 or guard.device != self.device):
            raise ValueError("GraphAdam.step: guard must be a 64-bit word on the optimiser's device")
        gp = ptr(guard)
        b1, b2 = self.betas
        # every tensor that has a gradient: sizes, the six columns of addresses, and the gradients themselves (copies live on)
        numel, cols, keep, params, f32 = [], ([], [], [], [], [], []), [], [], torch.float32
        add_p, add_g, add_m, add_v, add_lr, add_s = (c.append for c in cols)
        states, lr = self.state, self._lr_dev.data_ptr()
        for g in self.param_groups:
            for p in g["params"]:
                grad = p.grad
                if grad is None:
                    continue
                n = p.numel()
                if n == 0:
                    continue
                if grad.dtype is not f32 or not grad.is_contiguous():
                    grad = grad.float().contiguous()
                st = states[p]
                numel.append(n)
                keep.append(grad)
                params.append(p)
                add_p(p.data_ptr())
                add_g(grad.data_ptr())
                add_m(st["exp_avg"].data_ptr())
                add_v(st["exp_avg_sq"].data_ptr())
                add_lr(lr)
                add_s(st["state"].data_ptr())
            lr += 4
        if self.max_norm is not None:
            self._clipped_step(L, numel, cols, tick, gp, stream)
            increment_version(params)              # written in place: saved tensors and cached bindings of them are void
            return
        for k in range(0, len(numel), 16):                     # one launch per 16 tensors
            sizes = numel[k:k + 16]
            n = len(sizes)
            chunk = [(C.c_void_p * n)(*c[k:k + 16]) for c in cols]
            # step counts / bias corrections advance inside the update launch (the last workgroup of a tensor stores them)
            fn = L.ggs_adam_tick_step_multi if tick else L.ggs_adam_step_multi
            check(fn(n, (C.c_size_t * n)(*sizes), *chunk, b1, b2, self.eps, gp, stream),
                  "ggs_adam_tick_step_multi" if tick else "ggs_adam_step_multi")
        increment_version(params)

    def _clipped_step(self, L, numel, cols, tick: bool, gp, stream) -> None:
        n = len(numel)
        if len(set(cols[0])) != n:                 # the workgroups of both entries would update the same elements at once
            raise ValueError("GraphAdam: a parameter is listed twice (tied weights?): list it once")
        addresses = [(C.c_void_p * n)(*c) for c in cols]
        with on_device(self.device):
            # the partial sums of this step: allocated per step, so that two captured steps never share them
            nb = int(L.ggs_grad_norm_workspace_bytes(n))
            ws = torch.empty(nb, dtype=torch.uint8, device=self.device) if nb else None
            check(L.ggs_adam_clip_step(n, (C.c_size_t * n)(*numel), *addresses, self.betas[0], self.betas[1], self.eps,
                                       _checked_max_norm(self.max_norm), int(tick), gp, self.last_grad_norm.data_ptr(), ptr(ws), nb,
                                       stream), "ggs_adam_clip_step")
