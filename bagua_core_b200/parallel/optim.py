"""Optimizers that work on flat bucket memory with one fused kernel for all buckets.

The reference contains no optimizer (it is only the communication engine); the benchmarks
named for it train with SGD momentum 0.9, so the engine ships the obvious companion: since
gradients already live in flat buckets, parameters and momentum are laid out the same way
and `step()` is ONE sm_100a kernel over all buckets (read p, g, m; write p, m: 20 bytes per
parameter, the HBM minimum) instead of torch's multi-tensor loops.  `FlatAdamW` does the same
for AdamW, with moments in fp32 (28 bytes per parameter) or in 8 bits (16).
"""
from __future__ import annotations

from operator import is_
from typing import List, Tuple

import torch

from .._native import C as _C
from ..ops.adamw import MOMENT8_BLOCK, adamw_read8, adamw_state8, adamw_step


def _is_dense(t: torch.Tensor) -> bool:
    """True if the tensor's elements occupy one gap-free, non-overlapping block of memory."""
    if t.numel() <= 1:
        return True
    dims = sorted((st, sz) for st, sz in zip(t.stride(), t.shape) if sz > 1)
    expect = 1
    for st, sz in dims:
        if st != expect:
            return False
        expect *= sz
    return True


def _same_order(a: torch.Tensor, b: torch.Tensor) -> bool:
    """True if the elements of two dense tensors of one shape follow each other in memory alike."""
    return a.numel() <= 1 or all(n == 1 or s == t for n, s, t in zip(a.shape, a.stride(), b.stride()))


@torch.no_grad()
def _copy_moments8(to: dict, saved: dict) -> None:
    """8-bit moments into codes and scales whose elements may follow each other in another order.

    A block is 256 neighbours in memory: in another order it has other elements, whose values are read and rounded anew, each to the
    nearest code of its new block's scale."""
    m, v = saved["exp_avg"], saved["exp_avg_sq"]
    if _same_order(m, to["exp_avg"]):
        for k in ("exp_avg", "exp_avg_sq", "scales"):
            to[k].copy_(saved[k])
        return
    device, n = to["exp_avg"].device, m.numel()
    values = [torch.empty_like(m, dtype=torch.float32) for _ in range(2)]
    adamw_read8([m], [v], [saved["scales"]], values[:1], values[1:])
    codes = torch.arange(256, dtype=torch.uint8)
    tables = [torch.empty(256) for _ in range(2)]
    adamw_read8([codes], [codes], [torch.ones(2, 1)], tables[:1], tables[1:])
    blocks = to["scales"].shape[1]
    for row, (k, largest, last) in enumerate((("exp_avg", 480, 128), ("exp_avg_sq", 496, 256))):
        table = tables[row][:last].to(device)
        x = torch.empty_like(to[k], dtype=torch.float32).copy_(values[row]).as_strided((n,), (1,))
        x = torch.nn.functional.pad(x, (0, blocks * MOMENT8_BLOCK - n)).view(blocks, MOMENT8_BLOCK)
        top = x.abs().amax(1)
        scale = torch.where(top > 0, (top * (1.0 / largest)).clamp(min=2.0 ** -126), top)
        to["scales"][row].copy_(torch.where(top.isfinite(), scale, float("nan")))
        y = x.abs().double() / torch.where(scale > 0, scale, 1.0).double()[:, None]
        code = torch.bucketize(y, ((table[1:] + table[:-1]) / 2).double())
        if row:
            code = torch.where(x > 0, code.clamp(min=1), code)  # (not zero: the step divides by it)
        else:
            code = code + 128 * (x < 0)
        to[k].as_strided((n,), (1,)).copy_(code.flatten()[:n])


class _FlatOptimizer(torch.optim.Optimizer):
    """What optimizers on flat buckets have in common: parameters laid out as their gradients are, bf16 copies, the parameters
    that lie outside, and the gradients' zeroing.  A subclass keeps its state in the entries of `_flat` (`_lay_out_state`) and
    builds the native plan that steps them (`_make_plan`)."""

    def __init__(self, params, defaults, bf16_shadow: bool):
        super().__init__(params, defaults)
        self._flat: List[dict] = []
        self._attached_ids = set()
        self._plan = None   # the flat buffers, laid out for the native step
        self._loose = None  # (the groups' parameters, [(group index, parameter outside the flat buffers)])
        self._steps = 0
        self.kernel_launches = 0
        # bf16 copies of the weights, written by the step kernel (see bagua_core_b200.ops.shadow)
        self.bf16_shadow = bf16_shadow
        self.shadows_valid = False
        self._shadowed: List[torch.Tensor] = []

    def _group_runs(self, bucket):
        """[(start, end, group index)] over a bucket's flat elements: maximal runs of consecutive
        parameters that belong to the same parameter group, so that each run is stepped with its own
        group's learning rate, momentum and weight decay.  With one group (or a bucket whose parameters
        all share a group) that is one run over the whole bucket, padding included."""
        group_of = {id(p): gi for gi, g in enumerate(self.param_groups) for p in g["params"]}
        runs, off = [], 0
        for t in bucket.tensors:
            n = t.owner.numel()
            gi = group_of.get(id(t.owner))
            if gi is None:
                raise RuntimeError(f"parameter of bucket tensor `{t.name}` is not in this optimizer")
            if runs and runs[-1][2] == gi:
                runs[-1][1] = off + n
            else:
                runs.append([off, off + n, gi])
            off += n
        if runs:
            runs[-1][1] = bucket.flattened.numel()  # the padding (zero gradient, zero weights) rides along
        return [tuple(r) for r in runs]

    # called by BaguaModule after it has built gradient buckets
    def bagua_attach(self, bm):
        self._flat.clear()
        self._attached_ids.clear()
        self._loose = None
        for p in self._shadowed:
            p._bagua_bf16 = None
        self._shadowed.clear()
        self.shadows_valid = False
        for b in bm.bagua_buckets:
            if b.flattened is not None and b.flattened.dtype == torch.float32 and all(
                    t.kind == "weight" for t in b.tensors):
                # weights are the bucket: give the gradients the same flat layout
                flat_g = torch.zeros_like(b.flattened)
                off = 0
                for t in b.tensors:
                    p = t.owner
                    n = p.numel()
                    p.grad = flat_g[off:off + n].as_strided(tuple(p.shape), tuple(p.stride()))
                    self._attached_ids.add(id(p))
                    off += n
                self._flat.append({"p": b.flattened, "g": flat_g, "runs": self._group_runs(b)})
                self._lay_out_state(self._flat[-1], b)
                continue
            if b.flattened is None or any(t.kind != "grad" for t in b.tensors):
                continue
            if b.flattened.dtype != torch.float32:
                continue
            flat_p = torch.zeros_like(b.flattened)
            off = 0
            with torch.no_grad():
                for t in b.tensors:
                    p = t.owner
                    n = p.numel()
                    shape, stride = tuple(p.shape), tuple(p.stride())
                    if tuple(t.tensor.stride()) != stride:
                        raise RuntimeError("parameter and gradient layouts differ; cannot share a flat layout")
                    flat_p[off:off + n].as_strided(shape, stride).copy_(p)
                    p.set_(flat_p.untyped_storage(), off, shape, stride)
                    self._attached_ids.add(id(p))
                    off += n
            entry = {"p": flat_p, "g": b.flattened, "runs": self._group_runs(b)}
            self._lay_out_state(entry, b)
            if self.bf16_shadow:
                from ..ops.shadow import BF16Shadow

                flat_h = torch.zeros_like(flat_p, dtype=torch.bfloat16)
                off = 0
                for t in b.tensors:
                    p = t.owner
                    n = p.numel()
                    p._bagua_bf16 = BF16Shadow(flat_h[off:off + n].as_strided(tuple(p.shape), tuple(p.stride())), self)
                    self._shadowed.append(p)
                    off += n
                entry["h"] = flat_h
            self._flat.append(entry)
        self._plan = self._make_plan() if self._flat else None

    def _stream(self):
        return _C.current_stream(self._flat[0]["p"])

    def _loose_params(self):
        """[(group, parameter)] outside the flat buffers; looked up again when the groups' parameters are others than at
        the last look (an added, replaced or moved parameter, a loaded state)."""
        groups, known = self.param_groups, self._loose
        if known is None or len(groups) != len(known[0]):
            known = None
        else:
            for g, ps in zip(groups, known[0]):
                now = g["params"]
                if len(now) != len(ps) or not all(map(is_, now, ps)):
                    known = None
                    break
        if known is None:
            known = self._loose = ([list(g["params"]) for g in groups],
                                   [(gi, p) for gi, g in enumerate(groups) for p in g["params"] if id(p) not in self._attached_ids])
        return [(groups[gi], p) for gi, p in known[1]] if known[1] else ()

    def _validate_shadows(self):
        """The bf16 copies equal the parameters now: remember the parameters' versions."""
        for p in self._shadowed:
            p._bagua_bf16.version = p._version
        self.shadows_valid = True

    @torch.no_grad()
    def refresh_bf16(self):
        """Recomputes the bf16 copies from the parameters (after the weights were changed by something
        the copies cannot notice, or to use them before the first step)."""
        for f in self._flat:
            if "h" in f:
                f["h"].copy_(f["p"])
        if self._shadowed:
            self._validate_shadows()

    def zero_grad(self, set_to_none: bool = False):
        """Zero the flat gradient buffers in one launch; gradients stay views
        of the bucket (never set to None, which would detach them from the bucket)."""
        if self._plan is not None:
            self._plan.zero_grad(self._stream())
        for _, p in self._loose_params():
            if p.grad is not None:
                p.grad.zero_()


class FlatSGD(_FlatOptimizer):
    """torch.optim.SGD semantics (momentum, dampening, weight decay, Nesterov).

    Before `with_bagua` attaches it (or for parameters outside any bucket) it updates
    parameter by parameter with the same kernel.  A parameter that was laid out in a flat buffer is stepped
    with it, in the group that it was in then, as long as the buffer lives.

    `bf16_shadow=True`: for buckets of gradients (algorithms that do not communicate weights) the
    step kernel also writes every updated parameter rounded to bf16 into a second flat buffer, and
    each parameter gets a view of it (`bagua_core_b200.ops.shadow`); `ConvBiasReLU`,
    `ConvBiasReLUPool` and `ShadowLinear` under bf16 autocast then read their weights from there
    instead of casting the fp32 master weights in every forward pass.  After changing a parameter
    by other means than this optimizer or torch's in-place ops, call `refresh_bf16()`."""

    def __init__(self, params, lr: float = 1e-3, momentum: float = 0.0, dampening: float = 0.0,
                 weight_decay: float = 0.0, nesterov: bool = False, bf16_shadow: bool = False):
        if nesterov and (momentum <= 0 or dampening != 0):
            raise ValueError("Nesterov momentum requires a momentum and zero dampening")
        defaults = dict(lr=lr, momentum=momentum, dampening=dampening, weight_decay=weight_decay, nesterov=nesterov)
        super().__init__(params, defaults, bf16_shadow)

    def _lay_out_state(self, entry, bucket):
        entry["m"] = torch.zeros_like(entry["p"])

    def _make_plan(self):
        # one entry per run of parameters that share a parameter group (usually one per bucket), stepped with
        # its own group's hyperparameters as they are at the time (schedulers change them in place)
        plan = _C.SgdPlan()
        for f in self._flat:
            for lo, hi, gi in f["runs"]:
                plan.add(f["p"][lo:hi], f["g"][lo:hi], f["m"][lo:hi], f["h"][lo:hi] if "h" in f else None, gi)
        return plan

    @torch.no_grad()
    def step(self, closure=None):
        loss = closure() if closure is not None else None
        if self._plan is not None:
            self.kernel_launches += self._plan.step(
                [(g["lr"], g["momentum"], g["dampening"], g["weight_decay"], g["nesterov"]) for g in self.param_groups],
                self._stream())
        if self._shadowed and not self.shadows_valid:
            self._validate_shadows()
        for group, p in self._loose_params():
            if p.grad is None:
                continue
            st = self.state[p]
            first = "momentum_buffer" not in st
            if first:
                st["momentum_buffer"] = torch.zeros_like(p, memory_format=torch.preserve_format)
            buf = st["momentum_buffer"]
            same_layout = (p.dtype == torch.float32 and _is_dense(p) and p.grad.dtype == torch.float32
                           and p.grad.stride() == p.stride() and buf.stride() == p.stride())
            if not same_layout:
                # layouts differ (e.g. autograd produced a contiguous gradient for a
                # channels_last weight): element-wise torch math is layout-agnostic
                d = p.grad.add(p, alpha=group["weight_decay"]) if group["weight_decay"] else p.grad
                if group["momentum"]:
                    if first:
                        buf.copy_(d)
                    else:
                        buf.mul_(group["momentum"]).add_(d, alpha=1 - group["dampening"])
                    d = d.add(buf, alpha=group["momentum"]) if group["nesterov"] else buf
                p.add_(d, alpha=-group["lr"])
                continue
            s = torch.cuda.current_stream().cuda_stream if p.is_cuda else 0
            # dense tensors with equal strides can be updated as flat memory
            pv = torch.as_strided(p, (p.numel(),), (1,))
            gv = torch.as_strided(p.grad, (p.numel(),), (1,))
            mv = torch.as_strided(st["momentum_buffer"], (p.numel(),), (1,))
            _C.k_sgd_momentum_flat(pv, gv, mv, group["lr"], group["momentum"], group["dampening"],
                                   group["weight_decay"], group["nesterov"], first, s)
            self.kernel_launches += 1
        self._steps += 1
        return loss


class FlatAdamW(_FlatOptimizer):
    """torch.optim.AdamW semantics: Adam whose weight decay is taken from the weights, not through the gradient.

    Laid out by `with_bagua` as `FlatSGD` is: one kernel steps all buckets, and with `bf16_shadow=True` also writes the bf16
    copies of the weights.  Parameters outside any bucket are stepped as lists, a launch for each kind of them, and may be
    float32, float16 or bfloat16.  Each parameter counts its own steps.

    `state_bits=8`: the moments are held in 8 bits (`bagua_core_b200.ops.adamw`), 2 bytes per parameter instead of 8;
    `seed` is that of their rounding, the same on all ranks.  `moments(p)` reads a parameter's moments.

    The state of a parameter (`state[p]`, `state_dict()`, `load_state_dict()`) is `step` with `exp_avg` and `exp_avg_sq`, to which
    8 bits add `scales`; it goes along when a bucket is laid out (again).  Where a parameter's elements then follow each other in another
    order in memory, 8-bit moments are rounded anew, as other elements share their scales.

    `capturable=True`: the steps of the flat buffers are counted on the device, so that `step()` can be captured into a CUDA
    graph and replayed (with the learning rates that it was captured with).  It is captured again after a new layout, and after a
    loaded state whose parameters differ in their numbers of steps.  Otherwise, and for parameters outside any bucket, a step that
    is being captured is refused."""

    def __init__(self, params, lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, bf16_shadow: bool = False, state_bits: int = 32, seed: int = 0, capturable: bool = False):
        if lr < 0 or eps < 0 or weight_decay < 0 or not all(0 <= b < 1 for b in betas):
            raise ValueError("AdamW needs lr, eps and weight_decay of 0 or more and betas from 0 to below 1")
        if state_bits not in (8, 32):
            raise ValueError("moments are held in 8 or 32 bits")
        if not 0 <= seed < 1 << 64:
            raise ValueError("the seed is a number of 64 bits")
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay), bf16_shadow)
        self.state_bits = state_bits
        self.seed = seed
        self.capturable = capturable
        self._device_steps = None                # of the plan's groups, where they are counted on the device
        self._earlier_device_steps = []          # that a graph may still hold
        self._plan_groups: List[List[int]] = []  # [parameter group, steps done] of each group of the plan
        self._plan_group_of = {}                 # id(parameter in the flat buffers) -> index of its group there
        self._plan_tensors = 0

    # ---- state -----------------------------------------------------------------------
    def _new_state(self, p):
        if self.state_bits == 8:
            m, v, scales = adamw_state8(p)
            return {"step": 0, "exp_avg": m, "exp_avg_sq": v, "scales": scales}
        m, v = (torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format, requires_grad=False) for _ in range(2))
        return {"step": 0, "exp_avg": m, "exp_avg_sq": v}

    def bagua_attach(self, bm):
        self._sync_steps()
        super().bagua_attach(bm)

    @torch.no_grad()
    def _lay_out_state(self, entry, bucket):
        # a flat buffer for each moment; in 8 bits with scales for each parameter, whose blocks end where it ends
        dtype = torch.uint8 if self.state_bits == 8 else torch.float32
        flat = {k: torch.zeros_like(entry["p"], dtype=dtype) for k in ("exp_avg", "exp_avg_sq")}
        off = 0
        entry["owners"] = []
        for t in bucket.tensors:
            p, n = t.owner, t.owner.numel()
            state = {"step": 0, **{k: f[off:off + n].as_strided(tuple(p.shape), tuple(p.stride())) for k, f in flat.items()}}
            if self.state_bits == 8:
                state["scales"] = torch.zeros(2, (n + MOMENT8_BLOCK - 1) // MOMENT8_BLOCK, device=p.device)
            if p in self.state and "step" in self.state[p]:  # steps taken before, here or in another layout
                self._copy_state(state, self.state[p])
            self.state[p] = state
            entry["owners"].append((p, off, off + n))
            off += n
        entry["m"], entry["v"] = flat["exp_avg"], flat["exp_avg_sq"]

    def _make_plan(self):
        plan = _C.AdamWPlan()
        self._plan_groups, self._plan_group_of, self._plan_tensors = [], {}, 0
        known = {}
        group_of = {id(p): gi for gi, g in enumerate(self.param_groups) for p in g["params"]}

        def plan_group(gi, step):
            if (gi, step) not in known:
                known[gi, step] = len(self._plan_groups)
                self._plan_groups.append([gi, step])
            return known[gi, step]

        for f in self._flat:
            flats = [f["p"], f["g"], f["m"], f["v"]]
            pieces = []  # [from, to, group in the plan, scales]
            for p, lo, hi in f["owners"]:
                state = self.state[p]
                k = self._plan_group_of[id(p)] = plan_group(group_of[id(p)], state["step"])
                if self.state_bits == 32 and pieces and pieces[-1][2] == k:
                    pieces[-1][1] = hi  # a run of parameters that are stepped alike is one piece
                else:
                    pieces.append([lo, hi, k, state.get("scales")])
            for lo, hi, k, scales in pieces:
                plan.add(*(x[lo:hi] for x in flats), scales, f["h"][lo:hi] if "h" in f else None, k)
            self._plan_tensors += len(pieces)
            plan.add_grad_buffer(f["g"])
        if self.capturable:
            steps = torch.tensor([done for _, done in self._plan_groups], dtype=torch.int64, device=self._flat[0]["p"].device)
            if self._device_steps is not None and self._device_steps.shape == steps.shape and self._device_steps.device == steps.device:
                self._device_steps.copy_(steps)  # a captured step goes on counting there
            else:
                if self._device_steps is not None:
                    self._earlier_device_steps.append(self._device_steps)
                self._device_steps = steps
        return plan

    def _sync_steps(self):
        """The steps that the plan has counted, into the parameters' state."""
        if self._device_steps is not None and self._flat:
            for group, done in zip(self._plan_groups, self._device_steps.tolist()):
                group[1] = done
        for f in self._flat:
            for p, _, _ in f["owners"]:
                if p in self.state:
                    self.state[p]["step"] = self._plan_groups[self._plan_group_of[id(p)]][1]

    def _check_state(self, p, saved):
        """Throws unless `saved` can be the state of `p`."""
        held = torch.uint8 if self.state_bits == 8 else torch.float32
        want = {"exp_avg": (p.shape, held), "exp_avg_sq": (p.shape, held)}
        if self.state_bits == 8:
            want["scales"] = ((2, (p.numel() + MOMENT8_BLOCK - 1) // MOMENT8_BLOCK), torch.float32)
        if set(saved) != {"step", *want} or any(saved[k].shape != shape for k, (shape, _) in want.items()):
            raise ValueError(f"the saved state of a parameter is not that of moments in {self.state_bits} bits of its size")
        for k, (_, dtype) in want.items():
            if saved[k].dtype != dtype:
                raise ValueError(f"the saved moments are {saved[k].dtype}, not {dtype}")
        if self.state_bits == 8 and not (_is_dense(saved["exp_avg"]) and _same_order(saved["exp_avg"], saved["exp_avg_sq"])):
            raise ValueError("the saved codes of 8-bit moments have gaps, or two orders: which of them share a scale goes by their places in memory")
        if int(saved["step"]) < 0:
            raise ValueError(f"the saved state of a parameter has taken {int(saved['step'])} steps")

    def _copy_state(self, to, saved):
        if self.state_bits == 8:
            _copy_moments8(to, saved)
        else:
            for k in ("exp_avg", "exp_avg_sq"):
                to[k].copy_(saved[k])
        to["step"] = int(saved["step"])

    def state_dict(self):
        self._sync_steps()
        return super().state_dict()

    def load_state_dict(self, state_dict):
        """A state that does not fit is refused before anything has changed."""
        # The framework's own loads everything but the moments, which it would cast to the parameters' type: they are taken out behind
        # the hooks in front of it, and put in ahead of the hooks behind it.
        held, saved = dict(self.state), {}

        def take(_, state_dict):
            ids = [i for g in state_dict["param_groups"] for i in g["params"]]
            for i, p in zip(ids, (p for g in self.param_groups for p in g["params"])):
                if i in state_dict["state"]:
                    self._check_state(p, state_dict["state"][i])
                    saved[id(p)] = state_dict["state"][i]
            return {**state_dict, "state": {}}

        hooks = [self.register_load_state_dict_pre_hook(take),
                 self.register_load_state_dict_post_hook(lambda _: self._put_state(held, saved), prepend=True)]
        try:
            super().load_state_dict(state_dict)
        finally:
            for h in hooks:
                h.remove()

    @torch.no_grad()
    def _put_state(self, held, saved):
        for p in (p for g in self.param_groups for p in g["params"]):
            flat = id(p) in self._attached_ids
            if id(p) not in saved and not flat:
                continue  # made by its first step
            state = held[p] if flat else self._new_state(p)
            self._copy_state(state, saved[id(p)] if id(p) in saved else self._new_state(p))
            self.state[p] = state
        if self._flat:
            self._plan = self._make_plan()

    def moments(self, p) -> Tuple[torch.Tensor, torch.Tensor]:
        """(first, second) moment of a parameter that was stepped or laid out, in fp32."""
        s = self.state.get(p, {})
        if "step" not in s:
            raise KeyError("the parameter has no moments yet: it was neither stepped nor laid out")
        if self.state_bits == 32:
            return s["exp_avg"].clone(), s["exp_avg_sq"].clone()
        m, v = (torch.empty_like(s["exp_avg"], dtype=torch.float32) for _ in range(2))
        adamw_read8([s["exp_avg"]], [s["exp_avg_sq"]], [s["scales"]], [m], [v])
        return m, v

    # ---- stepping --------------------------------------------------------------------
    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        if self._plan is not None:
            values = []
            for gi, done in self._plan_groups:
                g = self.param_groups[gi]
                values.append((g["lr"], *g["betas"], g["eps"], g["weight_decay"]))
            if self.capturable:
                self.kernel_launches += self._plan.step(values, self._device_steps.add_(1), self.seed)
            else:
                self.kernel_launches += self._plan.step(values, [done + 1 for _, done in self._plan_groups], self.seed)
                for group in self._plan_groups:
                    group[1] += 1
        if self._shadowed and not self.shadows_valid:
            self._validate_shadows()
        self._step_loose()
        self._steps += 1
        return loss

    def _step_loose(self):
        kinds, back = {}, []  # one call for each kind of parameters
        for group, p in self._loose_params():
            if p.grad is None:
                continue
            if p not in self.state or "step" not in self.state[p]:
                self.state[p] = self._new_state(p)
            state, g, w = self.state[p], p.grad, p
            if not _is_dense(p):
                w = p.contiguous()
                back.append((p, w))
            m = state["exp_avg"]
            if m.stride() != w.stride():  # the parameter has been laid out anew since
                new = self._new_state(w)
                self._copy_state(new, state)
                state.update(new)
            if g.layout == torch.strided and g.stride() != w.stride():
                g = torch.empty_like(w, dtype=g.dtype).copy_(g)
            key = (id(group), state["step"], p.device, p.dtype, g.dtype)
            kinds.setdefault(key, (group, []))[1].append((w, g, state))
        first = self._plan_tensors
        for (_, done, *_), (group, parts) in kinds.items():
            self.kernel_launches += adamw_step(
                [w for w, _, _ in parts], [g for _, g, _ in parts], [s["exp_avg"] for _, _, s in parts], [s["exp_avg_sq"] for _, _, s in parts],
                step=done + 1, lr=group["lr"], betas=group["betas"], eps=group["eps"], weight_decay=group["weight_decay"],
                scales=[s["scales"] for _, _, s in parts] if self.state_bits == 8 else None, seed=self.seed, first_index=first)
            first += len(parts)
            for _, _, s in parts:
                s["step"] += 1
        for p, w in back:
            p.copy_(w)
