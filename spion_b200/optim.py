"""AdamW over many tensors at once (csrc/adamw.cu: a launch for the counts and one for the values), with moments in 32 or in 8 bits.

The moments of a set of tensors lie in two arrays, tensor after tensor, each from a multiple of ``BLOCK`` on (``places``); 8-bit moments have a scale per
``BLOCK`` values.  ``adamw_step`` is the step on such arrays, ``AdamW`` the optimizer that keeps them.  Beside the update a step can clip the gradients by
value and write 16-bit copies of the parameters (``layernorm.register_shadows``) in the same pass.
"""
from __future__ import annotations

import copy
from collections import defaultdict

import torch

from . import _ops
from ._lib import SpionError, check, lib

BLOCK = 256
# entries of torch.optim.AdamW's groups that say how it computes: a state is loaded without them
_SWITCHES = ("amsgrad", "maximize", "foreach", "capturable", "differentiable", "fused", "decoupled_weight_decay")


def places(tensors):
    """Where each tensor's moments begin, and how many places all of them take."""
    at, out = 0, []
    for t in tensors:
        out.append(at)
        at += -(-t.numel() // BLOCK) * BLOCK
    return out, at


def adamw_step(params, grads, exp_avg, exp_avg_sq, steps, *, scales=None, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2,
               clip_value=None, seed: int = 0, copies=None):
    """One step on params (contiguous tensors of one type), in place.  grads: a gradient of the parameter's type and shape each, or None (the tensor and its
    count are left alone).  exp_avg, exp_avg_sq: fp32 arrays of ``places(params)[1]`` values, or float8_e4m3fn and float8_e5m2 with ``scales``, the pair of
    their fp32 scales.  steps: fp32, one count per tensor, raised by the step.  lr: a number, or an fp32 CUDA scalar that is read when the step runs.
    copies: None, or per parameter a 16-bit tensor that receives it (or None).  ``seed`` and the counts decide how 8-bit moments are rounded.
    A step after a bounded wait of a kernel gave up changes nothing (``spion_linear_status``)."""
    lr_dev = None
    if isinstance(lr, torch.Tensor):
        lr, lr_dev = (0.0, lr) if lr.is_cuda else (float(lr), None)
    m_scale, v_scale = (None, None) if scales is None else scales
    if clip_value is not None and not clip_value >= 0:
        raise SpionError(f"adamw_step: clip_value is {clip_value}")
    _ops.ops.adamw_step(params, grads, exp_avg, exp_avg_sq, steps, m_scale, v_scale, lr_dev, copies, lr, betas[0], betas[1], eps, weight_decay,
                        -1.0 if clip_value is None else clip_value, seed & 0xFFFFFFFF)


class _Moments:
    """The arrays of one set of tensors: those of a parameter group that have the same type and device."""

    def __init__(self, params, bits):
        self.params, self.bits = params, bits
        dev = params[0].device
        self.at, total = places(params)
        eight = bits == 8
        self.exp_avg = torch.zeros(total, dtype=torch.float8_e4m3fn if eight else torch.float32, device=dev)
        self.exp_avg_sq = torch.zeros(total, dtype=torch.float8_e5m2 if eight else torch.float32, device=dev)
        self.scales = tuple(torch.ones(total // BLOCK, device=dev) for _ in range(2)) if eight else None
        self.steps = torch.zeros(len(params), device=dev)

    def __getstate__(self):                     # (torch does not pickle 8-bit floating-point types by themselves)
        bytes_ = {k: self.__dict__[k].view(torch.uint8) for k in ("exp_avg", "exp_avg_sq") if self.bits == 8}
        return self.__dict__ | bytes_

    def __setstate__(self, state):
        self.__dict__.update(state)
        if self.bits == 8:
            self.exp_avg, self.exp_avg_sq = self.exp_avg.view(torch.float8_e4m3fn), self.exp_avg_sq.view(torch.float8_e5m2)

    def state_of(self, i):
        p, at = self.params[i], self.at[i]
        s = {"step": self.steps[i], "exp_avg": self.exp_avg[at:at + p.numel()].view(p.shape), "exp_avg_sq": self.exp_avg_sq[at:at + p.numel()].view(p.shape)}
        if self.scales is not None:
            blocks = slice(at // BLOCK, (at + p.numel() + BLOCK - 1) // BLOCK)
            s["exp_avg_scales"], s["exp_avg_sq_scales"] = self.scales[0][blocks], self.scales[1][blocks]
        return s


class AdamW(torch.optim.Optimizer):
    """``torch.optim.AdamW`` on the library's kernels: two launches per parameter group, type and device (256 tensors each).

    ``state_bits=8``: moments in 8 bits with a scale per 256 values, 2 bytes a parameter instead of 8, rounded at random (repeatable: ``seed``).
    ``clip_value``: gradients are clipped to [-c, c] as they are read (``torch.nn.utils.clip_grad_value_``; ``.grad`` is left as it is).
    State dicts have one entry per parameter with torch's names; with 32 bits they are exchangeable with ``torch.optim.AdamW``'s (not those with amsgrad or
    maximize).  Moments belong to their parameters: groups may be added, removed and moved, not mixed anew.
    A step can be captured in a CUDA graph once a step has been taken; ``lr`` may be an fp32 CUDA scalar, which a replay reads."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, *, state_bits: int = 32, clip_value=None, seed: int = 0):
        if state_bits not in (8, 32):
            raise ValueError(f"AdamW: state_bits is {state_bits}, 8 or 32 are served")
        if not isinstance(lr, torch.Tensor) and not lr >= 0:
            raise ValueError(f"AdamW: lr is {lr}")
        if not all(0 <= b < 1 for b in betas) or not eps >= 0 or not weight_decay >= 0:
            raise ValueError(f"AdamW: betas {betas}, eps {eps}, weight_decay {weight_decay}")
        if clip_value is not None and not clip_value >= 0:
            raise ValueError(f"AdamW: clip_value is {clip_value}")
        self.state_bits, self.seed = state_bits, seed
        self._moments, self._copies = [], {}             # of each group that has taken a step: its parameters, their arrays by type and device
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, clip_value=clip_value))

    def __getstate__(self):                     # what the base class keeps, with the arrays in place of their views
        kept = super().__getstate__() | {k: self.__dict__[k] for k in ("state_bits", "seed", "_moments", "_copies")}
        kept["state"] = defaultdict(dict)
        return kept

    def __setstate__(self, state):
        super().__setstate__(state)
        for _, sets in self._moments:
            for m in sets:
                for i, p in enumerate(m.params):
                    self.state[p] = m.state_of(i)

    def write_copies(self, params, copies):
        """Every step also writes each of ``copies`` (16-bit, of its parameter's shape) for the parameter in ``params``."""
        for p, c in zip(params, copies, strict=True):
            self._copies[p] = c

    def _sets(self, g):
        """The moments of group number g, made at its first step (or when a state is loaded).  They belong to its parameters, not to its place among the groups."""
        params = self.param_groups[g]["params"]
        ids = [id(p) for p in params]                    # (of tensors that self._moments keeps)
        for held, have in self._moments:
            if [id(p) for p in held] == ids:
                return have
        if any(p in self.state for p in params):
            raise SpionError(f"AdamW: the parameters of group {g} have changed since its first step")
        kinds = {}
        for p in params:
            if not p.is_cuda:
                raise SpionError("AdamW: a parameter is not on a GPU (there is no CPU path)")
            kinds.setdefault((p.dtype, p.device), []).append(p)
        if torch.cuda.is_current_stream_capturing():
            raise SpionError("AdamW: take a step before one is captured (the moments would be made anew by every replay)")
        have = [_Moments(ps, self.state_bits) for ps in kinds.values()]
        self._moments.append((list(params), have))
        for m in have:
            for i, p in enumerate(m.params):
                self.state[p] = m.state_of(i)
        return have

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        number = 0
        for g, group in enumerate(self.param_groups):
            if not group["params"]:
                continue
            for m in self._sets(g):
                copies = [self._copies.get(p) for p in m.params] if self._copies else None
                adamw_step(m.params, [p.grad for p in m.params], m.exp_avg, m.exp_avg_sq, m.steps, scales=m.scales, lr=group["lr"], betas=group["betas"],
                           eps=group["eps"], weight_decay=group["weight_decay"], clip_value=group["clip_value"], seed=self.seed + 0x51ED270B * number,
                           copies=copies)
                number += 1
        return loss

    def check_device_status(self) -> None:
        """Raise if a bounded wait of the library's kernels has given up since it was last asked (steps after that changed nothing).  Synchronises;
        under a capture it asks nothing."""
        if torch.cuda.is_current_stream_capturing():
            return
        for device in {p.device for held, _ in self._moments for p in held}:
            with torch.cuda.device(device):
                check(lib.spion_linear_status(1), "device status")

    def state_dict(self):
        """As the base class's; raises if steps have been left out (``check_device_status``)."""
        self.check_device_status()
        return super().state_dict()

    def load_state_dict(self, state_dict):
        """Moments are copied into the arrays that this optimizer keeps; they have to be of its ``state_bits``."""
        state_dict = dict(state_dict)
        for hook in self._optimizer_load_state_dict_pre_hooks.values():
            other = hook(self, state_dict)
            state_dict = state_dict if other is None else other
        groups, state = state_dict["param_groups"], state_dict["state"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("the optimizer state is not that of these parameter groups")
        for g in groups:
            for k in ("amsgrad", "maximize"):
                if g.get(k):
                    raise ValueError(f"a state of AdamW with {k} cannot be continued: it is not served")
            if g.get("weight_decay") and not g.get("decoupled_weight_decay", True):
                raise ValueError("a state whose weight decay is not decoupled (Adam's) cannot be continued")
        want = {"step", "exp_avg", "exp_avg_sq"} | ({"exp_avg_scales", "exp_avg_sq_scales"} if self.state_bits == 8 else set())
        plan = []
        for g, saved in enumerate(groups):
            if not saved["params"]:
                continue
            sets = self._sets(g)
            mine = {p: m.state_of(i) for m in sets for i, p in enumerate(m.params)}
            for number, p in zip(saved["params"], self.param_groups[g]["params"]):
                entry = state.get(number)
                for k, dst in mine[p].items():
                    if entry is None:
                        plan.append((dst, None))
                        continue
                    src = torch.as_tensor(entry[k]) if k in entry and want <= set(entry) else None
                    # (torch's moments of 16-bit parameters are in their type)
                    types = (dst.dtype, torch.bfloat16, torch.float16) if self.state_bits == 32 else (dst.dtype,)
                    if src is None or src.shape != dst.shape or (k != "step" and src.dtype not in types):
                        raise ValueError(f"the state of parameter {number} ({k}) is not that of an AdamW of {self.state_bits} bits and this shape")
                    plan.append((dst, src))
        with torch.no_grad():
            for dst, src in plan:
                if src is None:                                       # a parameter that had taken no step
                    dst.copy_(torch.zeros_like(dst))
                else:
                    dst.copy_(src)
        for mine, saved in zip(self.param_groups, groups):
            mine.update({k: copy.deepcopy(v) for k, v in saved.items() if k != "params" and k not in _SWITCHES})
        for hook in self._optimizer_load_state_dict_post_hooks.values():
            hook(self)
