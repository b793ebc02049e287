"""AdamW over all tensors of a model in one launch, with states in 32 or 8 bits.

The reference trains with torch.optim.AdamW; this optimizer has its update rule
and its lr, betas, eps and weight_decay (no amsgrad, maximize, capturable or
differentiable).  States live in one allocation each for all parameters,
every tensor starting on a multiple of 128 elements.
"""
from __future__ import annotations

from typing import Optional

import torch

from .fp8 import BLOCK, F8, _ops
from .functional import _SUPPORTED


class AdamW(torch.optim.Optimizer):
    """p -= lr wd p; m = b1 m + (1 - b1) g; v = b2 v + (1 - b2) g^2;
    p -= lr / (1 - b1^t) m / (sqrt(v) / sqrt(1 - b2^t) + eps).

    params: float32 or bfloat16 CUDA tensors of one device, contiguous, with
      gradients of their own type; parameter groups may set lr, betas, eps and
      weight_decay.  A parameter without a gradient is left alone.
    state_bits: 32, or 8: m and the square root of v as e4m3 codes with a
      float32 scale for each 128 elements (2.06 bytes a parameter in place of
      8).  8-bit states and bfloat16 parameters are rounded up or down with the
      probability of the part cut off, so that changes smaller than a step of
      the format are not lost; a second moment above zero is never held as zero.
    seed: of that rounding; equal seeds and equal inputs give equal results.

    A step takes its count, learning rate and noise from the host, so it is refused
    while a CUDA graph is being captured: capture the passes before it alone.

    ``exp_avg``, ``exp_avg_sq`` and, with 8 bits, ``exp_avg_scale`` and
    ``exp_avg_sq_scale`` are the states of all parameters (``offsets`` says
    where each begins); with 8 bits ``exp_avg_sq`` holds the codes of sqrt(v)."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, state_bits: int = 32, seed: int = 0):
        if state_bits not in (8, 32):
            raise ValueError("state_bits must be 8 or 32")
        self._check_group({"lr": lr, "betas": betas, "eps": eps, "weight_decay": weight_decay})
        self.state_bits = state_bits
        self.seed = int(seed) & 0xFFFFFFFF
        self.offsets = {}
        self._total = 0
        self._plans = []          # of each group: where its states begin, sizes, steps taken
        self.exp_avg = self.exp_avg_sq = None
        self.exp_avg_scale = self.exp_avg_sq_scale = None
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay))

    @staticmethod
    def _check_group(g) -> None:
        if not g["lr"] >= 0 or not g["eps"] >= 0 or not g["weight_decay"] >= 0:
            raise ValueError("lr, eps and weight_decay must not be negative")
        if len(g["betas"]) != 2 or not all(0 <= b < 1 for b in g["betas"]):
            raise ValueError("betas must be two numbers in [0, 1)")

    def add_param_group(self, param_group) -> None:
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            self._check_group(group)
            for p in group["params"]:
                if not p.is_cuda:
                    raise ValueError("AdamW runs on CUDA parameters only (no CPU fallback)")
                if p.dtype not in _SUPPORTED:
                    raise ValueError("parameters must be float32 or bfloat16")
                if not p.is_contiguous():
                    raise ValueError("parameters must be contiguous")
                if p.device != self._device():
                    raise ValueError("all parameters must be on one device")
        except ValueError:
            self.param_groups.pop()
            raise
        before = self._total
        for p in group["params"]:
            self.offsets[p] = self._total
            self._total += -(-p.numel() // BLOCK) * BLOCK
        params = group["params"]
        steps = torch.zeros(len(params), dtype=torch.int32)
        self._plans.append(([self.offsets[p] for p in params], [p.numel() for p in params], steps))
        for p, s in zip(params, steps):
            self.state[p]["step"] = s      # a view: the step counts it up
        self._grow(self._total - before)

    def _device(self) -> Optional[torch.device]:
        return next((p.device for g in self.param_groups for p in g["params"]), None)

    def _grow(self, n: int) -> None:
        dev = self._device()
        if dev is None:                        # groups without parameters so far
            return
        dtype = torch.float32 if self.state_bits == 32 else F8
        new = {"exp_avg": torch.zeros(n, dtype=dtype, device=dev),
               "exp_avg_sq": torch.zeros(n, dtype=dtype, device=dev)}
        if self.state_bits == 8:
            new["exp_avg_scale"] = torch.zeros(n // BLOCK, dtype=torch.float32, device=dev)
            new["exp_avg_sq_scale"] = torch.zeros(n // BLOCK, dtype=torch.float32, device=dev)
        for name, t in new.items():
            old = getattr(self, name)
            if old is not None:
                b = old.view(torch.uint8) if old.dtype == F8 else old
                t = torch.cat((b, t.view(b.dtype))).view(dtype if old.dtype == F8 else old.dtype)
            setattr(self, name, t)

    _KEPT = ("state_bits", "seed", "offsets", "_total", "_plans", "exp_avg", "exp_avg_sq", "exp_avg_scale",
             "exp_avg_sq_scale")

    def __getstate__(self):
        kept = {name: getattr(self, name) for name in self._KEPT}
        if self.state_bits == 8:               # as bytes: pickle knows no 8-bit float storage
            kept.update({n: None if kept[n] is None else kept[n].view(torch.uint8) for n in ("exp_avg", "exp_avg_sq")})
        return {**super().__getstate__(), **kept}

    def __setstate__(self, state) -> None:
        super().__setstate__(state)
        if self.state_bits == 8 and self.exp_avg is not None:
            self.exp_avg, self.exp_avg_sq = self.exp_avg.view(F8), self.exp_avg_sq.view(F8)
        for group, (_, _, steps) in zip(self.param_groups, self._plans):
            for p, s in zip(group["params"], steps):
                self.state[p]["step"] = s      # views again: a copy of a view is none

    def set_state(self, step: int, exp_avg: torch.Tensor, exp_avg_sq: torch.Tensor,
                  exp_avg_scale: Optional[torch.Tensor] = None,
                  exp_avg_sq_scale: Optional[torch.Tensor] = None) -> None:
        """Takes over states of every parameter (in the layout of ``exp_avg``
        and the others, whose memory is kept and written) after ``step`` steps."""
        for name, t in (("exp_avg", exp_avg), ("exp_avg_sq", exp_avg_sq),
                        ("exp_avg_scale", exp_avg_scale), ("exp_avg_sq_scale", exp_avg_sq_scale)):
            have = getattr(self, name)
            if have is None and t is None:
                continue
            if (have is None or t is None or t.shape != have.shape or t.dtype != have.dtype
                    or t.device != have.device or not t.is_contiguous()
                    or t.data_ptr() % 16 != 0):
                raise ValueError(f"{name} must be a contiguous tensor like this optimizer's own")
        self.exp_avg, self.exp_avg_sq = exp_avg, exp_avg_sq
        self.exp_avg_scale, self.exp_avg_sq_scale = exp_avg_scale, exp_avg_sq_scale
        for _, _, steps in self._plans:
            steps.fill_(int(step))

    def state_dict(self):
        for hook in self._optimizer_state_dict_pre_hooks.values():
            hook(self)
        groups, index = [], {}
        for g in self.param_groups:
            for p in g["params"]:
                index[p] = len(index)
            groups.append({**{k: v for k, v in g.items() if k != "params"},
                           "params": [index[p] for p in g["params"]]})
        out = {"state": {index[p]: {"step": int(self.state[p]["step"]), "first": self.offsets[p]} for p in index},
               "param_groups": groups, "state_bits": self.state_bits, "seed": self.seed,
               "exp_avg": self.exp_avg, "exp_avg_sq": self.exp_avg_sq,
               "exp_avg_scale": self.exp_avg_scale, "exp_avg_sq_scale": self.exp_avg_sq_scale}
        for hook in self._optimizer_state_dict_post_hooks.values():
            other = hook(self, out)
            out = out if other is None else other
        return out

    def load_state_dict(self, state_dict) -> None:
        state_dict = dict(state_dict)          # a hook may change it
        for hook in self._optimizer_load_state_dict_pre_hooks.values():
            other = hook(self, state_dict)
            state_dict = state_dict if other is None else other
        if state_dict["state_bits"] != self.state_bits:
            raise ValueError(f"the states were kept in {state_dict['state_bits']} bits, this "
                             f"optimizer has {self.state_bits}")
        groups = state_dict["param_groups"]
        if [len(g["params"]) for g in groups] != [len(g["params"]) for g in self.param_groups]:
            raise ValueError("the parameter groups differ from this optimizer's")
        params = [p for g in self.param_groups for p in g["params"]]
        order = [i for g in groups for i in g["params"]]
        if any(state_dict["state"][i]["first"] != self.offsets[p] for i, p in zip(order, params)):
            raise ValueError("the parameters' sizes differ from this optimizer's")
        dev = self._device()
        names = ("exp_avg", "exp_avg_sq", "exp_avg_scale", "exp_avg_sq_scale")
        self.set_state(0, *(None if state_dict[n] is None else state_dict[n].to(dev, copy=True)
                            for n in names))
        for i, p in zip(order, params):
            self.state[p]["step"].fill_(int(state_dict["state"][i]["step"]))
        for g, s in zip(self.param_groups, groups):
            g.update({k: v for k, v in s.items() if k != "params"})
        self.seed = int(state_dict["seed"]) & 0xFFFFFFFF
        for hook in self._optimizer_load_state_dict_post_hooks.values():
            hook(self)

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group, (first, sizes, steps) in zip(self.param_groups, self._plans):
            if not sizes:
                continue
            b1, b2 = group["betas"]
            _ops.adamw(group["params"], first, sizes, steps, self.exp_avg, self.exp_avg_sq,
                       self.exp_avg_scale, self.exp_avg_sq_scale, group["lr"], b1, b2, group["eps"],
                       group["weight_decay"], self.seed, self.state_bits)
        return loss
