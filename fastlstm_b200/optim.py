"""AdamW over all of a model's tensors in one launch a data type, its states in 32 or 8 bits (csrc/adamw.cu; what a call does on the
host is csrc/host_adamw.cpp)."""
from __future__ import annotations

import math
from itertools import chain
from typing import Optional

import torch
import torch.optim.optimizer as _global_hooks

from . import _lib
from .language import _whole

_CAPTURE = "AdamW: take a step or load a state before a capture, which would begin with new states at every replay"
_LEAST, _MOST = torch.finfo(torch.float32).tiny, torch.finfo(torch.float32).max
BLOCK = 256                  # elements of a tensor, in row-major order, that share a scale in 8-bit states


def _check_group(group):
    """Refuses what a parameter group's step would be refused for."""
    lr, betas = group["lr"], group["betas"]
    if isinstance(lr, torch.Tensor):
        if lr.numel() != 1 or not lr.is_floating_point():
            raise ValueError("lr as a tensor must be one floating-point element")
    elif not 0 <= lr <= _MOST:
        raise ValueError(f"lr must be at least 0 and finite in 32 bits, got {lr!r}")
    if len(betas) != 2 or not all(0 <= b < 1 for b in betas):
        raise ValueError(f"betas must be two numbers in [0, 1), got {betas!r}")
    for name in ("eps", "weight_decay"):
        if not 0 <= group[name] <= _MOST:
            raise ValueError(f"{name} must be at least 0 and finite in 32 bits, got {group[name]!r}")
    if 0 < group["eps"] < _LEAST:
        raise ValueError(f"eps must be 0 or at least 2^-126 (its reciprocal is held in 32 bits), got {group['eps']!r}")
    _whole(group["seed"], "seed", 0, 2 ** 64 - 1)


class AdamW(torch.optim.Optimizer):
    """Adam with decoupled weight decay, on contiguous CUDA parameters in float32, float16 or bfloat16:

        m = beta1 m + (1 - beta1) g     v = beta2 v + (1 - beta2) g^2
        p = p (1 - lr weight_decay) - lr / (1 - beta1^t) m / (sqrt(v / (1 - beta2^t)) + eps)

    state_bits=32 keeps m and v as `exp_avg` and `exp_avg_sq` in float32; state dicts of torch.optim.AdamW can be loaded.
    state_bits=8 keeps m and sqrt(v) as `exp_avg` and `exp_avg_sq_root` in float8_e4m3fn, times `exp_avg_scale` and
    `exp_avg_sq_root_scale`, one for every 256 elements (their largest magnitude / 448).  Numbers between two of e4m3 go up with the
    probability of what would be cut off, a function of `seed`, step, tensor and element: means are kept, and a run repeats
    bit by bit.  A gradient that is not finite spoils the 256 elements that it shares scales with (see max_norm).
    master_weights: 16-bit parameters have their weight in float32 in the state (`master`) and are it, rounded.  Without, steps that
    are less than half the distance of two 16-bit numbers are lost.
    max_norm: gradients are multiplied by min(1, max_norm / (norm + 1e-6)), the norm taken over all parameters (on one device) and
    found in `grad_norm`.  Where it is not finite the step does nothing and does not count.
    eps is 0 or at least 2^-126; parameters share no memory.  A step that is refused (ValueError) is refused for all groups, before anything changes.
    lr may be a CUDA tensor of one float32, read when the step runs: a captured step can be replayed with another rate.  (Take a
    step, or load a state, before a capture; step counts lie in device memory and go on in replays.)"""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, *, state_bits: int = 32,
                 master_weights: bool = True, max_norm: Optional[float] = None, seed: int = 0):
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits!r}")
        if max_norm is not None and not (max_norm >= _LEAST and math.isfinite(max_norm)):
            raise ValueError(f"max_norm must be positive (at least 2^-126) and finite, got {max_norm!r}")
        self.state_bits, self.master_weights = int(state_bits), bool(master_weights)
        self.max_norm = None if max_norm is None else float(max_norm)
        super().__init__(params, dict(lr=lr, betas=tuple(betas), eps=eps, weight_decay=weight_decay, seed=_whole(seed, "seed", 0, 2 ** 64 - 1)))

    def add_param_group(self, param_group):
        if isinstance(param_group, dict):
            _check_group({**self.defaults, **param_group})
            if "seed" in param_group:
                param_group["seed"] = int(param_group["seed"])
        super().add_param_group(param_group)

    def __getstate__(self):
        return {**super().__getstate__(), "state_bits": self.state_bits, "master_weights": self.master_weights, "max_norm": self.max_norm}

    # ------------------------------------------------------------------ state
    def _format(self, p):
        """The state's tensors as {name: (shape, dtype)}."""
        moment = torch.float32 if self.state_bits == 32 else torch.float8_e4m3fn
        f = {"exp_avg": (p.shape, moment), "exp_avg_sq" if self.state_bits == 32 else "exp_avg_sq_root": (p.shape, moment), "step": ((), torch.int64)}
        if self.state_bits == 8:
            blocks = ((p.numel() + BLOCK - 1) // BLOCK,)
            f["exp_avg_scale"] = f["exp_avg_sq_root_scale"] = (blocks, torch.float32)
        if self.master_weights and p.dtype != torch.float32:
            f["master"] = (p.shape, torch.float32)
        return f

    def _start(self, p):
        if p.is_cuda and torch.cuda.is_current_stream_capturing():
            raise RuntimeError(_CAPTURE)
        self.state[p] = {name: p.detach().float() if name == "master" else torch.zeros(shape, dtype=dtype, device=p.device)
                         for name, (shape, dtype) in self._format(p).items()}
        return self.state[p]

    def load_state_dict(self, state_dict):
        """Takes copies in the types that this optimizer keeps.  Masters that the state does not have are the parameters."""
        state_dict = dict(state_dict)
        for hook in list(self._optimizer_load_state_dict_pre_hooks.values()):
            changed = hook(self, state_dict)
            state_dict = state_dict if changed is None else changed
        self._load(state_dict)
        for hook in list(self._optimizer_load_state_dict_post_hooks.values()):
            hook(self)

    @torch.no_grad()
    def _load(self, state_dict):
        ids = chain.from_iterable(g["params"] for g in state_dict["param_groups"])
        params = dict(zip(ids, chain.from_iterable(g["params"] for g in self.param_groups)))
        loaded = {}
        for k, saved in state_dict["state"].items():
            if k not in params:
                raise ValueError("loaded state dict has a state of a parameter that is in none of its groups")
            p, loaded[k] = params[k], {}
            for name, (shape, dtype) in self._format(p).items():
                if name == "master" and name not in saved:
                    loaded[k][name] = p.detach().float()
                    continue
                if name not in saved:
                    raise ValueError(f"loaded state has no {name}: it is of an optimizer with other state_bits")
                t = torch.as_tensor(saved[name])
                if tuple(t.shape) != tuple(shape):
                    raise ValueError(f"{name} of the loaded state has shape {tuple(t.shape)}, expected {tuple(shape)}")
                if (t.dtype == torch.float8_e4m3fn) != (dtype == torch.float8_e4m3fn):
                    raise ValueError(f"{name} of the loaded state has dtype {t.dtype}, expected {dtype}: it is of an optimizer with other state_bits")
                loaded[k][name] = torch.empty(shape, dtype=dtype, device=p.device).copy_(t)
        for g in state_dict["param_groups"]:
            _check_group({**self.defaults, **g})
            if g.get("amsgrad") or g.get("maximize"):
                raise ValueError("loaded state is of an optimizer with amsgrad or maximize, which are not there")
            if g.get("decoupled_weight_decay") is False and g.get("weight_decay"):
                raise ValueError("loaded state is of an optimizer that adds weight decay to its gradients")
        # (torch would cast states to the parameters' types; hooks run around all of this)
        hooks = self._optimizer_load_state_dict_pre_hooks, self._optimizer_load_state_dict_post_hooks
        self._optimizer_load_state_dict_pre_hooks, self._optimizer_load_state_dict_post_hooks = type(hooks[0])(), type(hooks[1])()
        try:
            super().load_state_dict({**state_dict, "state": {}})
        finally:
            self._optimizer_load_state_dict_pre_hooks, self._optimizer_load_state_dict_post_hooks = hooks
        for g in self.param_groups:
            for name, value in self.defaults.items():
                g.setdefault(name, value)
            g["seed"] = int(g["seed"])
        for k, s in loaded.items():
            self.state[params[k]] = s
            if params[k].is_cuda:
                self._scratch(params[k].device.index)

    # ------------------------------------------------------------------ step
    def _scratch(self, device):
        """(the counter that launches use, {norm, factor}) of a device."""
        kept = self.__dict__.setdefault("_kept", {})
        if device not in kept:
            if torch.cuda.is_current_stream_capturing():
                raise RuntimeError(_CAPTURE)
            at = torch.device("cuda", device)
            kept[device] = (torch.zeros(1, dtype=torch.int32, device=at), torch.zeros(2, dtype=torch.float32, device=at))
        return kept[device]

    @property
    def grad_norm(self) -> Optional[torch.Tensor]:
        """The norm of all gradients in the last step (before they were clipped), where max_norm is set; None before the first.  A copy: the
        next step writes its own."""
        return None if self.__dict__.get("_norm") is None else self._norm[0].clone()

    def _step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        norm = _lib.host().adamw_step(self.param_groups, self.state, self.state_bits, self.master_weights, self.max_norm, self._start, self._scratch)
        if norm is not None:
            self._norm = norm
        return loss

    _step_with_hooks = torch.optim.Optimizer.profile_hook_step(_step)

    def step(self, closure=None):
        # what torch puts around every step (a profiler's record, hooks: 12 us) only where it is listened to
        if (self._optimizer_step_pre_hooks or self._optimizer_step_post_hooks or _global_hooks._global_optimizer_pre_hooks
                or _global_hooks._global_optimizer_post_hooks or torch.autograd.profiler._is_profiler_enabled):
            return self._step_with_hooks(closure)
        return self._step(closure)

    step.hooked = True
