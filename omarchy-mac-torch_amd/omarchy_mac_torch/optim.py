"""Fused optimizers by default on the device (reference: omarchy_mac_torch/optim.py).

torch.optim.SGD, Adam and AdamW pick their per-tensor (foreach) implementation unless told otherwise; on this device
the fused one (`_fused_sgd_` / `_fused_adam_` / `_fused_adamw_`, one multi-tensor launch per step) is cheaper. PyTorch
has no hook for a device's preferred implementation, so `enable_fused_defaults` wraps the constructors: a call whose
parameters are all on the device, and that chose neither fused= nor foreach= (nor differentiable=, nor a tensor lr),
gets fused=True. `keeps_torch_default` says why a call is left alone. OMARCHY_MAC_TORCH_FUSED_OPTIM=0 leaves
torch.optim untouched.

AdamW is this package's own, for language models: parameters in float32 or bfloat16, these with float32 master copies, and
states in 8 bits or in 32 (no counterpart in the reference).
"""

import functools
import itertools
import os

import torch

from omarchy_mac_torch import hip_ops
from omarchy_mac_torch.native import DEVICE

_MARK = "_omarchy_mac_torch_fused_default"
DEFAULT_CLASSES = (torch.optim.SGD, torch.optim.Adam, torch.optim.AdamW)


def _tensors_of(params):
    """The tensors of a constructor's params argument: tensors, or param-group dicts (whose "params" is a tensor or
    an iterable of them)."""
    for item in params:
        if not isinstance(item, dict):
            yield item
        elif isinstance(item["params"], torch.Tensor):
            yield item["params"]
        else:
            yield from item["params"]


def keeps_torch_default(tensors, options):
    """Why a constructor call keeps torch's own choice of implementation, or None when it defaults to fused=True."""
    if not tensors:
        return "no parameters"
    if not all(isinstance(t, torch.Tensor) and t.device.type == DEVICE for t in tensors):
        return "parameters not all on the device"
    chosen = [k for k in ("fused", "foreach") if options.get(k) is not None]
    if chosen:
        return f"{chosen[0]}= given by the caller"
    if options.get("differentiable", False):
        return "differentiable=True"
    if isinstance(options.get("lr"), torch.Tensor):
        return "a tensor learning rate"
    return None


def fused_default(cls):
    """Wraps cls.__init__ (once) so that device-resident parameter sets default to fused=True."""
    original = cls.__init__
    if getattr(original, _MARK, False):
        return cls

    @functools.wraps(original)
    def __init__(self, params, *args, **kwargs):
        params = list(params)  # an iterator is consumed here and by the original constructor
        if keeps_torch_default(list(_tensors_of(params)), kwargs) is None:
            kwargs["fused"] = True
        original(self, params, *args, **kwargs)

    setattr(__init__, _MARK, True)
    cls.__init__ = __init__
    return cls


def enable_fused_defaults(classes=DEFAULT_CLASSES):
    """Applies fused_default to each class (the package does this on import unless OMARCHY_MAC_TORCH_FUSED_OPTIM=0);
    returns the classes."""
    return [fused_default(cls) for cls in classes]


class AdamW(torch.optim.Optimizer):
    """AdamW over hip_ops.adamw: one launch for each 32 parameters of a group and type. Parameters in float32 or bfloat16, on the
    device (or on torch.cuda); gradients of their type.

    state_bits: 8 (e4m3 with a scale for each block of 128, two bytes and 1/16 a parameter; the second moment as its root) or 32
    (eight bytes). masters: bfloat16 parameters keep a float32 copy, which is what is updated (so what else is written to a parameter
    after its first step is lost at the next); without one, an update below half a parameter's last place is lost. lr may be a
    one-element float32 tensor on the device. The step's counters are on the device, so a step may be captured into a graph once it
    has run eagerly (which makes the states).

    load_state_dict takes torch.optim.AdamW's too: its states go on in 32 bits, those of further parameters are of this optimizer's
    state_bits."""

    def __init__(self, params, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, weight_decay=0.01, *, state_bits=8, masters=True,
                 maximize=False):
        defaults = dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits, masters=masters,
                        maximize=maximize)
        self._check(defaults)
        super().__init__(params, defaults)

    @staticmethod
    def _check(g):
        if g["state_bits"] not in (8, 32):
            raise ValueError(f"state_bits: expected 8 or 32, got {g['state_bits']!r}")
        if not isinstance(g["lr"], torch.Tensor) and not g["lr"] >= 0:
            raise ValueError(f"lr: expected at least 0, got {g['lr']!r}")
        if not all(0 <= b < 1 for b in g["betas"]):
            raise ValueError(f"betas: expected from 0 to below 1, got {g['betas']!r}")
        if not g["eps"] >= 0 or not g["weight_decay"] >= 0:
            raise ValueError(f"eps, weight_decay: expected at least 0, got {g['eps']!r}, {g['weight_decay']!r}")

    def add_param_group(self, param_group):
        self._check({**self.defaults, **param_group})
        super().add_param_group(param_group)

    @staticmethod
    def _new_state(p, group):
        state = {"step": torch.zeros((), dtype=torch.float32, device=p.device)}
        held = torch.float8_e4m3fn if group["state_bits"] == 8 else torch.float32
        for name in ("exp_avg", "exp_avg_sq"):
            state[name] = torch.zeros_like(p, dtype=torch.float32).to(held)
            if group["state_bits"] == 8:
                state[name + "_scale"] = torch.zeros(-(-p.numel() // 128), dtype=torch.float32, device=p.device)
        if group["masters"] and p.dtype == torch.bfloat16:
            state["master"] = p.detach().float()
        return state

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            by_type = {}
            for p in group["params"]:
                if p.grad is None:
                    continue
                if p.grad.is_sparse:
                    raise TypeError("AdamW: sparse gradients are not covered")
                state = self.state[p]
                if not state:
                    state = self.state[p] = self._new_state(p, group)
                # (a state is in 8 bits or not, and with a master copy or not, as it was made or loaded)
                by_type.setdefault((p.dtype, p.device, "exp_avg_scale" in state, "master" in state), []).append(p)
            for ps in by_type.values():
                def of(name):
                    return [self.state[p][name] for p in ps] if name in self.state[ps[0]] else None

                steps = of("step")
                torch._foreach_add_(steps, 1)
                try:
                    hip_ops.adamw(ps, [p.grad for p in ps], of("exp_avg"), of("exp_avg_sq"), steps, of("exp_avg_scale"),
                                  of("exp_avg_sq_scale"), of("master"), lr=group["lr"], betas=group["betas"], eps=group["eps"],
                                  weight_decay=group["weight_decay"], maximize=group["maximize"])
                except Exception:  # refused: no step has been made
                    torch._foreach_add_(steps, -1)
                    raise
        return loss

    def __setstate__(self, state):
        super().__setstate__(state)
        for group in self.param_groups:  # (loaded ones may be torch.optim.AdamW's, without this class's options)
            for name, value in self.defaults.items():
                group.setdefault(name, value)

    def load_state_dict(self, state_dict):
        # (torch casts states to their parameter's type; these keep their own. Its hooks may put another dictionary in this one's place,
        # and what they do to the states afterwards stays.)
        taken = []

        def take(_, d):
            if any(g.get("amsgrad") for g in d["param_groups"]):
                raise ValueError("AdamW: amsgrad is not covered")
            taken.append(d)

        hooks = (self.register_load_state_dict_pre_hook(take),
                 self.register_load_state_dict_post_hook(lambda _: self._take_states(taken[-1]), prepend=True))
        try:
            super().load_state_dict(state_dict)
        finally:
            for hook in hooks:
                hook.remove()

    def _take_states(self, state_dict):
        ids = itertools.chain.from_iterable(g["params"] for g in state_dict["param_groups"])
        params = itertools.chain.from_iterable(g["params"] for g in self.param_groups)
        for i, p in zip(ids, params):
            for name, t in state_dict["state"].get(i, {}).items():
                t = t.detach().to(p.device, copy=True)
                self.state[p][name] = t if t.dtype in (torch.float32, torch.float8_e4m3fn) else t.float()


if os.environ.get("OMARCHY_MAC_TORCH_FUSED_OPTIM", "1") != "0":
    enable_fused_defaults()
