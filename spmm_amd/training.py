"""The operators beside the sparse product in a training step, on the GPU:
layer norm, softmax cross entropy and AdamW (include/tca_train.h).

    h = layer_norm(c, weight, bias, out_dtype=torch.bfloat16)   # C of a product -> B of the next
    loss = cross_entropy(logits, target)                        # differentiable; target -100: no label
    loss, dlogits = cross_entropy_grad(logits, target)          # both from one pass over the logits
    opt = AdamW(model.parameters(), lr=1e-3, state_bits=8)      # one launch per 48 tensors

They are torch operators of namespace spmm_amd (torch.ops.spmm_amd.layer_norm and
so on), defined with their autograd formulas in lib/libtcatorch.so
(csrc/torch_training.cpp); this module loads it, gives the operators their fake
kernels (so that torch.compile traces them as opaque nodes) and their Python
forms.  There is no fallback: without the library the import fails, and tensors
that are not on a GPU raise ValueError.  Derivatives are first derivatives in reverse
mode: second ones, forward mode (torch.autograd.forward_ad, torch.func.jvp) and
torch.func.grad raise an error.

Work runs on the current stream of the tensors' device; workspaces come from
torch's allocator.  No counterpart in the reference, which has no training path.
"""
from __future__ import annotations

import math
import os
from typing import Optional, Tuple

import torch

from . import _lib  # loads libtcaspmm.so, which the operators call
from ._lib import TCA_ADAMW_BLOCK, TCA_LOSS_MEAN, TCA_LOSS_NONE, TCA_LOSS_SUM

__all__ = ["layer_norm", "LayerNorm", "cross_entropy", "cross_entropy_grad", "AdamW"]

LIB_PATH = os.path.join(os.path.dirname(_lib.LIB_PATH), "libtcatorch.so")
if not os.path.exists(LIB_PATH):
    raise ImportError(f"libtcatorch.so not found at {LIB_PATH}; build it first (python -c 'import __graft_entry__ as g; "
                      "g.build()' or make -C spmm_amd). There is no CPU fallback.")
torch.ops.load_library(LIB_PATH)
_ops = torch.ops.spmm_amd

_REDUCTIONS = {"none": TCA_LOSS_NONE, "sum": TCA_LOSS_SUM, "mean": TCA_LOSS_MEAN}


# ------------------------------------------------------------------ layer norm
@torch.library.register_fake("spmm_amd::layer_norm")
def _layer_norm_fake(x, weight, bias, eps, out_dtype):
    return x.new_empty(x.shape, dtype=out_dtype)


@torch.library.register_fake("spmm_amd::layer_norm_stats")
def _layer_norm_stats_fake(x, weight, bias, eps, out_dtype):
    return x.new_empty(x.shape, dtype=out_dtype), x.new_empty((math.prod(x.shape[:-1]), 2), dtype=torch.float32)


@torch.library.register_fake("spmm_amd::layer_norm_backward")
def _layer_norm_backward_fake(dy, x, weight, stats, need_dx, need_dw, need_db, weight_dtype):
    return (x.new_empty(x.shape if need_dx else 0), x.new_empty(x.shape[-1] if need_dw else 0, dtype=weight_dtype),
            x.new_empty(x.shape[-1] if need_db else 0, dtype=weight_dtype))


def layer_norm(x: torch.Tensor, weight: Optional[torch.Tensor] = None, bias: Optional[torch.Tensor] = None,
               eps: float = 1e-5, out_dtype: Optional[torch.dtype] = None) -> torch.Tensor:
    """(x - mean) / sqrt(var + eps) * weight + bias over the last axis of x
    (1 to 16384 entries; any distance between rows), differentiable in x, weight
    and bias.  x is float32, float16 or bfloat16; weight and bias (each may be
    left out) have its dtype, the output's, or float32.  out_dtype: the output's
    dtype where x is float32 (a product's result going into 16 bits); else x's."""
    return _ops.layer_norm(x, weight, bias, eps, out_dtype)


class LayerNorm(torch.nn.Module):
    """layer_norm over a last axis of `width` entries, with weight and bias."""

    def __init__(self, width: int, eps: float = 1e-5, bias: bool = True, out_dtype: Optional[torch.dtype] = None,
                 device=None, dtype=None):
        super().__init__()
        self.eps, self.out_dtype = eps, out_dtype
        self.weight = torch.nn.Parameter(torch.ones(width, device=device, dtype=dtype))
        self.bias = torch.nn.Parameter(torch.zeros(width, device=device, dtype=dtype)) if bias else None

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        return layer_norm(x, self.weight, self.bias, self.eps, self.out_dtype)


# --------------------------------------------------------------- cross entropy
def _loss_fake(logits, reduction):
    return logits.new_empty((logits.shape[0],) if reduction == TCA_LOSS_NONE else (), dtype=torch.float32)


@torch.library.register_fake("spmm_amd::cross_entropy")
def _cross_entropy_fake(logits, target, ignore_index, reduction):
    return _loss_fake(logits, reduction)


@torch.library.register_fake("spmm_amd::cross_entropy_stats")
def _cross_entropy_stats_fake(logits, target, ignore_index, reduction):
    return (_loss_fake(logits, reduction), logits.new_empty((logits.shape[0], 2), dtype=torch.float32),
            logits.new_empty(() if reduction == TCA_LOSS_MEAN else (0,), dtype=torch.float32))


@torch.library.register_fake("spmm_amd::cross_entropy_backward")
def _cross_entropy_backward_fake(gloss, logits, target, ignore_index, stats, norm):
    return logits.new_empty(logits.shape)


@torch.library.register_fake("spmm_amd::cross_entropy_grad")
def _cross_entropy_grad_fake(logits, target, ignore_index, reduction, scale):
    return logits.new_empty((), dtype=torch.float32), logits.new_empty(logits.shape)


def _reduction(name: str, reduction: str, allowed) -> int:
    if reduction not in allowed:
        raise ValueError(f"{name}: reduction must be one of {', '.join(allowed)}; got {reduction!r}")
    return _REDUCTIONS[reduction]


def cross_entropy(logits: torch.Tensor, target: torch.Tensor, ignore_index: int = -100,
                  reduction: str = "mean") -> torch.Tensor:
    """Softmax cross entropy of logits (rows x classes) with int64 or int32
    targets, in float32, differentiable in the logits.  Rows whose target is
    ignore_index count for nothing and are not read; the mean is over the others
    (0 over none).  A target outside the classes gives NaN.  reduction: "mean",
    "sum" or "none"."""
    return _ops.cross_entropy(logits, target, ignore_index, _reduction("cross_entropy", reduction,
                                                                       ("mean", "sum", "none")))


def cross_entropy_grad(logits: torch.Tensor, target: torch.Tensor, ignore_index: int = -100, reduction: str = "mean",
                       scale: float = 1.0) -> Tuple[torch.Tensor, torch.Tensor]:
    """(loss, gradient of scale * loss with respect to the logits) in one pass
    over the logits, for a training step that needs both at once:

        loss, dlogits = cross_entropy_grad(logits, target)
        logits.backward(dlogits)

    The loss is not multiplied by `scale` (a loss scale of 16-bit training); the
    gradient is, before it is rounded to the logits' dtype.  reduction: "mean" or
    "sum".  Both results are constants to autograd, in reverse and in forward mode."""
    return _ops.cross_entropy_grad(logits, target, ignore_index,
                                   _reduction("cross_entropy_grad", reduction, ("mean", "sum")), scale)


# ----------------------------------------------------------------------- AdamW
class AdamW(torch.optim.Optimizer):
    """AdamW with decoupled weight decay, all tensors of one type and step count
    in one launch (48 tensors at most each).

    Parameters are contiguous GPU tensors in float32, float16 or bfloat16.  16-bit
    ones have a float32 master copy in the state, which the step updates and
    rounds into the parameter.  Arithmetic is float32.  Gradients are taken as they are:
    no factor undoes a loss scale, and no step is skipped for a gradient that is not
    finite.

    state_bits 32: state[p] holds "step" (int), "exp_avg" and "exp_avg_sq"
    (float32, p's shape), and "master" (float32) for 16-bit p.
    state_bits 8: "exp_avg" and "exp_avg_rms" (the root of the second moment) as
    float8_e4m3fn [blocks, 256], the last block padded with zeros, and their
    blocks' float32 scales "exp_avg_scale" and "exp_avg_rms_scale".

    A parameter whose gradient is None keeps its values, states and step count.
    Step counts live on the host, and a step cannot be captured into a graph, unless
    capturable is set: then "step" is an int64 GPU tensor, and a captured step goes
    on counting at each replay (the group's other settings are those of the
    capture).  Create the states before a capture, by a step or init_states()."""

    _STATES = {32: ("exp_avg", "exp_avg_sq"), 8: ("exp_avg", "exp_avg_rms", "exp_avg_scale", "exp_avg_rms_scale")}

    def __init__(self, params, lr: float = 1e-3, betas: Tuple[float, float] = (0.9, 0.999), eps: float = 1e-8,
                 weight_decay: float = 1e-2, state_bits: int = 32, capturable: bool = False):
        self._check_settings(lr, betas, eps, weight_decay, state_bits)
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay, state_bits=state_bits,
                                      capturable=capturable))

    def _check_settings(self, lr, betas, eps, weight_decay, state_bits) -> None:
        if state_bits not in self._STATES:
            raise ValueError(f"AdamW: state_bits must be 32 or 8, got {state_bits}")
        if not (eps >= 0 and lr >= 0 and weight_decay >= 0 and all(0 <= b < 1 for b in betas)):
            raise ValueError(f"AdamW: lr {lr}, betas {betas}, eps {eps}, weight_decay {weight_decay}")
        if state_bits == 8 and not eps > 0:
            raise ValueError("AdamW: states in 8 bits need eps above 0")

    def add_param_group(self, param_group) -> None:
        """torch.optim.Optimizer.add_param_group; a parameter given twice, of which torch
        only warns, is refused: a launch would update it twice at once."""
        super().add_param_group(param_group)
        group = self.param_groups[-1]
        try:
            self._check_settings(*(group[name] for name in ("lr", "betas", "eps", "weight_decay", "state_bits")))
            if len({id(p) for p in group["params"]}) != len(group["params"]):
                raise ValueError("AdamW: a parameter is in its group more than once")
        except ValueError:
            self.param_groups.pop()
            raise

    def _new_state(self, p: torch.Tensor, bits: int, capturable: bool) -> dict:
        if not p.is_cuda:
            raise ValueError(f"AdamW: parameters must be GPU tensors (no CPU fallback), got {p.device}")
        state = {"step": torch.zeros((), dtype=torch.int64, device=p.device) if capturable else 0}
        if p.dtype != torch.float32:
            state["master"] = p.detach().to(torch.float32)
        if bits == 32:
            for name in self._STATES[32]:
                state[name] = torch.zeros_like(p, dtype=torch.float32, requires_grad=False)
        else:
            blocks = -(-p.numel() // TCA_ADAMW_BLOCK)
            for name in ("exp_avg", "exp_avg_rms"):
                state[name] = torch.zeros((blocks, TCA_ADAMW_BLOCK), dtype=torch.uint8,
                                          device=p.device).view(torch.float8_e4m3fn)
                state[name + "_scale"] = torch.zeros(blocks, dtype=torch.float32, device=p.device)
        return state

    def init_states(self) -> None:
        """Creates the states of all parameters that have none yet."""
        for group in self.param_groups:
            for p in group["params"]:
                if not self.state[p]:
                    self.state[p].update(self._new_state(p, group["state_bits"], group["capturable"]))

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        for group in self.param_groups:
            batches = {}  # (device, dtype, step of the host) -> (parameters, gradients, states)
            bits, capturable = group["state_bits"], group["capturable"]
            for p in group["params"]:
                g = p.grad
                if g is None:
                    continue
                state = self.state[p]
                if not state:
                    if capturable and torch.cuda.is_current_stream_capturing():
                        raise RuntimeError("AdamW: states must be there before a capture: take a step or call init_states()")
                    state.update(self._new_state(p, bits, capturable))
                batch = batches.setdefault((p.device, p.dtype, None if capturable else state["step"]), ([], [], []))
                batch[0].append(p)
                batch[1].append(g)
                batch[2].append(state)
            for (device, dtype, step), (params, grads, states) in batches.items():
                names = self._STATES[bits] if dtype == torch.float32 else self._STATES[bits] + ("master",)
                held = [s[name] for name in names for s in states]
                settings = (group["lr"], *group["betas"], group["eps"], group["weight_decay"])
                if capturable:
                    _ops.adamw_step_device_(params, grads, held, [s["step"] for s in states], bits, *settings)
                    continue
                if torch.cuda.is_current_stream_capturing():
                    raise RuntimeError("AdamW: a step cannot be captured into a graph unless capturable is set")
                _ops.adamw_step_(params, grads, held, bits, step + 1, *settings)
                for state in states:
                    state["step"] = step + 1
        return loss

    # settings of torch's AdamW: those that would change a step and what they have to be here, and
    # those that say how torch computes it
    _FIXED = {"maximize": False, "amsgrad": False, "differentiable": False, "decoupled_weight_decay": True}
    _THEIRS = (*_FIXED, "foreach", "fused")

    def _check_loaded(self, state_dict) -> None:
        """ValueError where a saved state would mean something else here."""
        for group, saved in zip(self.param_groups, state_dict["param_groups"]):
            for name in ("lr", "betas", "eps", "weight_decay"):
                if name not in saved:
                    raise ValueError(f"AdamW: the loaded group has no {name}: it is not of an AdamW optimizer")
            for name, value in self._FIXED.items():
                if saved.get(name, value) != value:
                    raise ValueError(f"AdamW: a state with {name}={saved[name]} cannot be loaded: only {name}={value} is "
                                     "supported")
            bits = saved.get("state_bits", group["state_bits"])
            if bits not in self._STATES:
                raise ValueError(f"AdamW: state_bits must be 32 or 8, got {bits}")
            for i, p in zip(saved["params"], group["params"]):
                if not state_dict["state"].get(i):
                    continue
                names = {"step", *self._STATES[bits]} | ({"master"} if p.dtype != torch.float32 else set())
                if set(state_dict["state"][i]) != names:
                    raise ValueError(f"AdamW: the loaded state of a {p.dtype} parameter must hold {sorted(names)} for states "
                                     f"in {bits} bits, got {sorted(state_dict['state'][i])}")

    def load_state_dict(self, state_dict) -> None:
        """torch.optim.Optimizer.load_state_dict, with the states in their own
        dtypes (the base class casts them to their parameters').  Takes torch's
        AdamW's for float32 parameters and 32-bit states too: its step counts are
        tensors, state_bits and capturable stay this optimizer's, and options that
        change its step (maximize, amsgrad, differentiable, coupled decay) are refused."""
        self._check_loaded(state_dict)
        own = [{name: group[name] for name in ("state_bits", "capturable")} for group in self.param_groups]
        super().load_state_dict(state_dict)
        for group, settings in zip(self.param_groups, own):
            if "state_bits" not in group:  # torch's
                group.update(settings)
            group.setdefault("capturable", settings["capturable"])
            for name in self._THEIRS:
                group.pop(name, None)
        ids = [i for group in state_dict["param_groups"] for i in group["params"]]
        params = [p for group in self.param_groups for p in group["params"]]
        capturable = [group["capturable"] for group in self.param_groups for _ in group["params"]]
        for i, p, c in zip(ids, params, capturable):
            if i not in state_dict["state"]:
                continue
            state = {k: v.detach().to(device=p.device, copy=True) if isinstance(v, torch.Tensor) else v
                     for k, v in state_dict["state"][i].items()}
            if "step" in state:
                step = int(state["step"])
                state["step"] = torch.tensor(step, device=p.device) if c else step
            self.state[p] = state
