"""The dense layers around the embedding path on the library's kernels (csrc/dense_cuda.cu, called from csrc/dense_torch.cpp).

fused_linear   y = act(x W^T + b) + residual, differentiable
fused_mlp      a run of such layers as one node of the autograd graph: one call per direction
gave_up        whether a bounded wait inside the kernels has ever run out (outputs are then not numbers)
FusedMLP       the Sequential of Linear and activation modules that the reference's create_mlp builds
               (dlrm_s_pytorch.py:213-251), computed by fused_mlp; same parameters, same state_dict

Tensors are CUDA tensors of one type (fp32, bf16 or fp16); sums are fp32.  Kernels go to the current stream of the tensors'
device.  The gradients are those of first order: differentiating them again raises, and so do forward-mode derivatives
and calls that a trace (torch.jit.trace, make_fx) records.  Captured into a CUDA graph, forward and
backward follow torch's rules for whole-network capture (warm-up on a side stream, no autograd graph of the same leaves alive
from outside the capture)."""
from __future__ import annotations

import contextlib
import ctypes

import torch
import torch.nn as nn

from . import _lib

_lib.load()   # (the extension is linked against the library: what is wrong with that is said first)
try:
    from . import _dense_torch
except ImportError as e:
    raise ImportError(f"cafe_b200/_dense_torch.so cannot be loaded ({e}); run: python -m cafe_b200.build") from e

ACTIVATIONS = {"none": 0, "relu": 1, "sigmoid": 2, "gelu": 3, "silu": 4}


def fused_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, activation: str = "none",
                 residual: torch.Tensor | None = None) -> torch.Tensor:
    """act(x W^T + b) + residual.  x [..., K], weight [N, K], bias [N]; residual broadcasts to [..., N]; activation is one of
    none, relu, sigmoid, gelu (with erf) and silu.  x, weight and residual may be slices of wider tensors (any pitch
    between rows).  For the backward the call keeps x, weight and, with an activation, its derivative (16 bits beside bf16, with
    the range of bf16, else fp32); of a ReLU without residual the output.  In
    16 bits the gradient of the pre-activation is rounded to the tensors' type before its two products, as by torch's own layers (in
    fp16 it overflows with a gradient above 58 000 where a GELU's or SiLU's derivative is above 1)."""
    act = ACTIVATIONS.get(activation)
    if act is None:
        raise ValueError(f"fused_linear: activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    return _dense_torch.linear(x, weight, bias, residual, act)


def fused_mlp(x: torch.Tensor, weights, biases, activations) -> torch.Tensor:
    """Layer after layer of act(x W^T + b): weights [N_l, N_{l-1}], biases [N_l] or None, activations by name (see
    fused_linear).  The values are those of fused_linear layer by layer; between the layers they are held in x's type."""
    acts = [ACTIVATIONS.get(a) for a in activations]
    if None in acts:
        raise ValueError(f"fused_mlp: activations must be among {sorted(ACTIVATIONS)}, got {list(activations)!r}")
    return _dense_torch.mlp(x, list(weights), list(biases), acts)


def gave_up(device=None) -> int:
    """How many of the two kinds of kernel here have, since the library was loaded, ended a wait that ran out on this device (0: none).  Every
    wait inside them has an end, about a second; what it waited for is then stored as NaN, and this says that the NaN came from
    there.  Waits for the device; not while a stream of it is being captured."""
    count = ctypes.c_int32(0)
    with torch.cuda.device(device) if device is not None else contextlib.nullcontext():
        _lib.check(_lib.load().cafe_linear_gave_up(ctypes.byref(count)), "cafe_linear_gave_up")
    return count.value


_MODULES = {nn.ReLU: "relu", nn.Sigmoid: "sigmoid", nn.SiLU: "silu", nn.Identity: "none"}


def _module_activation(m: nn.Module) -> str:
    if type(m) is nn.GELU and m.approximate == "none":
        return "gelu"
    if type(m) not in _MODULES:
        raise ValueError(f"FusedMLP: no kernel for {m}")
    return _MODULES[type(m)]


def _check_plain(m: nn.Module) -> None:
    """FusedMLP takes what a module holds without calling it: what would run in a call of it must not be passed by."""
    if m._forward_hooks or m._forward_pre_hooks or m._backward_hooks or m._backward_pre_hooks:
        raise ValueError(f"FusedMLP does not call its modules: {m} has hooks (as of prune or weight_norm) that would not run")
    if "forward" in m.__dict__:
        raise ValueError(f"FusedMLP does not call its modules: {m} has a forward of its own that would not run")


class FusedMLP(nn.Sequential):
    """nn.Sequential of nn.Linear layers, each followed by an activation module or none, computed by fused_mlp.  Its modules hold the
    parameters and are not called: one with hooks is refused, when it comes in and in every call."""

    def __init__(self, *layers):
        super().__init__(*layers)
        self._plan()

    def _plan(self):
        linears, acts = [], []
        for m in self._modules.values():
            if type(m) is nn.Linear:
                linears.append(m)
                acts.append(None)
            elif not linears or acts[-1] is not None:
                raise ValueError("FusedMLP: every activation follows a Linear layer")
            else:
                acts[-1] = _module_activation(m)
            _check_plain(m)
        return linears, [a or "none" for a in acts]

    def forward(self, x):
        linears, acts = self._plan()
        return fused_mlp(x, [m.weight for m in linears], [m.bias for m in linears], acts)
