"""The dense layers around the embedding path on the library's kernels (csrc/dense_cuda.cu).

fused_linear   y = act(x W^T + b) + residual, differentiable
fused_mlp      a run of such layers as one node of the autograd graph: one call per direction
FusedMLP       the Sequential of Linear and activation modules that the reference's create_mlp builds
               (dlrm_s_pytorch.py:213-251), computed by fused_mlp; same parameters, same state_dict

Tensors are CUDA tensors of one type (fp32, bf16 or fp16); sums are fp32.  Kernels go to the current stream of the tensors'
device.  The gradients are those of first order: differentiating them again raises.  Captured into a CUDA graph, forward and
backward follow torch's rules for whole-network capture (warm-up on a side stream, no autograd graph of the same leaves alive
from outside the capture)."""
from __future__ import annotations

import ctypes
from functools import lru_cache

import torch
import torch.nn as nn
from torch.autograd.function import once_differentiable

from . import _lib
from .sketch import _stream

ACTIVATIONS = {"none": 0, "relu": 1, "sigmoid": 2, "gelu": 3, "silu": 4}
_NONE, _RELU = 0, 1
_SLOPE_NONE, _SLOPE_VALUES, _SLOPE_OUTPUT = 0, 1, 2
DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_SIZE, MAX_LAYERS = 8388608, 32
_LARGE, _FEW = 1 << 27, 16   # no call of fewer multiply-adds takes workspace (its size is 0), but a backward of few outputs: not asked


_get_device = getattr(torch._C, "_cuda_getDevice", torch.cuda.current_device)   # (without the checks of the public form)


class _on:
    """The tensors' device as the current one; `as` its current stream."""
    __slots__ = ("other",)

    def __init__(self, device):
        self.other = None if device.index == _get_device() else torch.cuda.device(device)

    def __enter__(self):
        if self.other is not None:
            self.other.__enter__()
        return _stream()

    def __exit__(self, *args):
        if self.other is not None:
            self.other.__exit__(*args)


def _rows(t: torch.Tensor, cols: int, repeated: bool = False):
    """t as rows of `cols` contiguous elements at one pitch: (tensor, rows, pitch).  Other layouts are copied; `repeated`:
    pitch 0 (a row that stands for all) is one."""
    if t.dim() != 2:
        t = t.reshape(-1, cols) if cols else t.reshape(t.numel(), 0)
    m = t.shape[0]
    if t.is_contiguous() or t.numel() == 0:
        return t, m, cols
    if cols == 1 or t.stride(1) == 1:
        ld = t.stride(0)
        if m == 1:
            return t, m, cols
        if ld >= cols or (repeated and ld == 0):
            return t, m, ld
    return t.contiguous(), m, cols


def _check(x, tensors, what):
    dtype = x.dtype
    if not x.is_cuda or dtype not in DTYPES:
        raise ValueError(f"{what} needs CUDA tensors of fp32, bf16 or fp16")
    device = x.get_device()
    for t in tensors:
        if t is not None and (t.dtype is not dtype or not t.is_cuda or t.get_device() != device):
            raise ValueError(f"{what}: all tensors must have one type and be on one device")


def _check_layer(cols, weight, bias, what):
    if weight.dim() != 2 or weight.shape[1] != cols:
        raise ValueError(f"{what}: weight must be [out, {cols}], got {list(weight.shape)}")
    if bias is not None and (bias.dim() != 1 or bias.shape[0] != weight.shape[0]):
        raise ValueError(f"{what}: bias must be [{weight.shape[0]}], got {list(bias.shape)}")
    if max(cols, weight.shape[0]) > MAX_SIZE:
        raise ValueError(f"{what}: sizes up to {MAX_SIZE}")


def _ptr(t):
    return None if t is None else t.data_ptr()


def _slope_type(dtype):
    return torch.float16 if dtype == torch.bfloat16 else torch.float32


def _work(size, like):
    """Workspace of one call, from torch's allocator: free again in the stream's order."""
    return torch.empty(size, dtype=torch.uint8, device=like.device) if size else None


def _contiguous(t):
    return t if t is None or t.is_contiguous() else t.contiguous()


def _saved_rows(t, cols):
    if t is None or t.is_contiguous():
        return t, cols
    t, _, ld = _rows(t, cols)
    return t, ld


def _linear(x, weight, bias, residual, act, keep):
    """The forward call: (x, weight as rows, y, what the backward needs of the activation)."""
    n, k = weight.shape
    x2, m, ldx = _rows(x, k)
    if m > MAX_SIZE:
        raise ValueError(f"fused_linear: up to {MAX_SIZE} rows")
    w2, _, ldw = _rows(weight, k)
    y = torch.empty(*x.shape[:-1], n, dtype=x.dtype, device=x.device)
    r2, ldr = None, 0
    if residual is not None:
        r2, _, ldr = _rows(residual, n, True)
    slope = None
    if keep and act != _NONE and not (act == _RELU and residual is None):
        slope = torch.empty(m, n, dtype=_slope_type(x.dtype), device=x.device)
    b = _contiguous(bias)
    lib, t, px, pw = _lib.load(), DTYPES[x.dtype], x2.data_ptr(), w2.data_ptr()
    size = lib.cafe_linear_forward_work(px, ldx, pw, ldw, m, n, k, t) if m * n * k >= _LARGE else 0
    with _on(x.device) as stream:
        status = lib.cafe_linear_forward(px, ldx, pw, ldw, _ptr(b), _ptr(r2), ldr, m, n, k, t, act, y.data_ptr(), n, _ptr(slope), n,
                                         _ptr(_work(size, x)), size, stream)
    if status:
        _lib.check(status, "cafe_linear_forward")
    return x2, w2, y, slope, (m, n, k)


class _FusedLinear(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, weight, bias, residual, act):
        x2, w2, y, slope, ctx.sizes = _linear(x, weight, bias, residual, act, True)
        need = ctx.needs_input_grad
        ctx.kind = kind = _SLOPE_NONE if act == _NONE else _SLOPE_VALUES if slope is not None else _SLOPE_OUTPUT
        ctx.shape = x.shape
        ctx.save_for_backward(x2 if need[1] else None, w2 if need[0] else None,
                              None if kind == _SLOPE_NONE else slope if kind == _SLOPE_VALUES else y)
        return y

    @staticmethod
    def backward(ctx, grad_y):
        # (differentiated with create_graph: gradients that refuse to be differentiated again)
        return _linear_backward_once(ctx, grad_y) if torch.is_grad_enabled() else _linear_backward(ctx, grad_y)


def _linear_backward(ctx, grad_y):
    x, w, slope = ctx.saved_tensors
    m, n, k = ctx.sizes
    need_x, need_w, need_b, need_r, _ = ctx.needs_input_grad
    gx = gw = gb = None
    if need_x or need_w or need_b:
        g, _, ldg = _rows(grad_y, n, True)
        dtype, device = g.dtype, g.device
        # (what was saved need not come back at the pitch that it was saved with)
        x, ldx = _saved_rows(x, k)
        w, ldw = _saved_rows(w, k)
        slope = _contiguous(slope)
        if need_x:
            gx = torch.empty(ctx.shape, dtype=dtype, device=device)
        if need_w:
            gw = torch.empty(n, k, dtype=dtype, device=device)
        if need_b:
            gb = torch.empty(n, dtype=dtype, device=device)
        lib, t, pg, px, pw = _lib.load(), DTYPES[dtype], g.data_ptr(), _ptr(x), _ptr(w)
        size = 0
        if n <= _FEW or m * n * k >= _LARGE:
            size = lib.cafe_linear_backward_work(pg, ldg, ctx.kind, px, ldx, pw, ldw, m, n, k, t, need_x, need_w, need_b)
        with _on(device) as stream:
            status = lib.cafe_linear_backward(pg, ldg, _ptr(slope), n, ctx.kind, px, ldx, pw, ldw, m, n, k, t, _ptr(gx), k, _ptr(gw), k, _ptr(gb),
                                              _ptr(_work(size, g)), size, stream)
        if status:
            _lib.check(status, "cafe_linear_backward")
    return gx, gw, gb, grad_y if need_r else None, None


_linear_backward_once = once_differentiable(_linear_backward)


def fused_linear(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None, activation: str = "none",
                 residual: torch.Tensor | None = None) -> torch.Tensor:
    """act(x W^T + b) + residual.  x [..., K], weight [N, K], bias [N]; residual broadcasts to [..., N]; activation is one of
    none, relu, sigmoid, gelu (with erf) and silu.  x, weight and residual may be slices of wider tensors (any pitch
    between rows).  For the backward the call keeps x, weight and, with an activation, its derivative (fp16 beside bf16, else
    fp32); of a ReLU without residual the output."""
    _check(x, (weight, bias, residual), "fused_linear")
    if activation not in ACTIVATIONS:
        raise ValueError(f"fused_linear: activation must be one of {sorted(ACTIVATIONS)}, got {activation!r}")
    if x.dim() < 1:
        raise ValueError("fused_linear: x must have a last dimension")
    _check_layer(x.shape[-1], weight, bias, "fused_linear")
    if residual is not None:
        shape = x.shape[:-1] + weight.shape[:1]
        if residual.shape != shape:
            residual = torch.broadcast_to(residual, shape)   # (raises if it cannot)
    act = ACTIVATIONS[activation]
    if torch.is_grad_enabled() and (x.requires_grad or weight.requires_grad or (bias is not None and bias.requires_grad) or
                                    (residual is not None and residual.requires_grad)):
        return _FusedLinear.apply(x, weight, bias, residual, act)
    return _linear(x, weight, bias, residual, act, False)[2]


# ---- a run of layers ---------------------------------------------------------------------------------------
def _pointers(tensors):
    return (ctypes.c_void_p * len(tensors))(*[None if t is None else t.data_ptr() for t in tensors])


class _Plan:
    """What a run of layers of these sizes needs besides its tensors: where the outputs between the layers and the slopes lie in
    one buffer (rows and starts on 16 bytes), and the arrays that describe it to the library."""

    def __init__(self, m, widths, acts, dtype, keep):
        n, size = len(acts), dtype.itemsize
        slope_size = _slope_type(dtype).itemsize
        pitch = [(v + 7) // 8 * 8 for v in widths[1:-1]] + [widths[-1]]
        at, self.y_at, self.slope_at = 0, [], []
        for p in pitch[:-1]:
            self.y_at.append(at)
            at += -(-m * p * size // 256) * 256
        for p, a in zip(pitch, acts):
            held = keep and a not in (_NONE, _RELU)
            self.slope_at.append(at if held else None)
            if held:
                at += -(-m * p * slope_size // 256) * 256
        self.bytes, self.n, self.type = at, n, DTYPES[dtype]
        self.widths, self.acts, self.pitch = (ctypes.c_int32 * (n + 1))(*widths), (ctypes.c_int32 * n)(*acts), (ctypes.c_int64 * n)(*pitch)

    def outputs(self, base, last):
        return (ctypes.c_void_p * self.n)(*[base + a for a in self.y_at], last)

    def slopes(self, base):
        return (ctypes.c_void_p * self.n)(*[None if a is None else base + a for a in self.slope_at])


_plan = lru_cache(maxsize=256)(_Plan)


def _weight_rows(weights):
    """(weights as rows of contiguous elements, their pitches for the library)."""
    ws, lds = [], []
    for w in weights:
        if w.is_contiguous():
            ws.append(w)
            lds.append(w.shape[1])
        else:
            w, _, ld = _rows(w, w.shape[1])
            ws.append(w)
            lds.append(ld)
    return ws, (ctypes.c_int64 * len(lds))(*lds)


def _mlp(x, weights, biases, acts, keep):
    """The forward call: (x and weights as rows, output, buffer of what lies between, plan, rows, pitches)."""
    widths = (weights[0].shape[1], *[w.shape[0] for w in weights])
    x2, m, ldx = _rows(x, widths[0])
    if m > MAX_SIZE:
        raise ValueError(f"fused_mlp: up to {MAX_SIZE} rows")
    plan = _plan(m, widths, acts, x.dtype, keep)
    ws, lds = _weight_rows(weights)
    bs = [_contiguous(b) for b in biases]
    device = x.device
    y = torch.empty(*x.shape[:-1], widths[-1], dtype=x.dtype, device=device)
    between = torch.empty(plan.bytes, dtype=torch.uint8, device=device)
    base = between.data_ptr()
    lib = _lib.load()
    call = (plan.n, plan.widths, m, x2.data_ptr(), ldx, _pointers(ws), lds)
    size = lib.cafe_mlp_forward_work(*call, plan.type)
    with _on(device) as stream:
        status = lib.cafe_mlp_forward(*call, _pointers(bs), plan.acts, plan.type, plan.outputs(base, y.data_ptr()), plan.pitch,
                                      plan.slopes(base) if keep else None, _ptr(_work(size, x)), size, stream)
    if status:
        _lib.check(status, "cafe_mlp_forward")
    return x2, ws, y, between, (plan, m)


class _FusedMLP(torch.autograd.Function):
    @staticmethod
    def forward(ctx, x, acts, *params):
        n = len(acts)
        x2, ws, y, between, ctx.sizes = _mlp(x, params[:n], params[n:], acts, True)
        ctx.shape = x.shape
        ctx.save_for_backward(x2, y, between, *ws)
        return y

    @staticmethod
    def backward(ctx, grad_y):
        return _mlp_backward_once(ctx, grad_y) if torch.is_grad_enabled() else _mlp_backward(ctx, grad_y)


def _mlp_backward(ctx, grad_y):
    x, y, between, *ws = ctx.saved_tensors
    plan, m = ctx.sizes
    n, need = plan.n, ctx.needs_input_grad
    # (what was saved need not come back at the pitch that it was saved with)
    x, ldx = _saved_rows(x, plan.widths[0])
    ws, lds = _weight_rows(ws)
    y, between = y.contiguous(), between.contiguous()
    g, _, ldg = _rows(grad_y, plan.widths[n], True)
    dtype, device = g.dtype, g.device
    gx = torch.empty(ctx.shape, dtype=dtype, device=device) if need[0] else None
    gws = [torch.empty(w.shape, dtype=dtype, device=device) if want else None for w, want in zip(ws, need[2:2 + n])]
    gbs = [torch.empty(w.shape[0], dtype=dtype, device=device) if want else None for w, want in zip(ws, need[2 + n:])]
    lib, base = _lib.load(), between.data_ptr()
    call = (n, plan.widths, m, g.data_ptr(), ldg, x.data_ptr(), ldx, _pointers(ws), lds)
    size = lib.cafe_mlp_backward_work(*call, plan.type)
    with _on(device) as stream:
        status = lib.cafe_mlp_backward(*call, plan.acts, plan.type, plan.outputs(base, y.data_ptr()), plan.pitch, plan.slopes(base), _ptr(gx),
                                       plan.widths[0], _pointers(gws), _pointers(gbs), _ptr(_work(size, g)), size, stream)
    if status:
        _lib.check(status, "cafe_mlp_backward")
    return (gx, None, *gws, *gbs)


_mlp_backward_once = once_differentiable(_mlp_backward)


def fused_mlp(x: torch.Tensor, weights, biases, activations) -> torch.Tensor:
    """Layer after layer of act(x W^T + b): weights [N_l, N_{l-1}], biases [N_l] or None, activations by name (see
    fused_linear).  The values are those of fused_linear layer by layer; between the layers they are held in x's type."""
    weights, biases, activations = tuple(weights), tuple(biases), tuple(activations)
    n = len(weights)
    if not 1 <= n <= MAX_LAYERS or len(biases) != n or len(activations) != n:
        raise ValueError(f"fused_mlp: one bias (or None) and one activation for each of 1 to {MAX_LAYERS} weights")
    _check(x, weights + biases, "fused_mlp")
    if x.dim() < 1:
        raise ValueError("fused_mlp: x must have a last dimension")
    cols = x.shape[-1]
    for w, b, a in zip(weights, biases, activations):
        if a not in ACTIVATIONS:
            raise ValueError(f"fused_mlp: activations must be among {sorted(ACTIVATIONS)}, got {a!r}")
        _check_layer(cols, w, b, "fused_mlp")
        cols = w.shape[0]
    acts = tuple([ACTIVATIONS[a] for a in activations])
    if torch.is_grad_enabled() and (x.requires_grad or any(w.requires_grad for w in weights) or any(b is not None and b.requires_grad for b in biases)):
        return _FusedMLP.apply(x, acts, *weights, *biases)
    return _mlp(x, weights, biases, acts, False)[2]


_MODULES = {nn.ReLU: "relu", nn.Sigmoid: "sigmoid", nn.SiLU: "silu", nn.Identity: "none"}


def _module_activation(m: nn.Module) -> str:
    if type(m) is nn.GELU and m.approximate == "none":
        return "gelu"
    if type(m) not in _MODULES:
        raise ValueError(f"FusedMLP: no kernel for {m}")
    return _MODULES[type(m)]


class FusedMLP(nn.Sequential):
    """nn.Sequential of nn.Linear layers, each followed by an activation module or none, computed by fused_mlp."""

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
        return linears, [a or "none" for a in acts]

    def forward(self, x):
        linears, acts = self._plan()
        return fused_mlp(x, [m.weight for m in linears], [m.bias for m in linears], acts)
