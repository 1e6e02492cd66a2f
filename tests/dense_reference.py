"""The dense layers in 64 bits, with bounds on how far a right result may be off, element by element.

Sums: a sum of n products in fp32, in any order, with every operation rounded or cut off, is off by at most (n + 8) 2^-23
times the sum of the products' magnitudes; an operand split into three 8-bit parts loses less than one further unit of 2^-23.
Results rounded to type t: eps(t) / 2 relative, or half the smallest step of fp16 / bf16.  Derivatives kept in fp16 beside bf16:
fp16 has 11 significant bits, so 2^-11 relative (finfo(fp16).eps / 2 = 2^-10 / 2), or 2^-25 near zero.  gz rounded to a 16-bit
type before its products: eps / 2 relative.  A rounding is relative to the value that is rounded, which is itself off already."""
import math

import torch

U = 2.0 ** -23
# (Lipschitz constant of the activation, of its derivative)
LIPSCHITZ = {"none": (1, 0), "relu": (1, 0), "sigmoid": (0.25, 0.1), "gelu": (1.13, 0.8), "silu": (1.1, 0.5)}
# the smallest step of each type near zero
LEAST = {torch.float32: 2.0 ** -149, torch.bfloat16: 2.0 ** -133, torch.float16: 2.0 ** -24}


def half_step(t, dtype):
    """What rounding to `dtype` may change."""
    return t.abs() * (torch.finfo(dtype).eps / 2) + LEAST[dtype] / 2


def activation(z, act):
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return z.clamp(min=0), (z > 0).to(z.dtype)
    if act == "gelu":
        c = 0.5 * torch.erfc(-z * math.sqrt(0.5))
        return z * c, c + z * torch.exp(-0.5 * z * z) / math.sqrt(2 * math.pi)
    s, t = torch.sigmoid(z), torch.sigmoid(-z)
    return (s, s * t) if act == "sigmoid" else (z * s, s + z * s * t)


def forward(x, w, b, act, r, dtype, x_off=None):
    """(y, bound, z, bound on z).  x_off: how far x itself may be off."""
    x, w = x.double(), w.double()
    z = x @ w.t()
    off = (x.abs() @ w.abs().t() + (b.double().abs() if b is not None else 0)) * ((x.shape[1] + 8) * U)
    if x_off is not None:
        off = off + x_off @ w.abs().t()
    if b is not None:
        z = z + b.double()
    a, _ = activation(z, act)
    # the activation's own evaluation: 8 units of 2^-23 of the value, plus 8 of |z| where it cancels (gelu, silu, sigmoid)
    far = off * LIPSCHITZ[act][0] + (8 * U) * (a.abs() + (0 if act in ("none", "relu") else z.abs() * 2.0 ** -10)) + 1e-37
    y = a if r is None else a + r.double()
    far = far + U * y.abs()
    return y, far + half_step(y.abs() + far, dtype), z, off


def backward(gy, z, z_off, x, w, act, dtype, mask=None, g_off=None, x_off=None):
    """{gx, gw, gb}: (value, bound).  mask: which derivative of a ReLU the forward took."""
    gy, x, w = gy.double(), x.double(), w.double()
    d = activation(z, act)[1] if mask is None else mask.double()
    gz = gy * d
    d_off = z_off * LIPSCHITZ[act][1] + (16 * U * (1 + z.abs()) if act not in ("none", "relu") else 0)
    if dtype == torch.bfloat16 and act not in ("none", "relu"):
        d_off = d_off + (d.abs() + d_off) * 2.0 ** -11 + 2.0 ** -25
    off = gy.abs() * d_off + U * gz.abs()
    if g_off is not None:
        off = off + g_off * (d.abs() + d_off)
    if dtype != torch.float32:
        off = off + half_step(gz.abs() + off, dtype)
    a = gz.abs() + off
    out = {}
    M, N = gz.shape
    for name, value, mag, far, n in (("gx", gz @ w, a @ w.abs(), off @ w.abs(), N),
                                     ("gw", gz.t() @ x, a.t() @ (x.abs() + (0 if x_off is None else x_off)),
                                      off.t() @ x.abs() + (0 if x_off is None else a.t() @ x_off), M),
                                     ("gb", gz.sum(0), a.sum(0), off.sum(0), M)):
        far = far + mag * ((n + 8) * U)
        out[name] = (value, far + half_step(value.abs() + far, dtype))
    return out


def assert_within(got, want, bound, what):
    far = (got.double() - want).abs()
    bad = ~(far <= bound)
    assert not bad.any(), (what, int(bad.sum()), "of", bad.numel(), "worst", float((far / bound.clamp(min=1e-300))[bad].max()),
                           [tuple(int(i) for i in at) for at in bad.nonzero()[:4]])
