"""Gradients where an activation's derivative is tiny and the gradient that meets it is large: a sigmoid under binary cross-entropy
has gy = -1 / y for a target of 1, so gz = -(1 - y), about -1 however far z is below zero.

The weight is an identity, so that z is x and gx is gz, element by element.  Bounds, relative to gz: the derivative's evaluation is off
by 2^-22 + 1.2 * 2^-24 |x| of exp(x) (|x| <= 85) and a few units of 2^-23 besides, less than 2^-16 together; beside bf16 it is kept with 11 bits
from 2^-14 on and with 8 below (2^-8 of it); gz is rounded to a 16-bit type once (2^-8, 2^-11) before its products with ones and
zeros, which are exact, and a sum of n of the same sign in fp32 adds (n + 8) 2^-23; gb is rounded once, of gz before or after its own
rounding."""
import pytest

pytestmark = pytest.mark.gpu

SMALL = [(7, 1, 24), (200, 16, 24), (300, 48, 64)]
LARGE = [(2048, 512, 512), (16384, 1024, 1024)]
# activation: ranges of z (each in quarters or halves, exact in all types)
RANGES = {"sigmoid": [(-80, -5), (5, 80)], "silu": [(-80, -5)], "gelu": [(-13, -3)]}


def _check(M, N, K, act, dtype, mlp):
    import torch
    import dense_reference as ref
    from cafe_b200 import fused_linear, fused_mlp
    half, least = torch.finfo(dtype).eps / 2, 2.0 ** -13 if dtype == torch.float16 else 0.0
    for lo, hi in RANGES[act]:
        # (whole numbers and halves up to 80.5 have 8 bits)
        z = (torch.arange(M * N, device="cuda") % (2 * (hi - lo) + 1)).double().view(M, N) / 2 + lo
        if dtype == torch.float16:   # (gy = 2^-6 / d has to stay below 65504, and sums of gz x too)
            z = z.clamp(-4, 4) if act == "gelu" else z.clamp(-8, 8)
        d = ref.activation(z, act)[1]
        gy = (-1 / d * (2.0 ** -6 if dtype == torch.float16 else 1)).to(dtype)
        assert bool(torch.isfinite(gy).all()) and bool((d.abs() > least).all())
        x = torch.zeros(M, K, dtype=dtype, device="cuda")
        x[:, :N] = z
        w = torch.eye(N, K, dtype=dtype, device="cuda")
        b = torch.zeros(N, dtype=dtype, device="cuda")
        leaves = [t.requires_grad_(True) for t in (x, w, b)]
        y = fused_mlp(x, [w], [b], [act]) if mlp else fused_linear(x, w, b, act)
        gx, gw, gb = torch.autograd.grad(y, leaves, gy)
        gz = gy.double() * d
        kept = 2.0 ** -8 if dtype == torch.bfloat16 else 0.0
        one = (1 + 2.0 ** -16) * (1 + kept) * (1 + half) - 1 + (N + 8) * 2.0 ** -23 + 2.0 ** -22
        far = ((gx[:, :N].double() - gz) / gz).abs()
        assert bool((far <= one).all()), (lo, hi, float(far.max()), one, float(z.reshape(-1)[far.argmax()]))
        assert bool((gx[:, N:] == 0).all())
        far = ((gb.double() - gz.sum(0)) / gz.sum(0)).abs()
        both = (1 + one) * (1 + half) - 1 + (M + 8) * 2.0 ** -23
        assert bool((far <= both).all()), (lo, hi, "gb", float(far.max()), both)
        # gw[n, k] = sum over rows of gz[m, n] x[m, k]: x's own range has one sign
        want = gz.t() @ x.double()
        far = ((gw.double() - want).abs() / (gz.abs().t() @ x.double().abs()).clamp(min=1e-300))
        assert bool((far <= both).all()), (lo, hi, "gw", float(far.max()), both)


@pytest.mark.parametrize("M,N,K", SMALL)
@pytest.mark.parametrize("act", ["sigmoid", "silu", "gelu"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_small_derivatives(M, N, K, act, dtype):
    import torch
    _check(M, N, K, act, getattr(torch, dtype), False)


@pytest.mark.parametrize("M,N,K", LARGE)
@pytest.mark.parametrize("act", ["sigmoid", "silu", "gelu"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_small_derivatives_of_large_layers(M, N, K, act, dtype):
    import torch
    _check(M, N, K, act, getattr(torch, dtype), False)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_small_derivatives_at_the_end_of_an_mlp(dtype):
    import torch
    _check(300, 48, 64, "sigmoid", getattr(torch, dtype), True)


def test_a_wrong_sample_still_teaches():
    """binary cross-entropy of a bf16 sigmoid: the gradient of every sample that is confidently wrong is -1 / rows."""
    import torch
    from cafe_b200 import fused_linear
    z = torch.arange(-80, -4, device="cuda").to(torch.bfloat16)[:, None].contiguous().requires_grad_(True)
    y = fused_linear(z, torch.ones(1, 1, dtype=torch.bfloat16, device="cuda"), None, "sigmoid")
    (-torch.log(y.float()).mean()).backward()
    got = z.grad.double() * len(z)
    # y, 1 / y and gy are bf16 or exact in fp32 and rounded to bf16: three roundings of 2^-8 beside the two of gz
    assert bool(((got + torch.sigmoid(-z.detach().double())).abs() <= 5.1 * 2.0 ** -8).all()), got.flatten().tolist()
