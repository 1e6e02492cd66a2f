"""How far sums are off as a whole.  dense_reference's bounds are those of the worst order of roundings, element by element, and grow
with the depth; here errors are averaged (norms, signed means), where a lost part of an operand or sums cut off for too long show."""
import pytest

pytestmark = pytest.mark.gpu

# (product, rows, out, in): the depth is `in` for y, `out` for gx, rows for gw.  The large ones are laid out first (two ways of sharing the
# tiles out, by estimate), the narrow ones are not.
SHAPES = [("y", 4096, 512, 512), ("y", 2048, 512, 4096), ("y", 1024, 512, 65536), ("y", 100, 50, 512), ("y", 100, 50, 65536), ("y", 100, 50, 400000),
          ("gx", 4096, 512, 512), ("gx", 1024, 4096, 512), ("gx", 1024, 65536, 512), ("gx", 100, 512, 50), ("gx", 100, 65536, 50),
          ("gw", 512, 512, 1024), ("gw", 4096, 1024, 2048), ("gw", 65536, 512, 1024), ("gw", 65536, 1024, 2048), ("gw", 131072, 1024, 2048),
          ("gw", 512, 48, 40), ("gw", 65536, 48, 40), ("gw", 400000, 48, 40)]


def _error(product, M, N, K, dtype, positive, seed=31):
    """(mean of the relative error, norm of the error over the result's) of 128 x 128 elements at most."""
    import torch
    from cafe_b200 import fused_linear
    g = torch.Generator(device="cuda").manual_seed(seed)
    u = lambda *s: torch.rand(s, device="cuda", generator=g) + 1   # noqa: E731
    # (rows and columns of different sizes, so that results do not share a place in their binade)
    make = (lambda r, c: (u(r, c) * u(r, 1) / 32)) if positive else (lambda r, c: torch.randn(r, c, device="cuda", generator=g) * u(r, 1) / 32)
    if product == "y":
        a, b = make(M, K).to(dtype), make(N, K).to(dtype)
        got = fused_linear(a, b)
    elif product == "gx":
        a, b = make(M, N).to(dtype), make(K, N).to(dtype)
        x = torch.zeros(M, K, dtype=dtype, device="cuda", requires_grad=True)
        got, = torch.autograd.grad(fused_linear(x, b.t().contiguous()), x, a)
    else:
        a, b = make(N, M).to(dtype), make(K, M).to(dtype)
        w = torch.zeros(N, K, dtype=dtype, device="cuda", requires_grad=True)
        got, = torch.autograd.grad(fused_linear(b.t().contiguous(), w), w, a.t().contiguous())
    got = got[:128, :128].double()
    want = a[:128].double() @ b[:128].double().t()
    return float(((got - want) / want).mean()), float((got - want).norm() / want.norm())


@pytest.mark.parametrize("product,M,N,K", SHAPES)
def test_fp32_sums_of_one_sign(product, M, N, K):
    """An instruction adds 16 of k and loses at most 2^-23 of the sum.  The upper parts' sums grow from zero over 256 of k: 16 of these, on
    half of the sum, half of the unit: 4.8e-7.  The others are at most 2^-7 of the result, five products over 4096 of k: 1280 of
    these, as above: 3.0e-7 (an instruction's own sixteen products are cut off too: twice that).  Sums of pieces are rounded, not cut off.
    Together below 1.1e-6; a lost pair of parts is 2^-18 of a product at least, 3.8e-6."""
    import torch
    mean, norm = _error(product, M, N, K, torch.float32, True)
    assert abs(mean) < 1.1e-6 and norm < 1.3e-6, (mean, norm)


@pytest.mark.parametrize("product,M,N,K", SHAPES)
def test_fp32_sums_of_both_signs(product, M, N, K):
    """Relative to the result's norm, which is that of a random walk: what a sum of pieces loses is of the same walk.  The three products
    that are left out are 2^-24 of a product each in the mean, the pieces' roundings 2^-25 sqrt(pieces / 3) of the walk's last place at
    most (1563 pieces of 400 000: 7e-7), cutting off as above."""
    import torch
    _, norm = _error(product, M, N, K, torch.float32, False)
    assert norm < 2e-6, norm


@pytest.mark.parametrize("product,M,N,K", SHAPES)
@pytest.mark.parametrize("dtype", ["bfloat16", "float16"])
def test_16_bit_norms(product, M, N, K, dtype):
    """One rounding of the result (its error's norm is at most half a step's), and the sums' cut-off beside it, below a quarter of it."""
    import torch
    dt = getattr(torch, dtype)
    for positive in (True, False):
        _, norm = _error(product, M, N, K, dt, positive)
        assert norm < 1.25 * torch.finfo(dt).eps / 2, (positive, norm)


@pytest.mark.parametrize("M,N,K", [(16384, 1024, 2048), (65536, 1024, 2048), (131072, 1024, 2048), (3 << 17, 1024, 512), (1 << 18, 512, 2048), (1 << 20, 256, 256)])
@pytest.mark.parametrize("dtype", ["float16", "bfloat16"])
def test_16_bit_long_sums_of_one_sign(M, N, K, dtype):
    """gW over many rows, all products positive: what is cut off adds up, 6.3e-9 of the sum for each row that is added in one go, so that no
    more than a fifth of what rounding the result may change is lost: 1.0e-4 in fp16, 7.6e-4 in bf16 (and a fifth of that for other
    values than the comment's).  Beside it the mean of n independent roundings, half a step / sqrt(3 n), 6 standard deviations."""
    import torch
    dt = getattr(torch, dtype)
    mean, _ = _error("gw", M, N, K, dt, True)
    assert abs(mean) < (1.0e-4 if dtype == "float16" else 7.6e-4) * 1.2 + 6 * torch.finfo(dt).eps / 2 / (3 * 128 * 128) ** 0.5, mean
