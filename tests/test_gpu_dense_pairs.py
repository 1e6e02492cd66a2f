"""Large layers, whose tiles are worked on by pairs of blocks: the same bits however the two blocks' copies fall in time."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("M,N,K", [(4096, 1024, 1024), (2500, 1100, 700), (40000, 300, 200)])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_the_same_bits_beside_other_work(M, N, K, dtype):
    """Whole numbers small enough that every product and sum is exact (fp32 below 2^24; 16-bit results rounded once), so that anything
    read too early or too late shows; copies on another stream take bandwidth at changing times."""
    import torch
    from cafe_b200 import fused_linear
    dt = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(11)
    r = lambda *s: torch.randint(-4, 5, s, device="cuda", generator=g).to(dt)   # noqa: E731
    x, w, b, gy = r(M, K), r(N, K), r(N), r(M, N)
    # (64-bit products are exact here; the sums fit 2^20; fp16 ends at 65504)
    xd, wd, gd = x.double(), w.double(), gy.double()
    want = [(xd @ wd.t() + b.double()).to(dt), (gd @ wd).to(dt), (gd.t() @ xd).to(dt), gd.sum(0).to(dt)]
    leaves = [t.requires_grad_(True) for t in (x, w, b)]
    other, noise, target = torch.cuda.Stream(), torch.ones(1 << 26, device="cuda"), torch.empty(1 << 26, device="cuda")
    for turn in range(12):
        with torch.cuda.stream(other):
            for _ in range(turn % 4):
                target[:1 << (20 + turn % 7)].copy_(noise[:1 << (20 + turn % 7)])
        y = fused_linear(*leaves)
        got = [y.detach(), *torch.autograd.grad(y, leaves, gy)]
        for name, a, e in zip(("y", "gx", "gw", "gb"), got, want):
            assert torch.equal(a, e), (name, turn)


def test_no_wait_has_run_out_here():
    import cafe_b200.dense
    assert cafe_b200.dense.gave_up() == 0
    assert cafe_b200.dense.gave_up(0) == 0
