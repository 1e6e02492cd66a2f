"""fused_linear and fused_mlp as parts of a graph: what may be written to afterwards."""
import pytest

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("act", ["none", "relu", "sigmoid", "gelu", "silu"])
@pytest.mark.parametrize("M,N,K", [(5, 20, 30), (300, 60, 70)])
def test_outputs_written_to_in_place(act, M, N, K):
    """As with the Linear and activation modules that it stands for: only a ReLU's output is needed by the backward.  (torch's own
    sigmoid keeps its output too; this one does not.)"""
    import torch
    from cafe_b200 import fused_linear, fused_mlp
    g = torch.Generator(device="cuda").manual_seed(3)
    x, w, b = (torch.randn(s, device="cuda", generator=g).requires_grad_(True) for s in ((M, K), (N, K), (N,)))
    gy = torch.randn(M, N, device="cuda", generator=g)
    for call in (lambda: fused_linear(x, w, b, act), lambda: fused_mlp(x, [w], [b], [act])):
        want = torch.autograd.grad(call(), (x, w, b), gy)
        y = call()
        y.mul_(2)
        if act == "relu":
            with pytest.raises(RuntimeError, match="inplace"):
                torch.autograd.grad(y, (x, w, b), gy)
        else:
            for a, e in zip(torch.autograd.grad(y, (x, w, b), gy), want):
                assert torch.equal(a, 2 * e)


def test_an_output_of_no_use_is_not_kept():
    import torch
    from cafe_b200 import fused_mlp
    x = torch.randn(1 << 14, 50, device="cuda", requires_grad=True)
    w = torch.randn(512, 50, device="cuda")
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    y = fused_mlp(x, [w], [None], ["none"])
    node = y.grad_fn
    del y
    assert torch.cuda.memory_allocated() - before < 1 << 20, node   # (the output has 32 MB)

