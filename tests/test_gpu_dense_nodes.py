"""fused_linear and fused_mlp as parts of a graph: what may be written to afterwards, views that carry a sign,
threads that have made no CUDA call yet."""
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


def test_views_that_carry_a_sign():
    """Tensors whose sign lies in their view (the imaginary part of a conjugate) are taken at their value, one column wide too."""
    import torch
    from cafe_b200 import fused_linear, fused_mlp
    g = torch.Generator(device="cuda").manual_seed(4)

    def signed(*shape):
        t = torch._neg_view(torch.randn(*shape, device="cuda", generator=g))
        assert t.is_neg()
        return t
    for M, N, K in ((40, 1, 1), (50, 30, 20)):
        x, w, b, r, gy = signed(M, K), signed(N, K), signed(N), signed(M, N), signed(M, N)
        plain = [(t + 0).detach() for t in (x, w, b, r, gy)]
        assert not any(t.is_neg() for t in plain)
        assert torch.equal(fused_linear(x, w, b, "silu", r), fused_linear(*plain[:3], "silu", plain[3]))
        assert torch.equal(fused_mlp(x, [w], [b], ["gelu"]), fused_mlp(plain[0], [plain[1]], [plain[2]], ["gelu"]))
        leaves = [t.requires_grad_(True) for t in plain[:4]]
        for call in (lambda: fused_linear(*leaves[:3], "silu", leaves[3]), lambda: fused_mlp(leaves[0], [leaves[1]], [leaves[2]], ["gelu"])):
            mine = leaves if "silu" in call.__code__.co_consts else leaves[:3]
            got, want = torch.autograd.grad(call(), mine, gy), torch.autograd.grad(call(), mine, plain[4])
            assert all(torch.equal(a, e) for a, e in zip(got, want))
    # as a program meets it: through a conjugate of a complex number made of the output
    x, w = torch.randn(40, 3, device="cuda", generator=g), torch.randn(1, 3, device="cuda", generator=g)
    c = torch.randn(40, 1, dtype=torch.complex64, device="cuda", generator=g)
    grads = []
    for f in (lambda x, w: fused_linear(x, w), lambda x, w: x @ w.t()):
        x1 = x.clone().requires_grad_(True)
        y = f(x1, w)
        (torch.complex(torch.zeros_like(y), y).conj() * c).abs().square().sum().backward()
        (torch.complex(y.detach() * 0, f(x1, w)).conj() * c).imag.sum().backward()
        grads.append(x1.grad)
    torch.testing.assert_close(*grads, rtol=1e-5, atol=1e-6)


def test_negative_views_as_gradients_of_adamw():
    import torch
    from cafe_b200 import AdamW
    p, q = (torch.nn.Parameter(torch.ones(500, device="cuda")) for _ in range(2))
    grad = torch.randn(500, device="cuda")
    p.grad, q.grad = torch._neg_view(grad), -grad
    a, b = AdamW([p]), AdamW([q])
    a.step()
    b.step()
    assert torch.equal(p, q)


def test_first_call_of_a_thread():
    """A thread that has made no CUDA call of its own has no context, which the description of operands in place asks for.  Memory comes
    from what the first pass left, so nothing else makes one."""
    import threading
    import torch
    from cafe_b200 import fused_linear
    x, w = (torch.randn(1024, 1024, device="cuda").bfloat16() for _ in range(2))
    with torch.no_grad():
        want = fused_linear(x, w)
        spare = fused_linear(x, w)
        torch.cuda.synchronize()
        del spare
        got = []

        def call():
            with torch.no_grad():
                try:
                    got.append(fused_linear(x, w))
                except RuntimeError as e:
                    got.append(e)
        for _ in range(2):
            t = threading.Thread(target=call)
            t.start()
            t.join()
    assert not isinstance(got[0], Exception), got[0]
    torch.cuda.synchronize()
    assert torch.equal(got[0], want) and torch.equal(got[1], want)


def test_first_backward_of_a_process():
    import subprocess
    import sys
    from pathlib import Path
    program = """
import torch
from cafe_b200 import fused_linear
x, w, gy = (torch.randn(1024, 1024, device="cuda").bfloat16() for _ in range(3))
w.requires_grad_(True)
gw, = torch.autograd.grad(fused_linear(x, w), w, gy)
want = gy.double().t() @ x.double()
assert float((gw.double() - want).norm() / want.norm()) < 2.0 ** -8
print("fine")
"""
    r = subprocess.run([sys.executable, "-c", program], cwd=Path(__file__).resolve().parents[1], capture_output=True, text=True, timeout=300)
    assert r.stdout.strip() == "fine", r.stderr[-2000:]


@pytest.mark.parametrize("M,widths", [(40, [30, 20, 10]), (70, [33, 40, 5]), (700, [300, 400, 600])])
def test_what_an_mlp_keeps(M, widths):
    """Whichever gradients are wanted, they are right, and the same tensors may be written to before the backward as with the layers one
    by one: a weight whose input needs no gradient is not needed, nor x where the first weight is frozen."""
    import itertools
    import torch
    from cafe_b200 import fused_mlp
    g = torch.Generator(device="cuda").manual_seed(9)
    r = lambda *s: torch.randn(s, device="cuda", generator=g) * 0.2   # noqa: E731
    values = [r(M, widths[0]), r(widths[1], widths[0]), r(widths[1]), r(widths[2], widths[1]), r(widths[2])]
    gy = r(M, widths[2])
    act = torch.nn.functional.silu

    def fused(x, w0, b0, w1, b1):
        return fused_mlp(x, [w0, w1], [b0, b1], ["silu", "none"])

    def stock(x, w0, b0, w1, b1):
        return act(x @ w0.t() + b0) @ w1.t() + b1
    for wanted in itertools.product((False, True), repeat=5):
        if not any(wanted):
            continue
        grads = []
        for f in (fused, stock):
            leaves = [v.double() if f is stock else v.clone() for v in values]
            leaves = [v.requires_grad_(n) for v, n in zip(leaves, wanted)]
            grads.append(torch.autograd.grad(f(*leaves), [v for v in leaves if v.requires_grad], gy.to(leaves[0].dtype)))
        for a, e in zip(*grads):
            # (norms: one layer's sums and evaluations are a few units of 2^-23 each)
            assert float((a.double() - e).norm() / e.norm()) < 1e-5, wanted
        for changed in range(5):
            raised = []
            for f in (fused, stock):
                leaves = [v.clone().requires_grad_(n) for v, n in zip(values, wanted)]
                y = f(*leaves)
                with torch.no_grad():
                    leaves[changed].mul_(2)
                try:
                    y.backward(gy)
                    raised.append(False)
                except RuntimeError as e:
                    assert "inplace" in str(e)
                    raised.append(True)
            assert raised[0] == raised[1], (wanted, changed, raised)


def test_tensors_without_memory_are_refused():
    import torch
    from torch._subclasses.fake_tensor import FakeTensorMode
    from cafe_b200 import fused_linear
    with FakeTensorMode():
        x, w = torch.empty(4, 8, device="cuda"), torch.empty(5, 8, device="cuda")
        with pytest.raises(RuntimeError):
            fused_linear(x, w)
