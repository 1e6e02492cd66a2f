"""What the dense entry points and FusedMLP refuse because they could not do it right; no GPU needed."""
import pytest


def test_forward_derivatives_are_refused():
    import torch
    import torch.autograd.forward_ad as fwad
    from cafe_b200 import fused_linear, fused_mlp
    x, w, b = torch.randn(3, 4), torch.randn(2, 4), torch.randn(2)
    r = torch.randn(3, 2)
    with fwad.dual_level():
        dual = lambda t: fwad.make_dual(t, torch.ones_like(t))   # noqa: E731
        for call in (lambda: fused_linear(dual(x), w, b), lambda: fused_linear(x, dual(w), b), lambda: fused_linear(x, w, dual(b)),
                     lambda: fused_linear(x, w, b, "relu", dual(r)), lambda: fused_mlp(dual(x), [w], [b], ["relu"]),
                     lambda: fused_mlp(x, [dual(w)], [None], ["relu"]), lambda: fused_mlp(x, [w], [dual(b)], ["relu"])):
            with pytest.raises(NotImplementedError, match="forward"):
                call()
        with pytest.raises(ValueError, match="needs CUDA tensors"):   # (none of them dual: the next check's turn)
            fused_linear(x, w, b)


def test_traces_are_refused():
    import torch
    from torch.fx.experimental.proxy_tensor import make_fx
    from cafe_b200 import fused_linear, fused_mlp
    x, w = torch.randn(3, 4), torch.randn(2, 4)
    for call in (lambda x: fused_linear(x, w), lambda x: fused_mlp(x, [w], [None], ["silu"])):
        with pytest.raises(NotImplementedError, match="trace"):
            torch.jit.trace(call, (x,), check_trace=False)
        with pytest.raises(NotImplementedError, match="trace"):
            make_fx(call)(x)


def test_layers_with_hooks_are_refused():
    """FusedMLP takes the weights of its modules without calling them, so what hangs on a call of one of them would be passed by."""
    import torch
    import torch.nn as nn
    from torch.nn.utils import prune
    from cafe_b200 import FusedMLP

    def hook(*a):
        return None
    hooks = ["register_forward_hook", "register_forward_pre_hook", "register_full_backward_hook", "register_full_backward_pre_hook"]
    for name in hooks:
        for at in (0, 1, 2):
            net = FusedMLP(nn.Linear(4, 3), nn.ReLU(), nn.Linear(3, 2))
            handle = getattr(net[at], name)(hook)
            with pytest.raises(ValueError, match="hook"):
                net(torch.zeros(2, 4))
            handle.remove()
            with pytest.raises(ValueError, match="CUDA"):
                net(torch.zeros(2, 4))
    net = FusedMLP(nn.Linear(4, 3), nn.ReLU())
    prune.l1_unstructured(net[0], "weight", 0.5)
    with pytest.raises(ValueError, match="hook"):
        net(torch.zeros(2, 4))
    net = FusedMLP(nn.Linear(4, 3), nn.ReLU())
    net[0].forward = lambda x: x
    with pytest.raises(ValueError, match="forward"):
        net(torch.zeros(2, 4))
    normed = prune.identity(nn.Linear(4, 3), "weight")
    with pytest.raises(ValueError, match="hook"):
        FusedMLP(normed)
    # hooks of the whole still run
    seen = []
    net = FusedMLP(nn.Linear(4, 3))
    net.register_forward_pre_hook(lambda m, a: seen.append(1))
    with pytest.raises(ValueError, match="CUDA"):
        net(torch.zeros(2, 4))
    assert seen == [1]


def test_waits_that_ran_out_are_told(monkeypatch):
    """What the library counts reaches the caller, and so does its error."""
    import types
    import pytest
    from cafe_b200 import CafeError, dense

    def library(status, kinds):
        def gave_up(count):
            count._obj.value = kinds
            return status
        return types.SimpleNamespace(cafe_linear_gave_up=gave_up, cafe_last_error=lambda: b"no device")
    for kinds in (0, 1, 2):
        monkeypatch.setattr(dense._lib, "load", lambda: library(0, kinds))
        assert dense.gave_up() == kinds
    monkeypatch.setattr(dense._lib, "load", lambda: library(dense._lib.ERR_CUDA, 0))
    with pytest.raises(CafeError):
        dense.gave_up()
