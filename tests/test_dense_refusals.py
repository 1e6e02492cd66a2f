"""What the dense and optimizer entry points refuse, without a GPU: arguments are checked before anything is launched."""
import ctypes

import pytest

ERR_ARG = 1
P = 4096   # (a pointer that is never followed: every call below is refused, or has nothing to do)


def _forward(lib, x=P, ldx=8, w=P, ldw=8, M=4, N=6, K=8, dtype=0, act=0, y=P, ldy=6, res=None, ldr=0, slope=None, lds=0, work=None):
    return lib.cafe_linear_forward(x, ldx, w, ldw, None, res, ldr, M, N, K, dtype, act, y, ldy, slope, lds, work, 0, None)


def test_linear_arguments():
    from cafe_b200 import _lib
    lib = _lib.load()
    for bad in [dict(M=-1), dict(N=-1), dict(K=-1), dict(dtype=3), dict(dtype=-1), dict(act=5), dict(act=-1), dict(x=None), dict(w=None),
                dict(y=None), dict(ldx=7), dict(ldw=7), dict(ldy=5), dict(res=P, ldr=5), dict(slope=P, lds=5), dict(M=8388609), dict(work=P + 8)]:
        assert _forward(lib, **bad) == ERR_ARG, bad

    def backward(gy=P, ldg=6, slope=P, lds=6, kind=1, x=P, ldx=8, w=P, ldw=8, M=4, N=6, K=8, dtype=0, gx=P, ldgx=8, gw=P, ldgw=8):
        return lib.cafe_linear_backward(gy, ldg, slope, lds, kind, x, ldx, w, ldw, M, N, K, dtype, gx, ldgx, gw, ldgw, P, None, 0, None)
    for bad in [dict(gy=None), dict(ldg=5), dict(slope=None), dict(lds=5), dict(kind=3), dict(kind=-1), dict(x=None), dict(ldx=7), dict(w=None),
                dict(ldw=7), dict(ldgx=7), dict(ldgw=7), dict(dtype=7), dict(M=-2)]:
        assert backward(**bad) == ERR_ARG, bad


def test_mlp_arguments():
    from cafe_b200 import _lib
    lib = _lib.load()
    i32, i64, vp = ctypes.c_int32, ctypes.c_int64, ctypes.c_void_p
    widths, acts = (i32 * 3)(4, 5, 6), (i32 * 2)(1, 2)
    ptrs, lds, pitch = (vp * 2)(P, P), (i64 * 2)(4, 5), (i64 * 2)(8, 6)
    assert lib.cafe_mlp_forward(0, widths, 3, P, 4, ptrs, lds, ptrs, acts, 0, ptrs, pitch, None, None, 0, None) == ERR_ARG
    assert lib.cafe_mlp_forward(33, widths, 3, P, 4, ptrs, lds, ptrs, acts, 0, ptrs, pitch, None, None, 0, None) == ERR_ARG
    assert lib.cafe_mlp_forward(2, widths, 3, P, 3, ptrs, lds, ptrs, acts, 0, ptrs, pitch, None, None, 0, None) == ERR_ARG
    assert lib.cafe_mlp_forward(2, widths, 3, P, 4, ptrs, lds, ptrs, acts, 0, ptrs, (i64 * 2)(4, 6), None, None, 0, None) == ERR_ARG
    need = lib.cafe_mlp_backward_work(2, widths, 3, P, 6, P, 4, ptrs, lds, 0)
    assert need >= 2 * 3 * 5 * 4
    slopes = (vp * 2)(None, P)

    def backward(work=P, size=need, slopes=slopes):
        return lib.cafe_mlp_backward(2, widths, 3, P, 6, P, 4, ptrs, lds, acts, 0, ptrs, pitch, slopes, P, 4, ptrs, ptrs, work, size, None)
    assert backward(size=2 * 3 * 5 * 4 - 1) == ERR_ARG   # (less than the gradients between the layers take)
    assert backward(work=None) == ERR_ARG
    assert backward(work=P + 4) == ERR_ARG
    assert backward(slopes=None) == ERR_ARG    # a sigmoid needs its slope


def test_adamw_arguments():
    from cafe_b200 import _lib
    lib = _lib.load()
    vp = ctypes.c_void_p
    one, none = (vp * 1)(P), (vp * 1)(None)

    def step(p=one, m=one, mtop=one, n=8, dtype=0, bits=32, b1=0.9, b2=0.999, eps=1e-8, ticket=P, steps=one, count=1):
        return lib.cafe_adamw_step(count, p, one, m, one, mtop, one, steps, (ctypes.c_int64 * 1)(n), None, dtype, bits, 1e-3, b1, b2, eps, 0.0, 0,
                                   ticket, None)
    for bad in [dict(p=none), dict(p=None), dict(m=none), dict(n=-1), dict(dtype=3), dict(bits=16), dict(b1=1.0), dict(b1=float("nan")), dict(b2=-0.1),
                dict(eps=-1.0), dict(ticket=None), dict(steps=none), dict(count=-1), dict(bits=8, mtop=none), dict(bits=8, mtop=None),
                dict(bits=8, m=(vp * 1)(P + 1))]:
        assert step(**bad) == ERR_ARG, bad
    assert step(count=0) == 0


def test_python_refusals_on_cpu_tensors():
    import torch
    import cafe_b200
    x, w = torch.randn(3, 4), torch.randn(2, 4)
    with pytest.raises(ValueError):
        cafe_b200.fused_linear(x, w)
    with pytest.raises(ValueError):
        cafe_b200.fused_mlp(x, [w], [None], ["relu"])
    with pytest.raises(ValueError):
        cafe_b200.AdamW([torch.nn.Parameter(w)])
    with pytest.raises(ValueError):
        cafe_b200.FusedMLP(torch.nn.ReLU(), torch.nn.Linear(3, 4))
    for bad in [dict(lr=-1), dict(betas=(0.9, 1.0)), dict(eps=-1e-8), dict(weight_decay=-1), dict(state_bits=16), dict(lr=float("nan"))]:
        with pytest.raises(ValueError):
            cafe_b200.AdamW([], **bad)


def test_torch_entry_points_without_a_gpu():
    """The messages of the extension module are formatted and come as ValueError."""
    import torch
    from cafe_b200 import fused_linear, fused_mlp
    x, w = torch.zeros(4, 6), torch.zeros(5, 6)
    with pytest.raises(ValueError, match="needs CUDA tensors"):
        fused_linear(x, w)
    with pytest.raises(ValueError, match="1 to 32 weights"):
        fused_mlp(x, [], [], [])
    with pytest.raises(ValueError, match="1 to 32 weights"):
        fused_mlp(x, [w], [], ["relu"])
    with pytest.raises(ValueError, match="activation"):
        fused_linear(x, w, activation="tanh")
    with pytest.raises(TypeError):
        fused_linear(x, None)
