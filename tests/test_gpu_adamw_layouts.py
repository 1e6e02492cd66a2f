"""AdamW and the order in which a parameter's elements lie: moments belong to elements, not to places in memory."""
import pytest

pytestmark = pytest.mark.gpu

CHANGES = {"transposed": ((40, 30), lambda t: t.t().contiguous().t()),
           "channels last": ((4, 3, 5, 6), lambda t: t.contiguous(memory_format=__import__("torch").channels_last)),
           "another shape": ((40, 30), lambda t: t.reshape(30, 40).t())}


def _fresh(shape, bits, layout=lambda t: t):
    import torch
    from cafe_b200 import AdamW
    g = torch.Generator(device="cuda").manual_seed(5)
    p = torch.nn.Parameter(layout(torch.randn(shape, device="cuda", generator=g)))
    opt = AdamW([p], state_bits=bits)
    p.grad = torch.randn(shape, device="cuda", generator=g)
    opt.step()
    return p, opt


@pytest.mark.parametrize("change", CHANGES)
@pytest.mark.parametrize("bits", [32, 8])
def test_a_new_order_of_elements_is_refused(bits, change):
    import torch
    shape, move = CHANGES[change]
    p, opt = _fresh(shape, bits)
    p.grad = None
    p.data = move(p.data)
    p.grad = torch.randn_like(p)
    before = p.detach().clone()
    with pytest.raises(RuntimeError, match="order"):
        opt.step()
    assert torch.equal(p, before)
    if bits == 8:
        with pytest.raises(RuntimeError, match="order"):
            opt.moments()


def test_moments_of_32_bits_are_laid_out_anew_by_loading():
    """What the message says: the state loaded again belongs to the elements in their new order."""
    import torch
    p, opt = _fresh((40, 30), 32)
    q, theirs = p.detach().clone().requires_grad_(True), None
    theirs = torch.optim.AdamW([q])
    theirs.load_state_dict(dict(state={0: {k: v.clone().float() if k == "step" else v.clone() for k, v in opt.state[p].items()}},
                                param_groups=theirs.state_dict()["param_groups"]))
    p.grad = None
    p.data = p.data.t().contiguous().t()
    opt.load_state_dict(opt.state_dict())
    g = torch.randn(40, 30, device="cuda")
    p.grad, q.grad = g, g.clone()
    opt.step()
    theirs.step()
    # (one step: corrections to 2^-19 of it, a rounding of the parameter each; a step is at most a few lr)
    assert bool(((p - q).abs() <= 10 * 1e-3 * 2 ** -18 + 2 ** -23 * q.abs()).all())


@pytest.mark.parametrize("bits", [32, 8])
def test_orders_that_are_the_same(bits):
    """Axes of one element have no order, a row-major parameter is one in any shape, and a layout of its own goes on."""
    import torch
    p, opt = _fresh((40, 1, 30), bits)
    p.grad = None
    p.data = p.data.as_strided((40, 1, 30), (30, 7, 1))
    p.grad = torch.randn_like(p)
    opt.step()
    p.grad = None
    p.data = p.data.reshape(1200)
    p.grad = torch.randn_like(p)
    opt.step()
    q, opt = _fresh((4, 3, 5, 6), bits, lambda t: t.contiguous(memory_format=torch.channels_last))
    opt.step()
    assert len(opt.moments()) == 1
    assert int(opt.state[q]["step"]) == 2


def test_codes_of_another_order_are_not_loaded():
    import copy
    import torch
    from cafe_b200 import AdamW
    p, opt = _fresh((4, 3, 5, 6), 8)
    kept = copy.deepcopy(opt.state_dict())
    last = torch.nn.Parameter(p.detach().contiguous(memory_format=torch.channels_last))
    other = AdamW([last], state_bits=8)
    with pytest.raises(ValueError, match="order"):
        other.load_state_dict(kept)
    assert not other.state.get(last)
    same = torch.nn.Parameter(p.detach().clone())
    again = AdamW([same], state_bits=8)
    again.load_state_dict(kept)
    p.grad = torch.randn_like(p)
    same.grad = p.grad.clone()
    opt.step()
    again.step()
    assert torch.equal(p, same)
    # channels last to channels last, through a pickle
    p, opt = _fresh((4, 3, 5, 6), 8, lambda t: t.contiguous(memory_format=torch.channels_last))
    import io
    file = io.BytesIO()
    torch.save(opt.state_dict(), file)
    file.seek(0)
    q = torch.nn.Parameter(p.detach().clone())
    again = AdamW([q], state_bits=8)
    again.load_state_dict(torch.load(file, weights_only=True))
    p.grad = torch.randn_like(p)
    q.grad = p.grad.clone()
    opt.step()
    again.step()
    assert q.stride() == p.stride() and torch.equal(p, q)
    # a state that does not say how its codes lie is one of row-major parameters
    for s in kept["state"].values():
        s.pop("layout", None)
    third = torch.nn.Parameter(p.detach().contiguous())
    AdamW([third], state_bits=8).load_state_dict(kept)
    with pytest.raises(ValueError, match="order"):
        AdamW([q], state_bits=8).load_state_dict(kept)


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_and_states_of_another_size_are_refused(bits):
    """torch checks a gradient's size when it is set, but not when .data is exchanged behind it."""
    import torch
    from cafe_b200 import AdamW
    for size in (5000, 3):
        p = torch.nn.Parameter(torch.zeros(10, device="cuda"))
        p.grad = torch.ones(10, device="cuda")
        p.data = torch.zeros(size, device="cuda")
        opt = AdamW([p], state_bits=bits)
        with pytest.raises(RuntimeError, match="gradient"):
            opt.step()
        assert bool((p == 0).all())
    for name in ("exp_avg", "exp_avg_sq", "step") if bits == 32 else ("exp_avg", "exp_avg_top", "root_avg_sq", "root_avg_sq_top", "step"):
        p, opt = _fresh((40, 30), bits)
        before = p.detach().clone()
        for bad in (lambda t: t.reshape(-1)[:0], lambda t: t.double(), lambda t: t.cpu()):
            kept = opt.state[p][name]
            opt.state[p][name] = bad(kept)
            with pytest.raises(RuntimeError, match="moments|order"):
                opt.step()
            opt.state[p][name] = kept
        assert torch.equal(p, before)
        opt.step()
        assert not torch.equal(p, before)


def test_states_that_a_trainer_moves():
    """Loops that move every tensor of a state to the parameter's device take the layouts along."""
    import torch
    p, opt = _fresh((40, 30), 8)
    q, other = _fresh((40, 30), 8)
    for s in opt.state.values():
        for k, t in s.items():
            s[k] = t.cuda()
    assert torch.equal(opt.moments()[0][0], other.moments()[0][0])
    for s in opt.state.values():
        for k, t in s.items():
            s[k] = t.cuda()
    p.grad = torch.randn_like(p)
    q.grad = p.grad.clone()
    opt.step()
    other.step()
    assert torch.equal(p, q)
    for size in ((0, 3), ()):            # nothing, and a number
        e = torch.nn.Parameter(torch.ones(size, device="cuda"))
        e.grad = torch.ones(size, device="cuda")
        opt = type(opt)([e], state_bits=8)
        opt.step()
        opt.step()
        assert int(opt.state[e]["step"]) == 2 and opt.moments()[0][0].shape == e.shape
