"""AdamW over many tensors against its formulas: parameters in 64 bits, 8-bit moments bit for bit against the code's definition
evaluated one fp32 operation after the other."""
import math

import pytest

pytestmark = pytest.mark.gpu

M32 = 0xFFFFFFFF
BLOCK = 256


def _mix(x):
    x = x & M32
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & M32
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & M32
    return x ^ (x >> 16)


def _random(n, seed, index, step):
    import torch
    key = _mix(_mix(seed + 0x9E3779B9 * (index + 1)) ^ (step & M32))
    at = torch.arange(n, device="cuda")
    return _mix((at & M32) ^ _mix(key + (at >> 32)))


def _pack(x, rnd, S):
    import torch
    drop, n = 23 - S, x.numel()
    bits = x.abs().view(torch.int32).to(torch.int64)
    blocks = torch.nn.functional.pad(bits, (0, -n % BLOCK)).view(-1, BLOCK)
    top = (((blocks + (1 << drop) - 1) >> drop).amax(1) >> S).clamp(16, 255)
    base = (top.repeat_interleave(BLOCK)[:n] - 15) << S
    code = ((bits + (rnd << (drop - 16))) >> drop) - base
    least = ((base + 1) << drop).to(torch.int32).view(torch.float32)
    low = (rnd.float() * (least * 2.0 ** -16) < x.abs()) if S == 3 else x > 0
    code = torch.where(x.abs() < least, low.to(torch.int64), code)
    if S == 3:
        code = code | (x < 0).to(torch.int64) << 7
    return code.to(torch.uint8), top.to(torch.uint8)


def _unpack(code, top, S):
    import torch
    n, c = code.numel(), code.to(torch.int64)
    low = c & 127 if S == 3 else c
    base = (top.to(torch.int64).repeat_interleave(BLOCK)[:n] - 15) << S
    x = torch.where(low > 0, ((low + base) << (23 - S)).to(torch.int32).view(torch.float32), torch.zeros((), device="cuda"))
    return torch.where(c > 127, -x, x) if S == 3 else x


SHAPES = [(1,), (255,), (256,), (257,), (3, 5), (64, 33), (4097,), (300, 1000), (2, 3, 4, 5), (8,), (1 << 20,)]


def _params(shapes, dtype, seed=0, offset=0):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    out = []
    for s in shapes:
        n = math.prod(s)
        p = torch.randn(n + offset, device="cuda", generator=g).to(dtype)[offset:].view(s)
        p = torch.nn.Parameter(p)
        p.grad = (torch.randn(n + offset, device="cuda", generator=g) * 1e-2).to(dtype)[offset:].view(s)
        out.append(p)
    return out


def _step_and_check(opt, params, group, t, bits, index0=0, seed=0):
    """One step of `opt` checked against the formulas from the state before it."""
    import torch
    before = [(p.detach().clone(), {k: v.clone() for k, v in opt.state[p].items()} if p in opt.state else None) for p in params]
    opt.step()
    b1, b2 = group["betas"]
    for i, (p, (old, s)) in enumerate(zip(params, before)):
        if p.grad is None:
            assert torch.equal(p, old)
            continue
        now = opt.state[p]
        assert int(now["step"]) == t
        g = p.grad.float()
        if bits == 32:
            m = s["exp_avg"] if s else torch.zeros_like(g)
            v = s["exp_avg_sq"] if s else torch.zeros_like(g)
        else:
            z = torch.zeros(p.numel(), dtype=torch.uint8, device="cuda")
            zt = torch.zeros(-(-p.numel() // BLOCK), dtype=torch.uint8, device="cuda")
            m = _unpack(*((s["exp_avg"], s["exp_avg_top"]) if s else (z, zt)), 3).view(p.shape)
            v = _unpack(*((s["root_avg_sq"], s["root_avg_sq_top"]) if s else (z, zt)), 4).view(p.shape).square()
        m1, v1 = m * b1 + g * (1 - b1), v * b2 + g * (1 - b2) * g
        root = v1.sqrt()
        if bits == 32:
            assert torch.equal(now["exp_avg"], m1) and torch.equal(now["exp_avg_sq"], v1)
        else:
            rnd = _random(p.numel(), seed, index0 + i, t)
            for names, x, r, S in ((("exp_avg", "exp_avg_top"), m1, rnd & 0xFFFF, 3), (("root_avg_sq", "root_avg_sq_top"), root, rnd >> 16, 4)):
                code, top = _pack(x.reshape(-1), r, S)
                assert torch.equal(now[names[1]], top) and torch.equal(now[names[0]], code), names
        # the new parameter in 64 bits from the same moments: the step itself is off by a few units of 2^-24, its corrections by
        # 2^-22 (exponentials of t log b in fp32), the sum is rounded to the parameter's type once
        m64, r64 = m1.double(), root.double()
        move = group["lr"] * group["weight_decay"] * old.double() + group["lr"] / (1 - b1 ** t) * m64 / (r64 / math.sqrt(1 - b2 ** t) + group["eps"])
        want = old.double() - move
        bound = move.abs() * 2.0 ** -18 + group["lr"] * group["weight_decay"] * old.double().abs() * 2.0 ** -20 + \
            group["lr"] / (1 - b1 ** t) * (m64 / (r64 / math.sqrt(1 - b2 ** t) + group["eps"])).abs() * 2.0 ** -19 + \
            want.abs() * torch.finfo(p.dtype).eps / 2 * (1.01 if p.dtype == torch.float32 else 1 + 2 ** -10) + 2.0 ** -24 * (old.double().abs() + 1e-30) + \
            (2.0 ** -25 if p.dtype == torch.float16 else 0)
        assert bool(((p.detach().double() - want).abs() <= bound).all()), (i, float(((p.detach().double() - want).abs() / bound).max()))


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("offset", [0, 1])
def test_steps(dtype, bits, offset):
    import torch
    from cafe_b200 import AdamW
    params = _params(SHAPES, getattr(torch, dtype), 3, offset)
    opt = AdamW(params, lr=2e-3, weight_decay=0.05, state_bits=bits, seed=99)
    g = torch.Generator(device="cuda").manual_seed(4)
    for t in range(1, 4):
        _step_and_check(opt, params, opt.param_groups[0], t, bits, seed=99)
        for p in params:
            p.grad = (torch.randn(p.shape, device="cuda", generator=g) * 10.0 ** -t).to(p.dtype)


def test_equals_torch_adamw_in_32_bits():
    """Ten steps beside torch.optim.AdamW: each step's corrections are off by 2^-19 of the step (see above) and both round each
    parameter at 2^-24, so after ten steps of at most lr they are within 10 (lr 2^-18 + 2^-23 |p|)."""
    import torch
    from cafe_b200 import AdamW
    a, b = _params(SHAPES, torch.float32, 5), _params(SHAPES, torch.float32, 5)
    mine, theirs = AdamW(a, lr=1e-2, weight_decay=0.1), torch.optim.AdamW(b, lr=1e-2, weight_decay=0.1)
    for t in range(10):
        for p, q in zip(a, b):
            g = torch.randn(p.shape, device="cuda") * (0.1 + t)
            p.grad, q.grad = g, g.clone()
        mine.step()
        theirs.step()
    for p, q in zip(a, b):
        # (a step can be several lr where the first moments meet small second ones: 10 lr is more than any here)
        assert bool(((p - q).abs() <= 10 * (10 * 1e-2 * 2 ** -18 + 2 ** -23 * q.abs())).all()), float((p - q).abs().max())


@pytest.mark.parametrize("bits", [32, 8])
def test_missing_gradients_and_groups(bits):
    import torch
    from cafe_b200 import AdamW
    params = _params([(40,), (300,), (7, 9)], torch.float32, 7) + _params([(64,)], torch.bfloat16, 8)
    opt = AdamW([dict(params=params[:2], lr=1e-3), dict(params=params[2:], lr=1e-2, betas=(0.0, 0.5), weight_decay=0.0, eps=1e-6)], state_bits=bits)
    keep = params[1].grad
    params[1].grad = None
    opt.step()
    params[1].grad = keep
    opt.step()
    assert [int(opt.state[p]["step"]) for p in params] == [2, 1, 2, 2]
    fresh = _params([(40,), (300,), (7, 9)], torch.float32, 7)[1]
    lone = AdamW([fresh], lr=1e-3, state_bits=bits)
    if bits == 32:     # (8-bit codes go by the tensor's place)
        lone.step()
        assert torch.equal(fresh, params[1])
    _step_and_check(opt, params[2:3], opt.param_groups[1], 3, bits, index0=2)


@pytest.mark.parametrize("count", [48, 49, 400, 431])
def test_many_tensors(count):
    """Lists on both sides of what one launch takes."""
    import torch
    from cafe_b200 import AdamW
    params = _params([(1 + (k * 37) % 600,) for k in range(count)], torch.float32, 9)
    opt = AdamW(params, state_bits=8, seed=1)
    _step_and_check(opt, params, opt.param_groups[0], 1, 8, seed=1)
    _step_and_check(opt, params, opt.param_groups[0], 2, 8, seed=1)


def test_rounding_keeps_the_mean():
    """Moments that change by less than a code's step move on average.  With a constant gradient v goes from its start towards
    g^2 by (1 - b2) of the way a step; the root's codes are 2^-4 apart relative to their own binade, each rounding's error is at
    most that step, independent from element to element, so the mean over n elements is within 6 standard deviations,
    6 * sqrt(steps) * 2^-4 / sqrt(n), of the recursion without rounding (rounding r up or down evenly raises r^2 by at most
    a quarter of a squared step: 2^-10 a step of the recursion, of which (1 - b2) stays)."""
    import torch
    from cafe_b200 import AdamW
    n, steps, b2 = 1 << 18, 200, 0.99
    p = torch.nn.Parameter(torch.zeros(n, device="cuda"))
    opt = AdamW([p], lr=0.0, betas=(0.9, b2), weight_decay=0.0, state_bits=8)
    p.grad = torch.full((n,), 0.75, device="cuda")
    p.grad[::2] *= 0.37
    want = torch.zeros(n, dtype=torch.double, device="cuda")
    mean = torch.zeros(n, dtype=torch.double, device="cuda")
    for _ in range(steps):
        opt.step()
        want = b2 * want + (1 - b2) * p.grad.double() ** 2
        mean = 0.9 * mean + 0.1 * p.grad.double()
    (m, r), = opt.moments()
    for half in (slice(0, None, 2), slice(1, None, 2)):
        got = float(r[half].double().square().mean() / want[half].mean())
        assert abs(got - 1) < 6 * math.sqrt(steps) * 2 * 2 ** -4 / math.sqrt(n / 2) + steps * 2 ** -10, got
        assert abs(float(m[half].double().mean() / mean[half].mean()) - 1) < 6 * math.sqrt(20) * 2 ** -3 / math.sqrt(n / 2)


def test_moments_are_the_codes_values():
    import torch
    from cafe_b200 import AdamW
    for bits in (8, 32):
        params = _params([(5, 7), (1000,), (0,)], torch.float32, 11)
        params[0].data = params[0].data.t().contiguous().t()      # columns contiguous
        params[0].grad = torch.randn(5, 7, device="cuda")         # rows contiguous
        opt = AdamW(params, state_bits=bits)
        for _ in range(3):
            opt.step()
        got = opt.moments()
        assert len(got) == 3
        for p, (m, v) in zip(params, got):
            assert m.shape == p.shape
            s = opt.state[p]
            if bits == 32:
                assert m is s["exp_avg"] and v is s["exp_avg_sq"]
            elif p.dim() == 1:
                assert torch.equal(m.float(), _unpack(s["exp_avg"], s["exp_avg_top"], 3))
                assert torch.equal(v.float(), _unpack(s["root_avg_sq"], s["root_avg_sq_top"], 4))
        # a constant gradient since the start: m = (1 - 0.9^3) g, within three roundings of 2^-3 (8 bits) or 2^-22
        m = got[0][0].float()
        assert float((m / (params[0].grad * (1 - 0.9 ** 3)) - 1).abs().max()) < (1.25 ** 3 - 1 if bits == 8 else 1e-5)


@pytest.mark.parametrize("bits", [32, 8])
def test_gradients_that_are_not_finite(bits):
    import torch
    from cafe_b200 import AdamW
    p = torch.nn.Parameter(torch.ones(1000, device="cuda"))
    p.grad = torch.ones(1000, device="cuda")
    p.grad[300] = float("inf")
    p.grad[700] = float("nan")
    opt = AdamW([p], state_bits=bits)
    opt.step()
    opt.step()
    bad = p.isnan()
    want = torch.zeros(1000, dtype=torch.bool, device="cuda")
    if bits == 32:
        want[[300, 700]] = True
    else:
        want[256:768] = True       # the blocks of 256 that share their exponent
    assert torch.equal(bad, want)


def test_extreme_magnitudes():
    """Zeros, a block whose elements are 2^40 apart, gradients near the ends of fp32."""
    import torch
    from cafe_b200 import AdamW
    g = torch.zeros(2048, device="cuda")
    g[256:512] = 2.0 ** torch.linspace(-60, 0, 256, device="cuda")
    g[512:768] = 1e-38
    g[768:1024] = 1e-25
    g[1024:1280] = 1e15
    g[1300] = 1.0
    p = torch.nn.Parameter(torch.ones(2048, device="cuda"))
    p.grad = g
    opt = AdamW([p], weight_decay=0.0, lr=1e-3, state_bits=8)
    for t in range(1, 4):
        _step_and_check(opt, [p], opt.param_groups[0], t, 8)
    assert bool(p.isfinite().all())
    assert bool((p[g == 0] == 1).all())
    # an element far below its block's largest moves no further than the others: lr a step with exact moments of a constant
    # gradient; each earlier rounding raises m by at most 2^-3 of it and lowers the root by at most 2^-4, so step k is at most
    # ((1 + 2^-3) / (1 - 2^-4))^(k-1) lr = 1, 1.2, 1.44 lr
    assert float((p.detach() - 1).abs().max()) < (1 + 1.2 + 1.44) * 1e-3 * 1.01


@pytest.mark.parametrize("bits", [32, 8])
def test_state_dict_round_trip(bits):
    import copy
    import torch
    from cafe_b200 import AdamW
    a = _params(SHAPES[:6], torch.bfloat16, 13)
    oa = AdamW(a, state_bits=bits, seed=5)
    oa.step()
    kept = copy.deepcopy(oa.state_dict())
    b = [torch.nn.Parameter(p.detach().clone()) for p in a]
    ob = AdamW(b, lr=7.0, state_bits=bits)
    ob.load_state_dict(kept)
    for p, q in zip(a, b):
        q.grad = p.grad.clone()
    oa.step()
    ob.step()
    for p, q in zip(a, b):
        assert torch.equal(p, q)
        for k in oa.state[p]:
            assert torch.equal(oa.state[p][k], ob.state[q][k]) and oa.state[p][k].dtype == ob.state[q][k].dtype, k
    other = AdamW(b, state_bits=40 - bits)
    with pytest.raises(ValueError):
        other.load_state_dict(kept)


def test_copies_and_pickles():
    import copy
    import pickle
    import torch
    from cafe_b200 import AdamW
    net = torch.nn.Linear(33, 9).cuda()
    opt = AdamW(net.parameters(), state_bits=8, seed=3)
    for p in net.parameters():
        p.grad = torch.ones_like(p)
    opt.step()
    for again in (copy.deepcopy((net, opt)), pickle.loads(pickle.dumps((net, opt)))):
        n2, o2 = again
        assert (o2.state_bits, o2.seed) == (8, 3)
        for p in n2.parameters():
            p.grad = torch.ones_like(p)
        o2.step()
    for p in net.parameters():
        p.grad = torch.ones_like(p)
    opt.step()
    for a, b in zip(net.parameters(), n2.parameters()):
        assert torch.equal(a, b)


def test_captured_steps_count_on():
    import torch
    from cafe_b200 import AdamW
    for bits in (32, 8):
        a, b = _params(SHAPES[:8], torch.float32, 15), _params(SHAPES[:8], torch.float32, 15)
        oa, ob = AdamW(a, state_bits=bits), AdamW(b, state_bits=bits)
        oa.step()
        ob.step()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            oa.step()
        for t in range(3):
            for p, q in zip(a, b):
                p.grad.normal_()
                q.grad.copy_(p.grad)
            graph.replay()
            ob.step()
            for p, q in zip(a, b):
                assert torch.equal(p, q)
                assert int(oa.state[p]["step"]) == t + 2
    c = _params([(8,)], torch.float32, 16)
    with pytest.raises(RuntimeError, match="one step before capturing"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            AdamW(c).step()


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_exchanged_behind_it(bits):
    """A parameter whose memory is not what its moments were made for is refused before anything is launched."""
    import torch
    from cafe_b200 import AdamW

    def fresh():
        p = torch.nn.Parameter(torch.randn(40, 30, device="cuda"))
        opt = AdamW([p], state_bits=bits)
        p.grad = torch.randn_like(p)
        opt.step()
        return p, opt
    for change in (lambda t: t.cpu(), lambda t: t.double(), lambda t: torch.cat([t, t]), lambda t: torch.cat([t, t], 1)[:, :30]):
        p, opt = fresh()
        p.grad = None
        p.data = change(p.data)
        p.grad = torch.randn_like(p)
        with pytest.raises(RuntimeError):
            opt.step()
    p, opt = fresh()            # another floating type of the same size goes on with the same moments
    p.grad = None
    p.data = p.data.bfloat16()
    p.grad = torch.randn_like(p)
    opt.step()
    assert torch.isfinite(p).all()
    if hasattr(p, "grad_dtype"):
        p, opt = fresh()
        p.grad = None
        p.grad_dtype = torch.bfloat16
        p.grad = torch.randn(40, 30, device="cuda", dtype=torch.bfloat16)
        with pytest.raises(RuntimeError):
            opt.step()


def test_a_step_between_forward_and_backward_is_noticed():
    import torch
    from cafe_b200 import AdamW
    p = torch.nn.Parameter(torch.randn(40, 30, device="cuda"))
    opt = AdamW([p])
    y = (p * p).sum()
    p.grad = torch.ones_like(p)
    opt.step()
    with pytest.raises(RuntimeError, match="inplace"):
        y.backward()


def test_refusals():
    import torch
    from cafe_b200 import AdamW
    e = torch.nn.Embedding(10, 4, sparse=True).cuda()
    e(torch.tensor([1, 2], device="cuda")).sum().backward()
    with pytest.raises(RuntimeError, match="sparse"):
        AdamW(e.parameters()).step()
    with pytest.raises(ValueError):
        AdamW([torch.nn.Parameter(torch.zeros(4, dtype=torch.double, device="cuda"))])
    with pytest.raises(ValueError):
        AdamW([torch.nn.Parameter(torch.zeros(4, 8, device="cuda")[:, :4])])
    with pytest.raises(ValueError):
        AdamW([torch.nn.Parameter(torch.zeros(4, device="cuda"))], lr=torch.tensor(1e-3))
    p = torch.nn.Parameter(torch.zeros(4, device="cuda"))
    opt = AdamW([p])
    opt.param_groups[0]["betas"] = (0.9, 1.0)
    p.grad = torch.ones(4, device="cuda")
    with pytest.raises(ValueError):
        opt.step()
