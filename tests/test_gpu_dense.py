"""fused_linear, fused_mlp and FusedMLP against the layers in 64 bits (dense_reference: every bound is derived there)."""
import pytest

pytestmark = pytest.mark.gpu

ACTS = ["none", "relu", "sigmoid", "gelu", "silu"]
#            rows, out, in: one row, one column, odd sizes, sizes around the kernels' tiles, long axes
SIZES = [(1, 1, 1), (1, 1024, 1024), (1, 5, 2000), (3, 700, 129), (7, 3, 5), (16, 1024, 479), (128, 512, 367), (130, 129, 65),
         (257, 16, 13), (64, 1, 256), (300, 511, 479), (2048, 256, 512), (5000, 8, 64), (4097, 40, 33), (255, 257, 1024), (20000, 1, 31),
         (9000, 130, 70)]


def _make(M, N, K, dtype, seed, pitch=0, bias=True, residual=None):
    import torch
    g = torch.Generator(device="cuda").manual_seed(seed)
    r = lambda *s: torch.randn(s, device="cuda", generator=g)   # noqa: E731
    x = r(M, K + pitch).to(dtype)[:, pitch:]
    w = (r(N, K + pitch) * (2 / (N + K)) ** 0.5).to(dtype)[:, :K]
    b = (r(N) * 0.1).to(dtype) if bias else None
    res = None
    if residual == "full":
        res = r(M, N + pitch).to(dtype)[:, pitch:]
    elif residual == "row":
        res = r(N).to(dtype)
    gy = (r(M, N) * 0.1).to(dtype)
    return x, w, b, res, gy


def _check(M, N, K, dtype, act, seed=1, pitch=0, bias=True, residual=None):
    import torch
    from cafe_b200 import fused_linear
    import dense_reference as ref
    x, w, b, r, gy = _make(M, N, K, dtype, seed, pitch, bias, residual)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b, r) if t is not None]
    it = iter(leaves)
    lx, lw = next(it), next(it)
    lb = next(it) if b is not None else None
    lr = next(it) if r is not None else None
    y = fused_linear(lx, lw, lb, act, lr)
    assert y.shape == (M, N) and y.dtype == dtype
    want, bound, z, z_off = ref.forward(x, w, b, act, r, dtype)
    ref.assert_within(y.detach(), want, bound, "y")
    with torch.no_grad():
        assert torch.equal(fused_linear(x, w, b, act, r), y)   # the form that keeps nothing
    grads = dict(zip(["gx", "gw"] + (["gb"] if b is not None else []) + (["gr"] if r is not None else []),
                     torch.autograd.grad(y, leaves, gy)))
    mask = None
    if act == "relu":
        # the derivative goes by the sign of the kernel's own pre-activation, which may differ where 64 bits cannot tell
        mask = (z > 0) if r is not None else y.detach() > 0
        near = z.abs() <= z_off + ref.LEAST[dtype]
        assert bool(((mask == (z > 0)) | near).all())
        if r is not None:   # the mask itself is not seen: leave out rows and columns that a near one could change
            gy = gy.masked_fill(near, 0)
            grads = dict(zip(grads, torch.autograd.grad(fused_linear(lx, lw, lb, act, lr), leaves, gy)))
    for name, (value, far) in ref.backward(gy, z, z_off, x, w, act, dtype, mask).items():
        if name in grads:
            ref.assert_within(grads[name], value, far, name)
    if r is not None:
        full = gy.double() if r.dim() == 2 else gy.double().sum(0)
        tol = ref.half_step(full, dtype) + gy.double().abs().sum(0) * (M + 8) * (ref.U if dtype == torch.float32 else torch.finfo(dtype).eps)
        ref.assert_within(grads["gr"], full, tol, "gr")


@pytest.mark.parametrize("M,N,K", SIZES)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_sizes(M, N, K, dtype):
    import torch
    i = SIZES.index((M, N, K))
    _check(M, N, K, getattr(torch, dtype), ACTS[i % 5], seed=i)


# rows, out, in, pitch, activation, residual: layers large enough for operands that are laid out first; ragged on every side, long
# in each axis, one tile wide, rows on and off 16 bytes
LARGE = [(2048, 512, 512, 0, "none", None), (2100, 700, 479, 0, "relu", None), (1030, 1100, 520, 8, "gelu", "full"), (300, 2000, 1000, 3, "silu", "row"),
         (70000, 130, 70, 0, "sigmoid", None), (130, 64, 70000, 2, "silu", None), (128, 70001, 64, 0, "gelu", None), (4100, 129, 1025, 0, "none", "full"),
         (1500, 640, 640, 8, "relu", "full")]


@pytest.mark.parametrize("M,N,K,pitch,act,residual", LARGE)
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_large_layers(M, N, K, pitch, act, residual, dtype):
    import torch
    _check(M, N, K, getattr(torch, dtype), act, seed=M, pitch=pitch, residual=residual)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_large_layers_one_gradient_alone(dtype):
    """Which gradients are wanted decides how the products are laid out and in what order they are summed: every subset within
    the bounds of 64 bits."""
    import torch
    from cafe_b200 import fused_linear
    import dense_reference as ref
    dt = getattr(torch, dtype)
    x, w, b, _, gy = _make(1100, 700, 800, dt, 12)
    _, _, z, z_off = ref.forward(x, w, b, "silu", None, dt)
    want = ref.backward(gy, z, z_off, x, w, "silu", dt)
    for keep in range(1, 8):
        leaves = [t.detach().requires_grad_(bool(keep >> i & 1)) for i, t in enumerate((x, w, b))]
        got = torch.autograd.grad(fused_linear(*leaves, "silu"), [t for t in leaves if t.requires_grad], gy)
        for a, name in zip(got, [n for i, n in enumerate(("gx", "gw", "gb")) if keep >> i & 1]):
            ref.assert_within(a, *want[name], f"{name} of {keep}")


@pytest.mark.parametrize("act", ACTS)
@pytest.mark.parametrize("residual", [None, "full", "row"])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
def test_activations_residuals_and_pitches(act, residual, dtype):
    import torch
    _check(200, 96, 64, getattr(torch, dtype), act, seed=3, pitch=0, residual=residual)
    _check(137, 61, 83, getattr(torch, dtype), act, seed=4, pitch=3, bias=residual is None, residual=residual)
    _check(65, 72, 40, getattr(torch, dtype), act, seed=5, pitch=8, residual=residual)


def test_layouts_that_are_copied_and_more_dimensions():
    import torch
    from cafe_b200 import fused_linear
    import dense_reference as ref
    g = torch.Generator(device="cuda").manual_seed(7)
    x = torch.randn(40, 3, 50, device="cuda", generator=g)
    w = torch.randn(50, 30, device="cuda", generator=g).t()          # not rows
    y = fused_linear(x, w)
    want, bound, *_ = ref.forward(x.reshape(-1, 50), w, None, "none", None, torch.float32)
    ref.assert_within(y.reshape(-1, 30), want, bound, "y")
    xt = torch.randn(50, 70, device="cuda", generator=g).t()         # columns contiguous
    want, bound, *_ = ref.forward(xt, w, None, "none", None, torch.float32)
    ref.assert_within(fused_linear(xt, w), want, bound, "y of a transposed x")
    xe = torch.randn(1, 50, device="cuda", generator=g).expand(20, 50)   # one row for all
    want, bound, *_ = ref.forward(xe, w, None, "none", None, torch.float32)
    ref.assert_within(fused_linear(xe, w), want, bound, "y of an expanded x")
    one = torch.randn(50, device="cuda", generator=g)
    assert fused_linear(one, w).shape == (30,)
    # a gradient that is one number for all
    lx = x.clone().requires_grad_(True)
    gx, = torch.autograd.grad(fused_linear(lx, w).sum(), lx)
    ref.assert_within(gx[0], w.double().sum(0).expand(3, 50), (w.double().abs().sum(0) * 38 * ref.U).expand(3, 50), "gx")


def test_empty_sizes():
    import torch
    from cafe_b200 import fused_linear, fused_mlp
    for M, N, K in [(0, 5, 3), (4, 0, 3), (4, 5, 0), (0, 0, 0)]:
        x = torch.randn(M, K, device="cuda", requires_grad=True)
        w = torch.randn(N, K, device="cuda", requires_grad=True)
        b = torch.randn(N, device="cuda", requires_grad=True)
        y = fused_linear(x, w, b, "relu")
        assert torch.equal(y, torch.relu(b).expand(M, N) if K == 0 else torch.zeros(M, N, device="cuda"))
        gx, gw, gb = torch.autograd.grad(y.sum(), [x, w, b])
        assert not gx.any() and not gw.any()
        assert torch.equal(gb, (b > 0).float() * M)
    x = torch.randn(2, 3, 0, device="cuda", requires_grad=True)   # no depth, more than two axes
    w, b = torch.randn(4, 0, device="cuda", requires_grad=True), torch.randn(4, device="cuda", requires_grad=True)
    y = fused_linear(x, w, b, "relu")
    assert torch.equal(y, b.clamp(min=0).expand(2, 3, 4))
    gb, = torch.autograd.grad(y.sum(), [b])
    assert torch.equal(gb, 6.0 * (b > 0))
    x = torch.randn(5, 3, device="cuda", requires_grad=True)      # a layer of nothing between two others
    w = [torch.randn(0, 3, device="cuda", requires_grad=True), torch.randn(2, 0, device="cuda", requires_grad=True)]
    b = torch.randn(2, device="cuda", requires_grad=True)
    y = fused_mlp(x, w, [None, b], ["gelu", "none"])
    assert torch.equal(y, b.expand(5, 2))
    gx, gb = torch.autograd.grad(y.sum(), [x, b])
    assert not gx.any() and torch.equal(gb, torch.full_like(gb, 5))
    x = torch.randn(0, 3, device="cuda", requires_grad=True)
    w = [torch.randn(4, 3, device="cuda", requires_grad=True), torch.randn(2, 4, device="cuda", requires_grad=True)]
    grads = torch.autograd.grad(fused_mlp(x, w, [None, None], ["relu", "none"]).sum(), [x, *w])
    assert not any(g.any() for g in grads)


def test_only_wanted_gradients():
    import torch
    from cafe_b200 import fused_linear
    x, w, b, _, gy = _make(70, 33, 45, torch.float32, 11)
    lx, lw, lb = (t.detach().requires_grad_(True) for t in (x, w, b))
    full = torch.autograd.grad(fused_linear(lx, lw, lb, "silu"), [lx, lw, lb], gy)
    for keep in range(1, 8):
        leaves = [t.detach().requires_grad_(bool(keep >> i & 1)) for i, t in enumerate((x, w, b))]
        got = torch.autograd.grad(fused_linear(*leaves, "silu"), [t for t in leaves if t.requires_grad], gy)
        for a, c in zip(got, [f for i, f in enumerate(full) if keep >> i & 1]):
            assert torch.equal(a, c)


def test_gradient_against_differences():
    """Central differences of a smooth function in 64 bits on the kernel's own outputs cannot resolve fp32; instead the step is
    large (2^-3) and the function quadratic in x (no activation), where central differences are exact up to rounding."""
    import torch
    from cafe_b200 import fused_linear
    x, w, b, _, gy = _make(9, 14, 21, torch.float32, 13)
    lx = x.clone().requires_grad_(True)
    gx, = torch.autograd.grad(fused_linear(lx, w, b), lx, gy)
    h = 0.125
    for i, j in [(0, 0), (3, 20), (8, 7)]:
        d = torch.zeros_like(x)
        d[i, j] = h
        up, down = (float((fused_linear(x + s * d, w, b).double() * gy.double()).sum()) for s in (1, -1))
        # each output off by (21 + 9) 2^-23 of the sum of magnitudes (< 8): 14 outputs of weight < 0.5 over 2h
        assert abs((up - down) / (2 * h) - float(gx[i, j])) < 14 * 0.5 * 30 * 2 ** -23 * 8 * 2 / (2 * h)


@pytest.mark.parametrize("act", ["none", "relu", "gelu"])
@pytest.mark.parametrize("M", [140, 40000])     # (both kernels)
def test_infinities_and_nans(act, M):
    """An element that is not finite reaches the outputs that a sum over it gives it, and no others."""
    import torch
    from cafe_b200 import fused_linear
    inf = float("inf")
    x, w, b, _, _ = _make(M, 150, 96, torch.float32, 17)
    w = w.to(torch.bfloat16).float()       # (values with few bits: their lower parts are zero)
    x[3, 5], x[50, 0], x[139, 95], x[20, 7], x[20, 8] = inf, -inf, float("nan"), inf, -inf
    w[10, 5] = 0
    w[77, 30] = inf
    got = fused_linear(x, w, b, act)
    z = x.double() @ w.double().t() + b.double()
    want = z if act == "none" else z.clamp(min=0) if act == "relu" else torch.nn.functional.gelu(z)
    if act == "gelu":   # (-inf * 0 of the formula: torch gives nan, as the formula does)
        assert torch.equal(got.isnan(), want.isnan())
    assert torch.equal(got.isnan(), want.isnan()) and torch.equal(got.isinf(), want.isinf())
    assert torch.equal(got[got.isinf()].double(), want[want.isinf()])
    fine = want.isfinite()
    assert float((got.double() - want)[fine].abs().max()) < 1e-4


@pytest.mark.parametrize("M,N,K", [(900, 40, 50), (60000, 150, 96), (5000, 300, 400)])
def test_gradients_that_are_not_finite(M, N, K):
    """An infinite gradient reaches its row of gx and of gW with the signs that the sums give it; a NaN with nothing but its lowest
    bit set (whose upper half alone would be an infinity) stays one."""
    import torch
    from cafe_b200 import fused_linear
    x, w, _, _, gy = _make(M, N, K, torch.float32, 71)
    x, w = x.sign() * 1.5, w.sign() * 0.25            # (few bits: lower parts that are zero)
    gy[M // 2, 3], gy[7, 20] = float("inf"), -float("inf")
    gy.view(torch.int32)[11, 9] = 0x7f800001
    leaves = [t.detach().requires_grad_(True) for t in (x, w)]
    gx, gw = torch.autograd.grad(fused_linear(*leaves), leaves, gy)
    for got, want in ((gx, gy.double() @ w.double()), (gw, gy.double().t() @ x.double())):
        assert torch.equal(got.isnan(), want.isnan())
        inf = want.isinf()
        assert torch.equal(got.isinf(), inf) and torch.equal(got[inf].double(), want[inf])


def test_large_and_small_magnitudes():
    """Products far from 1: every part of a split operand keeps its place."""
    import torch
    from cafe_b200 import fused_linear
    import dense_reference as ref
    for sx, sw in [(1e-17, 1e-13), (1e18, 1e15), (1e-25, 1e25), (3e38, 1e-30)]:
        x, w, _, _, _ = _make(130, 70, 90, torch.float32, 19)
        x, w = (x / x.abs().max()) * sx, (w / w.abs().max()) * sw
        want, bound, *_ = ref.forward(x, w, None, "none", None, torch.float32)
        # (products below the smallest normal number may be flushed: six per term, 1.2e-38 each)
        ref.assert_within(fused_linear(x, w), want, bound + 90 * 6 * 1.2e-38, f"y at {sx} {sw}")


@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
@pytest.mark.parametrize("M,N,K", [(90, 40, 24), (2000, 512, 640)])
def test_one_gradient_row_for_all(M, N, K, dtype):
    import torch
    from cafe_b200 import fused_linear
    import dense_reference as ref
    dt = getattr(torch, dtype)
    x, w, b, _, gy = _make(M, N, K, dt, 47)
    row = gy[:1].expand(M, N)
    _, _, z, z_off = ref.forward(x, w, b, "silu", None, dt)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    got = torch.autograd.grad(fused_linear(*leaves, "silu"), leaves, row)
    for a, (name, (value, far)) in zip(got, ref.backward(row, z, z_off, x, w, "silu", dt).items()):
        ref.assert_within(a, value, far, name)


def test_more_rows_than_the_laid_out_form_takes():
    import torch
    _check((1 << 20) + 77, 65, 64, torch.float32, "relu", seed=53)


@pytest.mark.parametrize("dtype", ["float32", "bfloat16", "float16"])
@pytest.mark.parametrize("M,N,K", [(3, 50, 70), (130, 70, 90), (5000, 3, 37), (2500, 500, 450)])
def test_what_lies_between_rows_is_left(M, N, K, dtype):
    """The C entry points with outputs that are slices of wider tensors: nothing but the slices is written, and nothing past the
    workspace that the library asked for."""
    import torch
    from cafe_b200 import _lib
    import dense_reference as ref
    dt, lib = getattr(torch, dtype), _lib.load()
    t = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}[dt]
    x, w, b, _, gy = _make(M, N, K, dt, 59)
    st = torch.cuda.current_stream().cuda_stream
    wide = lambda r, c: torch.full((r + 2, c + 5), 7.0, device="cuda", dtype=dt)   # noqa: E731
    cut = lambda a, r, c: a[1:1 + r, 2:2 + c]                                      # noqa: E731
    slope = torch.full((M + 2, N + 5), 7.0, device="cuda", dtype=torch.float16 if dt == torch.bfloat16 else torch.float32)
    y, gx, gw, gb = wide(M, N), wide(M, K), wide(N, K), torch.full((N + 4,), 7.0, device="cuda", dtype=dt)
    at = lambda a, r, c: cut(a, r, c).data_ptr()                                   # noqa: E731

    def work(size):
        return torch.full((size + 64,), 171, dtype=torch.uint8, device="cuda")
    size = lib.cafe_linear_forward_work(x.data_ptr(), K, w.data_ptr(), K, M, N, K, t)
    wf = work(size)
    assert lib.cafe_linear_forward(x.data_ptr(), K, w.data_ptr(), K, b.data_ptr(), None, 0, M, N, K, t, 4, at(y, M, N), N + 5, at(slope, M, N), N + 5,
                                   wf.data_ptr(), size, st) == 0
    size = lib.cafe_linear_backward_work(gy.data_ptr(), N, 1, x.data_ptr(), K, w.data_ptr(), K, M, N, K, t, 1, 1, 1)
    wb = work(size)
    assert lib.cafe_linear_backward(gy.data_ptr(), N, at(slope, M, N), N + 5, 1, x.data_ptr(), K, w.data_ptr(), K, M, N, K, t, at(gx, M, K), K + 5,
                                    at(gw, N, K), K + 5, gb[2:].data_ptr(), wb.data_ptr(), size, st) == 0
    torch.cuda.synchronize()
    assert bool((wf[-64:] == 171).all()) and bool((wb[-64:] == 171).all())
    want, bound, z, z_off = ref.forward(x, w, b, "silu", None, dt)
    ref.assert_within(cut(y, M, N), want, bound, "y")
    back = ref.backward(gy, z, z_off, x, w, "silu", dt)
    for name, got in (("gx", cut(gx, M, K)), ("gw", cut(gw, N, K)), ("gb", gb[2:2 + N])):
        ref.assert_within(got, *back[name], name)
    for a, r, c in ((y, M, N), (slope, M, N), (gx, M, K), (gw, N, K)):
        cut(a, r, c).fill_(7.0)
        assert bool((a == 7).all())
    gb[2:2 + N] = 7
    assert bool((gb == 7).all())


@pytest.mark.parametrize("M,N,K", [(60, 40, 50), (1500, 500, 450)])
def test_saved_tensors_that_come_back_at_another_pitch(M, N, K):
    """save_on_cpu brings slices of wider tensors back without what lay between their rows."""
    import torch
    from cafe_b200 import fused_linear, fused_mlp
    x, w, b, _, gy = _make(M, N, K, torch.float32, 67)
    wide = lambda t: torch.cat([t, torch.full((t.shape[0], 3), float("nan"), device="cuda")], 1)[:, :t.shape[1]]   # noqa: E731
    w2 = torch.randn(20, N, device="cuda")
    calls = {"linear": (lambda x, w, b: fused_linear(x, w, b, "gelu"), [x, w, b], gy),
             "relu": (lambda x, w, b: fused_linear(x, w, b, "relu"), [x, w, b], gy),
             "mlp": (lambda x, w, b, w2: fused_mlp(x, [w, w2], [b, None], ["silu", "none"]), [x, w, b, w2], gy[:, :20].contiguous())}
    for name, (call, leaves, grad) in calls.items():
        leaves = [t.detach().requires_grad_(True) for t in leaves]
        want = torch.autograd.grad(call(*leaves), leaves, grad)
        sliced = [wide(t.detach()).requires_grad_(True) if t.dim() == 2 else t for t in leaves]
        with torch.autograd.graph.save_on_cpu():
            y = call(*sliced)
        for a, e in zip(torch.autograd.grad(y, sliced, grad), want):
            torch.testing.assert_close(a, e, rtol=1e-4, atol=1e-4)   # (other kernels may take a slice: sums of 1500 terms in other orders)


def test_two_threads():
    """Calls of different sizes from two threads, each on its own stream."""
    import threading
    import torch
    from cafe_b200 import fused_linear
    sizes = [(3000, 600, 500), (40, 130, 90)]
    sets = [_make(M, N, K, torch.float32, 61 + i) for i, (M, N, K) in enumerate(sizes)]
    want = [fused_linear(x, w, b, "gelu") for x, w, b, _, _ in sets]
    torch.cuda.synchronize()
    got, errors = [[], []], []

    def go(i):
        try:
            x, w, b, _, _ = sets[i]
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(30):
                    got[i].append(fused_linear(x, w, b, "gelu"))
                torch.cuda.current_stream().synchronize()
        except Exception as e:   # noqa: BLE001
            errors.append(e)
    threads = [threading.Thread(target=go, args=(i,)) for i in range(2)]
    for q in threads:
        q.start()
    for q in threads:
        q.join()
    assert not errors, errors
    for i in range(2):
        assert all(torch.equal(a, want[i]) for a in got[i])


def test_offsets_past_32_bits():
    """A weight matrix of more than 2^31 elements apart: rows of one pitch of 2^21 elements."""
    import torch
    from cafe_b200 import fused_linear
    import dense_reference as ref
    big = torch.zeros(1100, 1 << 21, dtype=torch.bfloat16, device="cuda")     # 4.6 GB, 2.3e9 elements
    w = big[:, (1 << 21) - 40:]
    g = torch.Generator(device="cuda").manual_seed(23)
    w.copy_(torch.randn(1100, 40, device="cuda", generator=g))
    x = torch.randn(30, 40, device="cuda", generator=g).to(torch.bfloat16)
    want, bound, *_ = ref.forward(x, w, None, "none", None, torch.bfloat16)
    ref.assert_within(fused_linear(x, w), want, bound, "y")
    gy = torch.randn(1100, 30, device="cuda", generator=g).to(torch.bfloat16)
    lx = w.detach().requires_grad_(True)
    lw = torch.randn(30, 40, device="cuda", generator=g).to(torch.bfloat16).requires_grad_(True)
    gx, gw = torch.autograd.grad(fused_linear(lx, lw), [lx, lw], gy)
    for name, (value, far) in ref.backward(gy, torch.zeros(1100, 30, device="cuda").double(), torch.zeros((), device="cuda").double(), w, lw.detach(), "none", torch.bfloat16).items():
        if name != "gb":
            ref.assert_within(dict(gx=gx, gw=gw)[name], value, far, name)


@pytest.mark.parametrize("M,widths,acts", [(128, [13, 512, 256, 64, 16], ["relu"] * 4), (50, [367, 512, 256, 1], ["silu", "gelu", "sigmoid"]),
                                           (1, [479, 1024, 512, 1], ["relu", "relu", "sigmoid"]), (2049, [35, 24, 7], ["none", "sigmoid"]),
                                           (33, [40, 9], ["gelu"])])
@pytest.mark.parametrize("dtype", ["float32", "bfloat16"])
def test_mlp_equals_layer_by_layer(M, widths, acts, dtype):
    """A run of layers as one node against fused_linear layer by layer.  Values are those of the same kernels on the same
    operands (another pitch between rows may take another order of sums: the bounds of one layer, carried on)."""
    import torch
    from cafe_b200 import fused_linear, fused_mlp
    dt = getattr(torch, dtype)
    g = torch.Generator(device="cuda").manual_seed(29)
    x = torch.randn(M, widths[0], device="cuda", generator=g).to(dt).requires_grad_(True)
    ws = [(torch.randn(n, m, device="cuda", generator=g) * (2 / (n + m)) ** 0.5).to(dt).requires_grad_(True) for m, n in zip(widths, widths[1:])]
    bs = [(torch.randn(n, device="cuda", generator=g) * 0.1).to(dt).requires_grad_(True) for n in widths[1:]]
    bs[0] = None
    y = fused_mlp(x, ws, bs, acts)
    h, hidden = x, []
    for w, b, a in zip(ws, bs, acts):
        h = fused_linear(h, w, b, a)
        hidden.append(h)
    # relative to the whole: each layer adds (K + 8) 2^-23 (fp32) or half a step (bf16) to what came before, against norms
    # that grow by the layers' gain (< 4 in all here)
    tol = (sum(widths) * 2 ** -23 if dt == torch.float32 else len(ws) * 2 ** -8) * 4
    rel = lambda a, c: float(((a.double() - c.double()).norm() / c.double().norm().clamp(min=1e-30)).detach())   # noqa: E731
    assert rel(y, h) <= tol
    gy = torch.randn(M, widths[-1], device="cuda", generator=g).to(dt)
    leaves = [x, *ws, *[b for b in bs if b is not None]]
    ga, gb = torch.autograd.grad(y, leaves, gy), torch.autograd.grad(h, leaves, gy)
    flips = "relu" in acts    # (a ReLU whose pre-activation is within rounding of zero may differ: few of M x N)
    for a, c in zip(ga, gb):
        assert rel(a, c) <= (4 * tol if not flips else max(4 * tol, 0.02))
    with torch.no_grad():
        assert torch.equal(fused_mlp(x, ws, bs, acts), y)


def test_fused_mlp_module_is_the_reference_mlp():
    import numpy as np
    import torch
    import dense_reference as ref
    from cafe_b200 import FusedMLP
    from cafe_b200.dlrm_harness import create_mlp
    plain = create_mlp([13, 64, 32, 1], 2, np.random.default_rng(0)).cuda()
    fused = FusedMLP(*create_mlp([13, 64, 32, 1], 2, np.random.default_rng(0))).cuda()
    assert list(plain.state_dict()) == list(fused.state_dict())
    x = torch.randn(77, 13, device="cuda")
    want, off = x.double(), None
    for lin, act in zip([plain[0], plain[2], plain[4]], ["relu", "relu", "sigmoid"]):
        want, off, *_ = ref.forward(want, lin.weight, lin.bias, act, None, torch.float32, off)
    ref.assert_within(fused(x).detach(), want.detach(), off.detach(), "y")
    fused(x).sum().backward()
    assert all(p.grad is not None and p.grad.shape == p.shape for p in fused.parameters())


@pytest.mark.parametrize("M,N,K", [(150, 400, 300), (1500, 700, 900)])
def test_on_another_stream_and_two_calls_at_once(M, N, K):
    import torch
    from cafe_b200 import fused_linear
    x, w, b, _, gy = _make(M, N, K, torch.float32, 31)
    want = fused_linear(x, w, b, "gelu")
    streams = [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    got = []
    for s in streams:
        with torch.cuda.stream(s):
            leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
            y = fused_linear(*leaves, "gelu")
            got.append((y, torch.autograd.grad(y, leaves, gy)))
    torch.cuda.synchronize()
    for y, g in got:
        assert torch.equal(y, want)
        for a, c in zip(g, got[0][1]):
            assert torch.equal(a, c)


def test_repeated_calls_give_the_same_bits():
    import torch
    from cafe_b200 import fused_linear
    for M, N, K in [(9000, 130, 70), (64, 512, 1000), (30000, 16, 40), (20000, 200, 300), (2048, 1024, 1024)]:
        x, w, b, _, gy = _make(M, N, K, torch.float32, 37)
        leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
        first = None
        for _ in range(5):
            y = fused_linear(*leaves, "silu")
            now = (y, *torch.autograd.grad(y, leaves, gy))
            assert first is None or all(torch.equal(a, c) for a, c in zip(now, first))
            first = now


@pytest.mark.parametrize("M,N,K", [(700, 130, 260), (3000, 640, 900)])
def test_captured_and_replayed(M, N, K):
    """Two captured graphs of forward and backward, replayed in turn and on two streams at once with new inputs."""
    import torch
    from cafe_b200 import fused_linear, fused_mlp
    sets = []
    for seed in (41, 42):
        x, w, b, _, gy = _make(M, N, K, torch.float32, seed)
        w2 = torch.randn(40, N, device="cuda") * 0.1
        x, w, b, w2 = (t.detach().clone().requires_grad_(True) for t in (x, w, b, w2))
        gy = torch.randn(M, 40, device="cuda")

        def go(x=x, w=w, b=b, w2=w2, gy=gy):
            y = fused_linear(fused_linear(x, w, b, "gelu"), w2)
            z = fused_mlp(x, [w, w2], [b, None], ["gelu", "none"])
            return (y, z, *torch.autograd.grad(y, [x, w, b, w2], gy), *torch.autograd.grad(z, [x, w, b, w2], gy))
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            for _ in range(2):
                go()
        torch.cuda.current_stream().wait_stream(side)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = go()
        sets.append((x, go, graph, out))
    streams = [torch.cuda.Stream() for _ in sets]
    for round_ in range(3):
        for x, *_ in sets:
            with torch.no_grad():
                x.normal_()
        want = [[t.clone() for t in go()] for _, go, _, _ in sets]
        torch.cuda.synchronize()
        for (_, _, graph, _), s in zip(sets, streams):
            with torch.cuda.stream(s):
                graph.replay()
        torch.cuda.synchronize()
        for (_, _, _, out), exp in zip(sets, want):
            assert all(torch.equal(a, c) for a, c in zip(out, exp))


def test_refusals_with_cuda_tensors():
    import torch
    from cafe_b200 import FusedMLP, fused_linear, fused_mlp
    x, w, b = torch.randn(4, 6, device="cuda"), torch.randn(5, 6, device="cuda"), torch.randn(5, device="cuda")
    for bad in [lambda: fused_linear(x, w[:, :5], b), lambda: fused_linear(x, w, b[:4]), lambda: fused_linear(x, w, b, "tanh"),
                lambda: fused_linear(x.half(), w, b), lambda: fused_linear(x.double(), w.double()), lambda: fused_linear(x, w.cpu()),
                lambda: fused_linear(x, w, b.view(5, 1)), lambda: fused_mlp(x, [w, w], [None, None], ["relu", "relu"]),
                lambda: fused_mlp(x, [w], [], ["relu"]), lambda: fused_mlp(x, [], [], []), lambda: FusedMLP(torch.nn.Tanh()),
                lambda: FusedMLP(torch.nn.Linear(3, 3), torch.nn.Tanh()), lambda: fused_linear(torch.ones((), device="cuda"), w)]:
        with pytest.raises(ValueError):
            bad()
    with pytest.raises(RuntimeError):
        fused_linear(x, w, b, "none", torch.randn(3, 5, device="cuda"))
    lx = x.clone().requires_grad_(True)
    gx, = torch.autograd.grad(fused_linear(lx, w, b, "gelu").sum(), lx, create_graph=True)
    with pytest.raises(RuntimeError):
        gx.sum().backward()


@pytest.mark.parametrize("call", ["relu", "gelu", "mlp"])
def test_as_a_node_of_the_graph(call):
    """A second backward needs retain_graph, what was saved must not have been written to, nothing is left behind."""
    import gc
    import torch
    from cafe_b200 import fused_linear, fused_mlp
    x, w, b, _, gy = _make(70, 60, 50, torch.float32, 73)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]

    def forward():
        x, w, b = leaves
        return fused_mlp(x, [w], [b], ["silu"]) if call == "mlp" else fused_linear(x, w, b, call)
    y = forward()
    first = torch.autograd.grad(y, leaves, gy, retain_graph=True)
    again = torch.autograd.grad(y, leaves, gy)
    assert all(torch.equal(p, q) for p, q in zip(first, again))
    with pytest.raises(RuntimeError):
        torch.autograd.grad(y, leaves, gy)
    y = forward()
    with torch.no_grad():
        leaves[1].mul_(2)
    with pytest.raises(RuntimeError, match="inplace"):
        torch.autograd.grad(y, leaves, gy)
    y = forward()
    gw, = torch.autograd.grad(y, leaves[1], gy)
    assert torch.isfinite(gw).all()
    assert "Fused" in y.grad_fn.name()
    del y, gw, first, again
    gc.collect()
    torch.cuda.synchronize()
    before = torch.cuda.memory_allocated()
    for _ in range(20):
        y = forward()
        torch.autograd.grad(y, leaves, gy)
        forward()
    del y
    gc.collect()
    assert torch.cuda.memory_allocated() == before


def test_no_wait_has_run_out():
    """Last of the file: the count of waits that ran out in all that ran before."""
    import ctypes
    from cafe_b200 import _lib
    count = ctypes.c_int32(-1)
    assert _lib.load().cafe_linear_gave_up(ctypes.byref(count)) == 0
    assert count.value == 0
    assert _lib.load().cafe_linear_gave_up(None) == 1
