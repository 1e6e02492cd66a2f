"""The dense half of a training or serving step, as cases that can be timed and whose outputs can be compared.

Two operators, each through the entry points that a user's program calls:

  linear, mlp   cafe_b200.fused_linear / fused_mlp: a matrix product with bias, activation and residual in its epilogue,
                alone and as the layers of an MLP, forward only (serving) or forward and backward (training)
  adamw         cafe_b200.AdamW: one step over many tensors at once, moments held in 32 bits or in 8

Shapes are those of the click-log models of cafe_b200.dlrm_harness (layer widths, batches), or generic ones.

Inputs of a layer with a ReLU lie on a binary grid (x in sixteenths, weights in 512ths, biases in 8192ths), on which
every order of the sum gives the same pre-activation: the derivative of a ReLU jumps at zero, so that otherwise two right
results would differ wherever a pre-activation is within a rounding of it.

With `own` false the same is computed by elementary torch operations in 32 bits.
"""
import math

import torch

own = False

TYPES = {"fp32": torch.float32, "bf16": torch.bfloat16, "fp16": torch.float16}
BLOCK = 256          # elements that share the exponent of their 8-bit moments
MOST_FLOPS = 6 * 16384 * 1024 * 4096
MOST_ELEMENTS = 134_000_000

KAGGLE = "512x13,512,256x512,256,64x256,64,16x64,16,512x367,512,256x512,256,1x256,1"
TERABYTE = "512x13,512,256x512,256,128x256,128,1024x479,1024,1024x1024,1024,512x1024,512,256x512,256,1x256,1"
BLOCKS = ",".join(["4096x2048,4096,2048x4096,2048"] * 4)


def listed():
    def linear(name, rows, cols, out, act, dtype, train, residual=False, pitch=0):
        return dict(name=name, kind="linear", rows=rows, cols=cols, out=out, act=act, dtype=dtype, train=train, residual=residual, pitch=pitch)

    def mlp(name, rows, widths, act, last, train):
        return dict(name=name, kind="mlp", rows=rows, widths=widths, act=act, last=last, dtype="fp32", train=train)

    def adamw(name, sizes, dtype, bits):
        return dict(name=name, kind="adamw", sizes=sizes, dtype=dtype, bits=bits)
    return [
        # one request through one layer: latency is all there is
        linear("linear_serve_1x1024x1024", 1, 1024, 1024, "relu", "fp32", False),
        # the first top layer of the Kaggle model at its batch of 128: odd width, few tiles, two short products in the backward
        linear("linear_train_128x367x512", 128, 367, 512, "relu", "fp32", True),
        # the first top layer of the Terabyte model at the micro-benchmark's batch: a long axis to reduce over for the weights
        linear("linear_train_65536x479x1024", 65536, 479, 1024, "relu", "fp32", True),
        # a wide layer in bfloat16 with a smooth activation and a residual: the largest product
        linear("linear_train_bf16_16384x1024x4096", 16384, 1024, 4096, "gelu", "bf16", True, True),
        # ragged sizes in half precision, the input a slice of a wider tensor
        linear("linear_train_fp16_1777x367x511", 1777, 367, 511, "silu", "fp16", True, True, 13),
        # the Terabyte model's top MLP scoring a handful of candidates
        mlp("mlp_serve_16_terabyte", 16, "479-1024-1024-512-256-1", "relu", "sigmoid", False),
        # the same MLP in training, its batch of 2048 (smooth inner activations: see above)
        mlp("mlp_train_2048_terabyte", 2048, "479-1024-1024-512-256-1", "silu", "sigmoid", True),
        # the deep half of the Avazu DCN at its batch
        mlp("mlp_train_4096_avazu", 4096, "352-1024-1024", "gelu", "gelu", True),
        # all dense parameters of the Kaggle model: launches count
        adamw("adamw_kaggle_32bit", KAGGLE, "fp32", 32),
        # those of the Terabyte model, moments in 8 bits
        adamw("adamw_terabyte_8bit", TERABYTE, "fp32", 8),
        # large matrices: bandwidth counts
        adamw("adamw_large_bf16_32bit", BLOCKS, "bf16", 32),
        adamw("adamw_large_8bit", BLOCKS, "fp32", 8),
    ]


def _log_int(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi + 1)))))))


def draw(rng):
    kind = rng.choice(["linear"] * 4 + ["mlp"] * 2 + ["adamw"] * 3)
    dtype = rng.choice(["fp32", "fp32", "bf16", "fp16"])
    if kind == "adamw":
        n = rng.randint(2, 20)
        most = _log_int(rng, 1000, MOST_ELEMENTS // n)
        return dict(kind=kind, sizes=",".join(str(_log_int(rng, 1, most)) for _ in range(n)), dtype=dtype, bits=rng.choice([8, 32]))
    train = rng.random() < 0.7
    if kind == "mlp":
        widths = [_log_int(rng, 13, 1100) for _ in range(rng.randint(2, 5))] + [rng.choice([1, 16, 64, 256])]
        per_row = 6 * sum(a * b for a, b in zip(widths, widths[1:]))
        return dict(kind=kind, rows=_log_int(rng, 1, min(65536, MOST_FLOPS // per_row)), widths="-".join(map(str, widths)),
                    act=rng.choice(["silu", "gelu"] if train else ["relu", "silu", "gelu"]), last=rng.choice(["sigmoid", "none"]), dtype="fp32", train=train)
    cols, out = _log_int(rng, 13, 4096), _log_int(rng, 1, 4096)
    return dict(kind=kind, rows=_log_int(rng, 1, min(65536, MOST_FLOPS // (6 * cols * out))), cols=cols, out=out,
                act=rng.choice(["none", "relu", "sigmoid", "gelu", "silu"]), dtype=dtype, train=train, residual=rng.random() < 0.4,
                pitch=rng.choice([0, 0, 1, 8, 33]))


# ---- inputs ------------------------------------------------------------------------------------------------
def _randn(gen, *shape):
    return torch.randn(shape, device="cuda", generator=gen)


def _layer(gen, n, m, act):
    """Weight and bias of a layer from n to m, distributed as the models initialise them."""
    w, b = _randn(gen, m, n) * math.sqrt(2 / (m + n)), _randn(gen, m) * math.sqrt(1 / m)
    return ((w * 512).round() / 512, (b * 8192).round() / 8192) if act == "relu" else (w, b)


def _shapes(case):
    return [tuple(int(v) for v in s.split("x")) for s in case["sizes"].split(",")]


def _prepare_adamw(case, gen):
    dt, shapes = TYPES[case["dtype"]], _shapes(case)
    s = dict(case=case, lr=1e-3, betas=(0.9, 0.999), eps=1e-8, decay=0.01, seed=17, step=10)
    s["p"] = [(_randn(gen, *h) * 0.05).to(dt) for h in shapes]
    # gradients whose size differs from row to row, as those of a real layer do
    s["g"] = [(_randn(gen, *h) * 1e-3 * torch.exp(_randn(gen, h[0], *([1] * (len(h) - 1))))).to(dt) for h in shapes]
    m = [_randn(gen, *h) * 4e-4 for h in shapes]
    v = [(_randn(gen, *h) * 3e-4).square() + 1e-9 for h in shapes]
    if case["bits"] == 8:
        zero = [torch.zeros((), dtype=torch.int64, device="cuda")] * len(shapes)
        m, v = [_pack(x.reshape(-1), z, 3) for x, z in zip(m, zero)], [_pack(x.reshape(-1).sqrt(), z, 4) for x, z in zip(v, zero)]
    s["m"], s["v"] = m, v
    if own:
        import cafe_b200
        params = [torch.nn.Parameter(p) for p in s["p"]]
        opt = cafe_b200.AdamW(params, lr=s["lr"], betas=s["betas"], eps=s["eps"], weight_decay=s["decay"], state_bits=case["bits"], seed=s["seed"])
        kept = {}
        for i, (a, b) in enumerate(zip(m, v)):
            at = torch.tensor(s["step"], dtype=torch.int64, device="cuda")
            kept[i] = (dict(step=at, exp_avg=a, exp_avg_sq=b) if case["bits"] == 32 else
                       dict(step=at, exp_avg=a[0], exp_avg_top=a[1], root_avg_sq=b[0], root_avg_sq_top=b[1]))
        opt.load_state_dict(dict(state=kept, param_groups=opt.state_dict()["param_groups"]))
        for p, g in zip(params, s["g"]):
            p.grad = g
        s["params"], s["opt"], s["m"], s["v"] = params, opt, None, None
    return s


def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed) * 7919 + 5)
    if case["kind"] == "adamw":
        return _prepare_adamw(case, gen)
    dt = TYPES[case["dtype"]]
    widths = [int(v) for v in case["widths"].split("-")] if case["kind"] == "mlp" else [case["cols"], case["out"]]
    acts = [case["act"]] * (len(widths) - 2) + [case.get("last", case["act"])]
    M, pitch = case["rows"], case.get("pitch", 0)
    x = _randn(gen, M, widths[0] + pitch)
    if case["act"] == "relu":
        x = ((x * 16).round() / 16).clamp_(-4, 4)
    x = x.to(dt)[:, pitch:]
    layers = [_layer(gen, n, m, case["act"]) for n, m in zip(widths, widths[1:])]
    s = dict(case=case, acts=acts, w=[w.to(dt) for w, _ in layers], b=[b.to(dt) for _, b in layers], x=x, r=None, gy=None)
    if case.get("residual"):
        s["r"] = _randn(gen, M, widths[-1]).to(dt)
    if case["train"]:
        s["gy"] = (_randn(gen, M, widths[-1]) * 0.01).to(dt)
    if own and case["train"]:
        s["x"] = s["x"].requires_grad_(True)
        s["w"], s["b"] = [torch.nn.Parameter(w) for w in s["w"]], [torch.nn.Parameter(b) for b in s["b"]]
        if s["r"] is not None:
            s["r"].requires_grad_(True)
    return s


# ---- plain forms -------------------------------------------------------------------------------------------
def _erf_half(z):
    return 0.5 * (1 + torch.erf(z * math.sqrt(0.5)))


def _act(z, act):
    """act(z) and its derivative."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return torch.where(z > 0, z, torch.zeros_like(z)), (z > 0).to(z.dtype)
    if act == "gelu":
        c = _erf_half(z)
        return z * c, c + z * torch.exp(-0.5 * z * z) * (1 / math.sqrt(2 * math.pi))
    e = torch.exp(-z.abs())
    s, t = torch.where(z >= 0, 1 / (1 + e), e / (1 + e)), torch.where(z >= 0, e / (1 + e), 1 / (1 + e))   # sigmoid(z), 1 - sigmoid(z)
    return (s, s * t) if act == "sigmoid" else (z * s, s * (1 + z * t))


def _linear_plain(s):
    case, f = s["case"], torch.float32
    dt = TYPES[case["dtype"]]
    inputs, slopes, y = [], [], s["x"].to(f)
    for w, b, act in zip(s["w"], s["b"], s["acts"]):
        inputs.append(y)
        y, d = _act(y @ w.to(f).t() + b.to(f), act)
        slopes.append(d)
    out = dict(y=(y if s["r"] is None else y + s["r"].to(f)).to(dt))
    if not case["train"]:
        return out
    g, gw, gb = s["gy"].to(f), [], []
    for x, d, w in zip(reversed(inputs), reversed(slopes), reversed(s["w"])):
        gz = g * d
        gw.append((gz.t() @ x).to(dt))
        gb.append(gz.sum(0).to(dt))
        g = gz @ w.to(f)
    out.update(gx=g.to(dt), gw=gw[::-1], gb=gb[::-1])
    if s["r"] is not None:
        out["gr"] = s["gy"]
    return out


_M32 = 0xFFFFFFFF


def _mix(x):
    """A mixing of 32-bit integers (held in 64)."""
    x = x & _M32
    x = x ^ (x >> 16)
    x = (x * 0x7FEB352D) & _M32
    x = x ^ (x >> 15)
    x = (x * 0x846CA68B) & _M32
    return x ^ (x >> 16)


def _random(n, seed, index, step):
    """The 32 random bits of every element of tensor `index` at `step`."""
    key = _mix(_mix(seed + 0x9E3779B9 * (index + 1)) ^ (step & _M32))
    at = torch.arange(n, device="cuda")
    return _mix((at & _M32) ^ _mix(key + (at >> 32)))


def _blocks(x):
    return torch.nn.functional.pad(x, (0, -x.numel() % BLOCK)).view(-1, BLOCK)


def _pack(x, rnd, S):
    """fp32 values [n] -> (codes uint8 [n], exponent of the block's largest code uint8 [blocks]).

    A code keeps 4 bits of exponent, relative to its block's, and S of the mantissa; with S = 3 the eighth bit is the sign.
    Rounded up or down at random by the 16 bits `rnd`, so that the mean is the value; below the smallest code to it or to
    zero in the same way (S = 3), or up to it (S = 4: roots of second moments divide, so a value that is not zero stays)."""
    drop, n = 23 - S, x.numel()
    rnd = rnd.expand(n)
    bits = x.abs().view(torch.int32).to(torch.int64)
    top = (((_blocks(bits) + (1 << drop) - 1) >> drop).amax(1) >> S).clamp(16, 255)
    base = top.repeat_interleave(BLOCK)[:n]
    base = (base - 15) << S
    code = ((bits + (rnd << (drop - 16))) >> drop) - base
    least = ((base + 1) << drop).to(torch.int32).view(torch.float32)
    small = (rnd.to(torch.float32) * (least * 2.0 ** -16) < x.abs()) if S == 3 else x > 0
    code = torch.where(x.abs() < least, small.to(torch.int64), code)
    if S == 3:
        code = code | (x < 0).to(torch.int64) << 7
    return code.to(torch.uint8), top.to(torch.uint8)


def _unpack(code, top, S):
    n, c = code.numel(), code.to(torch.int64)
    low = c & 127 if S == 3 else c
    base = (top.to(torch.int64).repeat_interleave(BLOCK)[:n] - 15) << S
    x = torch.where(low > 0, ((low + base) << (23 - S)).to(torch.int32).view(torch.float32), torch.zeros((), device="cuda"))
    return torch.where(c > 127, -x, x) if S == 3 else x


def _adamw_tensor(s, i):
    """One tensor's step; the new state replaces the old one."""
    p, g, m, v, step = s["p"][i], s["g"][i].to(torch.float32), s["m"][i], s["v"][i], s["step"] + 1
    b1, b2 = s["betas"]
    packed = s["case"]["bits"] == 8
    if packed:
        m, v = _unpack(*m, 3).view(p.shape), _unpack(*v, 4).view(p.shape).square()
    m, v = m * b1 + g * (1 - b1), v * b2 + g * (1 - b2) * g
    root = v.sqrt()
    new = p.to(torch.float32) * (1 - s["lr"] * s["decay"]) - s["lr"] / (1 - b1 ** step) * m / (root / math.sqrt(1 - b2 ** step) + s["eps"])
    s["p"][i].copy_(new)
    if not packed:
        s["m"][i].copy_(m)
        s["v"][i].copy_(v)
        return s["p"][i], s["m"][i], s["v"][i]
    rnd = _random(p.numel(), s["seed"], i, step)
    s["m"][i], s["v"][i] = _pack(m.reshape(-1), rnd & 0xFFFF, 3), _pack(root.reshape(-1), rnd >> 16, 4)
    return s["p"][i], _unpack(*s["m"][i], 3).to(torch.bfloat16), _unpack(*s["v"][i], 4).to(torch.bfloat16)   # (4 and 5 bits: exact)


def _adamw_plain(s):
    out = [_adamw_tensor(s, i) for i in range(len(s["p"]))]
    s["step"] += 1
    return dict(p=[o[0] for o in out], m=[o[1] for o in out], v=[o[2] for o in out])


# ---- the framework's calls ---------------------------------------------------------------------------------
def _own(s):
    import cafe_b200
    if s["case"]["kind"] == "adamw":
        s["opt"].step()
        moments = s["opt"].moments()
        if s["case"]["bits"] == 8:   # (as the plain form holds them: one axis)
            moments = [(m.view(-1), v.view(-1)) for m, v in moments]
        return dict(p=[p.data for p in s["params"]], m=[m for m, _ in moments], v=[v for _, v in moments])
    mlp, train = s["case"]["kind"] == "mlp", s["case"]["train"]
    if not train:
        with torch.no_grad():
            return dict(y=cafe_b200.fused_mlp(s["x"], s["w"], s["b"], s["acts"]) if mlp else
                        cafe_b200.fused_linear(s["x"], s["w"][0], s["b"][0], s["acts"][0], s["r"]))
    y = (cafe_b200.fused_mlp(s["x"], s["w"], s["b"], s["acts"]) if mlp else
         cafe_b200.fused_linear(s["x"], s["w"][0], s["b"][0], s["acts"][0], s["r"]))
    n = len(s["w"])
    got = torch.autograd.grad(y, [s["x"], *s["w"], *s["b"]] + ([] if s["r"] is None else [s["r"]]), s["gy"])
    out = dict(y=y, gx=got[0], gw=list(got[1:1 + n]), gb=list(got[1 + n:1 + 2 * n]))
    if s["r"] is not None:
        out["gr"] = got[-1]
    return out


def run(state):
    if own:
        return _own(state)
    return _adamw_plain(state) if state["case"]["kind"] == "adamw" else _linear_plain(state)


# ---- what a pass has to move and compute -------------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "fp32" else 2
    if case["kind"] == "adamw":
        n = sum(math.prod(h) for h in _shapes(case))
        # parameters and moments in and out, gradients in; 8-bit moments also come out as the values they stand for
        return dict(bytes=n * (3 * size + (16 if case["bits"] == 32 else 8)), flops=15 * n)
    M = case["rows"]
    widths = [int(v) for v in case["widths"].split("-")] if case["kind"] == "mlp" else [case["cols"], case["out"]]
    weights = sum(a * b for a, b in zip(widths, widths[1:]))
    params, ends = weights + sum(widths[1:]), M * (widths[0] + widths[-1])
    more = M * widths[-1] if case.get("residual") else 0
    if not case["train"]:
        return dict(bytes=size * (params + ends + more), flops=2 * M * weights)
    return dict(bytes=size * 2 * (params + ends) + size * more, flops=6 * M * weights)


# ---- the same from the definition, in 64 bits --------------------------------------------------------------
def _exact_linear(case, s):
    h = s["x"].double()
    kept = []
    for w, b, act in zip(s["w"], s["b"], s["acts"]):
        z = torch.einsum("mk,nk->mn", h, w.double()) + b.double()
        if act == "relu":
            a, d = z.clamp(min=0), torch.heaviside(z, torch.zeros((), dtype=z.dtype, device="cuda"))
        elif act == "gelu":
            phi = 0.5 * torch.erfc(-z / math.sqrt(2.0))
            a, d = z * phi, phi + z * torch.exp(-z ** 2 / 2) / math.sqrt(2 * math.pi)
        elif act in ("sigmoid", "silu"):
            p, q = 1 / (1 + torch.exp(-z)), 1 / (1 + torch.exp(z))
            a, d = (p, p * q) if act == "sigmoid" else (z * p, p + z * p * q)
        else:
            a, d = z, torch.ones_like(z)
        kept.append((h, d, w))
        h = a
    out = dict(y=h + (0 if s["r"] is None else s["r"].double()))
    if case["train"]:
        g, gw, gb = s["gy"].double(), [], []
        for h, d, w in kept[::-1]:
            g = g * d
            gw.insert(0, torch.einsum("mn,mk->nk", g, h))
            gb.insert(0, torch.einsum("mn->n", g))
            g = torch.einsum("mn,nk->mk", g, w.double())
        out.update(gx=g, gw=gw, gb=gb)
        if s["r"] is not None:
            out["gr"] = s["gy"].double()
    return out


def exact(case, seed):
    global own
    was, own = own, False   # the inputs alone, without the framework's handle
    try:
        s = prepare(case, seed)
    finally:
        own = was
    if case["kind"] != "adamw":
        return _exact_linear(case, s)
    out, (b1, b2), t = dict(p=[], m=[], v=[]), s["betas"], s["step"] + 1
    for p, g, m, v in zip(s["p"], s["g"], s["m"], s["v"]):
        g = g.double()
        if case["bits"] == 8:
            m, v = _unpack(*m, 3).double().view(p.shape), _unpack(*v, 4).double().view(p.shape) ** 2
        m, v = torch.lerp(g, m.double(), b1), torch.lerp(g * g, v.double(), b2)
        p = p.double()
        p = p - s["lr"] * (s["decay"] * p + (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + s["eps"]))
        out["p"].append(p)
        # what the 8-bit moments are rounded to goes by random bits: no value of the definition alone
        out["m"].append(m if case["bits"] == 32 else None)
        out["v"].append(v if case["bits"] == 32 else None)
    return out
