"""AdamW over all tensors of a model in one launch (csrc/adamw_cuda.cu), moments in 32 bits or in 8."""
from __future__ import annotations

import torch

from .dense import _dense_torch

DTYPES = (torch.float32, torch.bfloat16, torch.float16)
BLOCK = 256   # elements that share the exponent of their 8-bit moments
_CODES = ("exp_avg", "exp_avg_top", "root_avg_sq", "root_avg_sq_top")


def _dense(t: torch.Tensor) -> bool:
    """Whether t's elements fill one piece of memory, each once."""
    if t.is_contiguous():
        return True
    at = 1
    for stride, size in sorted((s, n) for s, n in zip(t.stride(), t.shape) if n > 1):
        if stride != at:
            return False
        at *= size
    return True


def _layout(p: torch.Tensor) -> torch.Tensor:
    """p's sizes and strides: the order in which a flat array of codes goes through its elements."""
    return torch.tensor([tuple(p.shape), tuple(p.stride())], dtype=torch.int64)


def _layouts(states) -> list:
    found = [s["layout"] for s in states]
    for i, t in enumerate(found):
        if t.is_cuda:   # (moved there with the rest of a state)
            found[i] = states[i]["layout"] = t.cpu()
    return found


def _order(layout):
    """What two layouts whose elements come in the same order have in common: None if row-major, else their axes."""
    sizes, strides = layout.tolist()
    axes, at, rows = [(n, s) for n, s in zip(sizes, strides) if n != 1], 1, True
    for n, s in reversed(axes):
        rows &= s == at
        at *= n
    return None if rows or 0 in sizes else axes


class AdamW(torch.optim.Optimizer):
    """torch.optim.AdamW's update (decoupled weight decay, both moments corrected for their start at zero) for CUDA parameters
    of fp32, bf16 or fp16, computed in fp32.

    state_bits = 32 keeps exp_avg and exp_avg_sq in fp32.  state_bits = 8 keeps a byte per element for exp_avg and one for the
    root of exp_avg_sq, plus a byte per 256 elements for each; they are rounded at random (by `seed`, the tensor's place among
    the parameters, the step and the element), so that moments which change by less than a code's step still move on average.
    A gradient that is not finite, or whose square is not, makes its block of 256 moments not a number.

    A step counts on the device and reads nothing back, so it can be captured into a CUDA graph; lr and the other settings are
    then those of the capture, and the optimizer's state has to exist before it (one step outside).  Parameters without a
    gradient keep their moments and their step count.  Sparse gradients are refused, and so is a parameter whose elements have come to
    lie in another order than its moments (another memory format, exchanged .data)."""

    def __init__(self, params, lr: float = 1e-3, betas=(0.9, 0.999), eps: float = 1e-8, weight_decay: float = 1e-2, state_bits: int = 32,
                 seed: int = 0):
        self._check_settings(dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))
        if state_bits not in (8, 32):
            raise ValueError(f"state_bits must be 8 or 32, got {state_bits!r}")
        self.state_bits, self.seed = state_bits, int(seed) & 0xFFFFFFFF
        self._ticket = {}
        super().__init__(params, dict(lr=lr, betas=betas, eps=eps, weight_decay=weight_decay))

    def __getstate__(self):   # (torch's has the settings and the state alone: copies and pickles need the rest)
        return {**super().__getstate__(), "state_bits": self.state_bits, "seed": self.seed, "_ticket": {}}

    def __setstate__(self, state):
        super().__setstate__(state)
        if self.state_bits == 8:   # (pickles without layouts: the parameter came with its codes)
            for p, s in self.state.items():
                if isinstance(p, torch.Tensor) and "step" in s:
                    s.setdefault("layout", _layout(p))

    @staticmethod
    def _check_settings(group):
        if isinstance(group["lr"], torch.Tensor):
            raise ValueError("lr must be a number")
        for name in ("lr", "eps", "weight_decay"):
            if not 0 <= group[name] < float("inf"):
                raise ValueError(f"{name} must be a number that is not negative, got {group[name]!r}")
        if len(group["betas"]) != 2 or not all(0 <= b < 1 for b in group["betas"]):
            raise ValueError(f"betas must be two numbers in [0, 1), got {group['betas']!r}")

    def add_param_group(self, group):
        super().add_param_group(group)
        self._check_settings(self.param_groups[-1])
        for p in self.param_groups[-1]["params"]:
            if not p.is_cuda or p.dtype not in DTYPES:
                raise ValueError("AdamW needs CUDA parameters of fp32, bf16 or fp16")
            if not _dense(p):
                raise ValueError("AdamW needs parameters whose elements lie in one piece")

    def _start(self, p):
        s = self.state[p]
        if torch.cuda.is_current_stream_capturing():
            raise RuntimeError("AdamW: a parameter has no state yet; take one step before capturing")
        s["step"] = torch.zeros((), dtype=torch.int64, device=p.device)
        if self.state_bits == 32:
            for name in ("exp_avg", "exp_avg_sq"):
                s[name] = torch.zeros_like(p, dtype=torch.float32, memory_format=torch.preserve_format)
        else:
            n = p.numel()
            for name in _CODES:
                s[name] = torch.zeros(-(-n // BLOCK) if name.endswith("top") else n, dtype=torch.uint8, device=p.device)
            s["layout"] = _layout(p)
        return s

    def _launches(self):
        """Parameters with a gradient, by what one call takes: {(group, device, type): (parameters, gradients, states, numbers)}."""
        found, number, state = {}, 0, self.state
        for i, group in enumerate(self.param_groups):
            key = rows = None
            for p in group["params"]:
                g = p.grad
                if g is not None:
                    if g.is_sparse:
                        raise RuntimeError("AdamW does not take sparse gradients")
                    s = state[p]
                    if "step" not in s:
                        s = self._start(p)
                    if key != (p.device, p.dtype):
                        key = (p.device, p.dtype)
                        rows = found.setdefault((i, *key), ([], [], [], []))
                    rows[0].append(p)
                    rows[1].append(g)
                    rows[2].append(s)
                    rows[3].append(number)
                number += 1
        return found

    @torch.no_grad()
    def step(self, closure=None):
        loss = None
        if closure is not None:
            with torch.enable_grad():
                loss = closure()
        names = ("exp_avg", "root_avg_sq", "exp_avg_top", "root_avg_sq_top") if self.state_bits == 8 else ("exp_avg", "exp_avg_sq")
        for (i, device, _), (params, grads, states, numbers) in self._launches().items():
            group = self.param_groups[i]
            self._check_settings(group)
            ticket = self._ticket.get(device)
            if ticket is None:
                ticket = self._ticket[device] = torch.zeros(1, dtype=torch.int32, device=device)
            m, v, *tops = ([s[name] for s in states] for name in names)
            _dense_torch.adamw_step(params, grads, m, v, *(tops or ([], [])), _layouts(states) if tops else [],
                                    [s["step"] for s in states], numbers, group["lr"], *group["betas"], group["eps"], group["weight_decay"],
                                    self.seed, ticket)
        return loss

    @torch.no_grad()
    def moments(self):
        """The moments of every parameter that has some, in the parameters' order: (exp_avg, exp_avg_sq) themselves with 32
        bits; with 8 the values that their codes stand for, (exp_avg, root of exp_avg_sq), as new bf16 tensors (exact)."""
        params = [p for group in self.param_groups for p in group["params"] if "step" in self.state.get(p, ())]
        if self.state_bits == 32:
            return [(self.state[p]["exp_avg"], self.state[p]["exp_avg_sq"]) for p in params]
        by_device = {}
        for p in params:
            by_device.setdefault(p.device, []).append(p)
        out = {}
        for ps in by_device.values():
            states = [self.state[p] for p in ps]
            out.update(zip(ps, _dense_torch.adamw_moments(ps, *([s[name] for s in states] for name in _CODES), _layouts(states))))
        return [out[p] for p in params]

    def state_dict(self):
        return {**super().state_dict(), "state_bits": self.state_bits, "seed": self.seed}

    def load_state_dict(self, state_dict):
        """Takes a state_dict of this class.  Moments keep their own type (torch would give them the parameter's); those of 32 bits
        are laid out as the parameter is, codes of 8 bits have to lie in the parameter's order of elements (`layout` in the
        state; row-major where it is missing)."""
        if state_dict.get("state_bits", self.state_bits) != self.state_bits:
            raise ValueError(f"the state is in {state_dict['state_bits']} bits, this optimizer's in {self.state_bits}")
        names = ("exp_avg", "exp_avg_sq") if self.state_bits == 32 else _CODES
        params = [p for group in self.param_groups for p in group["params"]]
        places = [k for group in state_dict["param_groups"] for k in group["params"]]
        if len(places) == len(params):   # (otherwise torch says what does not fit)
            for k, p in zip(places, params):
                s = state_dict["state"].get(k)
                if s is None:
                    continue
                for name in names:
                    if name not in s:
                        raise ValueError(f"the state of parameter {k} has no {name}")
                    want = p.numel() if not name.endswith("top") else -(-p.numel() // BLOCK)
                    if s[name].numel() != want:
                        raise ValueError(f"{name} of parameter {k} has {s[name].numel()} elements, {want} are needed")
                if self.state_bits == 8 and _order(s["layout"] if "layout" in s else _layout(torch.empty(p.shape, device="meta"))) != _order(_layout(p)):
                    raise ValueError(f"the codes of parameter {k} go through its elements in another order than the parameter's")
        super().load_state_dict(dict(state={k: {n: v for n, v in s.items() if n != "layout"} for k, s in state_dict["state"].items()},
                                     param_groups=state_dict["param_groups"]))
        self.seed = state_dict.get("seed", self.seed)
        for k, p in zip(places, params):
            s = state_dict["state"].get(k)
            if s is None:
                continue
            mine = self.state[p] = {"step": torch.as_tensor(s["step"]).to(device=p.device, dtype=torch.int64, copy=True).reshape(())}
            for name in names:
                if self.state_bits == 32:   # in the parameter's own order of elements
                    mine[name] = torch.empty_like(p, dtype=torch.float32, memory_format=torch.preserve_format).copy_(s[name].reshape(p.shape))
                else:
                    mine[name] = s[name].reshape(-1).to(device=p.device, dtype=torch.uint8, copy=True)
            if self.state_bits == 8:
                mine["layout"] = _layout(p)
