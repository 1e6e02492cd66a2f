"""The dense operators where the harness calls them: --fused-mlp and --optimizer adamw, whole training steps of the DLRM and DCN
models beside the same models on stock PyTorch layers and optimizers.

The two sides' losses differ by rounding (fp32 sums in another order; a ReLU or a sketch decision that falls the other way) for as
long as the steps are few: each loss is a mean over the batch of values of order 1, whose relative error after s steps is below
s * 2^-10 here."""
import copy

import pytest

pytestmark = pytest.mark.gpu


def _args(extra, model="dlrm", shape="kaggle", batch=256):
    from cafe_b200 import dlrm_harness as H
    return H.make_parser().parse_args(["--sketch-flag", "--data-set", shape, "--model", model, "--compress-rate", "0.001" if shape != "avazu" else "0.1",
                                       "--hash-rate", "0.3", "--mini-batch-size", str(batch), *extra])


def _losses(args, steps, optimizer=None):
    import torch
    from cafe_b200 import dlrm_harness as H
    net = H.build_model(args, torch.device("cuda", 0))
    opt = (optimizer or H.build_optimizer)(args, net)
    out = []
    for s in range(steps):
        dense, lS_o, ids, y = H.synthetic_batch(args.data_set, args.mini_batch_size, 2024, s, "cuda")
        loss, _ = H.train_step(net, opt, dense, lS_o, ids, y)
        out.append(loss.detach())
    return [float(v) for v in out], net, opt


@pytest.mark.parametrize("model,shape,extra", [("dlrm", "kaggle", []), ("dlrm", "terabyte", ["--fused-interaction"]), ("dcn", "avazu", [])])
def test_fused_mlp_trains_like_the_stock_layers(model, shape, extra):
    from cafe_b200 import FusedMLP
    steps = 8
    a, net, _ = _losses(_args(["--fused-mlp", *extra], model, shape), steps)
    b, plain, _ = _losses(_args(extra, model, shape), steps)
    assert isinstance(net.top if model == "dlrm" else net.deep, FusedMLP)
    assert list(net.state_dict()) == list(plain.state_dict())
    for s, (x, y) in enumerate(zip(a, b)):
        assert abs(x - y) <= (s + 1) * 2 ** -10, (s, a, b)


class _StockTwo:
    """TableSGDDenseAdamW on torch.optim.AdamW."""

    def __init__(self, args, net):
        import torch
        from cafe_b200 import dlrm_harness as H
        mine = H.dense_and_plain_parameters(net)
        of_tables = {id(p) for p in net.emb.parameters()}
        self.tables = torch.optim.SGD([dict(params=[p for p in mine if id(p) in of_tables])], lr=args.learning_rate)
        self.dense = torch.optim.AdamW([p for p in mine if id(p) not in of_tables], lr=args.dense_learning_rate)
        self.param_groups = self.tables.param_groups + self.dense.param_groups

    def zero_grad(self):
        self.tables.zero_grad()
        self.dense.zero_grad()

    def step(self):
        self.tables.step()
        self.dense.step()


@pytest.mark.parametrize("model,shape", [("dlrm", "kaggle"), ("dcn", "avazu")])
def test_adamw_beside_table_sgd(model, shape):
    steps = 8
    a, net, opt = _losses(_args(["--fused-mlp", "--optimizer", "adamw"], model, shape), steps)
    b, plain, _ = _losses(_args([], model, shape), steps, _StockTwo)
    for s, (x, y) in enumerate(zip(a, b)):
        assert abs(x - y) <= (s + 1) * 2 ** -8, (s, a, b)   # (AdamW divides by the gradient's size: rounding of small gradients counts fully)
    assert opt.param_groups[0]["lr"] == 0.1 and all(g["lr"] == 1e-3 for g in opt.param_groups[1:])
    c, _, opt8 = _losses(_args(["--fused-mlp", "--optimizer", "adamw", "--adamw-state-bits", "8"], model, shape), steps)
    assert all(v == v for v in c)
    kept = copy.deepcopy(opt8.state_dict())
    opt8.load_state_dict(kept)
    assert all(int(s["step"]) == steps for s in opt8.dense.state.values())


def test_the_command_line_runs():
    from cafe_b200 import dlrm_harness as H
    args = _args(["--fused-mlp", "--fused-interaction", "--optimizer", "adamw", "--adamw-state-bits", "8", "--nbatches", "12", "--warmup-batches", "2"])
    res = H.run(args)
    assert res["steps"] == 12 and all(v == v for v in res["losses"])
