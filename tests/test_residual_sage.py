"""GraphSAGE with RMS norm and residual layers: the CPU model, its options and its CLI."""
import pytest
import torch
import torch.nn.functional as F

from grappa_b200.block import Block
from grappa_b200.infer import apply_layer
from grappa_b200.models import ACTIVATIONS, SAGE, get_model


def blocks(n=40, layers=3, seed=0):
    g = torch.Generator().manual_seed(seed)
    deg = torch.randint(0, 5, (n,), generator=g)
    indptr = torch.zeros(n + 1, dtype=torch.int64)
    indptr[1:] = torch.cumsum(deg, 0)
    ix = torch.randint(0, n, (int(indptr[-1]),), generator=g)
    return [Block(indptr, ix, torch.arange(n), n, n) for _ in range(layers)]


@pytest.mark.parametrize("act", list(ACTIVATIONS))
@pytest.mark.parametrize("norm,residual", [(None, False), ("rms", False), ("rms", True)])
def test_forward_is_the_formula(act, norm, residual):
    torch.manual_seed(0)
    m = get_model("sage", 10, 7, num_hidden=12, num_layers=4, dropout=0.0, activation=act, norm=norm, residual=residual)
    for w in (n.weight for n in getattr(m, "norms", ())):
        w.data.uniform_(0.5, 1.5)
    bs, x = blocks(layers=4), torch.randn(40, 10)
    f = {"relu": torch.relu, "gelu": lambda z: F.gelu(z, approximate="tanh"), "silu": F.silu}[act]
    h = x
    for l, b in enumerate(bs):
        n = h
        if norm and l > 0:
            n = h / torch.sqrt((h * h).mean(1, keepdim=True) + 1e-5) * m.norms[l - 1].weight
        u, v = b.edges()
        mean = torch.zeros_like(n).index_add(0, v, n[u]) / b.in_degrees().clamp(min=1).unsqueeze(1)
        lay = m.layers[l]
        z = n @ lay.fc_self.weight.t() + mean @ lay.fc_neigh.weight.t() + lay.bias
        if l < 3:
            z = f(z)
            if residual and l > 0:
                z = z + h
        h = z
    # fp32 sums of at most 24 terms in another order, four layers
    torch.testing.assert_close(m(bs, x), h, rtol=1e-4, atol=1e-5)
    m.eval()
    y = x
    for l, b in enumerate(bs):
        y = apply_layer(m, l, b, y)
    torch.testing.assert_close(y, m(bs, x))


def test_options_and_state():
    assert sorted(k for k in SAGE(8, 16, 4, 3).state_dict()) == sorted(
        f"layers.{i}.{k}" for i in range(3) for k in ("bias", "fc_neigh.weight", "fc_self.weight"))
    m = SAGE(8, 16, 4, 4, norm="rms", residual=True)
    assert [k for k in m.state_dict() if k.startswith("norms")] == [f"norms.{i}.weight" for i in range(3)]
    assert [m.has_residual(l) for l in range(4)] == [False, True, True, False]
    assert m.layer_buckets(4) is not None  # each layer's norm lies with its weights
    m2 = SAGE(8, 16, 4, 4, norm="rms", residual=True)
    m2.load_state_dict(m.state_dict())
    assert torch.equal(m2.flat, m.flat)
    with pytest.raises(ValueError, match="norm"):
        SAGE(8, 16, 4, 3, residual=True)
    with pytest.raises(ValueError, match="unknown norm"):
        SAGE(8, 16, 4, 3, norm="layer")
    with pytest.raises(ValueError, match="unknown activation"):
        get_model("sage", 8, 4, activation="elu")
    with pytest.raises(ValueError, match="sage"):
        get_model("gcn", 8, 4, norm="rms")


def test_command_line_options():
    from grappa_b200.train.t10n_train import build_parser, model_options

    base = ["--model", "sage", "--tag_id", "t"]
    a = build_parser().parse_args(base)
    assert model_options(a) == dict(activation="relu", norm=None, residual=False) and a.act_bits == 16
    a = build_parser().parse_args(base + ["--norm", "rms", "--residual", "--activation", "silu", "--act_bits", "8",
                                          "--num_gpus", "1"])
    assert model_options(a) == dict(activation="silu", norm="rms", residual=True) and a.act_bits == 8
    a.num_gpus = -1
    with pytest.raises(ValueError, match="act_bits"):
        model_options(a)


def test_gradients_against_differences():
    torch.manual_seed(1)
    m = SAGE(6, 8, 3, 3, ACTIVATIONS["silu"], 0.0, norm="rms", residual=True)
    m.flat = None
    md = m.double()
    bs, x = blocks(20), torch.randn(20, 6, dtype=torch.float64)
    y = torch.randint(0, 3, (20,))
    params = list(md.parameters())
    loss = F.cross_entropy(md(bs, x), y)
    grads = torch.autograd.grad(loss, params)
    for p, g in zip(params, grads):
        v = torch.randn_like(p)
        with torch.no_grad():
            p.add_(1e-5 * v)
            up = float(F.cross_entropy(md(bs, x), y))
            p.sub_(2e-5 * v)
            down = float(F.cross_entropy(md(bs, x), y))
            p.add_(1e-5 * v)
        # second-order error h^2 and rounding 1e-16 / h
        assert abs((up - down) / 2e-5 - float((g * v).sum())) < 1e-7
