"""Which activations the GPU engines take: an unknown one is refused, not replaced."""
import copy

import pytest
import torch
import torch.nn.functional as F
from torch import nn

from grappa_b200.engine import make_engine
from grappa_b200.models import GAT, GCN, SAGE, PinSAGE, activation_name
from grappa_b200.ops import ref

UNKNOWN = [F.gelu, F.elu, torch.tanh, F.leaky_relu, F.relu6, nn.PReLU(), nn.GELU()]


@pytest.mark.parametrize("act", UNKNOWN, ids=lambda a: getattr(a, "__name__", type(a).__name__))
@pytest.mark.parametrize("bits,norm", [(16, None), (16, "rms"), (8, None)])
def test_engine_refuses_an_unknown_activation(act, bits, norm):
    # refused before the device is touched, whatever else the model has
    m = SAGE(8, 16, 4, 3, copy.deepcopy(act), norm=norm)
    with pytest.raises(ValueError, match="activation"):
        make_engine(m, 100, [3, 3, 3], 10, "cuda:0", act_bits=bits)


@pytest.mark.parametrize("model", [lambda: GCN(8, 16, 4, 2, F.elu), lambda: GAT(8, 8, 4, 2, 2, F.elu),
                                   lambda: PinSAGE(8, 16, 4, 2, F.silu), lambda: GCN(8, 16, 4, 2, ref.gelu)])
def test_models_with_relu_alone_refuse_the_others(model):
    with pytest.raises(ValueError, match="activation"):
        make_engine(model(), 100, [3, 3], 10, "cuda:0")


def test_names_of_activation_functions():
    for want, fns in {"relu": [F.relu, torch.relu, nn.ReLU(), nn.ReLU(inplace=True), lambda x: x.clamp(min=0)],
                      "gelu": [ref.gelu, nn.GELU(approximate="tanh"), lambda x: F.gelu(x, approximate="tanh")],
                      "silu": [F.silu, nn.SiLU(), lambda x: x * torch.sigmoid(x)]}.items():
        assert [activation_name(f) for f in fns] == [want] * len(fns)
    # a learned slope may start as a ReLU's; it does not stay one
    assert [activation_name(f) for f in UNKNOWN + [nn.PReLU(init=0.0), lambda x: 1 / 0]] == [None] * (len(UNKNOWN) + 2)


def test_a_single_layer_applies_no_activation():
    from grappa_b200.models import model_activation

    assert model_activation(SAGE(8, 16, 4, 1, F.elu)) == "relu"
    assert model_activation(SAGE(8, 16, 4, 2, F.elu)) is None
    assert model_activation(PinSAGE(8, 16, 4, 2, F.elu)) is None


@pytest.mark.gpu
@pytest.mark.parametrize("act", [F.gelu, F.elu])
def test_layer_inference_refuses_an_unknown_activation(act):
    from grappa_b200.block import Block
    from grappa_b200.infer_gpu import infer_layer

    dev = torch.device("cuda", 0)
    n = 20
    b = Block(torch.arange(n + 1), torch.arange(n), torch.arange(n), n, n).to(dev)
    for make in (SAGE, GCN):
        m = make(8, 16, 4, 2, act)
        with pytest.raises(ValueError, match="activation"):
            infer_layer(m, 0, b, torch.randn(n, 8, device=dev))
        assert infer_layer(m, 1, b, torch.randn(n, 16, device=dev)).shape == (n, 4)


@pytest.mark.gpu
@pytest.mark.parametrize("name,fns", [("relu", [torch.relu, nn.ReLU()]), ("silu", [F.silu, nn.SiLU()]),
                                      ("gelu", [ref.gelu, nn.GELU(approximate="tanh")])])
def test_layer_inference_knows_a_function_by_another_name(name, fns):
    from grappa_b200.block import Block
    from grappa_b200.infer_gpu import infer_layer
    from grappa_b200.models import ACTIVATIONS

    dev = torch.device("cuda", 0)
    n = 20
    b = Block(torch.arange(n + 1), torch.arange(n), torch.arange(n), n, n).to(dev)
    x, outs = torch.randn(n, 8, device=dev), []
    for fn in [ACTIVATIONS[name]] + fns:
        torch.manual_seed(0)
        outs.append(infer_layer(SAGE(8, 16, 4, 2, fn), 0, b, x))
    assert all(torch.equal(o, outs[0]) for o in outs)
