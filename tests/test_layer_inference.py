"""Layer inference apart from training."""
import pytest
import torch
import torch.nn.functional as F
from torch import nn

from grappa_b200.block import Block
from grappa_b200.infer import apply_layer
from grappa_b200.models import SAGE


def block(n=30, seed=0):
    g = torch.Generator().manual_seed(seed)
    indptr = torch.zeros(n + 1, dtype=torch.int64)
    indptr[1:] = torch.cumsum(torch.randint(1, 5, (n,), generator=g), 0)
    return Block(indptr, torch.randint(0, n, (int(indptr[-1]),), generator=g), torch.arange(n), n, n)


@pytest.mark.parametrize("kw", [{}, dict(norm="rms"), dict(norm="rms", residual=True)])
def test_layer_inference_draws_no_dropout(kw):
    torch.manual_seed(0)
    m = SAGE(8, 16, 4, 4, F.relu, 0.5, **kw)
    b, x = block(), torch.randn(30, 8)
    want, h = [], x
    m.eval()
    for l in range(4):
        h = m.run_layer(l, b, h).detach()
        want.append(h)
    m.train()  # a model in the middle of its training
    h = x
    for l in range(4):
        h = apply_layer(m, l, b, h).detach()
        assert torch.equal(h, want[l])


def test_layer_inference_of_a_users_own_sage():
    """A module of the same name that has layers and an activation, and nothing else."""
    class Own(nn.Module):
        name = "sage"

        def __init__(self, of):
            super().__init__()
            self.layers, self.activation = of.layers, of.activation

    m = SAGE(8, 16, 4, 2, F.relu, 0.0)
    b, x = block(), torch.randn(30, 8)
    own = Own(m)
    h = apply_layer(own, 0, b, x)
    torch.testing.assert_close(apply_layer(own, 1, b, h), m([b, b], x))
