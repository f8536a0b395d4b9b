"""A NaN or an infinity in one column of a linear layer, among finite ones, on every tile shape."""
import math
import zlib

import pytest
import torch

from grappa_b200 import _native

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
HALF_BF16 = 2.0 ** -8
BF = torch.bfloat16


def cu():
    return _native.cuda()


def gen_for(*key):
    g = torch.Generator(device=DEV)
    g.manual_seed(zlib.crc32(repr(key).encode()))
    return g


def pad(n, m=8):
    return (n + m - 1) // m * m


def nd(n):
    return torch.tensor([n], dtype=torch.int32, device=DEV)


def err_word():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


def operands(g, n, cap, k, m):
    a = torch.full((cap, pad(k)), float("nan"), dtype=BF, device=DEV)[:, :k]
    a[:n] = torch.randn((n, k), generator=g, device=DEV).to(BF)
    w = (torch.randn((m, pad(k)), generator=g, device=DEV) / math.sqrt(k)).to(BF)[:, :k]
    b = 0.5 * torch.randn(m, generator=g, device=DEV)
    return a, w, b


def act_of(z, act):
    if act == 1:
        return z.clamp(min=0)
    if act == 2:
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return z * torch.sigmoid(z) if act == 3 else z


@pytest.mark.parametrize("n,cap,k,m", [(300, 320, 64, 97), (19990, 20000, 96, 161), (57001, 57100, 256, 249)])
@pytest.mark.parametrize("act", [0, 1, 2, 3])
@pytest.mark.parametrize("generic", [False, True])
def test_nan_in_a_column_stays_in_its_column(n, cap, k, m, act, generic):
    g = gen_for("nan", n, k, m, act)
    a, w, b = operands(g, n, cap, k, m)
    outs = []
    where = [0, 33, m - 1]  # an odd neighbour, an even one, and one whose neighbour is a pad column
    for bad in (False, True):
        bb, ww = b.clone(), w.clone()
        if bad:
            bb[where[0]] = float("nan")
            ww[where[1], 0] = float("nan")
            bb[where[2]] = float("nan")
        out = torch.full((cap, pad(m)), -5.0, dtype=BF, device=DEV)
        z = torch.zeros((cap, pad(m)), dtype=BF, device=DEV) if generic else None
        er = err_word()
        cu().linear_fwd(a, ww, nd(n), cap, out, er, bias=bb, act=act, z=z)
        assert int(er) == 0
        outs.append(out)
    isnan = torch.isnan(outs[1][:n].float())
    want = torch.zeros_like(isnan)
    want[:, where] = True
    assert torch.equal(isnan, want)
    x, y = outs[0][:n][~want].double(), outs[1][:n][~want].double()
    if act < 2:
        assert torch.equal(x, y)
    # GELU and SiLU take one reciprocal for a pair: v = z (b r), r = rcp(a b), b the neighbour's, so
    # that another neighbour changes v's roundings: 2^-23 of the approximate reciprocal and 2^-24
    # of a b, of b r and of the product each, in both runs, 5 * 2^-23 in all.  Then each run
    # rounds to bf16, off by half a step, 2^-8, each
    assert bool(((x - y).abs() <= (2 * HALF_BF16 + 5 * 2.0 ** -23 + 2.0 ** -24) * torch.maximum(x.abs(), y.abs())).all())
    assert bool((outs[1][:n, m:] == 0).all())


@pytest.mark.parametrize("act", [2, 3])
def test_infinities_of_one_row(act):
    """+inf and -inf beside finite values and beside each other: +inf stays, -inf goes to zero."""
    inf = float("inf")
    w = torch.eye(8, device=DEV).to(BF)
    b = torch.tensor([inf, 1.0, -inf, -2.0, inf, -inf, 3e38, -3e38], device=DEV)
    a = torch.zeros(4, 8, dtype=BF, device=DEV)
    out = torch.zeros(4, 8, dtype=BF, device=DEV)
    cu().linear_fwd(a, w, None, 4, out, err_word(), bias=b, act=act)
    f = act_of(torch.tensor([1.0, -2.0], dtype=torch.float64), act).tolist()
    got = out[0].double().tolist()
    assert got[0] == inf and got[4] == inf and got[6] == pytest.approx(3e38, rel=HALF_BF16)
    assert got[1] == pytest.approx(f[0], rel=HALF_BF16 + 1e-5) and got[3] == pytest.approx(f[1], rel=HALF_BF16 + 1e-5)
    assert all(abs(got[i]) < 1e-15 for i in (2, 5, 7))
