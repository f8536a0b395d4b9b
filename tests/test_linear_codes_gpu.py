"""The 8-bit pre-activation of long products: the same bits on every run, and the code of the exact
sum wherever that sum is not within the accumulator's truncation of the middle between two codes."""
import math
import zlib

import pytest
import torch

from grappa_b200 import _native

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
BF = torch.bfloat16


@pytest.mark.parametrize("n,k,m", [(3000, 208, 256), (20000, 512, 256), (57344, 256, 256), (20480, 1024, 1024),
                                   (9000, 2048, 512)])
@pytest.mark.parametrize("act,res", [(2, False), (3, True)])
def test_codes_of_long_products(n, k, m, act, res):
    g = torch.Generator(device=DEV)
    g.manual_seed(zlib.crc32(repr((n, k, m, act)).encode()))
    a = (torch.randn((n, k), generator=g, device=DEV) * torch.exp(0.5 * torch.randn((n, 1), generator=g, device=DEV))).to(BF)
    w = (torch.randn((m, k), generator=g, device=DEV) / math.sqrt(k)).to(BF)
    b = 0.1 * torch.randn(m, generator=g, device=DEV)
    r = torch.randn((n, m), generator=g, device=DEV).to(BF) if res else None
    err = torch.zeros(1, dtype=torch.int32, device=DEV)
    runs = []
    for _ in range(3):
        out = torch.zeros((n, m), dtype=BF, device=DEV)
        q = torch.zeros((n, m), dtype=torch.int8, device=DEV)
        e = torch.zeros((n, m // 32), dtype=torch.uint8, device=DEV)
        _native.cuda().linear_fwd(a, w, None, n, out, err, bias=b, act=act, residual=r, q=q, q_exp=e)
        runs.append((out, q, e))
    assert int(err) == 0
    assert all(torch.equal(x, y) for run in runs[1:] for x, y in zip(run, runs[0]))
    z = a.double() @ w.double().t() + b.double()
    # K / 16 additions by truncation, 2^-23 of the running magnitude each, and the bias in fp32
    tol = (k / 16 + 8) * 2.0 ** -23 * (a.double().abs() @ w.double().abs().t() + b.double().abs())
    z, tol = z.view(n, m // 32, 32), tol.view(n, m // 32, 32)
    top, slack = z.abs().amax(2), tol.amax(2)
    exponent = torch.ceil(torch.log2(top / 127))
    sure = torch.ceil(torch.log2((top + slack) / 127)) == torch.ceil(torch.log2((top - slack) / 127))
    assert torch.equal(exponent[sure], e.double()[sure] - 127)
    assert float(sure.double().mean()) > 0.99  # a group's largest value is seldom at a power's border
    unit = torch.exp2(e.double() - 127).unsqueeze(2)
    x = z / unit
    middle = (x - torch.floor(x) - 0.5).abs() <= tol / unit
    q = runs[0][1].double().view_as(z)
    assert torch.equal(q[~middle & sure.unsqueeze(2)], torch.round(x)[~middle & sure.unsqueeze(2)])
    assert bool(((q - x).abs() <= 0.5 + tol / unit)[sure].all())
