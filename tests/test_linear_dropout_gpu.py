"""Dropout of the linear layer on every tile shape, with the activation backward that draws its
mask again and both kept forms of the pre-activation.

Tolerances count roundings: a tensor-core sum adds 16 products at a time by truncation (2^-23 of
the running magnitude each), 2^-8 is half a bf16 step, the activations' exponential and
reciprocal are within 4e-6 of |z|."""
import math
import zlib

import pytest
import torch

from grappa_b200 import _native
from grappa_b200.ops import ref

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
HALF_BF16, U = 2.0 ** -8, 2.0 ** -24
BF = torch.bfloat16

# rows, capacity, K, N: 64-column tiles, 128-column tiles, 256-column tiles of CTA pairs
SHAPES = [(777, 800, 96, 47), (1, 1, 40, 1), (19990, 20000, 96, 161), (19969, 20100, 200, 128),
          (57001, 57100, 256, 250), (73001, 73216, 200, 200)]


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
    r = torch.full((cap, pad(m)), float("nan"), dtype=BF, device=DEV)
    r[:n, :m] = torch.randn((n, m), generator=g, device=DEV).to(BF)
    return a, w, b, r


def act_of(z, act):
    if act == 1:
        return z.clamp(min=0)
    if act == 2:
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    return z * torch.sigmoid(z) if act == 3 else z


@pytest.mark.parametrize("n,cap,k,m", SHAPES)
@pytest.mark.parametrize("act,res,kept", [(0, True, None), (1, False, "q8"), (2, True, "bf16"), (3, True, "q8"),
                                          (3, False, "bf16")])
def test_dropout_on_every_tile(n, cap, k, m, act, res, kept):
    g = gen_for("drop", n, k, m, act, kept)
    a, w, b, r = operands(g, n, cap, k, m)
    p, key = 0.4, (7, 3, 11, 5)
    ctr = torch.tensor([key[0], key[1], key[2], 0, 0, 0], dtype=torch.int64, device=DEV)
    out = torch.full((cap, pad(m) + 64), -5.0, dtype=BF, device=DEV)[:, :pad(m)]
    z = q = e = None
    if kept == "bf16":
        z = torch.full((cap, pad(m)), -5.0, dtype=BF, device=DEV)
    elif kept:
        q = torch.full((cap, pad(m, 32)), 77, dtype=torch.int8, device=DEV)
        e = torch.full((cap, pad(m, 32) // 32), 99, dtype=torch.uint8, device=DEV)
    er = err_word()
    cu().linear_fwd(a, w, nd(n), cap, out, er, bias=b, act=act, residual=r if res else None, z=z, q=q, q_exp=e,
                    dropout_p=p, counters=ctr, salt=key[3])
    assert int(er) == 0
    # the mask that the CPU model draws, its scale read off it (p is a multiple of 1 / 256 there)
    mask = ref.dropout(torch.ones(n, m), p, True, key=key, ld=out.stride(0)).to(DEV) != 0
    dz = torch.full((cap, pad(m)), -5.0, dtype=BF, device=DEV)
    cu().linear_act_bwd(torch.ones(cap, pad(m), device=DEV), m, nd(n), cap, 0, dz, None, dropout_p=p, counters=ctr,
                        salt=key[3], ld_mask=out.stride(0))
    assert torch.equal(dz[:n, :m] != 0, mask)
    scale = 256.0 / (256 - round(p * 256))
    A, W = a[:n].double(), w.double()
    zz = A @ W.t() + b.double()
    ztol = (k / 16 + 8) * 2.0 ** -23 * (A.abs() @ W.abs().t() + b.double().abs())
    want = torch.where(mask, act_of(zz, act) * scale, 0.0)
    tol = torch.where(mask, scale * (1.13 * ztol + 4e-6 * zz.abs()) + 4 * U * want.abs(), 0.0)
    if res:
        want = want + r[:n, :m].double()
        tol = tol + 4 * U * r[:n, :m].double().abs()
    tol = tol + HALF_BF16 * want.abs()
    bad = ~((out[:n, :m].double() - want).abs() <= tol)
    assert not bool(bad.any()), int(bad.sum())
    assert bool((out[:n, m:] == 0).all()) and bool((out[n:] == -5).all())
    # the kept pre-activation knows nothing of the mask, and the backward pass from it uses the same one
    if z is not None:
        assert bool(((z[:n, :m].double() - zz).abs() <= ztol + HALF_BF16 * (zz.abs() + ztol)).all())
        assert bool((z[n:] == -5).all())
    if q is not None:
        top = torch.nn.functional.pad(zz.abs() + ztol, (0, pad(m, 32) - m)).view(n, -1, 32).amax(2)
        back = torch.zeros((cap, pad(m)), dtype=BF, device=DEV)
        cu().ckpt8_load(q, e, m, nd(n), cap, back)
        half = (top / 127).repeat_interleave(32, 1)[:, :m] * (2 if act == 1 else 1)
        assert bool(((back[:n, :m].double() - zz).abs() <= half + 2 * ztol).all())
        assert bool((q[n:] == 77).all()) and bool((e[n:] == 99).all())


def test_dropout_scale_of_the_kernels():
    """The kernels keep a value with probability 1 - round(256 p) / 256 and scale by its inverse."""
    n, p = 64, 0.4
    eye = torch.eye(8, device=DEV).to(BF)
    a = torch.ones(n, 8, dtype=BF, device=DEV)
    out = torch.zeros(n, 8, dtype=BF, device=DEV)
    ctr = torch.tensor([7, 3, 11, 0, 0, 0], dtype=torch.int64, device=DEV)
    cu().linear_fwd(a, eye, None, n, out, err_word(), dropout_p=p, counters=ctr)
    want = torch.tensor(256.0 / (256 - round(p * 256))).to(BF)
    assert set(out.unique().tolist()) == {0.0, float(want)}
