"""RMS norm, linear with its epilogue and 8-bit rows (rmsnorm.cu, linear.cu, ckpt8.cu,
ckpt8_dw.cu) against plain 64-bit implementations.

Tolerances count roundings.  HALF_BF16 = 2^-8 is half a bf16 step relative to the value, U =
2^-24 half an fp32 step.  A row statistic is a sum of at most 32 terms a lane, five shuffles
and eight partial sums, each rounded: under 48 U of the sum of magnitudes; column sums take
at most a few rows a lane, 64 teams, 19 + 32 parts: under 256 U.  A tensor-core sum adds 16
products at a time by truncation (2^-23 of the running magnitude each).  The fast exponential
and division of the activations are within 8e-6 of the slope and 4e-6 |z| of the value
(2^-22 + |x| 2^-23 for exp(x), damped by p (1 - p))."""
import math

import pytest
import torch

from grappa_b200 import _native

pytestmark = pytest.mark.gpu
DEV = torch.device("cuda", 0)
HALF_BF16, U = 2.0 ** -8, 2.0 ** -24
BF, F32 = torch.bfloat16, torch.float32


def cu():
    return _native.cuda()


def pad(n, m=8):
    return (n + m - 1) // m * m


def nd(n):
    return torch.tensor([n], dtype=torch.int32, device=DEV)


def err_word():
    return torch.zeros(1, dtype=torch.int32, device=DEV)


def buf(cap, cols, dtype, fill, wide=0):
    """A [cap, cols] window of a buffer that is ``wide`` columns wider, all of it ``fill``."""
    b = torch.full((cap, cols + wide), fill, dtype=dtype, device=DEV)
    return b[:, wide // 2 // 32 * 32: wide // 2 // 32 * 32 + cols]


def rows(gen, n, cap, dim, dtype, scale=1.0, wide=0, junk=float("nan")):
    """n live rows; dead rows and pad columns hold ``junk``."""
    b = buf(cap, pad(dim), dtype, junk, wide)
    v = torch.randn((n, dim), generator=gen, device=DEV) * torch.exp(torch.randn((n, 1), generator=gen, device=DEV))
    b[:n, :dim] = (v * scale).to(dtype)
    return b


def gen_for(*key):
    g = torch.Generator(device=DEV)
    g.manual_seed(abs(hash(key)) % (1 << 31))
    return g


def quantise(x):
    """Codes [n, pad32] and exponents of fp32/fp64 rows, from the definition."""
    n, dim = x.shape
    w = pad(dim, 32)
    x = torch.cat([x.double(), torch.zeros((n, w - dim), dtype=torch.float64, device=x.device)], 1).view(n, w // 32, 32)
    top = x.abs().amax(2)
    e = torch.full(top.shape, -126, dtype=torch.int64, device=x.device)
    m, k = torch.frexp(top)
    want = torch.where(m * 128 <= 127, k.long() - 7, k.long() - 6)
    e = torch.where(top > 0, torch.maximum(e, want), e)
    unit = power(e).unsqueeze(2)
    assert bool((top <= 127 * unit[..., 0]).all())
    return torch.round(x / unit).view(n, w), e


def power(e):
    return ((e + 1023) << 52).view(torch.float64)


def stand(q, e):
    n, w = q.shape
    return (q.double().view(n, w // 32, 32) * power(e.long()).unsqueeze(2)).view(n, w)


def held(q, qe, n, dim):
    return stand(q[:n, :pad(dim, 32)], qe[:n, :pad(dim, 32) // 32].long() - 127)[:, :dim]


def coded(gen, n, cap, dim, scale=1.0, wide=0):
    q = buf(cap, pad(dim, 32), torch.int8, 77, wide)
    e = torch.full((cap, pad(dim, 32) // 32 + (3 if wide else 0)), 200, dtype=torch.uint8, device=DEV)
    c, ex = quantise((torch.randn((n, dim), generator=gen, device=DEV) * scale).float())
    q[:n] = c.to(torch.int8)
    e[:n, :ex.shape[1]] = (ex + 127).to(torch.uint8)
    return q, e


def code_buffers(cap, dim, wide=0):
    return (buf(cap, pad(dim, 32), torch.int8, 77, wide),
            torch.full((cap, pad(dim, 32) // 32 + (5 if wide else 0)), 99, dtype=torch.uint8, device=DEV))


def within(got, want, tol):
    got, want = got.double(), want.double()
    assert got.shape == want.shape
    bad = ~((got - want).abs() <= tol)
    assert not bool(bad.any()), (int(bad.sum()), float((got - want).abs()[bad].max()), want[bad][:4], got[bad][:4])


def untouched(t, n, fill):
    assert bool((t[n:] == fill).all())


def act_of(z, act):
    if act == 1:
        return z.clamp(min=0)
    if act == 2:
        return z * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (z + 0.044715 * z ** 3))
    if act == 3:
        return z * torch.sigmoid(z)
    return z


def slope_of(z, act):
    z = z.detach().clone().requires_grad_(True)
    if act == 1:
        return (z > 0).double().detach()
    act_of(z, act).sum().backward()
    return z.grad


# ------------------------------------------------------------------ 8-bit rows
SHAPES = [(1, 1, 1), (1, 3, 8), (5, 5, 31), (33, 64, 32), (64, 70, 33), (100, 100, 100), (1000, 1024, 208),
          (257, 300, 1000), (3, 9, 4097)]


@pytest.mark.parametrize("dtype", [BF, F32])
@pytest.mark.parametrize("n,cap,dim", SHAPES + [(0, 7, 40)])
@pytest.mark.parametrize("wide", [0, 64])
def test_ckpt8_store_and_load(n, cap, dim, dtype, wide):
    g = gen_for("ckpt", n, dim)
    x = rows(g, n, cap, dim, dtype, 3.0, wide)
    if n > 2:
        x[0, :dim] = 0
        x[1, :dim] = 1e-42 if dtype == F32 else 2.0 ** -130  # below the least unit
        x[2, :dim] *= 1e30
    q, e = code_buffers(cap, dim, wide)
    cu().ckpt8_store(x, dim, nd(n), cap, q, e)
    c, ex = quantise(x[:n, :dim].float())
    groups = ex.shape[1]
    assert torch.equal(q[:n].long(), c.long())
    assert torch.equal(e[:n, :groups].long(), ex + 127)
    untouched(q, n, 77)
    untouched(e, n, 99)
    assert bool((e[:, groups:] == 99).all())
    for out_t in (BF, F32):
        out = buf(cap, pad(dim), out_t, -5.0, wide)
        cu().ckpt8_load(q, e, dim, nd(n), cap, out)
        # 2^E times an integer of 7 bits: exact in both types
        assert torch.equal(out[:n, :dim].double(), stand(c, ex)[:, :dim])
        assert bool((out[:n, dim:] == 0).all())
        untouched(out, n, -5.0)


def test_ckpt8_group_that_is_not_finite():
    x = torch.randn(4, 96, device=DEV)
    x[0, 5] = float("nan")
    x[1, 40] = float("inf")
    x[2, 95] = -float("inf")
    q, e = code_buffers(4, 96)
    cu().ckpt8_store(x, 96, None, 4, q, e)
    out = torch.zeros(4, 96, device=DEV)
    cu().ckpt8_load(q, e, 96, None, 4, out)
    nan = torch.zeros(4, 96, dtype=torch.bool, device=DEV)
    nan[0, :32] = nan[1, 32:64] = nan[2, 64:] = True
    assert torch.equal(torch.isnan(out), nan)
    c, ex = quantise(x.masked_fill(nan, 0))
    assert torch.equal(out[~nan].double(), stand(c, ex)[~nan])
    # a cleared buffer stands for zeros
    cu().ckpt8_load(torch.zeros_like(q), torch.zeros_like(e), 96, None, 4, out)
    assert bool((out == 0).all())


# ------------------------------------------------------------------ RMS norm
NORM = [(1, 1, 1), (3, 5, 8), (2, 2, 31), (65, 100, 33), (100, 100, 64), (1000, 1024, 100), (129, 129, 128),
        (500, 600, 256), (77, 90, 257), (300, 300, 512), (65, 65, 1000), (17, 20, 1025), (9, 9, 2048), (12, 13, 2500),
        (5, 6, 4097), (4, 4, 8192), (0, 3, 16), (5000, 5003, 96)]


@pytest.mark.parametrize("n,cap,dim", NORM)
@pytest.mark.parametrize("dtype,res,q8,wide", [(BF, False, False, 0), (BF, True, True, 0), (F32, True, True, 64),
                                               (F32, False, False, 64), (BF, False, True, 64)])
def test_rmsnorm_fwd(n, cap, dim, dtype, res, q8, wide):
    g = gen_for("norm", n, dim, res)
    x = rows(g, n, cap, dim, dtype, 2.0, wide)
    r = rows(g, n, cap, dim, dtype, 1.0, wide) if res else None
    gamma = torch.randn(dim, generator=g, device=DEV)
    y = buf(cap, pad(dim), BF, -5.0, wide)
    s = buf(cap, pad(dim), dtype, -5.0, wide) if res else None
    rstd = torch.full((cap,), -5.0, device=DEV)
    q, e = code_buffers(cap, dim, wide) if q8 else (None, None)
    eps = 1e-5
    cu().rmsnorm_fwd(x, dim, nd(n), cap, gamma, eps, y, rstd, residual=r, s_out=s, q=q, q_exp=e)
    h = x[:n, :dim].double()
    if res:
        want = h + r[:n, :dim].double()
        within(s[:n, :dim], want, want.abs() * (HALF_BF16 if dtype == BF else U))
        assert bool((s[:n, dim:] == 0).all())
        untouched(s, n, -5.0)
        h = s[:n, :dim].double()  # the norm is that of the rounded rows
    rs = 1 / torch.sqrt(h.square().mean(1) + eps)
    within(rstd[:n], rs, 32 * U * rs)  # half of 48 U, and the root, the quotient and the mean
    xh = h * rs.unsqueeze(1)
    want = xh * gamma.double()
    within(y[:n, :dim], want, want.abs() * (HALF_BF16 + 40 * U))
    assert bool((y[:n, dim:] == 0).all())
    untouched(y, n, -5.0)
    untouched(rstd, n, -5.0)
    if q8:
        top = torch.nn.functional.pad(xh.abs(), (0, pad(dim, 32) - dim)).view(n, pad(dim, 32) // 32, 32).amax(2)
        half = (top / 127).repeat_interleave(32, 1)[:, :dim]
        within(held(q, e, n, dim), xh, half * (1 + 64 * U) + 64 * U * xh.abs())
        assert bool((q[:n, dim:] == 0).all())
        untouched(q, n, 77)
        untouched(e, n, 99)


@pytest.mark.parametrize("n,cap,dim", NORM)
@pytest.mark.parametrize("dy_t,x_t,dx_t,dr_t,wide", [(F32, BF, F32, None, 0), (BF, BF, BF, BF, 64),
                                                     (F32, F32, F32, F32, 0), (BF, "q8", BF, BF, 0),
                                                     (F32, "q8", F32, None, 64)])
def test_rmsnorm_bwd(n, cap, dim, dy_t, x_t, dx_t, dr_t, wide):
    g = gen_for("normb", n, dim)
    dy = rows(g, n, cap, dim, dy_t, 0.1, wide)
    gamma = torch.randn(dim, generator=g, device=DEV)
    rstd = torch.exp(torch.randn(cap, generator=g, device=DEV))
    x = q = e = None
    if x_t == "q8":
        q, e = coded(g, n, cap, dim, wide=wide)
        xh = held(q, e, n, dim)
    else:
        x = rows(g, n, cap, dim, x_t, 1.0, wide)
        xh = x[:n, :dim].double() * rstd[:n].double().unsqueeze(1)
    n_res = n * 2 // 3
    dr = rows(g, n_res, cap, dim, dr_t, 0.1, wide) if dr_t else None
    dx = buf(cap, pad(dim), dx_t, -5.0, wide)
    dgamma = torch.full((dim,), 3.0, device=DEV)
    cu().rmsnorm_bwd(dy, x, rstd, gamma, dim, nd(n), cap, dx, dgamma, dres=dr, n_res_dev=nd(n_res) if dr_t else None,
                     q=q, q_exp=e)
    d, gm, rs = dy[:n, :dim].double(), gamma.double(), rstd[:n].double().unsqueeze(1)
    gy = d * gm
    want = rs * (gy - xh * (gy * xh).mean(1, keepdim=True))
    size = rs * (gy.abs() + xh.abs() * (gy * xh).abs().mean(1, keepdim=True))
    if dr_t:
        want[:n_res] += dr[:n_res, :dim].double()
        size[:n_res] += dr[:n_res, :dim].double().abs()
    within(dx[:n, :dim], want, 64 * U * size + (HALF_BF16 * want.abs() if dx_t == BF else 0))
    assert bool((dx[:n, dim:] == 0).all())
    untouched(dx, n, -5.0)
    p = d * xh
    within(dgamma, 3.0 + p.sum(0), 256 * U * (3.0 + p.abs().sum(0)))
    # without accumulation, and the same bits again
    a, b = torch.full((dim,), 9.0, device=DEV), torch.full((dim,), 7.0, device=DEV)
    for out in (a, b):
        cu().rmsnorm_bwd(dy, x, rstd, gamma, dim, nd(n), cap, dx, out, dres=dr,
                         n_res_dev=nd(n_res) if dr_t else None, q=q, q_exp=e, accumulate=False)
    assert torch.equal(a, b)
    within(a, p.sum(0), 256 * U * p.abs().sum(0))


def test_rmsnorm_in_place_and_clearing():
    g = gen_for("inplace")
    n, dim = 300, 200
    x, r = rows(g, n, n, dim, BF), rows(g, n, n, dim, BF)
    gamma = torch.randn(dim, generator=g, device=DEV)
    y, y2 = torch.zeros(n, dim, dtype=BF, device=DEV), torch.zeros(n, dim, dtype=BF, device=DEV)
    rstd = torch.zeros(n, device=DEV)
    s = torch.zeros(n, dim, dtype=BF, device=DEV)
    cu().rmsnorm_fwd(x, dim, None, n, gamma, 1e-6, y, rstd, residual=r, s_out=s)
    r2 = r.clone()
    cu().rmsnorm_fwd(x, dim, None, n, gamma, 1e-6, y2, rstd, residual=r2, s_out=r2)
    assert torch.equal(r2, s) and torch.equal(y, y2)
    # dx over dres, dy cleared
    dy = rows(g, n, n, dim, F32)
    dr = rows(g, n, n, dim, F32)
    dx, dg = torch.zeros_like(dr), torch.zeros(dim, device=DEV)
    cu().rmsnorm_bwd(dy, s, rstd, gamma, dim, None, n, dx, dg, dres=dr)
    dr2, dg2 = dr.clone(), torch.zeros(dim, device=DEV)
    cu().rmsnorm_bwd(dy, s, rstd, gamma, dim, None, n, dr2, dg2, dres=dr2, clear_dy=True)
    assert torch.equal(dr2, dx) and torch.equal(dg, dg2) and bool((dy == 0).all())


def test_rmsnorm_zero_rows_and_huge_rows():
    dim = 64
    x = torch.zeros(3, dim, device=DEV)
    x[1] = 3e18  # the squares' sum stays below the fp32 range
    x[2, 7] = 1e-20
    y, rstd = torch.zeros(3, dim, dtype=BF, device=DEV), torch.zeros(3, device=DEV)
    cu().rmsnorm_fwd(x, dim, None, 3, torch.ones(dim, device=DEV), 1e-5, y, rstd)
    h = x.double()
    rs = 1 / torch.sqrt(h.square().mean(1) + 1e-5)
    within(rstd, rs, 32 * U * rs)
    within(y, h * rs.unsqueeze(1), (h * rs.unsqueeze(1)).abs() * (HALF_BF16 + 40 * U))


# ------------------------------------------------------------------ linear
LINEAR = [(1, 1, 8, 1), (3, 5, 16, 8), (31, 40, 24, 47), (127, 130, 64, 64), (129, 129, 100, 65), (200, 256, 208, 256),
          (1000, 3000, 512, 256), (1000, 20000, 72, 200), (20000, 20000, 40, 300), (257, 300, 1032, 129), (0, 10, 16, 16),
          (19000, 19000, 136, 136), (2000, 2001, 256, 1000),
          # enough products for the 256-column tiles of CTA pairs
          (75001, 75100, 200, 136), (8000, 8100, 1032, 520), (300, 20000, 1024, 256), (4097, 4200, 2056, 300)]


@pytest.mark.parametrize("n,cap,k,m", LINEAR)
@pytest.mark.parametrize("act,res,q8,z16,bias,wide", [(0, False, False, False, False, 0), (1, True, True, False, True, 0),
                                                      (2, False, True, True, True, 64), (3, True, False, True, True, 64),
                                                      (3, True, True, False, False, 0)])
def test_linear_fwd(n, cap, k, m, act, res, q8, z16, bias, wide):
    g = gen_for("lin", n, k, m, act)
    a = rows(g, n, cap, k, BF, 1.0, wide)
    a[:n, k:] = 0  # the row's pad columns are part of K
    w = torch.zeros((m, pad(k)), dtype=BF, device=DEV)
    w[:, :k] = (torch.randn((m, k), generator=g, device=DEV) / math.sqrt(k)).to(BF)
    b = torch.randn(m, generator=g, device=DEV) if bias else None
    r = rows(g, n, cap, m, BF, 1.0, wide) if res else None
    out = buf(cap, pad(m), BF, -5.0, wide)
    zb = buf(cap, pad(m), BF, -5.0, wide) if z16 else None
    q, e = code_buffers(cap, m, wide) if q8 else (None, None)
    er = err_word()
    cu().linear_fwd(a, w, nd(n), cap, out, er, bias=b, act=act, residual=r, z=zb, q=q, q_exp=e)
    assert int(er) == 0
    A, W = a[:n, :k].double(), w[:, :k].double()
    z = A @ W.t() + (b.double() if bias else 0)
    ztol = (k / 16 + 8) * 2.0 ** -23 * (A.abs() @ W.abs().t() + (b.abs().double() if bias else 0))
    want = act_of(z, act) + (r[:n, :m].double() if res else 0)
    within(out[:n, :m], want, 1.13 * ztol + 4e-6 * z.abs() + 4 * U * want.abs() + HALF_BF16 * want.abs()
           + (4 * U * r[:n, :m].double().abs() if res else 0))
    assert bool((out[:n, m:] == 0).all())
    untouched(out, n, -5.0)
    if z16:
        within(zb[:n, :m], z, ztol + HALF_BF16 * z.abs() + HALF_BF16 * ztol)
        untouched(zb, n, -5.0)
    if q8:
        top = torch.nn.functional.pad(z.abs(), (0, pad(m, 32) - m)).view(n, pad(m, 32) // 32, 32).amax(2)
        half = (top / 127).repeat_interleave(32, 1)[:, :m]
        zt = torch.nn.functional.pad(ztol, (0, pad(m, 32) - m)).view(n, pad(m, 32) // 32, 32).amax(2).repeat_interleave(32, 1)[:, :m]
        zq = held(q, e, n, m)
        # with ReLU a positive value below half a unit takes code 1: up to one unit off
        within(zq, z, half * (2 if act == 1 else 1) + 2 * zt)
        if act == 1:
            sure = z.abs() > 2 * ztol
            assert torch.equal((zq > 0)[sure], (z > 0)[sure])
        assert bool((q[:n, m:] == 0).all())
        untouched(q, n, 77)
        untouched(e, n, 99)


def test_linear_residual_in_place_and_gemm_agreement():
    g = gen_for("lin2")
    n, k, m = 1500, 96, 160
    a, w = rows(g, n, n, k, BF), (torch.randn((m, k), generator=g, device=DEV) / 10).to(BF)
    b = torch.randn(m, generator=g, device=DEV)
    r = rows(g, n, n, m, BF)
    out = torch.zeros(n, m, dtype=BF, device=DEV)
    cu().linear_fwd(a, w, None, n, out, err_word(), bias=b, act=1, residual=r)
    r2 = r.clone()
    cu().linear_fwd(a, w, None, n, r2, err_word(), bias=b, act=1, residual=r2)
    assert torch.equal(out, r2)
    # with dropout: the mask and the values of the framework's GEMM epilogue
    ctr = torch.tensor([11, 2, 5, 0, 0, 0], dtype=torch.int64, device=DEV)
    ref, got = torch.zeros(n, m, dtype=BF, device=DEV), torch.zeros(n, m, dtype=BF, device=DEV)
    er = err_word()
    cu().gemm(a, False, w, False, n, None, m, k, None, 1, ref, 0, b, 1, 0.3, ctr, 4, None, 0, None, None, None, None,
              None, None, er, 64, None, 1.0, 0)
    cu().linear_fwd(a, w, None, n, got, er, bias=b, act=1, dropout_p=0.3, counters=ctr, salt=4)
    assert torch.equal(ref, got) and int(er) == 0


def test_linear_nan_in_a_row_stays_in_its_row():
    g = gen_for("lin3")
    n, k, m = 300, 64, 96
    a, w = rows(g, n, n, k, BF), torch.randn((m, k), generator=g, device=DEV).to(BF)
    a[7, 3] = float("nan")
    out = torch.zeros(n, m, dtype=BF, device=DEV)
    q, e = code_buffers(n, m)
    cu().linear_fwd(a, w, None, n, out, err_word(), act=1, q=q, q_exp=e)
    assert bool(torch.isnan(out[7]).all()) and int(torch.isnan(out).sum()) == m
    assert bool((e[7] == 255).all()) and bool((e[:7] != 255).all()) and bool((e[8:] != 255).all())


# ------------------------------------------------------------------ activation backward
@pytest.mark.parametrize("n,cap,dim", [(1, 1, 1), (3, 70, 8), (64, 64, 33), (100, 130, 100), (1000, 1024, 256),
                                       (700, 701, 300), (65, 200, 1000), (0, 5, 24), (9000, 9001, 64)])
@pytest.mark.parametrize("act,g_t,kept,wide", [(0, F32, None, 0), (1, BF, "q8", 64), (2, F32, "q8", 0),
                                               (3, BF, "bf16", 64), (2, BF, "bf16", 0), (3, F32, "q8", 64)])
def test_linear_act_bwd(n, cap, dim, act, g_t, kept, wide):
    g = gen_for("act", n, dim, act)
    dout = rows(g, n, cap, dim, g_t, 0.1, wide)
    z = q = e = None
    if kept == "q8":
        q, e = coded(g, n, cap, dim, 2.0, wide)
        zv = held(q, e, n, dim)
    elif kept:
        z = rows(g, n, cap, dim, BF, 1.0, wide)
        zv = z[:n, :dim].double()
    else:
        zv = torch.zeros((n, dim), dtype=torch.float64, device=DEV)
    dz = buf(cap, pad(dim), BF, -5.0, wide)
    db = torch.full((dim,), 2.0, device=DEV)
    cu().linear_act_bwd(dout, dim, nd(n), cap, act, dz, db, z=z, q=q, q_exp=e)
    d = dout[:n, :dim].double()
    want = d * slope_of(zv, act)
    slack = 8e-6 * d.abs() if act >= 2 else torch.zeros_like(d)
    within(dz[:n, :dim], want, HALF_BF16 * want.abs() + 2 * slack)
    assert bool((dz[:n, dim:] == 0).all())
    end = min(cap, pad(n, 64))
    assert bool((dz[n:end] == 0).all())
    untouched(dz, end, -5.0)
    within(db, 2.0 + want.sum(0), 256 * U * (2.0 + want.abs().sum(0)) + slack.sum(0))
    db2 = torch.full((dim,), 8.0, device=DEV)
    d2 = dout.clone()
    cu().linear_act_bwd(d2, dim, nd(n), cap, act, dz, db2, z=z, q=q, q_exp=e, clear_dout=True, accumulate=False)
    within(db2, want.sum(0), 256 * U * want.abs().sum(0) + slack.sum(0))
    assert bool((d2[:n, :dim] == 0).all())


@pytest.mark.parametrize("act", [2, 3])
def test_activation_far_out(act):
    z = torch.tensor([[0.0, -0.0, 1e-30, -1e-30, 30.0, -30.0, 1e4, -1e4, 3e38, -3e38, 5.0, -5.0, -12.0, 12.0, 88.0, -88.0]],
                     device=DEV).to(BF)
    dim = z.shape[1]
    dout = torch.ones(1, dim, device=DEV)
    dz = torch.zeros(1, dim, dtype=BF, device=DEV)
    cu().linear_act_bwd(dout, dim, None, 1, act, dz, None, z=z)
    zd = z.double().clamp(-1e5, 1e5)  # the slope is 0 or 1 long before
    within(dz, slope_of(zd, act), HALF_BF16 * slope_of(zd, act).abs() + 16e-6)
    # forward through an identity weight
    w = torch.eye(dim, device=DEV).to(BF)
    zz = z.clone()
    zz[0, 8:10] = torch.tensor([1e18, -1e18], device=DEV).to(BF)
    out = torch.zeros(1, dim, dtype=BF, device=DEV)
    cu().linear_fwd(zz, w, None, 1, out, err_word(), act=act)
    want = act_of(zz.double().clamp(-1e5, 1e5), act) * torch.where(zz.double().abs() > 1e5, zz.double().abs() / 1e5, 1.0)
    within(out, want, HALF_BF16 * want.abs() + 4e-6 * torch.minimum(zz.double().abs(), want.abs() + 1))


def test_linear_act_bwd_draws_the_forward_mask():
    g = gen_for("drop")
    n, k, m = 500, 64, 104
    a, w = rows(g, n, n, k, BF), torch.randn((m, k), generator=g, device=DEV).to(BF)
    ctr = torch.tensor([3, 1, 9, 0, 0, 0], dtype=torch.int64, device=DEV)
    wide = torch.zeros(n, 200, dtype=BF, device=DEV)
    out = wide[:, :m]
    cu().linear_fwd(a, w, None, n, out, err_word(), dropout_p=0.5, counters=ctr, salt=2)
    dz = torch.zeros(n, m, dtype=BF, device=DEV)
    cu().linear_act_bwd(torch.ones(n, m, device=DEV), m, None, n, 0, dz, None, dropout_p=0.5, counters=ctr, salt=2,
                        ld_mask=out.stride(0))
    z = torch.zeros(n, m, dtype=BF, device=DEV)
    cu().linear_fwd(a, w, None, n, z, err_word())
    sure = z != 0
    assert torch.equal((out != 0)[sure], (dz != 0)[sure])
    assert set(dz.unique().tolist()) == {0.0, 2.0}


# ------------------------------------------------------------------ weight gradient
@pytest.mark.parametrize("n,cap,k,m", [(1, 1, 1, 1), (5, 9, 8, 8), (63, 64, 100, 47), (64, 64, 32, 128), (65, 200, 130, 129),
                                       (1000, 3000, 208, 256), (3250, 10240, 512, 256), (4097, 4100, 264, 40),
                                       (40000, 40000, 96, 200), (150001, 150016, 136, 64), (0, 64, 40, 40),
                                       (2048, 2048, 1000, 300),
                                       # enough rows for the 256 x 256 tiles of CTA pairs
                                       (40003, 40100, 300, 300), (152064, 152064, 512, 256), (160001, 170000, 136, 200),
                                       (40960, 41000, 520, 264),
                                       # few live rows of many in a cluster; several chains a share
                                       (100, 2048, 512, 256), (1999, 2000, 300, 65), (90000, 90010, 520, 100),
                                       (200001, 200064, 1000, 64)])
@pytest.mark.parametrize("wide", [0, 64])
def test_ckpt8_dw(n, cap, k, m, wide):
    g = gen_for("dw", n, k, m)
    dy = rows(g, n, cap, m, BF, 0.1, wide)
    q, e = coded(g, n, cap, k, 1.0, wide)
    gw = torch.full((m, k + 3), 4.0, device=DEV)[:, :k]
    er = err_word()
    cu().ckpt8_dw(dy, q, e, nd(n), cap, gw, er)
    D, X = dy[:n, :m].double(), held(q, e, n, k)
    want, size = D.t() @ X, D.abs().t() @ X.abs()
    # 16-row steps by truncation over at most 2048 rows, then fp32 sums of the chains and shares
    tol = (min(n, 2048) / 16 + 8) * 2.0 ** -23 * size + 256 * U * size
    within(gw, 4.0 + want, tol + 4 * U * (4.0 + want.abs()))
    assert int(er) == 0
    a, b = torch.full((m, k), 9.0, device=DEV), torch.full((m, k), 7.0, device=DEV)
    cu().ckpt8_dw(dy, q, e, nd(n), cap, a, er, accumulate=False)
    cu().ckpt8_dw(dy, q, e, nd(n), cap, b, er, accumulate=False)
    assert torch.equal(a, b)
    within(a, want, tol)


def test_ckpt8_dw_long_sums_of_one_sign():
    # every product positive: a truncating sum would drift by 1e-9 of itself a row
    n, k, m = 300000, 64, 64
    g = gen_for("dwpos")
    dy = torch.rand((n, m), generator=g, device=DEV).to(BF)
    q, e = code_buffers(n, k)
    cu().ckpt8_store(torch.rand((n, k), generator=g, device=DEV), k, None, n, q, e)
    gw = torch.zeros((m, k), device=DEV)
    cu().ckpt8_dw(dy, q, e, None, n, gw, err_word(), accumulate=False)
    want = dy.double().t() @ held(q, e, n, k)
    # 128 truncations of a growing sum, half of 2^-23 of half of it on average, and fp32 sums
    within(gw, want, (128 / 4 + 64) * 2.0 ** -23 * want)


def test_offsets_past_32_bits():
    """Rows whose element offset passes 2^31 (a long buffer with a wide row stride)."""
    stride, cap = 65536, 33000  # 2.16e9 bf16 elements
    if torch.cuda.get_device_properties(0).total_memory < 40 << 30:
        pytest.skip("needs 20 GB")
    g = gen_for("far")
    n, dim, lo = cap, 64, 32900
    wide = torch.zeros((cap, stride), dtype=BF, device=DEV)
    x = wide[:, 1024:1024 + dim]
    x[lo:] = torch.randn((cap - lo, dim), generator=g, device=DEV).to(BF)
    y, rstd = torch.zeros(cap, dim, dtype=BF, device=DEV), torch.zeros(cap, device=DEV)
    gamma = torch.ones(dim, device=DEV)
    cu().rmsnorm_fwd(x, dim, None, n, gamma, 1e-5, y, rstd)
    h = x[lo:].double()
    want = h / torch.sqrt(h.square().mean(1, keepdim=True) + 1e-5)
    within(y[lo:], want, want.abs() * (HALF_BF16 + 40 * U))
    w = torch.eye(dim, device=DEV).to(BF)
    out = wide[:, 4096:4096 + dim]
    cu().linear_fwd(x, w, None, n, out, err_word(), residual=x)
    within(out[lo:], 2 * h, HALF_BF16 * 2 * h.abs())
    q, e = code_buffers(cap, dim)
    cu().ckpt8_store(x, dim, None, n, q, e)
    gw = torch.zeros((dim, dim), device=DEV)
    cu().ckpt8_dw(x, q, e, None, n, gw, err_word(), accumulate=False)
    D, X = h, held(q[lo:], e[lo:], cap - lo, dim)
    within(gw, D.t() @ X, 64 * 2.0 ** -23 * (D.abs().t() @ X.abs()))


# ------------------------------------------------------------------ a layer of them, streams and graphs
class _Layer:
    """One residual layer s' = s + act(rmsnorm(s) W^T + b) and its backward, from the operators:
    the normalised rows, the pre-activation and the operand of W are kept in 8 bits or bf16."""

    def __init__(self, g, n, dim, act, bits):
        self.n, self.dim, self.act, self.bits = n, dim, act, bits
        self.gamma = 1 + 0.2 * torch.randn(dim, generator=g, device=DEV)
        self.W = (torch.randn((dim, dim), generator=g, device=DEV) / math.sqrt(dim)).to(BF)
        self.b = 0.1 * torch.randn(dim, generator=g, device=DEV)
        self.s = torch.randn((n, dim), generator=g, device=DEV).to(BF)
        self.dout = torch.randn((n, dim), generator=g, device=DEV) * 0.1
        self.err = err_word()
        z = dict(dtype=BF, device=DEV)
        self.y, self.out, self.dz, self.dX = (torch.zeros((n, dim), **z) for _ in range(4))
        self.zb = torch.zeros((n, dim), **z)
        self.rstd = torch.zeros(n, device=DEV)
        self.xq, self.zq, self.yq = (code_buffers(n, dim) for _ in range(3))
        self.ds = torch.zeros((n, dim), device=DEV)
        self.dgamma, self.db = torch.zeros(dim, device=DEV), torch.zeros(dim, device=DEV)
        self.dW = torch.zeros((dim, dim), device=DEV)

    def run(self):
        c, n, d, eight = cu(), self.n, self.dim, self.bits == 8
        kq = dict(q=self.xq[0], q_exp=self.xq[1]) if eight else {}
        kz = dict(q=self.zq[0], q_exp=self.zq[1]) if eight else dict(z=self.zb)
        c.rmsnorm_fwd(self.s, d, None, n, self.gamma, 1e-5, self.y, self.rstd, **kq)
        c.linear_fwd(self.y, self.W, None, n, self.out, self.err, bias=self.b, act=self.act, residual=self.s, **kz)
        c.linear_act_bwd(self.dout, d, None, n, self.act, self.dz, self.db, accumulate=False, **kz)
        if eight:
            c.ckpt8_store(self.y, d, None, n, *self.yq)
            c.ckpt8_dw(self.dz, *self.yq, None, n, self.dW, self.err, accumulate=False)
        else:  # every kept tensor in bf16: the framework's split-K GEMM
            c.zero_(self.dW)
            c.gemm(self.dz, True, self.y, True, d, None, d, n, None, 1, self.dW, 2, None, 0, 0.0, None, 0, None, 0,
                   None, None, None, None, None, None, self.err, 128, None, 1.0, 0)
        c.gemm(self.dz, False, self.W, True, n, None, d, d, None, 1, self.dX, 0, None, 0, 0.0, None, 0, None, 0, None,
               None, None, None, None, None, self.err, 64, None, 1.0, 0)
        c.rmsnorm_bwd(self.dX, None if eight else self.s, self.rstd, self.gamma, d, None, n, self.ds, self.dgamma,
                      dres=self.dout, accumulate=False, **kq)
        return self.out, self.ds, self.dW, self.db, self.dgamma

    def truth(self):
        s = self.s.double().requires_grad_(True)
        p = [t.double().requires_grad_(True) for t in (self.W, self.b, self.gamma)]
        y = s / torch.sqrt(s.square().mean(1, keepdim=True) + 1e-5) * p[2]
        out = s + act_of(y @ p[0].t() + p[1], self.act)
        out.backward(self.dout.double())
        return out.detach(), s.grad, p[0].grad, p[1].grad, p[2].grad


@pytest.mark.parametrize("act", [1, 2, 3])
@pytest.mark.parametrize("bits", [8, 16])
def test_residual_layer_gradients(act, bits):
    layer = _Layer(gen_for("layer", act), 700, 128, act, bits)
    got, want = layer.run(), layer.truth()
    assert int(layer.err) == 0
    # 2-norm: y, z, dz, dX are rounded to bf16 (2^-8 / sqrt(3) each, rms) and in 8 bits a code is
    # off by amax / 127 / sqrt(3) rms, with amax up to 3.5 of a group's rms: 0.016 for each of the
    # three kept tensors; a ReLU's mask flips only where z is within that of zero
    lim = 0.006 if bits == 16 else 0.03
    for k, (x, y) in enumerate(zip(got, want)):
        rel = float((x.double() - y).norm() / y.norm())
        flips = 0.08 if act == 1 and k in (1, 2, 3, 4) else 0.0
        assert rel <= lim + flips, (k, rel)
    # the loss's difference quotient along a direction of s, in 64 bits, against the operators' ds
    g = gen_for("dir", act)
    v = torch.randn(layer.s.shape, generator=g, device=DEV).double()

    def loss(s):
        y = s / torch.sqrt(s.square().mean(1, keepdim=True) + 1e-5) * layer.gamma.double()
        return float(((s + act_of(y @ layer.W.double().t() + layer.b.double(), act)) * layer.dout.double()).sum())

    h = 1e-5
    quot = (loss(layer.s.double() + h * v) - loss(layer.s.double() - h * v)) / (2 * h)
    # sum of n * dim products, each off by at most lim of its rms
    assert abs(quot - float((got[1].double() * v).sum())) <= 4 * (lim + 0.08 * (act == 1)) * float(got[1].norm())


def test_operators_on_a_side_stream_and_in_two_graphs():
    layers = [_Layer(gen_for("g", i), 300 + 50 * i, 96, 2, 8) for i in range(2)]
    want = [[t.clone() for t in layer.run()] for layer in layers]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in layers]
    for layer, st in zip(layers, streams):
        with torch.cuda.stream(st):
            for _ in range(3):
                layer.run()
    torch.cuda.synchronize()
    for layer, w in zip(layers, want):
        assert all(torch.equal(a, b) for a, b in zip(layer.run(), w))
    graphs = []
    for layer, st in zip(layers, streams):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.stream(st), torch.cuda.graph(gr, stream=st):
            layer.run()
        graphs.append(gr)
    torch.cuda.synchronize()
    for layer in layers:
        for t in (layer.out, layer.ds, layer.dW, layer.db, layer.dgamma):
            t.fill_(-1)
    torch.cuda.synchronize()
    for _ in range(3):  # both at once
        for gr, st in zip(graphs, streams):
            with torch.cuda.stream(st):
                gr.replay()
    torch.cuda.synchronize()
    for layer, w in zip(layers, want):
        assert all(torch.equal(a, b) for a, b in zip((layer.out, layer.ds, layer.dW, layer.db, layer.dgamma), w))
        assert int(layer.err) == 0


def test_live_count_changes_between_replays():
    layer = _Layer(gen_for("live"), 400, 64, 3, 8)
    n = nd(0)
    gr = torch.cuda.CUDAGraph()
    c = cu()
    c.ckpt8_store(layer.s, 64, None, 400, *layer.yq)

    def body():
        c.rmsnorm_fwd(layer.s, 64, n, 400, layer.gamma, 1e-5, layer.y, layer.rstd)
        c.ckpt8_dw(layer.s, *layer.yq, n, 400, layer.dW, layer.err, accumulate=False)

    body()
    torch.cuda.synchronize()
    with torch.cuda.graph(gr):
        body()
    xh = held(*layer.yq, 400, 64)
    for live in (0, 1, 63, 64, 65, 399, 400, 1000):
        n.fill_(live)
        layer.y.fill_(-5)
        gr.replay()
        k = min(live, 400)
        D = layer.s[:k].double()
        within(layer.dW, D.t() @ xh[:k], 40 * 2.0 ** -23 * (D.abs().t() @ xh[:k].abs()))
        untouched(layer.y, k, -5.0)
        assert k == 0 or bool((layer.y[:k] != -5).any())
