"""Refusals of the residual layer's operators: every argument is checked before the device
is touched, so CPU tensors show the same errors."""
import pytest
import torch

from grappa_b200 import _native

BF, F32 = torch.bfloat16, torch.float32


def cu():
    return _native.cuda()


def z(r, c, t=BF):
    return torch.zeros((r, c), dtype=t)


def norm_args(**kw):
    a = dict(x=z(4, 104), dim=100, n_dev=None, cap=4, gamma=torch.zeros(100), eps=1e-5, y=z(4, 104), rstd=torch.zeros(4))
    a.update(kw)
    return a


def bwd_args(**kw):
    a = dict(dy=z(4, 104), x=z(4, 104), rstd=torch.zeros(4), gamma=torch.zeros(100), dim=100, n_dev=None, cap=4,
             dx=z(4, 104), dgamma=torch.zeros(100))
    a.update(kw)
    return a


def lin_args(**kw):
    a = dict(A=z(4, 64), W=z(40, 64), n_dev=None, cap=4, out=z(4, 40), err=torch.zeros(1, dtype=torch.int32))
    a.update(kw)
    return a


def act_args(**kw):
    a = dict(dout=z(4, 40), dim=40, n_dev=None, cap=4, act=2, dz=z(4, 40), z=z(4, 40))
    a.update(kw)
    return a


def dw_args(**kw):
    a = dict(dy=z(4, 40), q=z(4, 64, torch.int8), q_exp=z(4, 2, torch.uint8), n_dev=None, cap=4, gw=z(40, 64, F32),
             err=torch.zeros(1, dtype=torch.int32))
    a.update(kw)
    return a


BUF = z(4, 208)
Q, E = z(4, 128, torch.int8), z(4, 4, torch.uint8)

CASES = [
    # shapes, types, strides
    ("rmsnorm_fwd", norm_args, dict(x=z(4, 100)), "columns"),
    ("rmsnorm_fwd", norm_args, dict(x=z(3, 104)), "rows"),
    ("rmsnorm_fwd", norm_args, dict(x=z(4, 104, torch.float16)), "dtype"),
    ("rmsnorm_fwd", norm_args, dict(x=z(104, 4).t()), "contiguous rows"),
    ("rmsnorm_fwd", norm_args, dict(x=z(4, 108)), "16-byte"),
    ("rmsnorm_fwd", norm_args, dict(x=z(4, 120)[:, 4:112]), "16-byte"),
    ("rmsnorm_fwd", norm_args, dict(dim=0), "dim must be"),
    ("rmsnorm_fwd", norm_args, dict(dim=8193), "dim must be"),
    ("rmsnorm_fwd", norm_args, dict(cap=-1), "cap must be"),
    ("rmsnorm_fwd", norm_args, dict(cap=2 ** 31), "cap must be"),
    ("rmsnorm_fwd", norm_args, dict(gamma=torch.zeros(99)), "gamma"),
    ("rmsnorm_fwd", norm_args, dict(gamma=torch.zeros(100, dtype=BF)), "gamma"),
    ("rmsnorm_fwd", norm_args, dict(rstd=torch.zeros(3)), "rstd"),
    ("rmsnorm_fwd", norm_args, dict(eps=-1.0), "eps"),
    ("rmsnorm_fwd", norm_args, dict(y=z(4, 104, F32)), "dtype"),
    ("rmsnorm_fwd", norm_args, dict(y=z(1, 104).expand(4, 104)), "overlap"),
    ("rmsnorm_fwd", norm_args, dict(s_out=z(4, 104)), "residual"),
    ("rmsnorm_fwd", norm_args, dict(residual=z(4, 104, F32)), "dtype"),
    ("rmsnorm_fwd", norm_args, dict(q=Q), "together"),
    ("rmsnorm_fwd", norm_args, dict(q=z(4, 104, torch.int8), q_exp=E), "columns"),
    ("rmsnorm_fwd", norm_args, dict(q=Q, q_exp=z(4, 3, torch.uint8)), "columns"),
    ("rmsnorm_fwd", norm_args, dict(n_dev=torch.zeros(1, dtype=torch.int64)), "n_dev"),
    # outputs over inputs
    ("rmsnorm_fwd", norm_args, dict(x=BUF[:, :104], y=BUF[:, :104]), "overlaps"),
    ("rmsnorm_fwd", norm_args, dict(x=BUF[:, :104], y=BUF[:, 96:200]), "overlaps"),
    ("rmsnorm_bwd", bwd_args, dict(x=None), "one of them"),
    ("rmsnorm_bwd", bwd_args, dict(q=Q, q_exp=E), "one of them"),
    ("rmsnorm_bwd", bwd_args, dict(n_res_dev=torch.zeros(1, dtype=torch.int32)), "dres"),
    ("rmsnorm_bwd", bwd_args, dict(dres=z(3, 104)), "rows"),
    ("rmsnorm_bwd", bwd_args, dict(dres=z(4, 104, F32)), "dtype"),
    ("rmsnorm_bwd", bwd_args, dict(dgamma=torch.zeros(99)), "dgamma"),
    ("rmsnorm_bwd", bwd_args, dict(dy=BUF[:, :104], dx=BUF[:, :104], clear_dy=True), "overlaps"),
    ("rmsnorm_bwd", bwd_args, dict(x=BUF[:, :104], dx=BUF[:, :104]), "overlaps"),
    ("linear_fwd", lin_args, dict(W=z(40, 72)), "share K"),
    ("linear_fwd", lin_args, dict(out=z(4, 32)), "columns"),
    ("linear_fwd", lin_args, dict(A=z(1, 64).expand(4, 64)), "overlap"),
    ("linear_fwd", lin_args, dict(A=z(4, 64, F32)), "dtype"),
    ("linear_fwd", lin_args, dict(act=4), "act must be"),
    ("linear_fwd", lin_args, dict(bias=torch.zeros(39)), "bias"),
    ("linear_fwd", lin_args, dict(dropout_p=0.5), "counters"),
    ("linear_fwd", lin_args, dict(dropout_p=1.0), "dropout_p"),
    ("linear_fwd", lin_args, dict(residual=z(4, 40, F32)), "dtype"),
    ("linear_fwd", lin_args, dict(A=BUF[:, :64], out=BUF[:, 56:96]), "overlaps"),
    ("linear_fwd", lin_args, dict(err=torch.zeros(1)), "err"),
    ("linear_act_bwd", act_args, dict(z=None), "needs z"),
    ("linear_act_bwd", act_args, dict(q=Q, q_exp=E), "not both"),
    ("linear_act_bwd", act_args, dict(dz=z(4, 40, F32)), "dtype"),
    ("linear_act_bwd", act_args, dict(ld_mask=-1), "ld_mask"),
    ("linear_act_bwd", act_args, dict(dout=BUF[:, :40], dz=BUF[:, :40], clear_dout=True), "overlaps"),
    ("ckpt8_dw", dw_args, dict(gw=z(41, 64, F32)), "columns"),
    ("ckpt8_dw", dw_args, dict(gw=z(40, 65, F32)), "columns"),
    ("ckpt8_dw", dw_args, dict(gw=z(40, 64)), "dtype"),
    ("ckpt8_dw", dw_args, dict(q=z(4, 72, torch.int8)[:, :64]), "16-byte"),
    ("ckpt8_dw", dw_args, dict(cap=5), "rows"),
    # sound arguments, on the CPU
    ("rmsnorm_fwd", norm_args, dict(x=BUF[:, :104], y=BUF[:, 104:]), "CUDA"),
    ("rmsnorm_fwd", norm_args, dict(residual=BUF[:, :104], s_out=BUF[:, :104], q=Q, q_exp=E), "CUDA"),
    ("rmsnorm_bwd", bwd_args, dict(dres=BUF[:, :104], dx=BUF[:, :104]), "CUDA"),
    ("linear_fwd", lin_args, dict(residual=BUF[:, :40], out=BUF[:, :40], bias=torch.zeros(40)), "CUDA"),
    ("linear_act_bwd", act_args, {}, "CUDA"),
    ("ckpt8_dw", dw_args, {}, "CUDA"),
]


@pytest.mark.parametrize("op,base,change,says", CASES, ids=[f"{c[0]}-{i}" for i, c in enumerate(CASES)])
def test_refusals(op, base, change, says):
    with pytest.raises(RuntimeError, match=says):
        getattr(cu(), op)(**base(**change))


def test_ckpt8_refusals():
    x, q, e = z(4, 104), z(4, 128, torch.int8), z(4, 4, torch.uint8)
    for args, says in [((x, 100, None, 5, q, e), "rows"), ((x, 105, None, 4, q, e), "columns"),
                       ((x, 100, None, 4, q.to(torch.uint8), e), "dtype"), ((x, 100, None, 4, q, e.to(torch.int8)), "dtype"),
                       ((x, 100, None, 4, q, e), "CUDA")]:
        with pytest.raises(RuntimeError, match=says):
            cu().ckpt8_store(*args)
    for args, says in [((q, e, 100, None, 4, z(4, 96)), "columns"), ((q, e, 129, None, 4, z(4, 136)), "columns"),
                       ((q, e, 100, None, 4, z(4, 104, torch.int32)), "dtype"), ((q, e, 100, None, 4, z(4, 104)), "CUDA")]:
        with pytest.raises(RuntimeError, match=says):
            cu().ckpt8_load(*args)
