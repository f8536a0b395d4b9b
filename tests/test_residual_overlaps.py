"""Vectors that an operator writes, or reads beside its outputs, share no memory with its other
arguments: refused before the device is touched, so CPU tensors show it."""
import pytest
import torch

from grappa_b200 import _native

BF, F32 = torch.bfloat16, torch.float32


def store():
    """fp32 words of which the arguments below are windows."""
    return torch.zeros(4096, dtype=F32)


def rows(t, at, n, cols, dtype=F32):
    return t[at:at + n * cols * (4 if dtype is F32 else 2) // 4].view(dtype).view(n, cols)


def fwd(**kw):
    a = dict(x=torch.zeros(4, 64), dim=64, n_dev=None, cap=4, gamma=torch.zeros(64), eps=1e-5,
             y=torch.zeros(4, 64, dtype=BF), rstd=torch.zeros(4))
    a.update(kw)
    return a


def bwd(**kw):
    a = dict(dy=torch.zeros(4, 64), x=torch.zeros(4, 64), rstd=torch.zeros(4), gamma=torch.zeros(64), dim=64, n_dev=None,
             cap=4, dx=torch.zeros(4, 64), dgamma=torch.zeros(64))
    a.update(kw)
    return a


def lin(**kw):
    a = dict(A=torch.zeros(4, 64, dtype=BF), W=torch.zeros(32, 64, dtype=BF), n_dev=None, cap=4,
             out=torch.zeros(4, 32, dtype=BF), err=torch.zeros(1, dtype=torch.int32))
    a.update(kw)
    return a


def act(**kw):
    a = dict(dout=torch.zeros(4, 64), dim=64, n_dev=None, cap=4, act=0, dz=torch.zeros(4, 64, dtype=BF))
    a.update(kw)
    return a


S = store()
CASES = [
    ("rmsnorm_fwd", fwd, dict(x=rows(S, 0, 4, 64), rstd=S[100:104])),
    ("rmsnorm_fwd", fwd, dict(gamma=S[0:64], rstd=S[60:64])),
    ("rmsnorm_fwd", fwd, dict(y=rows(S, 0, 4, 64, BF), rstd=S[124:128])),
    ("rmsnorm_fwd", fwd, dict(y=rows(S, 0, 4, 64, BF), gamma=S[100:164])),
    ("rmsnorm_fwd", fwd, dict(residual=torch.zeros(4, 64), s_out=rows(S, 0, 4, 64), gamma=S[255:319])),
    ("rmsnorm_fwd", fwd, dict(residual=rows(S, 0, 4, 64), rstd=S[255:259])),
    ("rmsnorm_bwd", bwd, dict(dx=rows(S, 0, 4, 64), dgamma=S[192:256])),
    ("rmsnorm_bwd", bwd, dict(dx=rows(S, 0, 4, 64), gamma=S[192:256])),
    ("rmsnorm_bwd", bwd, dict(dx=rows(S, 0, 4, 64), rstd=S[252:256])),
    ("rmsnorm_bwd", bwd, dict(dy=rows(S, 0, 4, 64), dgamma=S[0:64])),
    ("rmsnorm_bwd", bwd, dict(rstd=S[0:4], dgamma=S[3:67])),
    ("linear_fwd", lin, dict(out=rows(S, 0, 4, 32, BF), bias=S[60:92])),
    ("linear_act_bwd", act, dict(dz=rows(S, 0, 4, 64, BF), dbias=S[64:128])),
    ("linear_act_bwd", act, dict(dout=rows(S, 0, 4, 64), dbias=S[200:264])),
]


@pytest.mark.parametrize("op,base,change", CASES, ids=[f"{c[0]}-{i}" for i, c in enumerate(CASES)])
def test_overlapping_vectors_are_refused(op, base, change):
    with pytest.raises(RuntimeError, match="overlaps"):
        getattr(_native.cuda(), op)(**base(**change))


@pytest.mark.parametrize("op,base,change", [
    ("rmsnorm_fwd", fwd, dict(x=rows(S, 0, 4, 64), rstd=S[256:260], gamma=S[260:324])),
    ("rmsnorm_bwd", bwd, dict(dx=rows(S, 0, 4, 64), dgamma=S[256:320], gamma=S[320:384], rstd=S[384:388])),
    ("linear_fwd", lin, dict(out=rows(S, 0, 4, 32, BF), bias=S[64:96])),
    ("linear_act_bwd", act, dict(dz=rows(S, 0, 4, 64, BF), dbias=S[128:192])),
])
def test_neighbours_are_taken(op, base, change):
    with pytest.raises(RuntimeError, match="CUDA"):  # sound arguments, on the CPU
        getattr(_native.cuda(), op)(**base(**change))
