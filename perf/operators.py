"""What the operators of a residual, normalised layer cost, and what they compute.

The operators (rows are graph nodes, columns features; ``n`` live rows at the head of
buffers of ``cap`` rows):

  norm_fwd   s = x (+ r),  y = s / rms(s) * gamma,  rstd = 1 / rms(s), and optionally the
             normalised rows s / rms(s) kept in 8 bits
  norm_bwd   dx = rstd (gamma dy - xh mean(gamma dy xh)) (+ dr),  dgamma = sum_rows dy xh,
             with xh = s rstd from the kept rows s or from their 8-bit form
  linear     out = act(A W^T + b) (+ r), and optionally z = A W^T + b kept in 8 bits
  act_bwd    dz = dout act'(z),  db = sum_rows dz, with z from its 8-bit form
  ckpt       rows to 8 bits and back
  dw         dW = dY^T Xh, Xh the rows that the 8-bit form stands for

8-bit form: a row's columns in groups of 32; a group holds integer codes of -127 to 127
and one power of two, the smallest 2^E with max|x| <= 127 * 2^E (E at least -126);
x stands as round-half-even(x / 2^E) * 2^E, which a bfloat16 holds exactly.  Where a ReLU
reads the 8-bit form its positive values keep a code of at least 1.
"""
import math

import torch

own = False

GROUP = 32
EPS = 1e-5
ACTS = {"none": 0, "relu": 1, "gelu": 2, "silu": 3}


# ------------------------------------------------------------------ the cases
def listed():
    return [
        # the seeds of one small mini-batch: a handful of rows, latency counts; 100 raw
        # feature columns in rows padded to 104
        {"name": "norm_small", "op": "norm_fwd", "n": 1000, "cap": 1024, "dim": 100, "type": "bf16", "res": False,
         "q": False},
        # a hidden layer of the input hop: residual added, 8-bit rows kept for the backward pass
        {"name": "norm_graph", "op": "norm_fwd", "n": 139058, "cap": 139058, "dim": 256, "type": "bf16", "res": True,
         "q": True},
        # full-graph rows in 32 bits, an odd row count and a width that ends inside a group
        {"name": "norm_wide_f32", "op": "norm_fwd", "n": 65537, "cap": 65600, "dim": 1000, "type": "f32", "res": False,
         "q": True},
        # backward of a middle hop: fp32 gradient rows from the aggregation, residual gradient joined
        {"name": "norm_bwd", "op": "norm_bwd", "n": 20853, "cap": 33280, "dim": 256, "type": "f32", "res": True,
         "q": False},
        # backward over a whole partition from the 8-bit rows
        {"name": "norm_bwd_graph_8bit", "op": "norm_bwd", "n": 1000003, "cap": 1000064, "dim": 128, "type": "bf16",
         "res": True, "q": True},
        # the layer before the output layer of a mini-batch
        {"name": "linear_small", "op": "linear", "n": 3250, "cap": 10240, "k": 512, "m": 256, "act": "relu",
         "res": True, "q": False},
        # the input layer's rows: two halves of 104 columns
        {"name": "linear_graph", "op": "linear", "n": 139058, "cap": 139264, "k": 208, "m": 256, "act": "gelu",
         "res": False, "q": True},
        # a wide hidden layer, where the products dominate
        {"name": "linear_wide", "op": "linear", "n": 131072, "cap": 131072, "k": 1024, "m": 1024, "act": "silu",
         "res": True, "q": True},
        # its kind's backward over the input hop
        {"name": "act_bwd_graph", "op": "act_bwd", "n": 139058, "cap": 139264, "dim": 256, "type": "f32",
         "act": "gelu"},
        # the concatenated operand of a layer kept in 8 bits and brought back
        {"name": "ckpt_graph", "op": "ckpt", "n": 139058, "cap": 139264, "dim": 512, "type": "bf16"},
        # weight gradients from 8-bit rows: one mini-batch hop, and a whole partition
        {"name": "dw_small", "op": "dw", "n": 3250, "cap": 10240, "k": 512, "m": 256},
        {"name": "dw_graph", "op": "dw", "n": 500009, "cap": 500032, "k": 512, "m": 256},
    ]


def draw(rng):
    def size(lo, hi):
        return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))

    op = rng.choice(["norm_fwd", "norm_bwd", "linear", "linear", "act_bwd", "ckpt", "dw", "dw"])
    n = size(1, 1000000)
    c = {"op": op}
    if op in ("linear", "dw"):
        k, m = size(16, 2048), size(16, 1024)
        n = max(1, min(n, 131072 * 1024 * 1024 // (k * m), 260000000 // (k + 2 * m)))
        c.update(n=n, cap=n + rng.randrange(0, 65), k=k, m=m)
        if op == "linear":
            c.update(act=rng.choice(["none", "relu", "gelu", "silu"]), res=rng.random() < 0.5, q=rng.random() < 0.5)
        return c
    dim = size(8, 4096)
    n = max(1, min(n, 128000000 // dim))
    c.update(n=n, cap=n + rng.randrange(0, 65), dim=dim, type=rng.choice(["bf16", "f32"]))
    if op in ("norm_fwd", "norm_bwd"):
        c.update(res=rng.random() < 0.5, q=rng.random() < 0.5)
    if op == "act_bwd":
        c.update(act=rng.choice(["relu", "gelu", "silu"]))
    return c


def _pad(n, m):
    return (int(n) + m - 1) // m * m


def _t(name):
    return torch.bfloat16 if name == "bf16" else torch.float32


# ------------------------------------------------------------------ inputs
def _rows(g, n, cap, dim, dtype, scale=1.0, pad=8):
    """n live rows of unequal size at the head of a [cap, padded] buffer, zeros elsewhere."""
    x = torch.zeros((cap, _pad(dim, pad)), dtype=dtype, device="cuda")
    v = torch.randn((n, dim), generator=g, device="cuda")
    v *= scale * torch.exp(0.5 * torch.randn((n, 1), generator=g, device="cuda"))
    x[:n, :dim] = v.to(dtype)
    return x


def _coded(g, n, cap, dim, scale=1.0):
    """Rows in the 8-bit form: codes and exponents (biased by 127) as a forward pass left them."""
    w = _pad(dim, GROUP)
    q = torch.zeros((cap, w), dtype=torch.int8, device="cuda")
    e = torch.ones((cap, w // GROUP), dtype=torch.uint8, device="cuda")
    c, ex = _codes(torch.randn((n, dim), generator=g, device="cuda") * scale)
    q[:n] = c.to(torch.int8)
    e[:n] = (ex + 127).to(torch.uint8)
    return q, e


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(int(seed))
    op, n, cap = case["op"], case["n"], case["cap"]
    s = {"case": case, "n": n, "cap": cap, "n_dev": torch.tensor([n], dtype=torch.int32, device="cuda"),
         "err": torch.zeros(1, dtype=torch.int32, device="cuda")}
    bf, f32 = torch.bfloat16, torch.float32

    def coded_out(w):
        s["q"] = torch.zeros((cap, _pad(w, GROUP)), dtype=torch.int8, device="cuda")
        s["e"] = torch.zeros((cap, _pad(w, GROUP) // GROUP), dtype=torch.uint8, device="cuda")
        s["back"] = torch.zeros((cap, _pad(w, 8)), dtype=bf, device="cuda")

    if op in ("norm_fwd", "norm_bwd"):
        dim = case["dim"]
        s["gamma"] = 1.0 + 0.2 * torch.randn(dim, generator=g, device="cuda")
    if op == "norm_fwd":
        t = _t(case["type"])
        s["x"] = _rows(g, n, cap, dim, t)
        if case["res"]:
            s["res"] = _rows(g, n, cap, dim, t, 2.0)
            s["s"] = torch.zeros_like(s["x"])
        s["y"] = torch.zeros((cap, _pad(dim, 8)), dtype=bf, device="cuda")
        s["rstd"] = torch.zeros(cap, dtype=f32, device="cuda")
        if case["q"]:
            coded_out(dim)
    elif op == "norm_bwd":
        t = _t(case["type"])
        s["dy"] = _rows(g, n, cap, dim, t, 0.01)
        if case["q"]:
            s["q"], s["e"] = _coded(g, n, cap, dim)
            s["rstd"] = torch.exp(0.5 * torch.randn(cap, generator=g, device="cuda"))
        else:
            s["x"] = _rows(g, n, cap, dim, bf, 2.0)
            s["rstd"] = s["x"].float().square().sum(1).div_(dim).add_(EPS).rsqrt_()
        if case["res"]:
            s["dr"] = _rows(g, n, cap, dim, t, 0.01)
        s["dx"] = torch.zeros((cap, _pad(dim, 8)), dtype=t, device="cuda")
        s["dgamma"] = torch.zeros(dim, dtype=f32, device="cuda")
    elif op == "linear":
        k, m = case["k"], case["m"]
        s["a"] = _rows(g, n, cap, k, bf)
        w = torch.zeros((m, _pad(k, 8)), device="cuda")
        w[:, :k] = torch.randn((m, k), generator=g, device="cuda") / math.sqrt(k)
        s["w"] = w.to(bf)
        s["b"] = 0.1 * torch.randn(m, generator=g, device="cuda")
        if case["res"]:
            s["res"] = _rows(g, n, cap, m, bf, 2.0)
        s["out"] = torch.zeros((cap, _pad(m, 8)), dtype=bf, device="cuda")
        if case["q"]:
            coded_out(m)
    elif op == "act_bwd":
        s["dout"] = _rows(g, n, cap, case["dim"], _t(case["type"]), 0.01)
        s["q"], s["e"] = _coded(g, n, cap, case["dim"])
        s["dz"] = torch.zeros((cap, _pad(case["dim"], 8)), dtype=bf, device="cuda")
        s["db"] = torch.zeros(case["dim"], dtype=f32, device="cuda")
    elif op == "ckpt":
        s["x"] = _rows(g, n, cap, case["dim"], _t(case["type"]))
        coded_out(case["dim"])
    else:
        s["dy"] = _rows(g, n, cap, case["m"], bf, 0.01)
        s["q"], s["e"] = _coded(g, n, cap, case["k"])
        s["dw"] = torch.zeros((case["m"], _pad(case["k"], 8)), dtype=f32, device="cuda")
    return s


# ------------------------------------------------------------------ the plain form
def _two_to(ex):
    """2^ex in fp32, exact, for -126 <= ex <= 127."""
    return ((ex.int() + 127) << 23).view(torch.float32)


def _codes(x, keep_sign=False):
    """Codes [n, padded] and exponents [n, groups] of fp32 rows."""
    n, dim = x.shape
    w = _pad(dim, GROUP)
    if w != dim:
        x = torch.cat([x, x.new_zeros((n, w - dim))], 1)
    x = x.view(n, w // GROUP, GROUP)
    m, k = torch.frexp(x.abs().amax(2))
    ex = torch.where(m <= 127.0 / 128.0, k - 7, k - 6).clamp(min=-126)
    c = torch.round(x * _two_to(-ex).unsqueeze(2))
    if keep_sign:
        c = torch.where((x > 0) & (c < 1), torch.ones_like(c), c)
    return c.view(n, w), ex


def _stand(c, ex, dim):
    """The values that codes and exponents stand for, fp32 [n, dim]."""
    n, w = c.shape
    v = c.float().view(n, w // GROUP, GROUP) * _two_to(ex).unsqueeze(2)
    return v.view(n, w)[:, :dim]


def _act(z, act):
    if act == "relu":
        return z.clamp(min=0)
    if act == "gelu":
        return 0.5 * z * (1 + torch.tanh(math.sqrt(2 / math.pi) * (z + 0.044715 * z * z * z)))
    if act == "silu":
        return z / (1 + torch.exp(-z))
    return z


def _act_slope(z, act):
    if act == "relu":
        return (z > 0).float()
    if act == "gelu":
        c = math.sqrt(2 / math.pi)
        t = torch.tanh(c * (z + 0.044715 * z * z * z))
        return 0.5 * (1 + t) + 0.5 * z * (1 - t * t) * c * (1 + 3 * 0.044715 * z * z)
    if act == "silu":
        p = 1 / (1 + torch.exp(-z))
        return p * (1 + z * (1 - p))
    return torch.ones_like(z)


def _plain(s):
    case, n = s["case"], s["n"]
    op, bf = case["op"], torch.bfloat16
    if op == "norm_fwd":
        dim = case["dim"]
        out = {}
        h = s["x"][:n, :dim].float()
        if case["res"]:
            # the sum is rounded once to the rows' type; the norm is that of the rounded rows
            out["s"] = (h + s["res"][:n, :dim].float()).to(s["x"].dtype)
            h = out["s"].float()
        out["rstd"] = 1 / torch.sqrt((h * h).mean(1) + EPS)
        xh = h * out["rstd"].unsqueeze(1)
        out["y"] = (xh * s["gamma"]).to(bf)
        if case["q"]:
            out["xh"] = _stand(*_codes(xh), dim).to(bf)
        return out
    if op == "norm_bwd":
        dim = case["dim"]
        r = s["rstd"][:n].unsqueeze(1)
        xh = _stand(s["q"][:n], s["e"][:n].int() - 127, dim) if case["q"] else s["x"][:n, :dim].float() * r
        dy = s["dy"][:n, :dim].float()
        gy = dy * s["gamma"]
        dx = r * (gy - xh * (gy * xh).mean(1, keepdim=True))
        if case["res"]:
            dx = dx + s["dr"][:n, :dim].float()
        return {"dx": dx.to(s["dx"].dtype), "dgamma": (dy * xh).sum(0)}
    if op == "linear":
        k, m = case["k"], case["m"]
        z = s["a"][:n, :k].float() @ s["w"][:, :k].float().t() + s["b"]
        v = _act(z, case["act"])
        if case["res"]:
            v = v + s["res"][:n, :m].float()
        out = {"out": v.to(bf)}
        if case["q"]:
            out["z"] = _stand(*_codes(z, case["act"] == "relu"), m).to(bf)
        return out
    if op == "act_bwd":
        dim = case["dim"]
        z = _stand(s["q"][:n], s["e"][:n].int() - 127, dim)
        dz = s["dout"][:n, :dim].float() * _act_slope(z, case["act"])
        return {"dz": dz.to(bf), "db": dz.sum(0)}
    if op == "ckpt":
        dim = case["dim"]
        return {"x": _stand(*_codes(s["x"][:n, :dim].float()), dim).to(bf)}
    xh = _stand(s["q"][:n], s["e"][:n].int() - 127, case["k"])
    return {"dw": s["dy"][:n, :case["m"]].float().t() @ xh}


# ------------------------------------------------------------------ the framework's calls
def _own(s):
    from grappa_b200 import _native

    cu = _native.cuda()
    case, n, nd, cap = s["case"], s["n"], s["n_dev"], s["cap"]
    op = case["op"]
    if op == "norm_fwd":
        dim = case["dim"]
        cu.rmsnorm_fwd(s["x"], dim, nd, cap, s["gamma"], EPS, s["y"], s["rstd"], residual=s.get("res"),
                       s_out=s.get("s"), q=s.get("q"), q_exp=s.get("e"))
        out = {"y": s["y"][:n, :dim], "rstd": s["rstd"][:n]}
        if case["res"]:
            out["s"] = s["s"][:n, :dim]
        if case["q"]:
            cu.ckpt8_load(s["q"], s["e"], dim, nd, cap, s["back"])
            out["xh"] = s["back"][:n, :dim]
        return out
    if op == "norm_bwd":
        dim = case["dim"]
        cu.rmsnorm_bwd(s["dy"], s.get("x"), s["rstd"], s["gamma"], dim, nd, cap, s["dx"], s["dgamma"],
                       dres=s.get("dr"), q=s.get("q"), q_exp=s.get("e"), accumulate=False)
        return {"dx": s["dx"][:n, :dim], "dgamma": s["dgamma"]}
    if op == "linear":
        m = case["m"]
        cu.linear_fwd(s["a"], s["w"], nd, cap, s["out"], s["err"], bias=s["b"], act=ACTS[case["act"]],
                      residual=s.get("res"), q=s.get("q"), q_exp=s.get("e"))
        out = {"out": s["out"][:n, :m]}
        if case["q"]:
            cu.ckpt8_load(s["q"], s["e"], m, nd, cap, s["back"])
            out["z"] = s["back"][:n, :m]
        return out
    if op == "act_bwd":
        dim = case["dim"]
        cu.linear_act_bwd(s["dout"], dim, nd, cap, ACTS[case["act"]], s["dz"], s["db"], q=s["q"], q_exp=s["e"],
                          accumulate=False)
        return {"dz": s["dz"][:n, :dim], "db": s["db"]}
    if op == "ckpt":
        dim = case["dim"]
        cu.ckpt8_store(s["x"], dim, nd, cap, s["q"], s["e"])
        cu.ckpt8_load(s["q"], s["e"], dim, nd, cap, s["back"])
        return {"x": s["back"][:n, :dim]}
    cu.ckpt8_dw(s["dy"], s["q"], s["e"], nd, cap, s["dw"], s["err"], accumulate=False)
    return {"dw": s["dw"][:, :case["k"]]}


def run(state):
    return _own(state) if own else _plain(state)


# ------------------------------------------------------------------ the least work
def work(case):
    op, n = case["op"], case["n"]
    if op in ("linear", "dw"):
        k, m = case["k"], case["m"]
        flops = 2.0 * n * k * m
        if op == "dw":
            return {"bytes": n * (2 * m + k + _pad(k, GROUP) // GROUP) + 4 * m * k, "flops": flops}
        b = n * 2 * (k + m) + 2 * m * k + 4 * m
        b += n * 2 * m if case["res"] else 0
        b += n * (m + m // GROUP + 2 * m) if case["q"] else 0  # codes written, and the values they stand for
        return {"bytes": b, "flops": flops + 8.0 * n * m}
    dim = case["dim"]
    w = 2 if case["type"] == "bf16" else 4
    codes = dim + _pad(dim, GROUP) // GROUP
    if op == "norm_fwd":
        b = n * (dim * (w + 2) + 4) + 4 * dim
        b += n * dim * 2 * w if case["res"] else 0
        b += n * (codes + 2 * dim) if case["q"] else 0
        return {"bytes": b, "flops": 5.0 * n * dim}
    if op == "norm_bwd":
        b = n * (dim * 2 * w + 4) + n * (codes if case["q"] else 2 * dim) + 8 * dim
        b += n * dim * w if case["res"] else 0
        return {"bytes": b, "flops": 9.0 * n * dim}
    if op == "act_bwd":
        return {"bytes": n * (dim * (w + 2) + codes) + 4 * dim, "flops": 20.0 * n * dim}
    return {"bytes": n * (dim * w + codes + 2 * dim), "flops": 6.0 * n * dim}


# ------------------------------------------------------------------ 64 bits
def _power(ex):
    """2^ex, exact: the exponent field of a double."""
    return torch.bitwise_left_shift(ex.long() + 1023, 52).view(torch.float64)


def _eight(x, positive_stays=False):
    """Values that the 8-bit form of the rows x (fp64) holds, from the definition: the least
    power of two whose 127-fold reaches the group's largest magnitude."""
    n, dim = x.shape
    out = torch.empty_like(x)
    for lo in range(0, dim, GROUP):
        part = x[:, lo:lo + GROUP]
        top = part.abs().max(1, keepdim=True).values
        ex = torch.ceil(torch.log2(torch.clamp(top, min=1e-300) / 127.0)).clamp(min=-126.0)
        # the logarithm is rounded: its neighbours decide where 127 units meet the top exactly
        ex = torch.where((127.0 * _power(ex - 1) >= top) & (ex > -126), ex - 1, ex)
        unit = _power(torch.where(127.0 * _power(ex) < top, ex + 1, ex))
        code = torch.round(part / unit)
        if positive_stays:
            code[(part > 0) & (code == 0)] = 1.0
        out[:, lo:lo + GROUP] = code * unit
    return out


def _held(q, e, dim):
    unit = _power(e.double() - 127.0)
    return (q.double() * unit.repeat_interleave(GROUP, 1))[:, :dim]


def _phi(z, act):
    """(activation, its derivative) in 64 bits, through the logistic function."""
    if act == "none":
        return z, torch.ones_like(z)
    if act == "relu":
        return torch.maximum(z, torch.zeros_like(z)), torch.sign(torch.maximum(z, torch.zeros_like(z)))
    if act == "silu":
        p = torch.sigmoid(z)
        return z * p, p + z * p * torch.sigmoid(-z)
    # 0.5 (1 + tanh u) = sigmoid(2 u)
    a, b = 2 * math.sqrt(2 / math.pi), 0.044715
    u = a * z + a * b * z ** 3
    p = torch.sigmoid(u)
    return z * p, p + z * p * torch.sigmoid(-u) * (a + 3 * a * b * z ** 2)


def exact(case, seed):
    s = prepare(case, seed)
    op, n = case["op"], s["n"]
    if op in ("linear", "dw"):
        k, m = case["k"], case["m"]
        if op == "dw":
            total = torch.zeros((m, k), dtype=torch.float64, device="cuda")
            for lo in range(0, n, 65536):
                hi = min(n, lo + 65536)
                total += s["dy"][lo:hi, :m].double().t() @ _held(s["q"][lo:hi], s["e"][lo:hi], k)
            return {"dw": total}
        z = torch.addmm(s["b"].double(), s["a"][:n, :k].double(), s["w"][:, :k].double().t())
        v = _phi(z, case["act"])[0]
        out = {"out": v + s["res"][:n, :m].double() if case["res"] else v}
        if case["q"]:
            out["z"] = _eight(z, case["act"] == "relu")
        return out
    dim = case["dim"]
    if op == "norm_fwd":
        out = {}
        h = s["x"][:n, :dim].double()
        if case["res"]:
            h = h + s["res"][:n, :dim].double()
            out["s"] = h
            h = h.to(s["x"].dtype).double()  # the rows that are normalised are the rounded ones
        length = torch.linalg.vector_norm(h, dim=1, keepdim=True)
        rms = torch.hypot(length / math.sqrt(dim), torch.full_like(length, math.sqrt(EPS)))
        out["rstd"] = (1.0 / rms).squeeze(1)
        h = h / rms
        out["y"] = h * s["gamma"].double()
        if case["q"]:
            out["xh"] = _eight(h)
        return out
    if op == "norm_bwd":
        r = s["rstd"][:n].double().unsqueeze(1)
        xh = _held(s["q"][:n], s["e"][:n], dim) if case["q"] else s["x"][:n, :dim].double() * r
        dy, gamma = s["dy"][:n, :dim].double(), s["gamma"].double()
        along = torch.einsum("ij,ij,j->i", dy, xh, gamma) / dim
        dx = r * torch.addcmul(dy * gamma, xh, along.unsqueeze(1), value=-1.0)
        if case["res"]:
            dx += s["dr"][:n, :dim].double()
        return {"dx": dx, "dgamma": torch.einsum("ij,ij->j", dy, xh)}
    if op == "act_bwd":
        dz = s["dout"][:n, :dim].double() * _phi(_held(s["q"][:n], s["e"][:n], dim), case["act"])[1]
        return {"dz": dz, "db": dz.sum(0)}
    return {"x": _eight(s["x"][:n, :dim].double())}
