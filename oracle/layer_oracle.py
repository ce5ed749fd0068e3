"""64-bit restatement of the epilogue GEMM, the expert router and the MoE layer (torch, any
device), each with the bound its rounding allows.

Notation: u16 = 2^-11, half a step of fp16; every kernel sums in fp32 on tensor cores, which may
truncate, so one addition is off by at most 2^-23 of the running magnitude, and a sum of K products
taken 16 at a time by at most ``acc(K)`` of S = sum |a| |w|.
"""
from __future__ import annotations

import math

import torch

U16 = 2.0 ** -11
ACT = ("none", "relu", "silu", "gelu", "gelu_tanh")
# largest slopes: silu 1.0998, gelu 1.1290, gelu_tanh 1.1290
SLOPE = {"none": 1.0, "relu": 1.0, "silu": 1.1, "gelu": 1.13, "gelu_tanh": 1.13}


def acc(K: int) -> float:
    """Relative to S: K / 16 accumulations and the 16 products inside each, plus the 8 partial
    sums and the epilogue's few operations."""
    return (K / 16 + 16 + 16) * 2.0 ** -23


def dequant(W, s, z, group):
    if s is None:
        return W.double()
    if z is None:
        return W.double() * s.double()[..., None]
    ss = s.double().repeat_interleave(group, -2).transpose(-1, -2)
    zz = z.double().repeat_interleave(group, -2).transpose(-1, -2)
    return (W.double() - zz) * ss


def act(y, name):
    if name == "relu":
        return torch.where(y < 0, torch.zeros_like(y), y)
    if name == "silu":
        return y * torch.sigmoid(y)
    if name == "gelu":
        return 0.5 * y * torch.special.erfc(-y * math.sqrt(0.5))
    if name == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3)))
    return y


def epilogue(A, Wd, bias, name, res, weight_rounding=0.0):
    """(y, bound): y = act(A Wd^T + bias) + res; weight_rounding: what the path rounds the
    weights by (U16 where group-wise weights become fp16 operands, else 0)."""
    A = A.double()
    y = A @ Wd.t()
    S = A.abs() @ Wd.abs().t()
    if bias is not None:
        y = y + bias.double()
        S = S + bias.double().abs()
    v = act(y, name)
    out = v if res is None else v + res.double()
    tol = SLOPE[name] * (acc(A.shape[1]) + weight_rounding) * S + 2.0 ** -20 * v.abs()
    return out, tol + U16 * (out.abs() + tol) + 2.0 ** -24


def route(x, wr, k, normalize=True, bias=None):
    """(ids, weights, bound of the weights, smallest gap between the logits that decide in units
    of what the kernel's may be off by)."""
    z = x.double() @ wr.double().t()
    S = x.double().abs() @ wr.double().abs().t()
    if bias is not None:
        z = z + bias.double()
        S = S + bias.double().abs()
    # steps of 32 products added in fp32: H / 256 additions per warp, 8 warps, 32 products
    off = ((x.shape[1] / 256 + 8 + 32) * 2.0 ** -23 * S).amax(1)
    order = torch.argsort(-z, dim=-1, stable=True)
    ids = order[:, :k]
    zs = torch.gather(z, 1, order)
    gap = (zs[:, :-1] - zs[:, 1:])[:, :k]
    top = torch.gather(z, 1, ids)
    e = torch.exp(top - top[:, :1])
    w = e / (e.sum(1, keepdim=True) if normalize else torch.exp(z - top[:, :1]).sum(1, keepdim=True))
    bound = w * (2 * off[:, None] * 1.01 + 2.0 ** -20)
    far = float((gap / (2 * off[:, None])).min()) if gap.numel() else math.inf
    return ids.int(), w, bound, far


def experts(x, ids, w, Wgu, Wd, res=None, block=0, w_off=None):
    """(y, bound) for float64 weights Wgu [E, 2I, H], Wd [E, H, I]; w_off: bound of the weights."""
    E, I2, H = Wgu.shape
    I = I2 // 2
    T, k = ids.shape
    dev = x.device
    y = torch.zeros(T, H, dtype=torch.float64, device=dev)
    tol = torch.zeros_like(y)
    rows = torch.arange(I, device=dev)
    gr = rows if not block else (rows // block) * 2 * block + rows % block
    ur = gr + (block if block else I)
    for t in range(T):
        xt = x[t].double()
        for j in range(k):
            e = int(ids[t, j])
            if not 0 <= e < E:
                continue
            g, u = Wgu[e][gr] @ xt, Wgu[e][ur] @ xt
            Sg, Su = Wgu[e][gr].abs() @ xt.abs(), Wgu[e][ur].abs() @ xt.abs()
            sl = g * torch.sigmoid(g)
            wt = float(w[t, j])
            h = wt * sl * u
            wo = 0.0 if w_off is None else float(w_off[t, j]) / max(abs(wt), 1e-300)
            dh = abs(wt) * acc(H) * (1.1 * Sg * (u.abs() + acc(H) * Su) + Su * sl.abs()) \
                + (2.0 ** -20 + wo) * h.abs() + 2.0 ** -38 * h.abs().max()
            y[t] += Wd[e] @ h
            tol[t] += Wd[e].abs() @ (dh + acc(I * k) * h.abs())
    if res is not None:
        y = y + res.double()
    return y, tol + U16 * (y.abs() + tol) + 2.0 ** -24
