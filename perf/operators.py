"""What is measured of three operators: a matrix product with its epilogue, a mixture-of-experts
router, and a whole mixture-of-experts layer for a few tokens.

    epilogue   y = act(A W^T + bias) + residual, W fp16, int8 (a scale per output channel) or
               uint8 (scale and zero point per group along K)
    route      the top-k experts of each token and their softmax weights
    moe        y = residual + sum_j w_j down_j(silu(gate_j(x)) * up_j(x)) over a token's experts,
               the routing included

Sizes are the layer shapes of ``cuda_tempiler_b200/workloads.py`` (hidden 3840 with FFN 15360,
hidden 5120 with FFN 17408) and, for the experts, an eighth of those FFN widths (1920, 2176).
"""
from __future__ import annotations

import math

import torch

own = False

GROUP = 128


def listed():
    return [
        # a projection of a small draft model on four tokens: launch latency is most of it
        dict(name="epi_fp16_small", op="epilogue", kind="fp16", M=4, N=1024, K=1024, act="gelu",
             bias=True, res=False, group=0),
        # one decoded token: the attention output projection added to the residual stream
        dict(name="epi_fp16_o_proj_m1", op="epilogue", kind="fp16", M=1, N=3840, K=4096,
             act="none", bias=False, res=True, group=0),
        # sixteen sequences decoded together: W8A16 output projection with bias and residual
        dict(name="epi_int8_o_proj_m16", op="epilogue", kind="int8", M=16, N=5120, K=8192,
             act="none", bias=True, res=True, group=0),
        # a ragged short prompt through an up projection with its activation
        dict(name="epi_fp16_up_m100", op="epilogue", kind="fp16", M=100, N=15360, K=3840,
             act="gelu_tanh", bias=True, res=False, group=0),
        # a prompt chunk of odd length through the group-wise quantised down projection
        dict(name="epi_uint8_down_m333", op="epilogue", kind="uint8", M=333, N=5120, K=17408,
             act="none", bias=False, res=True, group=GROUP),
        # prefill: the down projection of a layer, bias and residual in the epilogue
        dict(name="epi_fp16_down_m4096", op="epilogue", kind="fp16", M=4096, N=3840, K=15360,
             act="none", bias=True, res=True, group=0),
        # routing of one decoded token
        dict(name="route_t1", op="route", T=1, E=64, H=3840, k=4),
        # routing of a prompt chunk
        dict(name="route_t509", op="route", T=509, E=128, H=5120, k=8),
        # one decoded token through a layer of fp16 experts
        dict(name="moe_fp16_t1", op="moe", kind="fp16", T=1, E=64, H=3840, I=1920, k=4, res=True,
             group=0),
        # one decoded token through a layer of int8 experts
        dict(name="moe_int8_t1", op="moe", kind="int8", T=1, E=128, H=5120, I=2176, k=8,
             res=False, group=0),
        # seven tokens (speculative decoding) through group-wise quantised experts of odd width
        dict(name="moe_uint8_t7", op="moe", kind="uint8", T=7, E=32, H=2048, I=1408, k=2,
             res=True, group=GROUP),
        # a decode batch that reaches nearly every expert
        dict(name="moe_fp16_t32", op="moe", kind="fp16", T=32, E=64, H=3840, I=1920, k=4,
             res=True, group=0),
    ]


def _log(rng, lo, hi, step):
    return max(lo, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi))) / step)) * step)


def draw(rng):
    op = rng.choice(("epilogue", "epilogue", "route", "moe", "moe"))
    kind = rng.choice(("fp16", "int8", "uint8"))
    if op == "route":
        return dict(op=op, T=_log(rng, 1, 2048, 1), E=rng.choice((8, 24, 60, 64, 128, 200, 256)),
                    H=_log(rng, 512, 5120, 16), k=rng.randint(1, 8))
    if op == "epilogue":
        group = rng.choice((64, 128)) if kind == "uint8" else 0
        M = _log(rng, 1, 4096, 1)
        N = _log(rng, 256, 17408, 16)
        K = _log(rng, 256, 17408, group or 16)
        while 2.0 * M * N * K > 4.8e11:
            M = max(1, M // 2)
        return dict(op=op, kind=kind, M=M, N=N, K=K, act=rng.choice(
            ("none", "relu", "silu", "gelu", "gelu_tanh")), bias=rng.random() < 0.5,
            res=rng.random() < 0.5, group=group)
    group = rng.choice((64, 128)) if kind == "uint8" else 0
    T = _log(rng, 1, 32, 1)
    E = rng.choice((8, 16, 32, 60, 64, 128))
    k = rng.randint(1, 8)
    H = _log(rng, 1024, 5120, group or 16)
    I = _log(rng, 256, 2176, group or 16)
    while E * 3.0 * I * H * (2 if kind == "fp16" else 1) > 2.8e9:
        E //= 2
    while T * k * 2.0 * I * H * 4 > 2.0e10:
        T = max(1, T // 2)
    return dict(op=op, kind=kind, T=T, E=max(E, k), H=H, I=I, k=k, res=rng.random() < 0.5,
                group=group)


# ------------------------------------------------------------------------------ inputs
def _weight(g, kind, rows, K, group, lead=()):
    """(W, scale, zero) of `rows` output channels: entries of variance about 1 / K."""
    dev = "cuda"
    if kind == "fp16":
        W = torch.randn(*lead, rows, K, generator=g, device=dev, dtype=torch.float16)
        return W.mul_(K ** -0.5), None, None
    if kind == "int8":
        W = torch.randint(-127, 128, (*lead, rows, K), generator=g, device=dev, dtype=torch.int8)
        s = (torch.rand(*lead, rows, generator=g, device=dev) + 0.5) * (K ** -0.5 / 73.0)
        return W, s.half(), None
    W = torch.randint(0, 256, (*lead, rows, K), generator=g, device=dev, dtype=torch.uint8)
    s = (torch.rand(*lead, K // group, rows, generator=g, device=dev) + 0.5) * (K ** -0.5 / 74.0)
    z = torch.randint(112, 145, (*lead, K // group, rows), generator=g, device=dev,
                      dtype=torch.uint8)
    return W, s.half(), z


def prepare(case, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    c = dict(case)

    def rand(*shape, scale=1.0):
        x = torch.randn(*shape, generator=g, device="cuda", dtype=torch.float32)
        return (x * scale).half()

    if c["op"] == "epilogue":
        M, N, K = c["M"], c["N"], c["K"]
        c["A"] = rand(M, K)
        c["W"], c["s"], c["z"] = _weight(g, c["kind"], N, K, c["group"])
        c["b"] = rand(N, scale=0.5) if c["bias"] else None
        c["r"] = rand(M, N) if c["res"] else None
        return c
    T, E, H = c["T"], c["E"], c["H"]
    c["x"] = rand(T, H)
    c["wr"] = rand(E, H, scale=1.5 * H ** -0.5)
    if c["op"] == "moe":
        I, kind, group = c["I"], c["kind"], c["group"]
        c["wgu"], c["sgu"], c["zgu"] = _weight(g, kind, 2 * I, H, group, (E,))
        c["wd"], c["sd"], c["zd"] = _weight(g, kind, H, I, group, (E,))
        c["r"] = rand(T, H) if c["res"] else None
    return c


# ------------------------------------------------------------------------------ plain forms
def _dequant(W, s, z, group, dt):
    """The weight's values, [..., rows, K], in type dt."""
    w = W.to(dt)
    if s is None:
        return w
    if z is None:
        return w.mul_(s.to(dt)[..., None])
    w = w.unflatten(-1, (-1, group))
    w.sub_(z.to(dt).transpose(-1, -2)[..., None]).mul_(s.to(dt).transpose(-1, -2)[..., None])
    return w.flatten(-2)


def _act(y, act):
    if act == "relu":
        return torch.where(y > 0, y, torch.zeros_like(y))
    if act == "silu":
        return y / (1 + torch.exp(-y))
    if act == "gelu":
        return 0.5 * y * (1 + torch.erf(y * math.sqrt(0.5)))
    if act == "gelu_tanh":
        return 0.5 * y * (1 + torch.tanh(math.sqrt(2 / math.pi) * (y + 0.044715 * y * y * y)))
    return y


def _plain_epilogue(c):
    y = c["A"].float() @ _dequant(c["W"], c["s"], c["z"], c["group"], torch.float32).t()
    if c["b"] is not None:
        y = y + c["b"].float()
    y = _act(y, c["act"])
    if c["r"] is not None:
        y = y + c["r"].float()
    return {"y": y.half()}


def _plain_route(x, wr, k):
    """Top-k softmax weights, scaled to a sum of one, in 64 bits: which of two near logits is
    larger is lost in 32.  Equal logits: the lower expert first."""
    p = torch.softmax(x.double() @ wr.double().t(), -1)
    v, i = torch.sort(p, dim=-1, descending=True, stable=True)
    v, i = v[:, :k], i[:, :k]
    return i.int(), (v / v.sum(-1, keepdim=True)).float()


def _of(t, ids):
    return None if t is None else t[ids.long()]


def _plain_moe(c):
    ids, w = _plain_route(c["x"], c["wr"], c["k"])
    x, I = c["x"].float(), c["I"]
    # [T, k, 2I, H] of the chosen experts, then [T, k, H, I]
    gu = torch.einsum("tnh,th->tn", _dequant(_of(c["wgu"], ids), _of(c["sgu"], ids), _of(
        c["zgu"], ids), c["group"], torch.float32).flatten(1, 2), x).unflatten(1, (c["k"], 2 * I))
    gate, up = gu[..., :I], gu[..., I:]
    h = gate / (1 + torch.exp(-gate)) * up
    d = torch.einsum("tjhi,tji->tjh", _dequant(_of(c["wd"], ids), _of(c["sd"], ids), _of(
        c["zd"], ids), c["group"], torch.float32), h)
    y = (d * w[..., None]).sum(1)
    if c["r"] is not None:
        y = y + c["r"].float()
    return {"y": y.half(), "ids": ids, "weights": w}


# ------------------------------------------------------------------------------ one pass
def run(state):
    c = state
    if own:
        from cuda_tempiler_b200 import ops
        if c["op"] == "epilogue":
            if c["kind"] == "fp16":
                y = ops.gemm_fp16_epilogue(c["A"], c["W"], bias=c["b"], activation=c["act"],
                                           residual=c["r"])
            else:
                y = ops.gemm_w8a16_epilogue(c["A"], c["W"], c["s"], c["z"], c["group"],
                                            bias=c["b"], activation=c["act"], residual=c["r"])
            return {"y": y}
        if c["op"] == "route":
            ids, w = ops.moe_route(c["x"], c["wr"], c["k"])
            return {"ids": ids, "weights": w}
        y, ids, w = ops.moe_layer(
            c["x"], c["wr"], c["wgu"], c["wd"], c["k"], s_gate_up=c["sgu"], z_gate_up=c["zgu"],
            s_down=c["sd"], z_down=c["zd"], group_size=c["group"], residual=c["r"],
            return_routing=True)
        return {"y": y, "ids": ids, "weights": w}
    if c["op"] == "epilogue":
        return _plain_epilogue(c)
    if c["op"] == "route":
        ids, w = _plain_route(c["x"], c["wr"], c["k"])
        return {"ids": ids, "weights": w}
    return _plain_moe(c)


# ------------------------------------------------------------------------------ 64 bits
def _exact_weight(W, s, z, group):
    """One weight matrix [rows, K] in 64 bits, written out from the definition."""
    if s is None:
        return W.to(torch.float64)
    if z is None:
        return W.double() * s.double().reshape(-1, 1)
    zz = z.double().repeat_interleave(group, 0).t()
    ss = s.double().repeat_interleave(group, 0).t()
    return (W.double() - zz) * ss


def _exact_act(y, act):
    if act == "relu":
        return y.clamp(min=0)
    if act == "silu":
        return y * torch.sigmoid(y)
    if act == "gelu":
        return y * torch.special.ndtr(y)
    if act == "gelu_tanh":
        return y * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (y + 0.044715 * y ** 3))
    return y


def _exact_route(x, wr, k):
    z = torch.einsum("th,eh->te", x.double(), wr.double())
    order = torch.argsort(-z, dim=-1, stable=True)[:, :k]
    top = torch.gather(z, 1, order)
    e = torch.exp(top - top[:, :1])
    return order, e / e.sum(1, keepdim=True)


def exact(case, seed):
    c = prepare(case, seed)
    if c["op"] == "epilogue":
        y = torch.mm(c["A"].double(), _exact_weight(c["W"], c["s"], c["z"], c["group"]).t())
        y = _exact_act(y + (0 if c["b"] is None else c["b"].double()), c["act"])
        return {"y": y if c["r"] is None else y + c["r"].double()}
    ids, w = _exact_route(c["x"], c["wr"], c["k"])
    if c["op"] == "route":
        return {"ids": None, "weights": w}
    I, x = c["I"], c["x"].double()
    y = torch.zeros_like(x) if c["r"] is None else c["r"].double()

    def of(name, e):
        return None if c[name] is None else c[name][e]

    for e in sorted(set(ids.flatten().tolist())):
        t, j = torch.nonzero(ids == e, as_tuple=True)
        gu = x[t] @ _exact_weight(of("wgu", e), of("sgu", e), of("zgu", e), c["group"]).t()
        h = gu[:, :I] * torch.sigmoid(gu[:, :I]) * gu[:, I:]
        d = h @ _exact_weight(of("wd", e), of("sd", e), of("zd", e), c["group"]).t()
        y[t] += d * w[t, j][:, None]
    return {"y": y, "ids": None, "weights": w}


# ------------------------------------------------------------------------------ work
def _weight_bytes(kind, rows, K, group):
    if kind == "fp16":
        return 2.0 * rows * K
    return rows * K + (2.0 * rows if kind == "int8" else 3.0 * rows * K / group)


def work(case):
    c = case
    if c["op"] == "epilogue":
        M, N, K = c["M"], c["N"], c["K"]
        b = _weight_bytes(c["kind"], N, K, c["group"]) + 2.0 * M * K + 2.0 * M * N
        b += (2.0 * N if c["bias"] else 0) + (2.0 * M * N if c["res"] else 0)
        return {"bytes": b, "flops": 2.0 * M * N * K}
    T, E, H, k = c["T"], c["E"], c["H"], c["k"]
    b = 2.0 * (T + E) * H + 8.0 * T * k
    f = 2.0 * T * E * H
    if c["op"] == "moe":
        I = c["I"]
        # the experts that T tokens reach, if each chooses its k at random
        reached = E * (1 - (1 - k / E) ** T)
        b += reached * (_weight_bytes(c["kind"], 2 * I, H, c["group"])
                        + _weight_bytes(c["kind"], H, I, c["group"]))
        b += 2.0 * T * H * (2 if c["res"] else 1)
        f += 6.0 * T * k * I * H
    return {"bytes": b, "flops": f}
