"""GPU parity of the expert router and the few-token MoE layer against their 64-bit restatement:
every weight kind, token counts of every width of the kernels, ragged experts and sizes, ties,
tokens without an expert, infinities that must stay with their own token."""
import math

import pytest
import torch

from oracle import layer_oracle as L

pytestmark = pytest.mark.gpu


def rand(*shape, seed=0, scale=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).half()


def expert_weights(kind, E, rows, K, group, seed):
    g = torch.Generator("cuda").manual_seed(seed)
    if kind == "fp16":
        return (torch.randn(E, rows, K, generator=g, device="cuda") * K ** -0.5).half(), None, None
    if kind == "int8":
        W = torch.randint(-128, 128, (E, rows, K), generator=g, device="cuda", dtype=torch.int8)
        s = (torch.rand(E, rows, generator=g, device="cuda") + 0.5) * K ** -0.5 / 73
        return W, s.half(), None
    W = torch.randint(0, 256, (E, rows, K), generator=g, device="cuda", dtype=torch.uint8)
    s = (torch.rand(E, K // group, rows, generator=g, device="cuda") + 0.5) * K ** -0.5 / 74
    z = torch.randint(100, 157, (E, K // group, rows), generator=g, device="cuda",
                      dtype=torch.uint8)
    return W, s.half(), z


def whole(T, H, seed=0):
    """Tokens of small whole numbers: with router_weights their logits are multiples of 2^-s below
    2^23 of it, which fp32 sums hold exactly in any order, so the choice is decided alike in 32 and
    in 64 bits, equal logits included."""
    g = torch.Generator("cuda").manual_seed(seed)
    return torch.randint(-3, 4, (T, H), generator=g, device="cuda").half()


def router_weights(E, H, seed=0):
    g = torch.Generator("cuda").manual_seed(seed)
    s = round(math.log2(2 * 4.9 * H ** 0.5 / 1.5))
    return torch.randint(-8, 9, (E, H), generator=g, device="cuda").half() * 2.0 ** -s


class Layer:
    def __init__(self, kind, E, H, I, group=0, block=0, seed=0):
        self.kind, self.E, self.H, self.I, self.group, self.block = kind, E, H, I, group, block
        self.gu = expert_weights(kind, E, 2 * I, H, group, seed + 1)
        self.dn = expert_weights(kind, E, H, I, group, seed + 2)
        self.wr = router_weights(E, H, seed + 3)

    def kw(self):
        return dict(s_gate_up=self.gu[1], z_gate_up=self.gu[2], s_down=self.dn[1],
                    z_down=self.dn[2], group_size=self.group, gu_block=self.block)

    def __call__(self, x, k, **kw):
        from cuda_tempiler_b200 import ops
        return ops.moe_layer(x, self.wr, self.gu[0], self.dn[0], k, **self.kw(), **kw)

    def experts(self, x, ids, w, **kw):
        from cuda_tempiler_b200 import ops
        return ops.moe_experts(x, ids, w, self.gu[0], self.dn[0], **self.kw(), **kw)

    def ref(self, x, ids, w, res=None, w_off=None):
        return L.experts(x, ids, w, L.dequant(*self.gu, self.group),
                         L.dequant(*self.dn, self.group), res, self.block, w_off)


def assert_close(y, ref, tol):
    bad = ((y.double() - ref).abs() > tol) | ~torch.isfinite(y)
    assert not bad.any(), (int(bad.sum()), float(((y.double() - ref).abs() / tol).max()))


def routed(x, wr, k, **kw):
    ids, w, off, _ = L.route(x, wr, k, **kw)
    return ids, w, off


# ------------------------------------------------------------------------------ router
@pytest.mark.parametrize("T,E,H,k", [(1, 1, 8, 1), (1, 8, 64, 2), (1, 64, 3840, 4), (2, 7, 72, 7),
                                     (5, 60, 1000, 6), (8, 128, 2048, 8), (9, 33, 520, 3),
                                     (31, 200, 264, 16), (32, 512, 512, 16), (33, 16, 136, 1),
                                     (100, 129, 776, 8), (257, 24, 1032, 5)])
@pytest.mark.parametrize("normalize", [True, False])
def test_route(dev, T, E, H, k, normalize):
    from cuda_tempiler_b200 import ops
    x, wr = whole(T, H, seed=T), router_weights(E, H, seed=E)
    bias = (rand(E, seed=3) * 8).round() / 8 if T % 2 else None
    ids, w, off = routed(x, wr, k, normalize=normalize, bias=bias)
    i, v = ops.moe_route(x, wr, k, normalize, bias)
    assert i.dtype == torch.int32 and v.dtype == torch.float32
    assert torch.equal(i, ids)
    assert ((v.double() - w).abs() <= off + 2.0 ** -24).all()


@pytest.mark.parametrize("T,E,H,k", [(1, 64, 3840, 4), (16, 128, 5120, 8), (300, 60, 2064, 6)])
def test_route_of_normal_values(dev, T, E, H, k):
    """Tokens whose logits are decided by more than fp32 can be off by: nearly all of them."""
    from cuda_tempiler_b200 import ops
    x, wr = rand(T, H, seed=T), rand(E, H, seed=E, scale=1.5 * H ** -0.5)
    ids, w = ops.moe_route(x, wr, k)
    decided = 0
    for t in range(T):
        want, v, off, far = L.route(x[t:t + 1], wr, k)
        if far <= 1:
            continue
        decided += 1
        assert torch.equal(ids[t:t + 1], want)
        assert ((w[t:t + 1].double() - v).abs() <= off + 2.0 ** -24).all()
    assert decided >= 0.9 * T


@pytest.mark.parametrize("T", [1, 8, 20, 40])
def test_route_ties_go_to_the_lower_expert(dev, T):
    from cuda_tempiler_b200 import ops
    x = rand(T, 256, seed=1)
    one = rand(4, 256, seed=2)
    wr = one.repeat(10, 1)  # expert e equals e % 4
    ids, w = ops.moe_route(x, wr, 10)
    z = x.double() @ one.double().t()
    best = z.argmax(1)
    want = best[:, None] + 4 * torch.arange(10, device="cuda")[None]
    assert torch.equal(ids.long(), want)
    assert (w - 0.1).abs().max() < 2.0 ** -22
    ids, w = ops.moe_route(torch.zeros_like(x), wr, 5)  # logits of -0 and +0 are equal
    assert torch.equal(ids.long(), torch.arange(5, device="cuda").expand(T, 5))


def test_route_of_infinite_and_nan_logits(dev):
    from cuda_tempiler_b200 import ops
    x, wr = rand(9, 128, seed=4), rand(40, 128, seed=5)
    good_ids, good_w = ops.moe_route(x, wr, 6)
    bad = x.clone()
    bad[2, 7] = float("nan")
    bad[5, 0] = float("inf")
    for normalize in (True, False):
        good_ids, good_w = ops.moe_route(x, wr, 6, normalize)
        ids, w = ops.moe_route(bad, wr, 6, normalize)
        rest = [0, 1, 3, 4, 6, 7, 8]
        assert torch.equal(ids[rest], good_ids[rest]) and torch.equal(w[rest], good_w[rest])
        assert torch.isnan(w[2]).all() and torch.isnan(w[5]).any()
        for t in (2, 5):
            assert len(set(ids[t].tolist())) == 6 and 0 <= ids[t].min() and ids[t].max() < 40
    # a bias of the type's lowest value, and of -inf, shuts an expert
    bias = torch.zeros(40, dtype=torch.float16, device="cuda")
    bias[::2] = -65504.0
    bias[1] = float("-inf")
    ids, w = ops.moe_route(x, wr, 16, bias=bias)
    assert (ids % 2 == 1).all() and (ids != 1).all() and torch.isfinite(w).all()


def test_route_strided(dev):
    from cuda_tempiler_b200 import ops
    x, wr = rand(12, 512, seed=6), rand(16, 512, seed=7)
    ids, w = ops.moe_route(x[:, :256], wr[:, 256:], 3)
    i2, w2 = ops.moe_route(x[:, :256].contiguous(), wr[:, 256:].contiguous(), 3)
    assert torch.equal(ids, i2) and torch.equal(w, w2)


# ------------------------------------------------------------------------------ layer
CASES = [  # T, E, H, I, k
    (1, 1, 64, 64, 1), (1, 4, 128, 192, 2), (1, 16, 1024, 704, 4), (2, 8, 320, 64, 8),
    (7, 6, 2048, 128, 2), (8, 32, 576, 448, 5), (9, 12, 192, 320, 3), (16, 40, 448, 256, 8),
    (17, 8, 128, 576, 2), (31, 64, 256, 192, 16), (32, 5, 704, 128, 4)]


@pytest.mark.parametrize("kind,group", [("fp16", 0), ("int8", 0), ("uint8", 64)])
@pytest.mark.parametrize("T,E,H,I,k", CASES)
def test_layer(dev, kind, group, T, E, H, I, k):
    ly = Layer(kind, E, H, I, group, seed=T)
    x, res = whole(T, H, seed=20 + T), rand(T, H, seed=5)
    ids, w, off = routed(x, ly.wr, k)
    out = torch.empty(T, H, dtype=torch.float16, device="cuda")
    out.view(torch.int16).fill_(0x7F7F)
    y, i, v = ly(x, k, residual=res, out=out, return_routing=True)
    assert y is out and torch.equal(i, ids)
    assert_close(y, *ly.ref(x, ids, w, res, off))
    assert torch.equal(ly.experts(x, i, v, residual=res), y)
    plain = ly(x, k)
    assert_close(plain, *ly.ref(x, ids, w, None, off))


@pytest.mark.parametrize("kind", ["fp16", "int8"])
@pytest.mark.parametrize("H,I", [(16, 16), (80, 48), (1040, 336), (3856, 80)])
def test_odd_widths(dev, kind, H, I):
    for T in (1, 6, 20):
        ly = Layer(kind, 6, H, I, seed=H)
        x = whole(T, H, seed=T)
        ids, w, off = routed(x, ly.wr, 2)
        assert_close(ly(x, 2), *ly.ref(x, ids, w, None, off))


@pytest.mark.parametrize("kind,group", [("fp16", 0), ("int8", 0), ("uint8", 128)])
@pytest.mark.parametrize("block", [8, 64])
def test_interleaved_gate_up(dev, kind, group, block):
    ly = Layer(kind, 6, 256, 256 if group else 192, group, block, seed=30)
    x = whole(5, 256, seed=31)
    ids, w, off = routed(x, ly.wr, 3)
    assert_close(ly(x, 3), *ly.ref(x, ids, w, None, off))


@pytest.mark.parametrize("T", [1, 5, 13, 32])
def test_experts_with_a_given_routing(dev, T):
    """Ids that name no expert, experts named twice, weights of any size and sign."""
    ly = Layer("fp16", 5, 128, 64, seed=40)
    g = torch.Generator().manual_seed(T)
    ids = torch.randint(-2, 8, (T, 6), generator=g).int().cuda()
    w = torch.randn(T, 6, generator=g).cuda() * 3
    ids[0] = torch.tensor([-1, 5, 7, 2 ** 31 - 1, -2 ** 31, 100])
    x, res = rand(T, 128, seed=41), rand(T, 128, seed=42)
    y = ly.experts(x, ids, w, residual=res)
    assert_close(y, *ly.ref(x, ids, w, res))
    assert torch.equal(y[0], res[0])
    assert (ly.experts(x, ids, w)[0] == 0).all()
    ids.fill_(-1)
    assert (ly.experts(x, ids, w) == 0).all()


@pytest.mark.parametrize("T", [2, 12, 32])
@pytest.mark.parametrize("kind", ["fp16", "int8"])
def test_infinities_stay_with_their_token(dev, kind, T):
    ly = Layer(kind, 4, 128, 64, seed=50)
    x = rand(T, 128, seed=51)
    ids = torch.tensor([[0, 1], [2, 1]] * 16, device="cuda")[:T].int()
    w = torch.full((T, 2), 0.5, device="cuda")
    y = ly.experts(x, ids, w)
    bad = x.clone()
    bad[0, 5] = float("inf")
    bad[1, 6] = float("nan")
    z = ly.experts(bad, ids, w)
    assert torch.equal(z[2:], y[2:])
    assert not torch.isfinite(z[0]).any() and torch.isnan(z[1]).all()
    if kind == "fp16":  # an infinite weight of an expert reaches its own tokens only
        ly.dn[0][2, :, 3] = float("inf")
        z = ly.experts(x, ids, w)
        assert torch.equal(z[0::2], y[0::2]) and not torch.isfinite(z[1::2]).any()


def test_hidden_values_of_every_size(dev):
    """h far above fp16's range and far below it: the rows are scaled before they are split."""
    ly = Layer("fp16", 3, 128, 64, seed=60)
    x = rand(6, 128, seed=61)
    ids = torch.tensor([[0, 1]] * 6, device="cuda").int()
    for scale in (1e-12, 1e-3, 1.0, 3e3):
        w = torch.full((6, 2), scale, device="cuda")
        big = (x.float() * 30).half()
        y = ly.experts(big, ids, w)
        ref, tol = ly.ref(big, ids, w)
        small = ref.abs() < 65000
        assert (((y.double() - ref).abs() <= tol) | ~small).all()
    # 2e5 * 1e-4 through the layer: the hidden row alone would overflow fp16
    x2 = torch.full((1, 128), 200.0, dtype=torch.float16, device="cuda")
    ly.gu[0].abs_()
    ly.dn[0].mul_(2.0 ** -11)
    i1, w1 = torch.zeros(1, 1, dtype=torch.int32, device="cuda"), torch.ones(1, 1, device="cuda")
    ref, tol = ly.ref(x2, i1, w1)
    assert_close(ly.experts(x2, i1, w1), ref, tol)


def test_in_place_residual_and_strides(dev):
    ly = Layer("int8", 8, 192, 64, seed=70)
    buf = rand(11, 256, seed=71)
    keep = buf.clone()
    x = whole(9, 200, seed=72)[:, :192]
    stream = buf[1:10, 32:224]
    ids, w, off = routed(x, ly.wr, 2)
    ly(x, 2, residual=stream, out=stream)
    assert_close(stream, *ly.ref(x, ids, w, keep[1:10, 32:224], off))
    keep[1:10, 32:224] = stream
    assert torch.equal(buf, keep)


def test_no_tokens(dev):
    ly = Layer("fp16", 4, 64, 64, seed=80)
    x = torch.empty(0, 64, dtype=torch.float16, device="cuda")
    y, ids, w = ly(x, 2, return_routing=True)
    assert y.shape == (0, 64) and ids.shape == (0, 2) and w.shape == (0, 2)


def test_graphs_and_streams(dev):
    """A captured layer replays with new inputs; two graphs side by side keep apart; eager calls
    on several streams at once too."""
    ly = Layer("fp16", 16, 512, 256, seed=90)
    xs = [rand(4, 512, seed=91 + i) for i in range(4)]
    want = [ly(x, 4) for x in xs]
    side = torch.cuda.Stream()
    bufs, outs, graphs = [], [], []
    for i in range(2):
        b = xs[0].clone()
        side.wait_stream(torch.cuda.current_stream())
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            outs.append(ly(b, 4))
        bufs.append(b)
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in range(4)]
    for rep in range(6):
        bufs[0].copy_(xs[rep % 4])
        bufs[1].copy_(xs[(rep + 1) % 4])
        torch.cuda.synchronize()
        for st, gr in zip(streams, graphs):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        assert torch.equal(outs[0], want[rep % 4]) and torch.equal(outs[1], want[(rep + 1) % 4])
    for rep in range(4):
        ys = []
        for st, x in zip(streams, xs):
            with torch.cuda.stream(st):
                ys.append(ly(x, 4))
        torch.cuda.synchronize()
        for y, r in zip(ys, want):
            assert torch.equal(y, r)


@pytest.mark.parametrize("kind,group", [("fp16", 0), ("uint8", 64)])
def test_half_a_decoder_layer(dev, kind, group):
    """Output projection onto the residual stream, then experts onto it, as a decode step runs
    them; each operator's inputs are the outputs of the one before it."""
    from cuda_tempiler_b200 import ops
    H, I, E, k, T = 512, 256, 16, 4, 6
    ly = Layer(kind, E, H, I, group, seed=100)
    W, s, z = expert_weights(kind, 1, H, 768, group, 101)
    W, s, z = W[0], None if s is None else s[0], None if z is None else z[0]
    attn, stream = rand(T, 768, seed=102), rand(T, H, seed=103)
    before = stream.clone()
    if kind == "fp16":
        ops.gemm_fp16_epilogue(attn, W, residual=stream, out=stream)
    else:
        ops.gemm_w8a16_epilogue(attn, W, s, z, group, residual=stream, out=stream)
    assert_close(stream, *L.epilogue(attn, L.dequant(W, s, z, group), None, "none", before))
    mid = stream.clone()
    x = (mid.float() / mid.float().square().mean(1, keepdim=True).sqrt()).round().half()
    _, ids, w = ly(x, k, residual=stream, out=stream, return_routing=True)
    want_ids, want_w, off = routed(x, ly.wr, k)
    assert torch.equal(ids, want_ids)
    assert_close(stream, *ly.ref(x, want_ids, want_w, mid, off))
    assert ops.device_status() == [0, 0, 0, 0]


def test_refusals(dev):
    from cuda_tempiler_b200 import ops
    ly, ly8 = Layer("fp16", 4, 64, 64, seed=1), Layer("uint8", 4, 128, 64, 64, seed=1)
    x, x8 = rand(3, 64), rand(3, 128)
    ids = torch.zeros(3, 2, dtype=torch.int32, device="cuda")
    w = torch.ones(3, 2, device="cuda")
    with pytest.raises(ValueError, match="top_k"):
        ly(x, 5)
    with pytest.raises(ValueError, match="top_k"):
        ops.moe_route(x, ly.wr, 0)
    with pytest.raises(ValueError, match="hidden"):
        ops.moe_route(x, rand(4, 72), 1)
    with pytest.raises(ValueError, match="bias"):
        ops.moe_route(x, ly.wr, 1, bias=rand(5))
    with pytest.raises(ValueError, match="experts"):
        ops.moe_layer(x, rand(5, 64), ly.gu[0], ly.dn[0], 1)
    with pytest.raises(ValueError, match="expert weights"):
        ops.moe_layer(x, ly.wr, ly.gu[0], ly.dn[0].float(), 1)
    with pytest.raises(ValueError, match="expert weights"):
        ops.moe_layer(x, ly.wr, ly.gu[0][:, :120], ly.dn[0], 1)
    with pytest.raises(ValueError, match="expert weights"):
        ops.moe_layer(x, ly.wr, ly.gu[0].transpose(1, 2), ly.dn[0], 1)
    with pytest.raises(ValueError, match="scale"):
        ops.moe_layer(x8, ly8.wr, ly8.gu[0], ly8.dn[0], 1, group_size=64)
    with pytest.raises(ValueError, match="gu_block"):
        ly.block = 12
        ly(x, 2)
    ly.block = 0
    with pytest.raises(ValueError, match="ids"):
        ly.experts(x, ids.long(), w)
    with pytest.raises(ValueError, match="ids"):
        ly.experts(x, ids[:2], w)
    with pytest.raises(ValueError, match="weights"):
        ly.experts(x, ids, w.half())
    with pytest.raises(ValueError, match="weights"):
        ly.experts(x, ids, w.cpu())
    with pytest.raises(ValueError, match="overlaps x"):
        ly(x, 2, out=x)
    with pytest.raises(ops.NotCovered):
        ly(rand(33, 64), 2)
    with pytest.raises(ops.NotCovered):
        ops.moe_route(rand(3, 60), rand(4, 60), 2)


@pytest.mark.parametrize("kind", ["fp16", "int8"])
@pytest.mark.parametrize("M", [1, 9, 300])
def test_tensor_parallel_helpers(dev, kind, M):
    """One rank of tp: the MLP with the residual in its last epilogue, the sharded experts summed
    by hand over the ranks."""
    from cuda_tempiler_b200 import ops, tp
    H, I, E, k = 256, 256, 8, 2
    gu, dn = expert_weights(kind, E, 2 * I, H, 0, 7), expert_weights(kind, E, H, I, 0, 8)
    half = lambda t, i: None if t is None else t[:, i * I:(i + 1) * I]  # noqa: E731
    one = lambda t, e: None if t is None else t[e]  # noqa: E731
    x, res = whole(M, H, seed=9), rand(M, H, seed=10)
    m = tp.shard_mlp(half(gu[0], 0)[0], half(gu[0], 1)[0], dn[0][0], 1, 0,
                     one(half(gu[1], 0), 0), one(half(gu[1], 1), 0), one(dn[1], 0))
    y = tp.mlp_forward(x, m, residual=res)
    # the same two GEMMs by hand: the residual goes into the second one's epilogue
    h = tp._default_fused(x, m.w_gate_up, m.s_gate_up) if M > 256 else None
    if h is None:
        h = ops.silu_mul(tp._default_gemm(x, m.w_gate_up, m.s_gate_up), block=m.gu_block)
    assert torch.equal(y, tp._down_residual(h, m.w_down, m.s_down, res))
    assert_close(y, *L.epilogue(h, L.dequant(m.w_down, m.s_down, None, 0), None, "none", res))
    if M > 32:
        return
    wr = router_weights(E, H, 11)
    ids, w, off = routed(x, wr, k)
    ref, tol = L.experts(x, ids, w, L.dequant(*gu, 0), L.dequant(*dn, 0), res, 0, off)
    parts = [tp.moe_forward(x, wr, tp.shard_moe(half(gu[0], 0), half(gu[0], 1), dn[0], 2, r,
                                                half(gu[1], 0), half(gu[1], 1), dn[1]), k,
                            residual=res if r == 0 else None) for r in range(2)]
    # each of the two partials is rounded once
    total = parts[0].double() + parts[1].double()
    assert ((total - ref).abs() <= 2 * tol + 2.0 ** -10 * (parts[1].double().abs() +
                                                          parts[0].double().abs())).all()


def test_packed_scales_and_zero_points(dev):
    """Scales and zero points as views into one buffer: taken at any word, refused off one."""
    from cuda_tempiler_b200 import ops
    ly = Layer("uint8", 6, 128, 192, 64, seed=110)
    x = whole(5, 128, seed=111)
    want = ly(x, 3)

    def at(t, off):  # t's values from `off` elements behind a 16-byte boundary
        buf = torch.empty(t.numel() + 16, dtype=t.dtype, device="cuda")
        return buf[off:off + t.numel()].view(t.shape).copy_(t)

    gu, dn = ly.gu, ly.dn
    ly.gu, ly.dn = (gu[0], at(gu[1], 2), at(gu[2], 4)), (dn[0], at(dn[1], 6), at(dn[2], 12))
    assert torch.equal(ly(x, 3), want)
    for i, off in ((1, 1), (1, 3), (2, 1), (2, 2), (2, 3)):
        for which in "gu", "dn":
            ly.gu, ly.dn = gu, dn
            w = list(getattr(ly, which))
            w[i] = at(w[i], off)
            setattr(ly, which, w)
            with pytest.raises(ops.NotCovered):
                ly(x, 3)


@pytest.mark.parametrize("kind,group", [("int8", 0), ("uint8", 64)])
@pytest.mark.parametrize("T", [1, 7, 24])
def test_one_signed_tokens_and_narrow_weights(dev, kind, group, T):
    """Tokens of one sign (their sum over k is far from zero) and weights of a few steps around
    zero, the zero points anywhere."""
    E, H, I = 4, 4096, 256
    g = torch.Generator("cuda").manual_seed(T)

    def small(rows, K):
        q = torch.randint(-3, 4, (E, rows, K), generator=g, device="cuda", dtype=torch.int16)
        c = (0.75, 0.5) if K == H else (0.5, 0.25)  # scales that keep h near one
        if kind == "int8":
            s = (torch.rand(E, rows, generator=g, device="cuda") * c[0] + c[1]) * K ** -0.5
            return q.to(torch.int8), s.half(), None
        z = torch.randint(3, 253, (E, K // group, rows), generator=g, device="cuda",
                          dtype=torch.int16)
        W = (q + z.repeat_interleave(group, 1).transpose(1, 2)).to(torch.uint8)
        s = (torch.rand(E, K // group, rows, generator=g, device="cuda") * c[0] + c[1]) * K ** -0.5
        return W, s.half(), z.to(torch.uint8)

    ly = Layer(kind, E, H, I, group, seed=T)
    ly.gu, ly.dn = small(2 * I, H), small(H, I)
    x = rand(T, H, seed=T).abs()
    ids = torch.randint(0, E, (T, 2), generator=g, device="cuda").int()
    w = torch.rand(T, 2, generator=g, device="cuda") + 0.5
    y = ly.experts(x, ids, w)
    # acc(K) counts K / 16 truncations of the whole sum; here at most a step of 64 k is added on the
    # tensor core (20), the steps of a warp and the warps in fp32: K / 256 + 16 at 4 warps or more
    full, L.acc = L.acc, lambda K: (20 + K / 256 + 16) * 2.0 ** -23
    try:
        ref, tol = ly.ref(x, ids, w)
    finally:
        L.acc = full
    assert_close(y, ref, tol)


@pytest.mark.parametrize("kind", ["fp16", "int8"])
def test_tensor_parallel_residuals_in_any_layout(dev, kind):
    """One that the epilogue does not read as it lies is laid out first: a rank must not raise
    where the others go on to the all-reduce."""
    from cuda_tempiler_b200 import tp
    H, I, E, M = 256, 128, 4, 5
    gu, dn = expert_weights(kind, E, 2 * I, H, 0, 7), expert_weights(kind, E, H, I, 0, 8)
    x = whole(M, H, seed=9)
    one = lambda t: None if t is None else t[0]  # noqa: E731
    m = tp.MLPShard(gu[0][0], one(gu[1]), dn[0][0], one(dn[1]), I)
    e = tp.MoEShard(gu[0], gu[1], dn[0], dn[1])
    wr = router_weights(E, H, 11)
    buf = rand(M + 1, H + 16, seed=12)
    for res in (buf[:M, 3:3 + H], buf[1:2, 8:8 + H].expand(M, H), rand(H, M, seed=13).t()):
        flat = res.contiguous()
        assert torch.equal(tp.mlp_forward(x, m, residual=res), tp.mlp_forward(x, m, residual=flat))
        assert torch.equal(tp.moe_forward(x, wr, e, 2, residual=res),
                           tp.moe_forward(x, wr, e, 2, residual=flat))
    for bad in (buf[:M, :H].float(), buf[:M, :H].cpu(), buf[:M, :H + 8], buf[0, :H]):
        with pytest.raises(ValueError, match="residual"):
            tp.mlp_forward(x, m, residual=bad)
        with pytest.raises(ValueError, match="residual"):
            tp.moe_forward(x, wr, e, 2, residual=bad)


def test_threads_on_one_stream(dev):
    """A layer, its caller-routed form and GEMMs of several host threads on the same stream."""
    import threading
    from cuda_tempiler_b200 import ops
    ly = Layer("int8", 16, 512, 256, seed=120)
    x = rand(6, 512, seed=121)
    y, ids, w = ly(x, 3, return_routing=True)
    a, b, r = rand(300, 2048, seed=1), rand(784, 2048, seed=2, scale=0.02), rand(300, 784, seed=3)
    c = torch.randint(-128, 128, (1024, 2048), device="cuda", dtype=torch.int8)
    sc = torch.full((1024,), 1e-3, device="cuda", dtype=torch.float16)
    calls = [lambda: ly(x, 3), lambda: ly.experts(x, ids, w),
             lambda: ops.gemm_fp16_epilogue(a, b, residual=r), lambda: ops.gemm_fp16(a, b),
             lambda: ops.gemm_w8a16(a.repeat(5, 1), c, sc)]
    want = [f() for f in calls]
    torch.cuda.synchronize()
    bad = []

    def work(i):
        try:
            for _ in range(300):
                if not torch.equal(calls[i](), want[i]):
                    bad.append(i)
        except Exception as e:
            bad.append(e)

    ts = [threading.Thread(target=work, args=(i,)) for i in range(len(calls))]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    torch.cuda.synchronize()
    assert not bad, bad
