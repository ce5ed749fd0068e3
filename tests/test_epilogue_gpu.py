"""GPU parity of the GEMM with a fused epilogue against its 64-bit restatement: every path (the
weight stream, the swapped tiles whole and in shares, the 2-CTA tiles with and without a split
tail, the expanded prefill), every activation, ragged sizes, strides, in-place residuals."""
import itertools

import pytest
import torch

from oracle import layer_oracle as L

pytestmark = pytest.mark.gpu


def weights(kind, N, K, group, seed=0):
    g = torch.Generator("cuda").manual_seed(seed + 1000)
    if kind == "fp16":
        return (torch.randn(N, K, generator=g, device="cuda") * K ** -0.5).half(), None, None
    if kind == "int8":
        W = torch.randint(-128, 128, (N, K), generator=g, device="cuda", dtype=torch.int8)
        return W, ((torch.rand(N, generator=g, device="cuda") + 0.5) * K ** -0.5 / 73).half(), None
    W = torch.randint(0, 256, (N, K), generator=g, device="cuda", dtype=torch.uint8)
    s = ((torch.rand(K // group, N, generator=g, device="cuda") + 0.5) * K ** -0.5 / 74).half()
    z = torch.randint(0, 256, (K // group, N), generator=g, device="cuda", dtype=torch.uint8)
    return W, s, z


def rand(*shape, seed=0, scale=1.0):
    g = torch.Generator("cuda").manual_seed(seed)
    return (torch.randn(*shape, generator=g, device="cuda") * scale).half()


def call(A, w, group, **kw):
    from cuda_tempiler_b200 import ops
    W, s, z = w
    if s is None:
        return ops.gemm_fp16_epilogue(A, W, **kw)
    return ops.gemm_w8a16_epilogue(A, W, s, z, group, **kw)


def check(y, A, w, group, bias, act, res):
    rounding = L.U16 if w[2] is not None and A.shape[0] > 16 else 0.0
    ref, tol = L.epilogue(A, L.dequant(*w, group), bias, act, res, rounding)
    bad = ((y.double() - ref).abs() > tol) | ~torch.isfinite(y)
    assert not bad.any(), (int(bad.sum()), float(((y.double() - ref).abs() / tol).max()))


def poison(M, N):
    out = torch.empty(M, N, dtype=torch.float16, device="cuda")
    out.view(torch.int16).fill_(0x7F7F)
    return out


KINDS = [("fp16", 0), ("int8", 0), ("uint8", 64), ("uint8", 128)]
# rows of every band of the dispatch, with N and K ragged against every tile
SHAPES = [(1, 8, 16), (1, 136, 272), (2, 1000, 528), (3, 2504, 1040), (8, 5008, 784),
          (9, 264, 2064), (16, 9480, 400), (17, 272, 1040), (33, 1040, 2064), (64, 528, 4112),
          (65, 784, 1040), (100, 2064, 528), (128, 1296, 784), (129, 1040, 2064), (200, 528, 4112),
          (256, 4112, 272), (257, 784, 1040), (333, 2064, 2064), (600, 528, 4112),
          (1025, 1040, 1296)]


@pytest.mark.parametrize("kind,group", KINDS)
@pytest.mark.parametrize("M,N,K", SHAPES)
def test_shapes(dev, kind, group, M, N, K):
    if group:
        K = max(group, K // group * group)
        N = -(-N // 16) * 16
    A, w = rand(M, K, seed=M), weights(kind, N, K, group, seed=N)
    bias, res = rand(N, seed=3), rand(M, N, seed=4)
    out = poison(M, N)
    y = call(A, w, group, bias=bias, activation="silu", residual=res, out=out)
    assert y is out
    check(y, A, w, group, bias, "silu", res)


@pytest.mark.parametrize("kind,group", [("fp16", 0), ("int8", 0), ("uint8", 128)])
@pytest.mark.parametrize("M", [1, 12, 40, 96, 160, 300])
@pytest.mark.parametrize("act", L.ACT)
def test_activations_and_terms(dev, kind, group, M, act):
    N, K = 400, 512
    A, w = rand(M, K, seed=M, scale=3.0), weights(kind, N, K, group)
    for has_b, has_r in itertools.product((False, True), repeat=2):
        bias = rand(N, seed=3) if has_b else None
        res = rand(M, N, seed=4) if has_r else None
        check(call(A, w, group, bias=bias, activation=act, residual=res), A, w, group, bias, act,
              res)


@pytest.mark.parametrize("kind,group", [("fp16", 0), ("int8", 0), ("uint8", 128)])
@pytest.mark.parametrize("M", [5, 16, 50, 128, 256, 700, 1100])
def test_strides_and_in_place(dev, kind, group, M):
    """Row strides wider than the rows (what lies between stays as it was), the residual stream
    updated in place."""
    N, K = 656, 1152
    A = rand(M, K + 24, seed=1)[:, :K]
    w = list(weights(kind, N, K, group))
    wide = torch.zeros(N, K + 32, dtype=w[0].dtype, device="cuda")
    wide[:, :K] = w[0]
    w[0] = wide[:, :K]
    buf = rand(M + 2, N + 16, seed=2)
    keep = buf.clone()
    x = buf[1:M + 1, 8:N + 8]
    call(A, w, group, residual=x, out=x)
    check(x, A, (w[0].contiguous(), *w[1:]), group, None, "none", keep[1:M + 1, 8:N + 8])
    keep[1:M + 1, 8:N + 8] = x
    assert torch.equal(buf, keep)


@pytest.mark.parametrize("M,N,K", [(300, 768, 8192), (512, 3840, 4096), (2048, 3840, 1024)])
def test_split_tail(dev, M, N, K):
    """Shapes whose last wave runs as k-slices: the epilogue applies once, to the whole sum."""
    A, w = rand(M, K, seed=5), weights("fp16", N, K, 0)
    bias, res = rand(N, seed=6), rand(M, N, seed=7)
    for _ in range(2):
        check(call(A, w, 0, bias=bias, activation="relu", residual=res), A, w, 0, bias, "relu", res)


@pytest.mark.parametrize("kind,group", [("fp16", 0), ("int8", 0), ("uint8", 128)])
@pytest.mark.parametrize("M", [16, 17, 100, 256, 257, 340, 384, 385, 512, 768, 769, 1100, 1279, 1280])
@pytest.mark.parametrize("N,K", [(3840, 2048), (528, 8192)])
def test_long_shares(dev, kind, group, M, N, K):
    """Rows around every edge of the dispatch, k ranges that go round each ring of buffers often:
    right, and the same in every run."""
    A, w = rand(M, K, seed=M), weights(kind, N, K, group, seed=5)
    res = rand(M, N, seed=6)
    y = call(A, w, group, residual=res)
    check(y, A, w, group, None, "none", res)
    for _ in range(5):
        assert torch.equal(y, call(A, w, group, residual=res))


@pytest.mark.parametrize("kind,group", [("fp16", 0), ("int8", 0), ("uint8", 128)])
@pytest.mark.parametrize("M,N", [(1, 7168), (5, 15360), (8, 8192), (9, 5120), (16, 7680), (16, 20480)])
def test_few_rows_many_columns(dev, kind, group, M, N):
    """Up to 16 rows on both sides of the choice between the stream and the tiles, and the answer
    without a workspace."""
    from cuda_tempiler_b200 import _lib
    K = 1152
    A, w = rand(M, K, seed=M), weights(kind, N, K, group, seed=5)
    bias, res = rand(N, seed=7), rand(M, N, seed=6)
    check(call(A, w, group, bias=bias, activation="gelu_tanh", residual=res), A, w, group, bias,
          "gelu_tanh", res)
    out, lib = poison(M, N), _lib.load()
    st = torch.cuda.current_stream().cuda_stream
    tail = (out.data_ptr(), bias.data_ptr(), res.data_ptr(), M, N, K, K, K, N, N)
    act = 4  # TEMPO_ACT_GELU_TANH
    if kind == "fp16":
        rc = lib.tempo_sm100_gemm_fp16_epilogue(A.data_ptr(), w[0].data_ptr(), *tail, act, None, 0,
                                                st)
    else:
        rc = lib.tempo_sm100_gemm_w8a16_epilogue(
            A.data_ptr(), w[0].data_ptr(), w[1].data_ptr(),
            None if w[2] is None else w[2].data_ptr(), *tail, 1 if kind == "int8" else 2, group,
            act, None, 0, st)
    assert rc == 0
    check(out, A, w, group, bias, "gelu_tanh", res)


@pytest.mark.parametrize("kind,group", [("fp16", 0), ("int8", 0), ("uint8", 128)])
@pytest.mark.parametrize("M,N,K", [(40, 528, 4096), (300, 272, 2048), (700, 400, 1152)])
def test_without_a_workspace(dev, kind, group, M, N, K):
    """The tiles run whole; 8-bit weights are not expanded."""
    from cuda_tempiler_b200 import _lib
    A, w = rand(M, K, seed=M), weights(kind, N, K, group, seed=5)
    res = rand(M, N, seed=6)
    out, lib = poison(M, N), _lib.load()
    st = torch.cuda.current_stream().cuda_stream
    tail = (out.data_ptr(), None, res.data_ptr(), M, N, K, K, K, N, N)
    if kind == "fp16":
        rc = lib.tempo_sm100_gemm_fp16_epilogue(A.data_ptr(), w[0].data_ptr(), *tail, 0, None, 0, st)
    else:
        rc = lib.tempo_sm100_gemm_w8a16_epilogue(
            A.data_ptr(), w[0].data_ptr(), w[1].data_ptr(),
            None if w[2] is None else w[2].data_ptr(), *tail, 1 if kind == "int8" else 2, group, 0,
            None, 0, st)
    assert rc == 0
    check(out, A, w, group, None, "none", res)


@pytest.mark.parametrize("M", [40, 300])
def test_infinite_rows_stay_apart_in_tiles(dev, M):
    """As above for the tiles, whose MMA has the rows as its N side; k is cut into shares."""
    N, K = 264, 4096
    A, w = rand(M, K, seed=8), weights("fp16", N, K, 0)
    clean = call(A, w, 0)
    A[1, 3], A[M - 1, K - 1] = float("inf"), float("nan")
    y = call(A, w, 0)
    rest = [m for m in range(M) if m not in (1, M - 1)]
    assert torch.equal(y[rest], clean[rest])
    assert torch.isnan(y[M - 1]).all() and not torch.isfinite(y[1]).any()


@pytest.mark.parametrize("kind,group", [("fp16", 0), ("int8", 0), ("uint8", 64)])
@pytest.mark.parametrize("M", [1, 7, 16])
def test_infinite_rows_stay_apart(dev, kind, group, M):
    """An infinite or NaN activation reaches its own row only."""
    N, K = 264 if kind != "uint8" else 272, 512
    A, w = rand(M, K, seed=8), weights(kind, N, K, group)
    clean = call(A, w, group)
    A2 = A.clone()
    A2[0, 3] = float("inf")
    A2[M // 2, K - 1] = float("nan")
    y = call(A2, w, group)
    hit = {0, M // 2}
    rest = [m for m in range(M) if m not in hit]
    assert torch.equal(y[rest], clean[rest])
    assert torch.isnan(y[M // 2]).all() and not torch.isfinite(y[0]).any()


def test_extremes_of_the_activations(dev):
    """relu keeps NaN, large arguments neither overflow nor lose their sign."""
    from cuda_tempiler_b200 import ops
    K, N = 16, 8
    A = torch.zeros(6, K, dtype=torch.float16, device="cuda")
    A[:, 0] = torch.tensor([60000.0, -60000.0, 30.0, -30.0, float("nan"), 0.0])
    B = torch.zeros(N, K, dtype=torch.float16, device="cuda")
    B[:, 0] = 1.0
    for M, act in itertools.product((6, 48), L.ACT):
        X = A.repeat(M // 6, 1)
        y = ops.gemm_fp16_epilogue(X, B, activation=act)
        ref = L.act(X[:, :1].double().expand(M, N), act)
        assert torch.isnan(y[4::6]).all(), act
        y, ref = y.double(), ref
        keep = [i for i in range(M) if i % 6 != 4]
        assert torch.allclose(y[keep], ref[keep], rtol=2.0 ** -10, atol=2.0 ** -23), act


def test_results_do_not_change_between_runs(dev):
    for kind, group, M in (("fp16", 0, 3), ("uint8", 128, 16), ("int8", 0, 90), ("fp16", 0, 512)):
        A, w = rand(M, 2048, seed=9), weights(kind, 1040, 2048, group)
        y = call(A, w, group, activation="gelu")
        for _ in range(5):
            assert torch.equal(y, call(A, w, group, activation="gelu"))


@pytest.mark.parametrize("kind,group,M", [("fp16", 0, 4), ("fp16", 0, 300), ("int8", 0, 1100),
                                          ("uint8", 128, 200)])
def test_graph_capture(dev, kind, group, M):
    """Two graphs captured on one stream replay with their own workspaces, on other streams."""
    N, K = 3840, 2048
    A, w = rand(M, K, seed=10), weights(kind, N, K, group)
    res = [rand(M, N, seed=11 + i) for i in range(2)]
    want = [call(A, w, group, residual=r) for r in res]
    side = torch.cuda.Stream()
    graphs, outs = [], []
    with torch.cuda.stream(side):
        call(A, w, group, residual=res[0])
    side.synchronize()
    for r in res:
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr, stream=side):
            outs.append(call(A, w, group, residual=r))
        graphs.append(gr)
    streams = [torch.cuda.Stream() for _ in graphs]
    for _ in range(4):
        for o in outs:
            o.zero_()
        torch.cuda.synchronize()
        for st, gr in zip(streams, graphs):
            with torch.cuda.stream(st):
                gr.replay()
        torch.cuda.synchronize()
        for o, r in zip(outs, want):
            assert torch.equal(o, r)


def test_linear_layers_keep_gradients(dev, monkeypatch):
    """With gradients to record a fused layer takes the stock path, which has them."""
    from cuda_tempiler_b200 import bind
    monkeypatch.setenv("TEMPO_KERNELS", "1")
    W = rand(272, 512, seed=1, scale=512 ** -0.5)
    res, bias = rand(8, 272, seed=2), rand(272, seed=3)
    for leaf in range(4):
        args = [rand(8, 512, seed=4), W.clone(), bias.clone(), res.clone()]
        args[leaf].requires_grad_()
        bind.route_counts(reset=True)
        y = bind.linear_fp16(args[0], args[1], args[2], activation="silu", residual=args[3])
        assert bind.route_counts()["fallback"] == 1
        y.sum().backward()
        assert args[leaf].grad is not None and torch.isfinite(args[leaf].grad).all()
        with torch.no_grad():
            bind.linear_fp16(args[0], args[1], args[2], activation="silu", residual=args[3])
        assert bind.route_counts()["tempo"] == 1


def test_calls_at_the_same_time(dev):
    """Calls on several streams at once, each with the workspace of its stream: shares of k whose
    parts meet there, split tails with their counters."""
    shapes = [("fp16", 0, 90, 784, 4096), ("uint8", 128, 300, 528, 4096), ("fp16", 0, 512, 3840, 4096)]
    jobs = []
    for i, (kind, group, M, N, K) in enumerate(shapes):
        A, w, res = rand(M, K, seed=i), weights(kind, N, K, group, seed=i), rand(M, N, seed=9 + i)
        jobs.append((A, w, group, res, call(A, w, group, residual=res)))
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(4)]
    got = []
    for _ in range(6):
        for st in streams:
            with torch.cuda.stream(st):
                got.append([call(A, w, group, residual=res) for A, w, group, res, _ in jobs])
    torch.cuda.synchronize()
    for ys in got:
        for y, job in zip(ys, jobs):
            assert torch.equal(y, job[4])


def test_linear_layers_use_the_epilogue(dev, monkeypatch):
    """bind.linear_* with an activation or a residual: the kernels when they are switched on, the
    stock path otherwise, the same values within fp16's rounding."""
    from cuda_tempiler_b200 import bind
    A = rand(5, 8, 512, seed=12)
    bias, res = rand(272, seed=13), rand(5, 8, 272, seed=14)
    for kind, group in (("fp16", 0), ("int8", 0), ("uint8", 128)):
        w = weights(kind, 272, 512, group)
        ys = []
        for on in ("1", "0"):
            monkeypatch.setenv("TEMPO_KERNELS", on)
            bind.route_counts(reset=True)
            if kind == "fp16":
                y = bind.linear_fp16(A, w[0], bias, activation="gelu", residual=res)
            else:
                y = bind.linear_w8a16(A, *w, group, bias, activation="gelu", residual=res)
            assert bind.route_counts()["tempo"] == int(on)
            ys.append(y)
        check(ys[0].reshape(40, 272), A.reshape(40, 512), w, group, bias, "gelu",
              res.reshape(40, 272))
        # the stock path rounds the weight, the product, the bias sum, the activation and the sum
        assert torch.allclose(ys[0].float(), ys[1].float(), rtol=0, atol=2.0 ** -6)


def test_refusals(dev):
    from cuda_tempiler_b200 import ops
    A, B = rand(8, 64), rand(48, 64)
    W, s, z = weights("uint8", 48, 64, 64)
    with pytest.raises(ValueError, match="activation"):
        ops.gemm_fp16_epilogue(A, B, activation="tanh")
    with pytest.raises(ValueError, match="bias"):
        ops.gemm_fp16_epilogue(A, B, bias=rand(47))
    with pytest.raises(ValueError, match="bias"):
        ops.gemm_fp16_epilogue(A, B, bias=rand(48).float())
    with pytest.raises(ValueError, match="bias"):
        ops.gemm_fp16_epilogue(A, B, bias=rand(96)[::2])
    with pytest.raises(ValueError, match="residual"):
        ops.gemm_fp16_epilogue(A, B, residual=rand(8, 64))
    with pytest.raises(ValueError, match="residual"):
        ops.gemm_fp16_epilogue(A, B, residual=rand(48, 8).t())
    with pytest.raises(ValueError, match="residual"):
        ops.gemm_fp16_epilogue(A, B, residual=rand(8, 48).cpu())
    with pytest.raises(ValueError, match="K mismatch"):
        ops.gemm_fp16_epilogue(A, rand(48, 72))
    with pytest.raises(ValueError, match="out"):
        ops.gemm_fp16_epilogue(A, B, out=rand(8, 56))
    with pytest.raises(ValueError, match="scale"):
        ops.gemm_w8a16_epilogue(A, W, s.float(), z, 64)
    with pytest.raises(ValueError, match="zero"):
        ops.gemm_w8a16_epilogue(A, W, s, z[:, :40], 64)
    with pytest.raises(ValueError, match="group"):
        ops.gemm_w8a16_epilogue(A, W, s, None, 64)
    buf = rand(10, 64)
    with pytest.raises(ValueError, match="overlaps A"):
        ops.gemm_fp16_epilogue(buf[:8], rand(64, 64), out=buf[2:])
    with pytest.raises(ValueError, match="overlaps residual"):
        ops.gemm_fp16_epilogue(A, rand(64, 64), residual=buf[:8], out=buf[1:9])
    flat = rand(8 * 48 + 8)
    with pytest.raises(ops.NotCovered):  # residual not 16-byte aligned
        ops.gemm_fp16_epilogue(A, B, residual=flat[1:8 * 48 + 1].view(8, 48))
    with pytest.raises(ops.NotCovered):
        ops.gemm_fp16_epilogue(A, B, bias=rand(56)[1:49])
    with pytest.raises(ops.NotCovered):
        ops.gemm_fp16_epilogue(A, rand(44, 64))
    with pytest.raises(ops.NotCovered):
        ops.gemm_fp16_epilogue(A[:0], B)


def narrow(kind, N, K, group, seed=0):
    """8-bit weights of a few steps around zero (one outlier of the channel or group has set the
    scale), the zero points anywhere."""
    g = torch.Generator("cuda").manual_seed(seed + 2000)
    q = torch.randint(-3, 4, (N, K), generator=g, device="cuda", dtype=torch.int16)
    if kind == "int8":
        return q.to(torch.int8), ((torch.rand(N, generator=g, device="cuda") + 0.5) * 0.01).half(), \
            None
    z = torch.randint(3, 253, (K // group, N), generator=g, device="cuda", dtype=torch.int16)
    W = (q + z.repeat_interleave(group, 0).t()).to(torch.uint8)
    s = ((torch.rand(K // group, N, generator=g, device="cuda") + 0.5) * 0.01).half()
    return W, s, z.to(torch.uint8)


@pytest.mark.parametrize("kind,group", [("int8", 0), ("uint8", 64), ("uint8", 128)])
@pytest.mark.parametrize("M", [1, 8, 16])
@pytest.mark.parametrize("K", [1024, 4096, 16384])
def test_one_signed_activations_times_narrow_weights(dev, kind, group, M, K):
    """Up to 16 rows the products of an 8-bit weight enter the sum as they are: nothing in it is
    larger than S = sum |a| |w|.  A warp's step adds 4 times 16 products on the tensor core (20
    truncations of at most 2^-23 S at the most), the K / 1024 steps of a warp and the 16 warps are
    added in fp32."""
    N = 272
    A, w = rand(M, K, seed=M).abs(), narrow(kind, N, K, group, seed=K)
    y = call(A, w, group)
    Wd = L.dequant(*w, group)
    ref, S = A.double() @ Wd.t(), A.double() @ Wd.abs().t()
    tol = (20 + K / 1024 + 16) * 2.0 ** -23 * S
    tol = tol + L.U16 * (ref.abs() + tol) + 2.0 ** -25
    bad = ~((y.double() - ref).abs() <= tol)
    assert not bad.any(), (int(bad.sum()), float(((y.double() - ref).abs() / tol).max()))


@pytest.mark.parametrize("kind,group", [("int8", 0), ("uint8", 64)])
def test_an_infinite_activation_times_8_bit_weights(dev, kind, group):
    """Its row is infinite with the sign of the weight, NaN where the weight is zero, on every path."""
    N, K = 272, 512
    W, s, z = weights(kind, N, K, group)
    if kind == "int8":
        W[:, 7] = torch.arange(N, device="cuda").remainder(3).sub(1).to(torch.int8)
    else:
        W[:, 7] = (z[0].int().clamp(1, 254) + torch.arange(N, device="cuda") % 3 - 1).to(torch.uint8)
        z[0] = z[0].clamp(1, 254)
    sign = torch.arange(N, device="cuda") % 3 - 1
    for M in (1, 4, 16, 40):
        A = rand(M, K, seed=M)
        clean = call(A, (W, s, z), group)
        A[M // 2, 7] = float("inf")
        y = call(A, (W, s, z), group)
        row = y[M // 2].float()
        assert torch.isnan(row[sign == 0]).all()
        assert (row[sign > 0] == float("inf")).all() and (row[sign < 0] == -float("inf")).all()
        rest = [m for m in range(M) if m != M // 2]
        assert torch.equal(y[rest], clean[rest])


@pytest.mark.parametrize("kind,group", [("int8", 0), ("uint8", 64)])
def test_linear_layers_keep_the_gradient_of_a_scale(dev, monkeypatch, kind, group):
    from cuda_tempiler_b200 import bind
    monkeypatch.setenv("TEMPO_KERNELS", "1")
    W, s, z = weights(kind, 272, 512, group)
    x, res = rand(8, 512, seed=4), rand(8, 272, seed=2)
    grads = []
    for on in ("1", "0"):
        monkeypatch.setenv("TEMPO_KERNELS", on)
        leaf = s.clone().requires_grad_()
        bind.linear_w8a16(x, W, leaf, z, group, activation="silu", residual=res).sum().backward()
        grads.append(leaf.grad)
    assert torch.equal(*grads) and grads[0].abs().sum() > 0


def test_fused_layers_under_a_trace(dev, monkeypatch):
    """The custom ops a trace records give what the layers give, and keep their fake shapes."""
    from cuda_tempiler_b200 import bind
    from torch.fx.experimental.proxy_tensor import make_fx
    monkeypatch.setenv("TEMPO_KERNELS", "1")
    x, res, bias = rand(6, 512, seed=1), rand(6, 272, seed=2), rand(272, seed=3)
    for kind, group in (("fp16", 0), ("int8", 0), ("uint8", 64)):
        w = weights(kind, 272, 512, group)

        def f(x, res):
            if kind == "fp16":
                return bind.linear_fp16(x, w[0], bias, activation="silu", residual=res)
            return bind.linear_w8a16(x, *w, group, bias, activation="silu", residual=res)
        y = f(x, res)
        for mode in ("real", "fake"):
            bind.route_counts(reset=True)
            traced = make_fx(f, tracing_mode=mode, _allow_non_fake_inputs=True)(x, res)
            assert bind.route_counts()["tempo"] >= 1
            assert any("epilogue" in str(n.target) for n in traced.graph.nodes)
            assert torch.equal(traced(x, res), y)
    args = (x, weights("fp16", 272, 512, 0)[0], bias, "relu", res)
    torch.library.opcheck(torch.ops.tempo.gemm_fp16_epilogue, args)
    W, s, z = weights("uint8", 272, 512, 64)
    torch.library.opcheck(torch.ops.tempo.gemm_w8a16_epilogue, (x, W, s, z, 64, None, "none", res))


@pytest.mark.parametrize("M", [3, 40])
def test_scales_laid_out_as_for_the_plain_gemm(dev, monkeypatch, M):
    """Scales and zero points with other values between theirs, taken as gemm_w8a16 takes them."""
    from cuda_tempiler_b200 import bind, ops
    monkeypatch.setenv("TEMPO_KERNELS", "1")
    A = rand(M, 512, seed=1)
    for kind, group in (("int8", 0), ("uint8", 64)):
        W, s, z = weights(kind, 272, 512, group)
        want = ops.gemm_w8a16_epilogue(A, W, s, z, group, activation="relu")
        wide = torch.stack([s, s], -1).flatten(-2)[..., ::2]
        zt = None if z is None else z.t().contiguous().t()
        assert not wide.is_contiguous()
        assert torch.equal(ops.gemm_w8a16_epilogue(A, W, wide, zt, group, activation="relu"), want)
        bind.route_counts(reset=True)
        assert torch.equal(bind.linear_w8a16(A, W, wide, zt, group, activation="relu"), want)
        assert bind.route_counts()["tempo"] == 1
        # types that only the stock path takes, and a bias that broadcasts
        bias = rand(1, seed=3)
        y = bind.linear_w8a16(A, W, s.float(), z, group, bias, activation="relu")
        assert bind.route_counts()["fallback"] == 1
        monkeypatch.setenv("TEMPO_KERNELS", "0")
        assert torch.equal(y, bind.linear_w8a16(A, W, s.float(), z, group, bias, activation="relu"))
        monkeypatch.setenv("TEMPO_KERNELS", "1")


@pytest.mark.parametrize("M", [4, 40, 500])
def test_columns_of_one_buffer(dev, M):
    """Activations, residual and output side by side in one buffer."""
    from cuda_tempiler_b200 import ops
    K, N = 256, 128
    buf, W = rand(M, K + 2 * N, seed=1), rand(N, K, seed=2, scale=1 / 16)
    A, res, out = buf[:, :K], buf[:, K:K + N], buf[:, K + N:]
    keep = buf.clone()
    want = ops.gemm_fp16_epilogue(A, W, residual=res)
    assert ops.gemm_fp16_epilogue(A, W, residual=res, out=out) is out
    assert torch.equal(out, want) and torch.equal(buf[:, :K + N], keep[:, :K + N])
    with pytest.raises(ValueError, match="overlaps A"):
        ops.gemm_fp16_epilogue(A, W, out=buf[:, K - 8:K - 8 + N])


@pytest.mark.parametrize("which", ["fp16 epilogue", "int8 epilogue", "plain fp16", "plain int8"])
def test_first_call_of_a_host_thread(dev, which):
    """A thread that has made no CUDA call yet: nothing is current in it."""
    import threading

    from cuda_tempiler_b200 import _lib
    lib = _lib.load()
    M, N, K = 40, 272, 64
    kind = which.split()[0] if "epilogue" in which else which.split()[1]
    A, w = rand(M, K, seed=1), weights(kind, N, K, 0)
    out = poison(M, N)
    st = torch.cuda.current_stream().cuda_stream
    a, b, c = A.data_ptr(), w[0].data_ptr(), out.data_ptr()
    s = None if w[1] is None else w[1].data_ptr()
    torch.cuda.synchronize()
    rc = []

    def work():
        if which == "fp16 epilogue":
            rc.append(lib.tempo_sm100_gemm_fp16_epilogue(a, b, c, None, None, M, N, K, K, K, N, N, 0,
                                                         None, 0, st))
        elif which == "int8 epilogue":
            rc.append(lib.tempo_sm100_gemm_w8a16_epilogue(a, b, s, None, c, None, None, M, N, K, K,
                                                          K, N, N, 1, 0, 0, None, 0, st))
        elif which == "plain fp16":
            rc.append(lib.tempo_sm100_gemm_fp16(a, b, c, M, N, K, K, K, N, None, 0, st))
        else:
            rc.append(lib.tempo_sm100_gemm_w8a16(a, b, s, None, c, M, N, K, K, K, N, 1, 0, None, 0,
                                                 st))

    t = threading.Thread(target=work)
    t.start()
    t.join()
    assert rc == [0]
    torch.cuda.synchronize()
    check(out, A, w, 0, None, "none", None) if "epilogue" in which else None
    assert torch.isfinite(out).all()


def test_threads_on_one_stream(dev):
    """Calls of several host threads on the same stream: the launches of one call and the workspace
    they share stay together."""
    import threading
    shapes = [("fp16", 0, 90, 784, 4096), ("int8", 0, 200, 528, 4096), ("uint8", 128, 300, 528, 4096)]
    jobs = []
    for i, (kind, group, M, N, K) in enumerate(shapes):
        A, w, res = rand(M, K, seed=i), weights(kind, N, K, group, seed=i), rand(M, N, seed=9 + i)
        jobs.append((A, w, group, res, call(A, w, group, residual=res)))
    bad = []

    def work(i):
        A, w, group, res, want = jobs[i]
        try:
            for _ in range(400):
                if not torch.equal(call(A, w, group, residual=res), want):
                    bad.append(i)
        except Exception as e:
            bad.append(e)

    ts = [threading.Thread(target=work, args=(i % len(jobs),)) for i in range(6)]
    for t in ts:
        t.start()
    for t in ts:
        t.join()
    torch.cuda.synchronize()
    assert not bad, (len(bad), bad[:3])


@pytest.mark.parametrize("M", [4, 16, 64, 512])
def test_tails_of_the_activations(dev, M):
    """Small outputs of large negative arguments.  Relative to the value: the rounding to fp16, 2^-11;
    of the exponential 2 + 1.2 |y| units of 2^-23 at the most, with y = -x (silu, -11 < x), -2 u
    (gelu_tanh, u > -8) or -x^2 / 2 (gelu, -5.7 < x), each up to 16, before the result is below half
    of fp16's smallest value: 22 units, 2^-18.5; as much for the tail's fit; argument and quotient
    less than 8 units: 2^-17 covers them."""
    from cuda_tempiler_b200 import ops
    N, K = 512, 64
    A = torch.zeros(M, K, dtype=torch.float16, device="cuda")
    A[:, 0] = 1.0
    B = torch.zeros(N, K, dtype=torch.float16, device="cuda")
    B[:, 0] = torch.linspace(-9, 9, N, device="cuda").half()
    x = B[:, 0].double()
    for act in L.ACT:
        y = ops.gemm_fp16_epilogue(A, B, activation=act).double()
        if act == "gelu_tanh":  # without the cancellation of 1 + tanh
            ref = x * torch.sigmoid(2 * (2 / torch.pi) ** 0.5 * (x + 0.044715 * x ** 3))
        else:
            ref = L.act(x, act)
        tol = (L.U16 + 2.0 ** -17) * ref.abs() + 2.0 ** -25
        bad = (y - ref).abs() > tol
        assert not bad.any(), (act, int(bad.sum()), float(((y - ref).abs() / tol).max()))
