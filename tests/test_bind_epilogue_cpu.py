"""The linear layers' fused path without a GPU: fake CUDA tensors go through the layers' own checks
and the custom ops' fake implementations, so which way a call goes and what it returns shows here."""
import pytest
import torch
import torch.autograd.forward_ad as fwAD
from torch._subclasses.fake_tensor import FakeTensorMode

from cuda_tempiler_b200 import bind, ops

pytestmark = pytest.mark.filterwarnings("error:Accessing the data pointer of FakeTensor")
M, N, K = 6, 48, 128


@pytest.fixture
def fake(monkeypatch):
    monkeypatch.setenv("TEMPO_KERNELS", "1")
    bind.route_counts(reset=True)
    with FakeTensorMode():
        yield


def half(*shape):
    return torch.empty(*shape, dtype=torch.float16, device="cuda")


def layer(kind, x, w, bias, res, **kw):
    """A fused linear layer of an 8-bit or fp16 weight, and how it went."""
    bind.route_counts(reset=True)
    if kind == "fp16":
        y = bind.linear_fp16(x, w[0], bias, activation="silu", residual=res)
    else:
        y = bind.linear_w8a16(x, *w, bias=bias, activation="silu", residual=res)
    return y, bind.route_counts()


def operands(kind):
    if kind == "fp16":
        w = [half(N, K)]
    elif kind == "int8":
        w = [torch.empty(N, K, dtype=torch.int8, device="cuda"), half(N), None, 0]
    else:
        w = [torch.empty(N, K, dtype=torch.uint8, device="cuda"), half(K // 64, N),
             torch.empty(K // 64, N, dtype=torch.uint8, device="cuda"), 64]
    return half(M, K), w, half(N), half(M, N)


def refuse(monkeypatch):
    """The kernels are never entered."""
    def no(*a, **k):
        raise AssertionError("the kernels have no derivatives")
    monkeypatch.setattr(ops, "gemm_fp16_epilogue", no)
    monkeypatch.setattr(ops, "gemm_w8a16_epilogue", no)


@pytest.mark.parametrize("kind", ["int8", "uint8"])
def test_a_scale_that_is_learned_keeps_its_gradient(fake, monkeypatch, kind):
    refuse(monkeypatch)
    x, w, bias, res = operands(kind)
    w[1].requires_grad_()
    y, routes = layer(kind, x, w, bias, res)
    assert routes == {"tempo": 0, "fallback": 1} and y.requires_grad


@pytest.mark.parametrize("kind", ["fp16", "int8", "uint8"])
@pytest.mark.parametrize("leaf", ["x", "scale", "bias", "residual"])
def test_forward_mode_tangents_are_kept(fake, monkeypatch, kind, leaf):
    refuse(monkeypatch)
    x, w, bias, res = operands(kind)
    if leaf == "scale" and kind == "fp16":
        leaf = "weight"
    with fwAD.dual_level():
        def dual(t):
            return fwAD.make_dual(t, torch.empty_like(t))
        x = dual(x) if leaf == "x" else x
        bias = dual(bias) if leaf == "bias" else bias
        res = dual(res) if leaf == "residual" else res
        if leaf in ("scale", "weight"):
            i = 0 if leaf == "weight" else 1
            w[i] = dual(w[i])
        with torch.no_grad():
            y, routes = layer(kind, x, w, bias, res)
        assert routes["fallback"] == 1
        assert fwAD.unpack_dual(y).tangent is not None


def test_function_transforms_take_the_stock_path(monkeypatch):
    refuse(monkeypatch)
    monkeypatch.setenv("TEMPO_KERNELS", "1")
    monkeypatch.setattr(bind, "covered_fp16", lambda x, w: True)
    x, W, res = (torch.randn(*s).half() for s in ((M, K), (N, K), (M, N)))

    def f(x):
        return bind.linear_fp16(x, W, activation="silu", residual=res)

    y, dy = torch.func.jvp(f, (x,), (torch.ones_like(x),))
    assert dy.abs().sum() > 0
    assert torch.allclose(torch.func.vmap(lambda a, r: bind.linear_fp16(
        a[None], W, activation="silu", residual=r[None])[0])(x, res), y, rtol=2.0 ** -9,
                          atol=2.0 ** -9)


@pytest.mark.parametrize("kind", ["fp16", "int8", "uint8"])
def test_fused_layers_trace_as_opaque_ops(fake, kind):
    x, w, bias, res = operands(kind)
    for b, r in ((bias, res), (None, None), (bias, None), (None, res)):
        y, routes = layer(kind, x, w, b, r)
        assert routes == {"tempo": 1, "fallback": 0}
        assert y.shape == (M, N) and y.dtype == torch.float16 and y.is_cuda


def test_fused_layers_in_a_traced_graph(monkeypatch):
    from torch.fx.experimental.proxy_tensor import make_fx
    monkeypatch.setenv("TEMPO_KERNELS", "1")
    with FakeTensorMode():
        x, w, bias, res = operands("uint8")

        def f(x, res):
            return bind.linear_w8a16(x, *w, bias=bias, activation="gelu", residual=res)
        graph = make_fx(f)(x, res).graph
    assert [n.target for n in graph.nodes if n.op == "call_function"
            and "tempo" in str(n.target)] == [torch.ops.tempo.gemm_w8a16_epilogue.default]


def test_operands_that_only_the_stock_path_takes(fake, monkeypatch):
    """A bias or a residual that broadcasts, scales of another type or layout: the layer computes
    them in either setting of the switch."""
    refuse(monkeypatch)
    monkeypatch.setattr(bind, "_op", lambda name, x: getattr(ops, name))
    x, w, bias, res = operands("fp16")
    for b, r in ((half(1), res), (half(1, N), res), (half(M, N), res), (bias, half(N)),
                 (bias, half(M, 1)), (bias, half(1, N))):
        y, routes = layer("fp16", x, w, b, r)
        assert routes["fallback"] == 1 and y.shape == (M, N)
    for kind in ("int8", "uint8"):
        x, w, bias, res = operands(kind)
        for i in (1, 2) if kind == "uint8" else (1,):
            v = list(w)
            v[i] = w[i].float()
            y, routes = layer(kind, x, v, bias, res)
            assert routes["fallback"] == 1 and y.shape == (M, N)


def test_fused_layers_under_torch_compile(monkeypatch, recwarn):
    """The counter's lock breaks the graph, as it does in a layer without an epilogue; nothing else
    does, and the value is the layer's."""
    monkeypatch.setenv("TEMPO_KERNELS", "1")
    x, W, res = (torch.randn(*s).half() for s in ((M, K), (N, K), (M, N)))
    torch._dynamo.reset()
    y = torch.compile(lambda x: bind.linear_fp16(x, W, activation="silu", residual=res),
                      backend="eager")(x)
    assert torch.equal(y, bind.linear_fp16(x, W, activation="silu", residual=res))
    assert not [w for w in recwarn if "does not know how to trace" in str(w.message)]
