"""CPU checks of the epilogue GEMM, the router and the MoE layer: what the C entry points refuse
(before anything is launched), the sharding of the experts over gloo ranks, the stock path of the
linear layers, the 64-bit restatement against itself."""
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp

NOT_COVERED, BAD = 9, 1
P = 1 << 20  # a pointer that is never read: every call below is refused on the host


def lib():
    from cuda_tempiler_b200 import _lib
    return _lib.load()


def fp16_epilogue(**kw):
    a = dict(A=P, B=P, C=P, bias=P, res=P, M=4, N=64, K=64, lda=64, ldb=64, ldc=64, ldr=64, act=0,
             ws=None, ws_bytes=0)
    a.update(kw)
    return lib().tempo_sm100_gemm_fp16_epilogue(*a.values(), None)


@pytest.mark.parametrize("kw,rc", [
    (dict(A=None), NOT_COVERED), (dict(B=P + 2), NOT_COVERED), (dict(C=P + 8), NOT_COVERED),
    (dict(M=0), NOT_COVERED), (dict(N=60), NOT_COVERED), (dict(K=60), NOT_COVERED),
    (dict(lda=60), NOT_COVERED), (dict(ldc=56), NOT_COVERED), (dict(bias=P + 2), NOT_COVERED),
    (dict(res=P + 4), NOT_COVERED), (dict(ldr=56), NOT_COVERED), (dict(ldr=68), NOT_COVERED),
    (dict(act=5), BAD), (dict(act=-1), BAD), (dict(ws=P + 8, ws_bytes=1 << 20), BAD)])
def test_fp16_epilogue_refuses(kw, rc):
    assert fp16_epilogue(**kw) == rc


def w8_epilogue(**kw):
    a = dict(A=P, W=P, scale=P, zero=P, C=P, bias=None, res=None, M=4, N=64, K=128, lda=128,
             ldw=128, ldc=64, ldr=0, kind=2, group=64, act=0, ws=None, ws_bytes=0)
    a.update(kw)
    return lib().tempo_sm100_gemm_w8a16_epilogue(*a.values(), None)


@pytest.mark.parametrize("kw,rc", [
    (dict(kind=0), NOT_COVERED), (dict(kind=3), NOT_COVERED), (dict(scale=None), NOT_COVERED),
    (dict(zero=None), NOT_COVERED), (dict(group=48), NOT_COVERED), (dict(group=0), NOT_COVERED),
    (dict(K=192, lda=192, ldw=192, group=128), NOT_COVERED), (dict(ldw=120), NOT_COVERED),
    (dict(kind=1, scale=P + 2), NOT_COVERED), (dict(N=72, ldc=72), NOT_COVERED),
    (dict(act=9), BAD)])
def test_w8_epilogue_refuses(kw, rc):
    assert w8_epilogue(**kw) == rc


def route(**kw):
    a = dict(x=P, wr=P, bias=None, ids=P, w=P, T=4, E=16, H=64, k=2, ldx=64, ldw=64, norm=1)
    a.update(kw)
    import ctypes as C
    vals = [C.cast(v, C.c_void_p) if n in ("ids", "w") and v else v for n, v in a.items()]
    return lib().tempo_sm100_moe_route(*vals, None)


@pytest.mark.parametrize("kw,rc", [
    (dict(x=None), BAD), (dict(wr=None), BAD), (dict(ids=None), BAD), (dict(w=None), BAD),
    (dict(T=0), BAD), (dict(E=0), BAD), (dict(k=0), BAD), (dict(k=17), BAD),
    (dict(E=64, k=17), NOT_COVERED), (dict(E=513), NOT_COVERED), (dict(H=60), NOT_COVERED),
    (dict(ldx=56), NOT_COVERED), (dict(ldw=68), NOT_COVERED), (dict(x=P + 2), NOT_COVERED)])
def test_route_refuses(kw, rc):
    assert route(**kw) == rc


def layer(**kw):
    a = dict(x=P, wr=P, bias=None, wgu=P, wd=P, sgu=P, zgu=P, sd=P, zd=P, res=None, y=P, ids=P,
             w=P, T=4, E=16, H=128, I=128, k=2, ldx=128, ldw=128, ldr=0, ldy=128, kind=2, group=64,
             block=0, norm=1, ws=P, ws_bytes=1 << 30)
    a.update(kw)
    return lib().tempo_sm100_moe_layer(*a.values(), None)


@pytest.mark.parametrize("kw,rc", [
    (dict(T=33), NOT_COVERED), (dict(T=0), BAD), (dict(E=513), NOT_COVERED), (dict(H=136), NOT_COVERED),
    (dict(I=72, kind=0), NOT_COVERED), (dict(wgu=None), BAD), (dict(wd=P + 4), NOT_COVERED),
    (dict(sgu=None), BAD), (dict(zd=None), BAD), (dict(kind=1, sd=None), BAD), (dict(kind=3), BAD),
    (dict(group=32), NOT_COVERED), (dict(group=256), NOT_COVERED), (dict(block=12), NOT_COVERED),
    (dict(block=-8), NOT_COVERED), (dict(block=48), NOT_COVERED), (dict(ldy=120), NOT_COVERED),
    (dict(res=P, ldr=64), NOT_COVERED), (dict(ws=None), BAD), (dict(ws=P + 8), BAD),
    (dict(ws_bytes=64), BAD), (dict(k=17, E=32), NOT_COVERED)])
def test_layer_refuses(kw, rc):
    assert layer(**kw) == rc


@pytest.mark.parametrize("name", ["sgu", "zgu", "sd", "zd"])
@pytest.mark.parametrize("off", [1, 2, 3])
def test_group_scales_off_a_word_are_refused(name, off):
    """The experts read group-wise scales and zero points in 4-byte words."""
    assert layer(**{name: P + off}) == NOT_COVERED
    assert layer(**{name: P + 4, "ws": None}) == BAD  # a word's boundary passes that check
    a = dict(x=P, ids=P, w=P, wgu=P, wd=P, sgu=P, zgu=P, sd=P, zd=P, res=None, y=P, T=4, E=16,
             H=128, I=128, k=2, ldx=128, ldr=0, ldy=128, kind=2, group=64, block=0, ws=P,
             ws_bytes=1 << 30)
    a[name] += off
    assert lib().tempo_sm100_moe_experts(*a.values(), None) == NOT_COVERED


@pytest.mark.parametrize("kw", [dict(res=P + 1, ldr=128), dict(y=P + 1), dict(bias=P + 1),
                                dict(ids=P + 2), dict(w=P + 2), dict(kind=1, sgu=P + 1),
                                dict(kind=1, sd=P + 1)])
def test_elements_off_their_own_size_are_refused(kw):
    assert layer(**kw) == NOT_COVERED
    kw = {n: v for n, v in kw.items() if n in ("bias", "ids", "w")}
    assert not kw or route(**kw) == NOT_COVERED


def test_experts_refuse():
    def experts(**kw):
        a = dict(x=P, ids=P, w=P, wgu=P, wd=P, sgu=None, zgu=None, sd=None, zd=None, res=None, y=P,
                 T=4, E=16, H=128, I=128, k=2, ldx=128, ldr=0, ldy=128, kind=0, group=0, block=0,
                 ws=P, ws_bytes=1 << 30)
        a.update(kw)
        return lib().tempo_sm100_moe_experts(*a.values(), None)
    assert experts(ids=None) == BAD and experts(w=None) == BAD and experts(y=None) == BAD
    assert experts(k=17) == NOT_COVERED and experts(k=0) == BAD and experts(T=40) == NOT_COVERED


def test_moe_workspace_grows_with_the_rows():
    f = lib().tempo_sm100_moe_workspace_bytes
    assert f(0, 1, 1) == 0 and f(1, 0, 64) == 0
    base = f(1, 1, 16) - 64
    assert base % 256 == 0 and f(32, 16, 2176) == base + 32 * 16 * 2176 * 4


def test_wrappers_refuse_host_tensors():
    from cuda_tempiler_b200 import ops
    x, w = torch.zeros(2, 64).half(), torch.zeros(64, 64).half()
    e = torch.zeros(64, 128, 64).half(), torch.zeros(64, 64, 64).half()
    with pytest.raises(ValueError, match="CUDA"):
        ops.gemm_fp16_epilogue(x, w)
    with pytest.raises(ValueError, match="CUDA"):
        ops.gemm_w8a16_epilogue(x, w.to(torch.int8), w[0])
    with pytest.raises(ValueError, match="CUDA"):
        ops.moe_route(x, w, 2)
    with pytest.raises(ValueError, match="CUDA"):
        ops.moe_layer(x, w, *e, 2)
    with pytest.raises(ValueError, match="CUDA"):
        ops.moe_experts(x, torch.zeros(2, 2).int(), torch.zeros(2, 2), *e)


def test_stock_path_of_the_linear_layers():
    from cuda_tempiler_b200 import bind
    from oracle import layer_oracle as L
    g = torch.Generator().manual_seed(0)
    x = torch.randn(2, 3, 32, generator=g).half()
    w = (torch.randn(16, 32, generator=g) * 32 ** -0.5).half()
    b, r = torch.randn(16, generator=g).half(), torch.randn(2, 3, 16, generator=g).half()
    for act in L.ACT:
        y = bind.linear_fp16(x, w, b, activation=act, residual=r)
        ref, _ = L.epilogue(x.reshape(6, 32), w.double(), b, act, r.reshape(6, 16))
        # four fp16 roundings of values below 8
        assert (y.reshape(6, 16).double() - ref).abs().max() < 4 * 2.0 ** -9
    assert torch.equal(bind.linear_fp16(x, w, b), torch.nn.functional.linear(x, w, b))
    with pytest.raises(ValueError):
        bind.linear_fp16(x, w, activation="tanh", residual=r)


def test_only_tensors_that_share_bytes_overlap():
    """Against the sets of their bytes, for slices of one buffer."""
    import itertools
    from cuda_tempiler_b200 import ops
    buf = torch.zeros(6, 32, dtype=torch.float16)
    other = buf.view(torch.int8).view(6, 64)
    flat = buf.view(-1)
    slices = [buf[:, :16], buf[:, 16:], buf[:, 8:24], buf[:3, :16], buf[3:, :16], buf[2:5, 16:],
              buf[1:4], buf[:, :8], buf[:, 24:], buf[2, 8:16], flat[10:20], other[:, 20:40],
              other[:, :32], flat[:96].view(2, 48)[:, :16], buf[::2, :16], buf[1::2, :16]]

    def bytes_of(t):
        n, a = t.element_size(), t.data_ptr()
        at = torch.zeros(t.shape, dtype=torch.int64)
        for d, (size, st) in enumerate(zip(t.shape, t.stride())):
            at += (torch.arange(size) * st).view([-1 if i == d else 1 for i in range(t.dim())])
        return {a + int(x) * n + i for x in at.flatten() for i in range(n)}

    refused_apart = []
    for o, t in itertools.product(slices, slices):
        if o.dim() != 2 or o.dtype != torch.float16:
            continue
        meet = bool(bytes_of(o) & bytes_of(t))
        try:
            ops._check_alias(o, None, A=t)
            assert not meet, (o.shape, o.stride(), t.shape, t.stride())
        except ValueError:
            if not meet:
                refused_apart.append((o.stride(), t.stride()))
        same = o.data_ptr() == t.data_ptr() and o.stride() == t.stride()
        if same:
            ops._check_alias(o, t)  # the residual in place
    # column slices of the same rows are told apart; other strides may be refused
    assert all(a != b for a, b in refused_apart)


def test_whole_warps_give_up_together():
    """Where all lanes of a warp wait and then act as a warp, no lane leaves by its own wait's outcome:
    the warp votes (warp_wait, __all_sync) or the barrier group does (named_barrier_and); a lane that
    waits by itself does so under `lane == 0`."""
    import re
    from pathlib import Path

    import cuda_tempiler_b200
    text = (Path(cuda_tempiler_b200.__file__).parent / "csrc" / "swap_tile.cuh").read_text()
    kernel = text[text.index("k_epi_swap(const __grid_constant__"):text.index("k_swap_finish(const")]
    parts = re.split(r"// -{20,} (.*)\n", kernel)
    roles = dict(zip(parts[1::2], parts[2::2]))
    assert list(roles) == ["TMA", "TMA: raw weights", "MMA", "epilogue", "unpacking"]
    for name, body in roles.items():
        waits = re.findall(r"\bmbar_wait\(", body)
        if name.startswith("TMA"):
            assert body.lstrip().startswith("if (lane == 0) {") and len(waits) == 1
        elif name == "epilogue":
            assert len(waits) == 1 and "named_barrier_and(bar, 128, mbar_wait(" in body
        else:
            own = re.findall(r"ok (?:&)?= mbar_wait\(", body)
            assert len(own) == len(waits) and "ok = __all_sync(" in body.replace("if (!", "ok = ")
            # every way out of the loops is a vote's
            for line in body.splitlines():
                assert "break;" not in line or re.search(r"if \(!(warp_wait|__all_sync)\(", line)


def test_epilogue_warps_of_the_pair_tiles_give_up_together():
    """The 2-CTA tiles that the epilogue GEMM runs on: all four warps or none."""
    import re

    from cuda_tempiler_b200 import build
    text = (build.SKELETON / "kernel.cuh").read_text()
    kernel = text[text.index("    k_gemm_sm100_pair(const"):text.index("// k_gemm_sm100_pair_w8: W8A16")]
    epilogue = kernel[kernel.index("epilogue (both)"):]
    waits = re.findall(r"[^\n]*\bmbar_wait\(", epilogue)
    assert len(waits) == 1 and "named_barrier_and(1, 128, mbar_wait(" in waits[0]
    others = kernel[:kernel.index("epilogue (both)")]
    for role in re.split(r"// -{20,} ", others)[1:]:  # the producer's and the issuer's waits
        assert "mbar_wait" not in role or "lane == 0) {" in role.split("mbar_wait")[0]


# ------------------------------------------------------------------------------ sharding
def _port():
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    p = s.getsockname()[1]
    s.close()
    return p


def _inputs():
    g = torch.Generator().manual_seed(3)
    E, H, I, T = 6, 32, 48, 5
    wg, wu = torch.randn(E, I, H, generator=g), torch.randn(E, I, H, generator=g)
    wd = torch.randn(E, H, I, generator=g)
    sg, su = torch.rand(E, I, generator=g), torch.rand(E, I, generator=g)
    return (torch.randn(T, H, generator=g), torch.randn(E, H, generator=g), wg, wu, wd, sg, su,
            torch.rand(E, H, generator=g), torch.randn(T, H, generator=g))


def _layer(x, wr, sh, k, normalize, residual):
    from oracle import layer_oracle as L
    ids, w, _, _ = L.route(x, wr, k, normalize)
    y, _ = L.experts(x, ids, w, sh.w_gate_up.double() * sh.s_gate_up.double()[..., None],
                     sh.w_down.double() * sh.s_down.double()[..., None], residual)
    return y.float()


def _gemm(x, w, s):
    return (x.float() @ w.float().t()) * (1 if s is None else s.float())


def _swiglu(gu, block):
    from cuda_tempiler_b200 import tp
    return tp.swiglu_ref(gu, block)


def _worker(rank, world, port, q):
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=world)
    from cuda_tempiler_b200 import tp
    x, wr, wg, wu, wd, sg, su, sd, res = _inputs()
    sh = tp.shard_moe(wg, wu, wd, world, rank, sg, su, sd)
    y = tp.moe_forward(x, wr, sh, 3, layer=_layer, residual=res)
    m = tp.shard_mlp(wg[0], wu[0], wd[0], world, rank, sg[0], su[0], sd[0])
    z = tp.mlp_forward(x, m, gemm=_gemm, swiglu=_swiglu, residual=res)
    if rank == 0:
        q.put((y.numpy(), z.numpy()))
    dist.destroy_process_group()


@pytest.mark.parametrize("world", [2, 3])
def test_ranks_sum_to_the_whole_layer(world):
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = _port()
    ps = [ctx.Process(target=_worker, args=(r, world, port, q)) for r in range(world)]
    for p in ps:
        p.start()
    y, z = q.get(timeout=120)
    for p in ps:
        p.join(timeout=120)
        assert p.exitcode == 0
    from cuda_tempiler_b200 import tp
    x, wr, wg, wu, wd, sg, su, sd, res = _inputs()
    whole = tp.shard_moe(wg, wu, wd, 1, 0, sg, su, sd)
    assert whole.w_gate_up.shape == (6, 96, 32) and torch.equal(whole.w_gate_up[:, 48:], wu)
    ref = tp.moe_forward(x, wr, whole, 3, layer=_layer, residual=res)
    assert torch.allclose(torch.from_numpy(y), ref, rtol=1e-5, atol=1e-5 * float(ref.abs().max()))
    m = tp.shard_mlp(wg[0], wu[0], wd[0], 1, 0, sg[0], su[0], sd[0])
    ref = tp.mlp_forward(x, m, gemm=_gemm, swiglu=_swiglu, residual=res)
    bare = tp.mlp_forward(x, m, gemm=_gemm, swiglu=_swiglu)
    assert torch.allclose(ref, bare + res)
    assert torch.allclose(torch.from_numpy(z), ref, rtol=1e-5, atol=1e-5 * float(ref.abs().max()))
