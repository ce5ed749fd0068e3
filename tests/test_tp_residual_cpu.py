"""Who adds the residual of a tensor-parallel layer: once among the ranks that are summed over,
whichever way their group is given (four gloo ranks in two groups; the products are plain torch)."""
import os
import socket

import pytest
import torch
import torch.distributed as dist
import torch.multiprocessing as mp


def _port():
    s = socket.socket()
    s.bind(("127.0.0.1", 0))
    p = s.getsockname()[1]
    s.close()
    return p


class Reducer:
    """As PeerAllReduce: sums over the group it carries."""

    def __init__(self, group):
        self.group = group

    def __call__(self, y):
        dist.all_reduce(y, group=self.group)
        return y


def _gemm(x, w, s):
    return x @ w.t()


def _swiglu(gu, block):
    from cuda_tempiler_b200 import tp
    return tp.swiglu_ref(gu, block)


def _layer(x, wr, shard, k, normalize, residual):
    y = (x @ shard.w_gate_up[0].t())[:, :shard.w_down.shape[2]] @ shard.w_down[0].t()
    return y if residual is None else y + residual


def _inputs():
    g = torch.Generator().manual_seed(5)
    H, I, T = 32, 64, 3
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    return r(T, H), r(2, H), r(2, I, H), r(2, I, H), r(2, H, I), r(T, H)


def _worker(rank, port, q):
    os.environ["MASTER_ADDR"] = "127.0.0.1"
    os.environ["MASTER_PORT"] = str(port)
    dist.init_process_group("gloo", rank=rank, world_size=4)
    from cuda_tempiler_b200 import tp
    groups = [dist.new_group([0, 1]), dist.new_group([2, 3])]
    mine = groups[rank // 2]
    x, wr, wg, wu, wd, res = _inputs()
    m = tp.shard_mlp(wg[0], wu[0], wd[0], 2, rank % 2)
    e = tp.shard_moe(wg, wu, wd, 2, rank % 2)

    def opaque(y):
        dist.all_reduce(y, group=mine)
        return y

    got = {}
    for name, kw in (("carried", dict(all_reduce=Reducer(mine))), ("opaque", dict(all_reduce=opaque)),
                     ("given", dict(group=mine)),
                     ("both", dict(group=mine, all_reduce=opaque))):
        y = tp.mlp_forward(x, m, gemm=_gemm, swiglu=_swiglu, residual=res, **kw)
        z = tp.moe_forward(x, wr, e, 1, layer=_layer, residual=res, **kw)
        y0 = tp.mlp_forward(x, m, gemm=_gemm, swiglu=_swiglu, **kw)
        z0 = tp.moe_forward(x, wr, e, 1, layer=_layer, **kw)
        got[name] = [float((a - b - res).abs().max()) for a, b in ((y, y0), (z, z0))]
    # a residual that does not fit is refused by every rank, not by the one that would add it
    refused = 0
    for f in (lambda r: tp.mlp_forward(x, m, gemm=_gemm, swiglu=_swiglu, residual=r, group=mine),
              lambda r: tp.moe_forward(x, wr, e, 1, layer=_layer, residual=r, group=mine)):
        for bad in (res[:2], res[:, :16], res[0]):
            try:
                f(bad)
            except ValueError:
                refused += 1
    q.put((rank, got, refused))
    dist.destroy_process_group()


def test_the_residual_is_added_once_in_every_group():
    ctx = mp.get_context("spawn")
    q = ctx.Queue()
    port = _port()
    ps = [ctx.Process(target=_worker, args=(r, port, q)) for r in range(4)]
    for p in ps:
        p.start()
    out = [q.get(timeout=120) for _ in ps]
    for p in ps:
        p.join(timeout=120)
        assert p.exitcode == 0
    for rank, got, refused in out:
        for name, off in got.items():
            assert max(off) < 1e-4, (rank, name, off)
        assert refused == 6


def test_a_reducer_without_process_groups():
    """A callable over ranks that torch.distributed knows nothing of: every one of them is rank 0
    here, and the residual is still added once."""
    from cuda_tempiler_b200 import tp
    x, wr, wg, wu, wd, res = _inputs()
    shards = [tp.shard_moe(wg, wu, wd, 2, r) for r in range(2)]
    parts = [tp.moe_forward(x, wr, s, 1, layer=_layer, all_reduce=False) for s in shards]
    for s in shards:
        y = tp.moe_forward(x, wr, s, 1, layer=_layer, all_reduce=lambda p: parts[0] + parts[1],
                           residual=res)
        assert torch.allclose(y, parts[0] + parts[1] + res, atol=1e-5)


def test_group_wise_experts_are_refused():
    from cuda_tempiler_b200 import tp
    w, s = torch.zeros(2, 64, 64, dtype=torch.uint8), torch.ones(2, 1, 64).half()
    with pytest.raises(ValueError, match="group-wise"):
        tp.shard_moe(w, w, w, 1, 0, s, s, s)
