"""Serving-side binding: torch custom ops over the sm_100a kernels and a gated linear layer.

The reference's host integration (kernels/shipped/gemm_fp16/sm_70/INTEGRATION.md:83-103) is
tensor -> POD -> launch(), with the framework's own path taken when the shipped dispatcher does
not cover a shape, and the whole thing behind an environment switch that is OFF by default
(``TEMPO_KERNELS=1`` turns it on).  This module is that template for PyTorch:

* ``torch.ops.tempo.gemm_fp16(A, B)`` and ``torch.ops.tempo.gemm_w8a16(A, W, scale, zero,
  group_size)``, and with a bias, an activation and a residual ``gemm_fp16_epilogue`` and
  ``gemm_w8a16_epilogue``, are strict: they run the library's kernels or raise (``NotCovered`` for
  a shape the dispatcher does not cover, RuntimeError for a CUDA error or a missing library).  They
  have fake (meta) implementations, so they trace under torch.compile / export as opaque ops.
* ``linear_fp16`` / ``linear_w8a16`` are what a model's linear layer calls.  With the switch
  off they are the framework's stock path (``F.linear`` on the dequantised weight for W8A16);
  with it on they call the custom op when ``covered()`` says the shape is shipped and fall back
  to the stock path otherwise -- the caller's fallback, never a CPU path inside this library.
* ``route_counts()`` counts which way each call went (the reference's "entry proof": prove the
  kernels are entered before trusting an end-to-end number).
"""
from __future__ import annotations

import os
import threading

import torch
import torch.autograd.forward_ad as fwAD
import torch.nn.functional as F
from torch._subclasses.fake_tensor import FakeTensor

from . import ops
from ._lib import NotCovered

_lock = threading.Lock()
_routes = {"tempo": 0, "fallback": 0}


def enabled() -> bool:
    """The switch, read on every call: ``TEMPO_KERNELS=1`` turns the kernels on (default 0)."""
    return os.environ.get("TEMPO_KERNELS", "0") == "1"


def route_counts(reset: bool = False) -> dict:
    with _lock:
        out = dict(_routes)
        if reset:
            for k in _routes:
                _routes[k] = 0
    return out


def _count(route: str) -> None:
    with _lock:
        _routes[route] += 1


# ------------------------------------------------------------------------------ custom ops
@torch.library.custom_op("tempo::gemm_fp16", mutates_args=())
def gemm_fp16(A: torch.Tensor, B: torch.Tensor) -> torch.Tensor:
    """C[M, N] = A[M, K] @ B[N, K]^T on the tcgen05 kernels (fp16, fp32 accumulate)."""
    return ops.gemm_fp16(A, B)


@gemm_fp16.register_fake
def _(A, B):
    return A.new_empty((A.shape[0], B.shape[0]))


@torch.library.custom_op("tempo::gemm_w8a16", mutates_args=())
def gemm_w8a16(A: torch.Tensor, W: torch.Tensor, scale: torch.Tensor,
               zero: torch.Tensor | None, group_size: int) -> torch.Tensor:
    """C[M, N] = A[M, K] @ dequant(W)[N, K]^T; W int8 with scale [N] (per-channel) or uint8 with
    scale / zero [K / group_size, N] (group-wise, GPTQ orientation)."""
    return ops.gemm_w8a16(A, W, scale, zero, group_size)


@gemm_w8a16.register_fake
def _(A, W, scale, zero, group_size):
    return A.new_empty((A.shape[0], W.shape[0]))


@torch.library.custom_op("tempo::gemm_fp16_epilogue", mutates_args=())
def gemm_fp16_epilogue(A: torch.Tensor, B: torch.Tensor, bias: torch.Tensor | None,
                       activation: str, residual: torch.Tensor | None) -> torch.Tensor:
    """C = act(A @ B^T + bias) + residual, one rounding (``ops.gemm_fp16_epilogue``)."""
    return ops.gemm_fp16_epilogue(A, B, bias, activation, residual)


@gemm_fp16_epilogue.register_fake
def _(A, B, bias, activation, residual):
    return A.new_empty((A.shape[0], B.shape[0]))


@torch.library.custom_op("tempo::gemm_w8a16_epilogue", mutates_args=())
def gemm_w8a16_epilogue(A: torch.Tensor, W: torch.Tensor, scale: torch.Tensor,
                        zero: torch.Tensor | None, group_size: int, bias: torch.Tensor | None,
                        activation: str, residual: torch.Tensor | None) -> torch.Tensor:
    """``tempo::gemm_fp16_epilogue`` with an 8-bit weight (kinds of ``tempo::gemm_w8a16``)."""
    return ops.gemm_w8a16_epilogue(A, W, scale, zero, group_size, bias, activation, residual)


@gemm_w8a16_epilogue.register_fake
def _(A, W, scale, zero, group_size, bias, activation, residual):
    return A.new_empty((A.shape[0], W.shape[0]))


# ------------------------------------------------------------------------------ coverage
def _aligned(t: torch.Tensor) -> bool:
    # under a trace there is no address yet: the strict op raises NotCovered if the real one is off
    return isinstance(t, FakeTensor) or t.data_ptr() % 16 == 0


def covered_fp16(x2: torch.Tensor, weight: torch.Tensor) -> bool:
    """Whether the shipped fp16 dispatcher takes this problem (the reference's applicable())."""
    if not (x2.is_cuda and weight.is_cuda and x2.dtype == weight.dtype == torch.float16):
        return False
    if x2.dim() != 2 or weight.dim() != 2 or x2.stride(1) != 1 or weight.stride(1) != 1:
        return False
    M, K = x2.shape
    N = weight.shape[0]
    if weight.shape[1] != K or M == 0:
        return False
    if K % 8 or N % 8 or x2.stride(0) % 8 or weight.stride(0) % 8:
        return False
    return _aligned(x2) and _aligned(weight)


def covered_w8a16(x2, W, scale, zero, group_size) -> bool:
    if not (x2.is_cuda and W.is_cuda and x2.dtype == torch.float16):
        return False
    if W.dtype not in (torch.int8, torch.uint8) or x2.dim() != 2 or W.dim() != 2:
        return False
    if x2.stride(1) != 1 or W.stride(1) != 1:
        return False
    M, K = x2.shape
    N = W.shape[0]
    if W.shape[1] != K or M == 0 or K % 16 or N % 8 or x2.stride(0) % 8 or W.stride(0) % 16:
        return False
    if W.dtype == torch.uint8:
        if zero is None or group_size <= 0 or group_size % 64 or K % group_size or N % 16:
            return False
    return _aligned(x2) and _aligned(W)


# ------------------------------------------------------------------------------ linear layers
def _stock_epilogue(y, activation, residual):
    """The epilogue of the stock path, on the layer's fp16 output."""
    if activation not in ops.ACTIVATIONS:
        raise ValueError(f"activation {activation!r}")
    if activation == "relu":
        y = F.relu(y)
    elif activation == "silu":
        y = F.silu(y)
    elif activation in ("gelu", "gelu_tanh"):
        y = F.gelu(y, approximate="tanh" if activation == "gelu_tanh" else "none")
    return y if residual is None else y + residual


def _differentiated(*tensors) -> bool:
    """Whether any of them takes part in reverse- or forward-mode differentiation, or in a
    function transform (torch.func): the epilogue kernels have no rules for those."""
    grad, dual = torch.is_grad_enabled(), fwAD._current_level >= 0
    wrapped = not torch.compiler.is_compiling() \
        and torch._C._functorch.peek_interpreter_stack() is not None
    if not (grad or dual or wrapped):
        return False
    return any(t is not None and (
        grad and t.requires_grad or dual and fwAD.unpack_dual(t).tangent is not None
        or wrapped and torch._C._functorch.is_functorch_wrapped_tensor(t)) for t in tensors)


def _op(name: str, x):
    """The strict function, or under a trace (fake tensors, a dispatch mode, torch.compile) its custom
    op, which costs 17 us of host time a call (19 us without, 36 with)."""
    if type(x) in (torch.Tensor, torch.nn.Parameter) and not torch._C._len_torch_dispatch_stack() \
            and not torch.compiler.is_compiling():
        return getattr(ops, name)
    return getattr(torch.ops.tempo, name)


def _fused(x, weight, bias, residual, run):
    """run(residual rows) where the epilogue kernels cover the extra operands, else None."""
    N = weight.shape[0]
    if residual is not None and residual.shape != (*x.shape[:-1], N):
        return None
    res = None if residual is None else residual.reshape(-1, N)
    if res is not None and (res.dtype != torch.float16 or res.device != x.device
                            or res.stride(1) != 1 or res.stride(0) % 8 or not _aligned(res)):
        return None
    if bias is not None and (bias.dtype != torch.float16 or bias.device != x.device
                             or bias.shape != (N,) or not bias.is_contiguous()
                             or not _aligned(bias)):
        return None
    try:
        return run(res)
    except NotCovered:
        return None


def _scales_fit(x, W, scale, zero, group_size) -> bool:
    """Whether scale and zero point have the types and shapes the kernels read."""
    N, K = W.shape
    group = W.dtype == torch.uint8
    want = (K // group_size, N) if group else (N,)
    if scale.dtype != torch.float16 or scale.shape != want or scale.device != x.device:
        return False
    return not group or (zero.dtype == torch.uint8 and zero.shape == want
                         and zero.device == x.device)


def linear_fp16(x: torch.Tensor, weight: torch.Tensor, bias: torch.Tensor | None = None,
                activation: str | None = None,
                residual: torch.Tensor | None = None) -> torch.Tensor:
    """y = act(x @ weight^T (+ bias)) (+ residual) for x [..., K], weight [N, K], residual
    [..., N].  With an activation or a residual the kernels fuse the whole epilogue
    (``ops.gemm_fp16_epilogue``), unless a derivative is asked for; a bias alone is added to the
    rounded product."""
    fuse = activation not in (None, "none") or residual is not None
    if enabled() and not (fuse and _differentiated(x, weight, bias, residual)):
        x2 = x.reshape(-1, x.shape[-1])
        if covered_fp16(x2, weight):
            N = weight.shape[0]
            if fuse:
                y = _fused(x, weight, bias, residual,
                           lambda res: _op("gemm_fp16_epilogue", x2)(
                               x2, weight, bias, activation or "none", res))
                if y is not None:
                    _count("tempo")
                    return y.reshape(*x.shape[:-1], N)
            else:
                try:
                    y = torch.ops.tempo.gemm_fp16(x2, weight)
                except NotCovered:
                    y = None
                if y is not None:
                    _count("tempo")
                    y = y.reshape(*x.shape[:-1], N)
                    return y + bias if bias is not None else y
    _count("fallback")
    return _stock_epilogue(F.linear(x, weight, bias), activation, residual)


def dequantize(W, scale, zero=None, group_size: int = 0) -> torch.Tensor:
    """The fp16 weight the W8A16 op multiplies by (the stock path's operand): q * s[n], or
    (q - z[g][n]) * s[g][n] with g = k // group_size (reference bench/gemm_baseline.py:214-231)."""
    if W.dtype == torch.int8:
        return (W.float() * scale.float()[:, None]).half()
    s = scale.float().repeat_interleave(group_size, 0).t()
    z = zero.float().repeat_interleave(group_size, 0).t()
    return ((W.float() - z) * s).half()


def linear_w8a16(x: torch.Tensor, W: torch.Tensor, scale: torch.Tensor,
                 zero: torch.Tensor | None = None, group_size: int = 0,
                 bias: torch.Tensor | None = None, activation: str | None = None,
                 residual: torch.Tensor | None = None) -> torch.Tensor:
    """``linear_fp16`` with an 8-bit weight."""
    fuse = activation not in (None, "none") or residual is not None
    if enabled() and not (fuse and _differentiated(x, W, scale, bias, residual)):
        x2 = x.reshape(-1, x.shape[-1])
        if covered_w8a16(x2, W, scale, zero, group_size):
            N = W.shape[0]
            if fuse:
                y = None
                if _scales_fit(x, W, scale, zero, group_size):
                    y = _fused(x, W, bias, residual,
                               lambda res: _op("gemm_w8a16_epilogue", x2)(
                                   x2, W, scale, zero, group_size, bias, activation or "none", res))
                if y is not None:
                    _count("tempo")
                    return y.reshape(*x.shape[:-1], N)
            else:
                try:
                    y = torch.ops.tempo.gemm_w8a16(x2, W, scale, zero, group_size)
                except NotCovered:
                    y = None
                if y is not None:
                    _count("tempo")
                    y = y.reshape(*x.shape[:-1], N)
                    return y + bias if bias is not None else y
    _count("fallback")
    return _stock_epilogue(F.linear(x, dequantize(W, scale, zero, group_size), bias), activation,
                           residual)
