"""PyTorch-facing wrappers of the sm_100a kernels (device memory and streams come from torch;
the arithmetic runs only in ``libtempo_sm100.so``).

``gemm_fp16(A, B)`` computes ``A @ B.T`` for A [M,K], B [N,K] fp16 (the reference's k/k/n op,
kernels/shipped/gemm_fp16/sm_70/launch.cuh:20-26).  ``gemm_w8a16`` takes an 8-bit weight
[N,K] with per-channel or group-wise scales.  A problem the dispatcher does not cover raises
``NotCovered``; nothing falls back silently.
"""
from __future__ import annotations

import contextlib
import ctypes as C

import torch

from . import _lib
from ._lib import NotCovered, W8_INT8_PER_CHANNEL, W8_UINT8_GROUP  # noqa: F401

_ws_cache: dict = {}
# the W8A16 prefill's fp16 weight copy starts after the workspace's 64 KiB counter prefix
EXPAND_OFFSET = 65536
# a product with an epilogue of at most so many rows and columns streams its weights: no workspace
STREAM_MAX_M, STREAM_MAX_N = 16, 4096


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _stream(dev: torch.device) -> int:
    # the handle alone: building a Stream object takes 2 us, as long as a small kernel
    return torch._C._cuda_getCurrentRawStream(
        torch.cuda.current_device() if dev.index is None else dev.index)


def workspace(dev: torch.device, nbytes: int) -> torch.Tensor | None:
    """A zero-filled split-K workspace for (device, current stream), grown on demand.
    The kernels leave it zero-filled after every launch."""
    if nbytes <= 0:
        return None
    key = (dev.index, _stream(dev))
    ws = _ws_cache.get(key)
    if ws is None or ws.numel() < nbytes:
        ws = torch.zeros(max(nbytes, 1 << 20), dtype=torch.uint8, device=dev)
        _ws_cache[key] = ws
    return ws


def _check_2d(t: torch.Tensor, name: str, dtype) -> None:
    if t.dim() != 2 or t.dtype != dtype or not t.is_cuda or t.stride(1) != 1:
        raise ValueError(f"{name}: expected a row-major 2-D {dtype} CUDA tensor, got "
                         f"{tuple(t.shape)} {t.dtype} stride {t.stride()} on {t.device}")


def gemm_fp16(A: torch.Tensor, B: torch.Tensor, out: torch.Tensor | None = None,
              use_workspace: bool = True) -> torch.Tensor:
    lib = _lib.load()
    _check_2d(A, "A", torch.float16)
    _check_2d(B, "B", torch.float16)
    M, K = A.shape
    N = B.shape[0]
    if B.shape[1] != K:
        raise ValueError(f"K mismatch: A {tuple(A.shape)} B {tuple(B.shape)}")
    if out is None:
        out = torch.empty((M, N), dtype=torch.float16, device=A.device)
    _check_2d(out, "C", torch.float16)
    nb = lib.tempo_sm100_workspace_bytes(M, N, K, 0) if use_workspace else 0
    ws = workspace(A.device, nb)
    rc = lib.tempo_sm100_gemm_fp16(
        _ptr(A), _ptr(B), _ptr(out), M, N, K, A.stride(0), B.stride(0), out.stride(0),
        _ptr(ws), 0 if ws is None else ws.numel(), _stream(A.device))
    _lib.check(rc, "tempo_sm100_gemm_fp16")
    return out


def gemm_w8a16(A: torch.Tensor, W: torch.Tensor, scale: torch.Tensor,
               zero: torch.Tensor | None = None, group_size: int = 0,
               out: torch.Tensor | None = None, use_workspace: bool = True) -> torch.Tensor:
    """kind: int8 W with scale [N] -> per-channel symmetric; uint8 W with scale/zero
    [K/group_size, N] (GPTQ orientation) -> group-wise asymmetric."""
    lib = _lib.load()
    _check_2d(A, "A", torch.float16)
    M, K = A.shape
    N = W.shape[0]
    if W.dtype == torch.int8:
        kind = W8_INT8_PER_CHANNEL
        _check_2d(W, "W", torch.int8)
    elif W.dtype == torch.uint8:
        kind = W8_UINT8_GROUP
        _check_2d(W, "W", torch.uint8)
        if zero is None or group_size <= 0:
            raise ValueError("uint8 group-wise weights need zero and group_size")
    else:
        raise ValueError(f"W dtype {W.dtype}: expected int8 or uint8")
    if out is None:
        out = torch.empty((M, N), dtype=torch.float16, device=A.device)
    nb = lib.tempo_sm100_workspace_bytes(M, N, K, kind) if use_workspace else 0
    ws = workspace(A.device, nb)
    rc = lib.tempo_sm100_gemm_w8a16(
        _ptr(A), _ptr(W), _ptr(scale.contiguous()), _ptr(zero.contiguous() if zero is not None else None),
        _ptr(out), M, N, K, A.stride(0), W.stride(0), out.stride(0), kind, group_size,
        _ptr(ws), 0 if ws is None else ws.numel(), _stream(A.device))
    _lib.check(rc, "tempo_sm100_gemm_w8a16")
    return out


def gemm_hyperform(A: torch.Tensor, W: torch.Tensor, *, bn: int, swap: bool, splits: int = 1,
                   group_m: int = 8, max_ctas: int = 0, cta_group: int = 1,
                   scale: torch.Tensor | None = None,
                   zero: torch.Tensor | None = None, group_size: int = 0,
                   out: torch.Tensor | None = None) -> torch.Tensor:
    """Launch one explicit hyperform (search-space point) of the skeleton family; bn=0 is the
    decode GEMV (M <= 16), whose variant group_m selects: 1 CUDA-core FMAs, 2 warp tensor-core
    MMAs, anything else by M as the dispatcher does."""
    lib = _lib.load()
    M, K = A.shape
    N = W.shape[0]
    kind = 0 if W.dtype == torch.float16 else (W8_INT8_PER_CHANNEL if W.dtype == torch.int8
                                               else W8_UINT8_GROUP)
    if out is None:
        out = torch.empty((M, N), dtype=torch.float16, device=A.device)
    tiles = -(-(N if swap else M) // 128) * -(-(M if swap else N) // max(bn, 1))
    nb = 0
    if splits > 1 and cta_group == 2:
        # stream-K bound: 2 counters per tile of at most 2 waves, (3 x clusters) slot pairs
        P = torch.cuda.get_device_properties(A.device).multi_processor_count // 2
        nb = 65536 + 3 * P * 2 * 128 * bn * 4
    elif splits > 1:  # the fixed 64 KiB counter prefix, then the partials
        nb = 65536 + tiles * splits * 128 * bn * 4
    ws = workspace(A.device, nb)
    rc = lib.tempo_sm100_gemm_hyperform_cg(
        kind, _ptr(A), _ptr(W), _ptr(scale), _ptr(zero), _ptr(out), M, N, K, A.stride(0),
        W.stride(0), out.stride(0), group_size, bn, int(swap), splits, group_m, max_ctas,
        cta_group, _ptr(ws), 0 if ws is None else ws.numel(), _stream(A.device))
    _lib.check(rc, f"hyperform bn={bn} swap={swap} splits={splits}")
    return out


def naive_gemm_fp16(A: torch.Tensor, B: torch.Tensor) -> torch.Tensor:
    """The naive INPUT bar (one thread per output)."""
    lib = _lib.load()
    M, K = A.shape
    N = B.shape[0]
    out = torch.empty((M, N), dtype=torch.float16, device=A.device)
    rc = lib.tempo_sm100_naive_gemm_fp16(_ptr(A), _ptr(B), _ptr(out), M, N, K, A.stride(0),
                                         B.stride(0), out.stride(0), _stream(A.device))
    _lib.check(rc, "naive_gemm_fp16")
    return out


def naive_gemm_w8a16(A, W, scale, zero=None, group_size=0) -> torch.Tensor:
    lib = _lib.load()
    M, K = A.shape
    N = W.shape[0]
    kind = W8_INT8_PER_CHANNEL if W.dtype == torch.int8 else W8_UINT8_GROUP
    out = torch.empty((M, N), dtype=torch.float16, device=A.device)
    rc = lib.tempo_sm100_naive_gemm_w8a16(_ptr(A), _ptr(W), _ptr(scale), _ptr(zero), _ptr(out),
                                          M, N, K, A.stride(0), W.stride(0), out.stride(0), kind,
                                          group_size, _stream(A.device))
    _lib.check(rc, "naive_gemm_w8a16")
    return out


def select(kind: int, M: int, N: int, K: int, ws_bytes: int = 1 << 40) -> dict:
    lib = _lib.load()
    out = (C.c_int * 5)()
    rc = lib.tempo_sm100_select(kind, M, N, K, ws_bytes, out)
    _lib.check(rc, "select")
    return dict(bn=out[0], swap=out[1], splits=out[2], group_m=out[3], stages=out[4])


def device_status(reset: bool = True) -> list:
    lib = _lib.load()
    out = (C.c_int * 4)()
    rc = lib.tempo_sm100_device_status(out, int(reset))
    _lib.check(rc, "device_status")
    return list(out)


def silu_mul(gu: torch.Tensor, out: torch.Tensor | None = None, block: int = 0) -> torch.Tensor:
    """SwiGLU step: gu [M, 2I] holds [gate | up] (block 0) or gate and up alternating in blocks
    of `block` columns; returns silu(gate) * up as [M, I] fp16."""
    lib = _lib.load()
    _check_2d(gu, "gu", torch.float16)
    M, I2 = gu.shape
    I = I2 // 2
    if out is None:
        out = torch.empty((M, I), dtype=torch.float16, device=gu.device)
    rc = lib.tempo_sm100_silu_mul(_ptr(gu), _ptr(out), M, I, gu.stride(0), out.stride(0), block,
                                  _stream(gu.device))
    _lib.check(rc, "tempo_sm100_silu_mul")
    return out


def gemm_fp16_swiglu(A: torch.Tensor, W: torch.Tensor,
                     out: torch.Tensor | None = None) -> torch.Tensor:
    """silu(A Wg^T) * (A Wu^T) with gate/up rows of W interleaved in blocks of 64 (see
    ``tp.interleave_rows``); raises NotCovered for M <= 256."""
    lib = _lib.load()
    _check_2d(A, "A", torch.float16)
    _check_2d(W, "W", torch.float16)
    M, K = A.shape
    N = W.shape[0]
    if out is None:
        out = torch.empty((M, N // 2), dtype=torch.float16, device=A.device)
    rc = lib.tempo_sm100_gemm_fp16_swiglu(_ptr(A), _ptr(W), _ptr(out), M, N, K, A.stride(0),
                                          W.stride(0), out.stride(0), _stream(A.device))
    _lib.check(rc, "tempo_sm100_gemm_fp16_swiglu")
    return out


def gemm_w8a16_swiglu(A: torch.Tensor, W: torch.Tensor, scale: torch.Tensor,
                      zero: torch.Tensor | None = None, group_size: int = 0,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """The W8A16 form of ``gemm_fp16_swiglu`` (rows, scales and zero points interleaved alike);
    raises NotCovered below M = 512."""
    lib = _lib.load()
    _check_2d(A, "A", torch.float16)
    M, K = A.shape
    N = W.shape[0]
    kind = W8_INT8_PER_CHANNEL if W.dtype == torch.int8 else W8_UINT8_GROUP
    if out is None:
        out = torch.empty((M, N // 2), dtype=torch.float16, device=A.device)
    ws = workspace(A.device, EXPAND_OFFSET + N * K * 2)
    rc = lib.tempo_sm100_gemm_w8a16_swiglu(
        _ptr(A), _ptr(W), _ptr(scale.contiguous()),
        _ptr(zero.contiguous() if zero is not None else None), _ptr(out), M, N, K, A.stride(0),
        W.stride(0), out.stride(0), kind, group_size, _ptr(ws), 0 if ws is None else ws.numel(),
        _stream(A.device))
    _lib.check(rc, "tempo_sm100_gemm_w8a16_swiglu")
    return out


# ------------------------------------------------------------------------------ fused epilogue
ACTIVATIONS = {None: 0, "none": 0, "relu": 1, "silu": 2, "gelu": 3, "gelu_tanh": 4}
COUNTER_BYTES = 65536  # the workspace's arrival counters, which have to start at zero
MOE_MAX_TOKENS = 32


def _on(dev: torch.device):
    """Launches go to the tensors' device, whichever is current."""
    if dev.index == torch.cuda.current_device():
        return contextlib.nullcontext()
    return torch.cuda.device(dev)


def _rows(t: torch.Tensor, name: str, dtype=torch.float16) -> int:
    """``_check_2d``, and the row stride."""
    st = t.stride()
    if len(st) != 2 or st[1] != 1 or t.dtype is not dtype or not t.is_cuda:
        _check_2d(t, name, dtype)
    return st[0]


def _check_same_device(dev: torch.device, **tensors) -> None:
    for name, t in tensors.items():
        if t is not None and t.get_device() != dev.index:
            raise ValueError(f"{name}: on {t.device}, the activations on {dev}")


def _call_workspace(dev: torch.device, nbytes: int) -> torch.Tensor | None:
    """The cached workspace of the current stream, or under graph capture one of the graph's own:
    two graphs captured on one stream may replay side by side on others."""
    if nbytes <= 0:
        return None
    if not torch.cuda.is_current_stream_capturing():
        return workspace(dev, nbytes)
    ws = torch.empty(nbytes, dtype=torch.uint8, device=dev)
    ws[:min(nbytes, COUNTER_BYTES)].zero_()
    return ws


def _check_out(out: torch.Tensor | None, M: int, N: int, dev, name: str) -> torch.Tensor:
    if out is None:
        return torch.empty((M, N), dtype=torch.float16, device=dev)
    _check_2d(out, name, torch.float16)
    if out.shape != (M, N):
        raise ValueError(f"{name}: expected ({M}, {N}), got {tuple(out.shape)}")
    return out


def _span(t: torch.Tensor) -> tuple:
    a = t.data_ptr()
    return a, a + (sum((n - 1) * s for n, s in zip(t.shape, t.stride())) + 1) * t.element_size()


def _interleaved(a: torch.Tensor, b: torch.Tensor) -> bool:
    """Column ranges of one buffer: rows at the same distance whose bytes do not meet."""
    if a.dim() != 2 or b.dim() != 2 or a.stride(1) != 1 or b.stride(1) != 1:
        return False
    (ea, eb), ld = (a.element_size(), b.element_size()), a.stride(0) * a.element_size()
    if ld <= 0 or ld != b.stride(0) * eb:
        return False
    d = (b.data_ptr() - a.data_ptr()) % ld
    return a.shape[1] * ea <= d and d + b.shape[1] * eb <= ld


def _check_alias(out: torch.Tensor, residual: torch.Tensor | None, **inputs) -> None:
    """out may be the residual itself; any other overlap would be read after it is written."""
    lo, hi = _span(out)
    for name, t in dict(inputs, residual=residual).items():
        if t is None:
            continue
        a, b = _span(t)
        if a < hi and lo < b and not _interleaved(out, t):
            if name == "residual" and a == lo and t.stride() == out.stride():
                continue
            raise ValueError(f"out overlaps {name}")


def _epilogue_args(N: int, M: int, bias, activation, residual):
    if activation not in ACTIVATIONS:
        raise ValueError(f"activation {activation!r}: expected one of "
                         f"{sorted(a for a in ACTIVATIONS if a)}")
    if bias is not None and (bias.dtype is not torch.float16 or bias.shape != (N,)
                             or bias.stride(0) != 1 and N > 1):
        raise ValueError(f"bias: expected a contiguous float16 ({N},), got {tuple(bias.shape)} "
                         f"{bias.dtype} stride {bias.stride()}")
    if residual is None:
        return ACTIVATIONS[activation], 0
    ldr = _rows(residual, "residual")
    if residual.shape != (M, N):
        raise ValueError(f"residual: expected ({M}, {N}), got {tuple(residual.shape)}")
    return ACTIVATIONS[activation], ldr


def gemm_fp16_epilogue(A: torch.Tensor, B: torch.Tensor, bias: torch.Tensor | None = None,
                       activation: str | None = None, residual: torch.Tensor | None = None,
                       out: torch.Tensor | None = None) -> torch.Tensor:
    """``act(A @ B.T + bias) + residual`` in one kernel, the epilogue in fp32 before the single
    rounding to fp16.  activation: None / "none", "relu", "silu", "gelu" (exact) or "gelu_tanh".
    ``out`` may be ``residual``.  Shapes and strides as ``gemm_fp16``; bias and residual 16-byte
    aligned."""
    lib = _lib.load()
    lda, ldb = _rows(A, "A"), _rows(B, "B")
    M, K = A.shape
    N, k = B.shape
    if k != K:
        raise ValueError(f"K mismatch: A {tuple(A.shape)} B {tuple(B.shape)}")
    act, ldr = _epilogue_args(N, M, bias, activation, residual)
    dev = A.device
    _check_same_device(dev, B=B, bias=bias, residual=residual, out=out)
    if dev.index != torch.cuda.current_device():  # launches go to the tensors' device
        with torch.cuda.device(dev):
            return gemm_fp16_epilogue(A, B, bias, activation, residual, out)
    if out is None:
        out, ldc = A.new_empty((M, N)), N
    else:
        _check_out(out, M, N, dev, "out")
        _check_alias(out, residual, A=A, B=B, bias=bias)
        ldc = out.stride(0)
    ws, ws_bytes = None, 0
    if M > STREAM_MAX_M or N > STREAM_MAX_N:
        ws = _call_workspace(dev, lib.tempo_sm100_epilogue_workspace_bytes(M, N, K, 0))
        ws_bytes = 0 if ws is None else ws.numel()
    rc = lib.tempo_sm100_gemm_fp16_epilogue(
        A.data_ptr(), B.data_ptr(), out.data_ptr(), _ptr(bias), _ptr(residual), M, N, K, lda, ldb,
        ldc, ldr, act, _ptr(ws), ws_bytes, _stream(dev))
    if rc:
        _lib.check(rc, "tempo_sm100_gemm_fp16_epilogue")
    return out


def _check_scales(name: str, lead: tuple, rows: int, K: int, kind: int, group: int, scale, zero):
    """Scales of a [*lead, rows, K] weight: int8 [*lead, rows], uint8 [*lead, K/group, rows]."""
    if kind == W8_UINT8_GROUP:
        if zero is None or scale is None or group <= 0 or K % group:
            raise ValueError(f"{name}: uint8 group-wise weights need scale, zero and a group_size "
                             f"that divides {K}")
        want = (*lead, K // group, rows)
        if zero.dtype is not torch.uint8 or zero.shape != want or not zero.is_contiguous():
            raise ValueError(f"{name} zero: expected a contiguous uint8 {want}, got "
                             f"{tuple(zero.shape)} {zero.dtype}")
    else:
        want = (*lead, rows)
    if scale is None or scale.dtype is not torch.float16 or scale.shape != want \
            or not scale.is_contiguous():
        raise ValueError(f"{name} scale: expected a contiguous float16 {want}, got "
                         f"{None if scale is None else (tuple(scale.shape), scale.dtype)}")


def gemm_w8a16_epilogue(A: torch.Tensor, W: torch.Tensor, scale: torch.Tensor,
                        zero: torch.Tensor | None = None, group_size: int = 0,
                        bias: torch.Tensor | None = None, activation: str | None = None,
                        residual: torch.Tensor | None = None,
                        out: torch.Tensor | None = None) -> torch.Tensor:
    """``gemm_fp16_epilogue`` with an 8-bit weight (kinds and layouts as ``gemm_w8a16``)."""
    lib = _lib.load()
    if W.dtype not in (torch.int8, torch.uint8):
        raise ValueError(f"W dtype {W.dtype}: expected int8 or uint8")
    kind = W8_INT8_PER_CHANNEL if W.dtype == torch.int8 else W8_UINT8_GROUP
    lda, ldw = _rows(A, "A"), _rows(W, "W", W.dtype)
    M, K = A.shape
    N, k = W.shape
    if k != K:
        raise ValueError(f"K mismatch: A {tuple(A.shape)} W {tuple(W.shape)}")
    scale, zero = (None if t is None else t.contiguous() for t in (scale, zero))
    _check_scales("W", (), N, K, kind, group_size, scale, zero)
    act, ldr = _epilogue_args(N, M, bias, activation, residual)
    dev = A.device
    _check_same_device(dev, W=W, scale=scale, zero=zero, bias=bias, residual=residual, out=out)
    if dev.index != torch.cuda.current_device():
        with torch.cuda.device(dev):
            return gemm_w8a16_epilogue(A, W, scale, zero, group_size, bias, activation, residual,
                                       out)
    if out is None:
        out, ldc = A.new_empty((M, N)), N
    else:
        _check_out(out, M, N, dev, "out")
        _check_alias(out, residual, A=A, W=W, scale=scale, zero=zero, bias=bias)
        ldc = out.stride(0)
    ws, ws_bytes = None, 0
    if M > STREAM_MAX_M or N > STREAM_MAX_N:
        ws = _call_workspace(dev, lib.tempo_sm100_epilogue_workspace_bytes(M, N, K, kind))
        ws_bytes = 0 if ws is None else ws.numel()
    rc = lib.tempo_sm100_gemm_w8a16_epilogue(
        A.data_ptr(), W.data_ptr(), scale.data_ptr(), _ptr(zero), out.data_ptr(), _ptr(bias),
        _ptr(residual), M, N, K, lda, ldw, ldc, ldr, kind, group_size, act, _ptr(ws), ws_bytes,
        _stream(dev))
    if rc:
        _lib.check(rc, "tempo_sm100_gemm_w8a16_epilogue")
    return out


# ------------------------------------------------------------------------------ experts
def _check_router(x, w_router, top_k, bias):
    ldx, ldw = _rows(x, "x"), _rows(w_router, "w_router")
    E, H = w_router.shape
    if x.shape[1] != H:
        raise ValueError(f"hidden size mismatch: x {tuple(x.shape)} w_router {tuple(w_router.shape)}")
    if not 1 <= top_k <= E:
        raise ValueError(f"top_k {top_k}: expected 1 .. {E}")
    if bias is not None and (bias.dtype is not torch.float16 or bias.shape != (E,)
                             or not bias.is_contiguous()):
        raise ValueError(f"bias: expected a contiguous float16 ({E},), got {tuple(bias.shape)} "
                         f"{bias.dtype}")
    _check_same_device(x.device, w_router=w_router, bias=bias)
    return E, H, ldx, ldw


def moe_route(x: torch.Tensor, w_router: torch.Tensor, top_k: int, normalize: bool = True,
              bias: torch.Tensor | None = None) -> tuple:
    """Expert choice of each token: ``logits = x @ w_router.T + bias`` in fp32, the ``top_k``
    largest in descending order (equal logits: the lower expert first).  Returns ids [T, top_k]
    int32 and weights [T, top_k] fp32: the softmax over the chosen logits (normalize), or over all
    of them.  Any number of tokens; up to 512 experts, top_k <= 16."""
    lib = _lib.load()
    E, H, ldx, ldw = _check_router(x, w_router, top_k, bias)
    T, dev = x.shape[0], x.device
    with _on(dev):
        ids = x.new_empty((T, top_k), dtype=torch.int32)
        weights = x.new_empty((T, top_k), dtype=torch.float32)
        if T == 0:
            return ids, weights
        rc = lib.tempo_sm100_moe_route(
            x.data_ptr(), w_router.data_ptr(), _ptr(bias), ids.data_ptr(), weights.data_ptr(), T,
            E, H, top_k, ldx, ldw, int(normalize), _stream(dev))
    _lib.check(rc, "tempo_sm100_moe_route")
    return ids, weights


EXPERT_KINDS = {torch.float16: 0, torch.int8: W8_INT8_PER_CHANNEL, torch.uint8: W8_UINT8_GROUP}


def _check_experts(x, w_gate_up, w_down, s_gate_up, z_gate_up, s_down, z_down, group_size,
                   gu_block, residual, out):
    _check_2d(x, "x", torch.float16)
    T, H = x.shape
    dt = w_gate_up.dtype
    kind = EXPERT_KINDS.get(dt)
    if kind is None or w_down.dtype is not dt:
        raise ValueError(f"expert weights: float16, int8 or uint8, both alike, got {dt} and "
                         f"{w_down.dtype}")
    if w_gate_up.dim() != 3 or w_down.dim() != 3 or not w_gate_up.is_contiguous() \
            or not w_down.is_contiguous():
        raise ValueError("expert weights: expected contiguous [E, 2I, H] and [E, H, I]")
    E, I2, k = w_gate_up.shape
    I = I2 // 2
    if I2 % 2 or k != H or w_down.shape != (E, H, I):
        raise ValueError(f"expert weights: [E, 2I, H] and [E, H, I] with H = {H}, got "
                         f"{tuple(w_gate_up.shape)} and {tuple(w_down.shape)}")
    if kind:
        _check_scales("gate_up", (E,), I2, H, kind, group_size, s_gate_up, z_gate_up)
        _check_scales("down", (E,), H, I, kind, group_size, s_down, z_down)
    if gu_block < 0 or gu_block and (gu_block % 8 or I % gu_block):
        raise ValueError(f"gu_block {gu_block}: a multiple of 8 that divides {I}, or 0")
    ldr = 0
    if residual is not None:
        ldr = _rows(residual, "residual")
        if residual.shape != (T, H):
            raise ValueError(f"residual: expected ({T}, {H}), got {tuple(residual.shape)}")
    _check_same_device(x.device, w_gate_up=w_gate_up, w_down=w_down, s_gate_up=s_gate_up,
                       z_gate_up=z_gate_up, s_down=s_down, z_down=z_down, residual=residual,
                       out=out)
    if out is not None:
        _check_out(out, T, H, x.device, "out")
        _check_alias(out, residual, x=x, w_gate_up=w_gate_up, w_down=w_down, s_gate_up=s_gate_up,
                     z_gate_up=z_gate_up, s_down=s_down, z_down=z_down)
    return T, H, E, I, kind, ldr


def moe_layer(x: torch.Tensor, w_router: torch.Tensor, w_gate_up: torch.Tensor,
              w_down: torch.Tensor, top_k: int, normalize: bool = True,
              bias: torch.Tensor | None = None, s_gate_up: torch.Tensor | None = None,
              z_gate_up: torch.Tensor | None = None, s_down: torch.Tensor | None = None,
              z_down: torch.Tensor | None = None, group_size: int = 0, gu_block: int = 0,
              residual: torch.Tensor | None = None, out: torch.Tensor | None = None,
              return_routing: bool = False):
    """A whole mixture-of-experts layer for up to 32 tokens x [T, H] (NotCovered above):
    routing as ``moe_route``, then ``residual + sum_j w_j down_j(silu(gate_j(x)) * up_j(x))``
    over each token's experts.  w_gate_up [E, 2I, H] holds gate rows then up rows (gu_block 0) or
    alternates them in blocks of gu_block; w_down [E, H, I].  fp16, int8 with a scale per output
    channel (s_gate_up [E, 2I], s_down [E, H]) or uint8 with scale and zero point per group
    ([E, H / group_size, 2I], [E, I / group_size, H]), both 4-byte aligned (else NotCovered).
    ``out`` may be ``residual``.  Returns y, or
    (y, ids, weights) with return_routing."""
    lib = _lib.load()
    T, H, E, I, kind, ldr = _check_experts(x, w_gate_up, w_down, s_gate_up, z_gate_up, s_down,
                                           z_down, group_size, gu_block, residual, out)
    n_routed, _, ldx, ldw = _check_router(x, w_router, top_k, bias)
    if n_routed != E:
        raise ValueError(f"w_router names {w_router.shape[0]} experts, w_gate_up {E}")
    dev = x.device
    with _on(dev):
        if out is None:
            out = x.new_empty((T, H))
        ids = x.new_empty((T, top_k), dtype=torch.int32)
        weights = x.new_empty((T, top_k), dtype=torch.float32)
        if T:
            # a call's own workspace: nothing in it outlives the call or has to be cleared
            ws = x.new_empty(lib.tempo_sm100_moe_workspace_bytes(T, top_k, I), dtype=torch.uint8)
            rc = lib.tempo_sm100_moe_layer(
                x.data_ptr(), w_router.data_ptr(), _ptr(bias), w_gate_up.data_ptr(),
                w_down.data_ptr(), _ptr(s_gate_up), _ptr(z_gate_up), _ptr(s_down), _ptr(z_down),
                _ptr(residual), out.data_ptr(), ids.data_ptr(), weights.data_ptr(), T, E, H, I,
                top_k, ldx, ldw, ldr, out.stride(0), kind, group_size, gu_block, int(normalize),
                ws.data_ptr(), ws.numel(), _stream(dev))
            _lib.check(rc, "tempo_sm100_moe_layer")
    return (out, ids, weights) if return_routing else out


def moe_experts(x: torch.Tensor, ids: torch.Tensor, weights: torch.Tensor,
                w_gate_up: torch.Tensor, w_down: torch.Tensor,
                s_gate_up: torch.Tensor | None = None, z_gate_up: torch.Tensor | None = None,
                s_down: torch.Tensor | None = None, z_down: torch.Tensor | None = None,
                group_size: int = 0, gu_block: int = 0, residual: torch.Tensor | None = None,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """The experts' part of ``moe_layer`` with the caller's routing: ids [T, k] int32, weights
    [T, k] fp32.  An id outside [0, E) names no expert (a token with none gets its residual, or
    zero); an expert a token names twice counts with the sum of the two weights."""
    lib = _lib.load()
    T, H, E, I, kind, ldr = _check_experts(x, w_gate_up, w_down, s_gate_up, z_gate_up, s_down,
                                           z_down, group_size, gu_block, residual, out)
    dev = x.device
    if ids.dtype != torch.int32 or ids.dim() != 2 or ids.shape[0] != T or ids.shape[1] < 1 \
            or not ids.is_contiguous():
        raise ValueError(f"ids: expected a contiguous int32 ({T}, k), got {tuple(ids.shape)} "
                         f"{ids.dtype}")
    if weights.dtype != torch.float32 or weights.shape != ids.shape \
            or not weights.is_contiguous():
        raise ValueError(f"weights: expected a contiguous float32 {tuple(ids.shape)}, got "
                         f"{tuple(weights.shape)} {weights.dtype}")
    _check_same_device(dev, ids=ids, weights=weights)
    top_k = ids.shape[1]
    with _on(dev):
        if out is None:
            out = x.new_empty((T, H))
        if T:
            ws = x.new_empty(lib.tempo_sm100_moe_workspace_bytes(T, top_k, I), dtype=torch.uint8)
            rc = lib.tempo_sm100_moe_experts(
                x.data_ptr(), ids.data_ptr(), weights.data_ptr(), w_gate_up.data_ptr(),
                w_down.data_ptr(), _ptr(s_gate_up), _ptr(z_gate_up), _ptr(s_down), _ptr(z_down),
                _ptr(residual), out.data_ptr(), T, E, H, I, top_k, x.stride(0), ldr,
                out.stride(0), kind, group_size, gu_block, ws.data_ptr(), ws.numel(), _stream(dev))
            _lib.check(rc, "tempo_sm100_moe_experts")
    return out
