"""Causal attention over a sliding window and a few first tokens (sinks), forward and backward.

Query i of q [B, H, Nq, D] is at position p = Nk - Nq + i of the keys k, v [B, Hkv, Nk, D] and
sees key j when 0 <= j <= p and (window == 0, or p - j < window, or j < sinks). H is a multiple of
Hkv: query head h reads key/value head h // (H // Hkv). A query that sees nothing gives O = 0. What is hidden
weighs 0 exactly, but infinities and NaN of v (in the gradients: of any input) reach rows of the same tile of 128.
float16 or bfloat16, D in {64, 128}; the last dim is contiguous, the other strides are multiples
of 8 elements (a [B, N, H, D] tensor's transpose(1, 2) is fine). Not in the reference, whose
attention is over all keys or all keys up to the query's own, and forward only.
"""

from __future__ import annotations

import ctypes
import math
import struct

import torch

from torch._C import _cuda_getCurrentRawStream as _raw_stream

from fa import _C

# FaWindowParams (include/fa_b200.h): 9 pointers, 8 x 3 strides, 8 ints, the scale, the dtype.
_PARAMS = struct.Struct("@9P24q8ifB3x")


_NO_GRADS = (0,) * 4
_NO_STRIDES = (0,) * 3


def _packed(block: struct.Struct, *values) -> bytes:
    """A parameter block. What its types do not hold is the caller's window or sinks: sizes of tensors that exist fit
    or are refused by the library, as is a softmax_scale that becomes infinite."""
    try:
        return block.pack(*values)
    except struct.error as e:
        raise ValueError(f"window and sinks must be 32-bit integers: {e}") from None


def _tensor_strides(t: torch.Tensor) -> tuple[int, int, int]:
    """{batch, head, row} strides; 0 for a dim of one element, whose stride means nothing."""
    s0, s1, s2, s3 = t.stride()
    if s3 != 1:
        raise RuntimeError("tensors must have a contiguous last dimension")
    n0, n1, n2, _ = t.shape
    return (s0 if n0 > 1 else 0, s1 if n1 > 1 else 0, s2 if n2 > 1 else 0)


def _check(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor) -> None:
    dtype, device = q.dtype, q.device
    for t in (q, k, v):
        if not t.is_cuda:
            raise RuntimeError("q, k, v must be CUDA tensors")
        if t.dtype not in _C.DTYPES:
            raise RuntimeError("q, k, v must be float16 (or bfloat16)")
        if t.dtype != dtype:
            raise RuntimeError("q, k, v must have the same dtype")
        if t.dim() != 4:
            raise RuntimeError("q, k, v must have shape [B, H, N, D]")
        if t.device != device:
            raise RuntimeError("q, k, v must be on the same device")
    if k.shape != v.shape or q.shape[0] != k.shape[0] or q.shape[3] != k.shape[3]:
        raise RuntimeError("q must have shape [B, H, Nq, D], k and v [B, Hkv, Nk, D]")


def _pack(q, k, v, o, lse, grads, grad_strides, window, sinks, softmax_scale) -> bytes:
    (b, h, nq, d), (_, hk, nk, _) = q.shape, k.shape
    scale = 1.0 / math.sqrt(d) if softmax_scale is None else float(softmax_scale)
    return _packed(
        _PARAMS, q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), 0 if lse is None else lse.data_ptr(), *grads,
        *_tensor_strides(q), *_tensor_strides(k), *_tensor_strides(v), *_tensor_strides(o), *grad_strides,
        b, h, hk, nq, nk, d, window, sinks, scale, _C.DTYPES[q.dtype])


def _on_device(index: int, call, *args) -> None:
    """call(*args, stream) with device `index` and its current stream; raises the library's error."""
    stream = _raw_stream(index)
    if torch.cuda.current_device() == index:
        rc = call(*args, stream)
    else:
        with torch.cuda.device(index):
            rc = call(*args, stream)
    if rc != _C.FA_OK:
        _C._raise(rc)


def _run_bwd(params: bytes, device: torch.device, stream: int) -> int:
    """fa_window_bwd with a workspace from torch."""
    nbytes = ctypes.c_uint64(0)
    rc = _C.lib.fa_window_bwd_workspace_size(params, ctypes.byref(nbytes))
    if rc == _C.FA_OK:
        ws = torch.empty(nbytes.value, dtype=torch.uint8, device=device)
        rc = _C.lib.fa_window_bwd(params, ws.data_ptr(), nbytes.value, stream)
    return rc


def forward_window(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    window: int,
    sinks: int = 0,
    softmax_scale: float | None = None,
    return_lse: bool = False,
):
    """O [B, H, Nq, D] of window attention with sinks (see the module's first lines; window 0 is no
    window: plain causal attention). return_lse: (O, LSE), LSE [B, H, Nq] float32 the natural log
    of each row's sum of exp(scale * score), -inf for a row that sees nothing. The result carries
    no gradient: window_attention does."""
    _check(q, k, v)
    o = torch.empty_like(q, memory_format=torch.contiguous_format)
    lse = o.new_empty(q.shape[:3], dtype=torch.float32) if return_lse else None
    if q.numel() > 0 and k.numel() > 0:
        params = _pack(q, k, v, o, lse, _NO_GRADS, _NO_STRIDES * 4, window, sinks, softmax_scale)
        _on_device(q.get_device(), _C.lib.fa_window_fwd, params)
    else:
        o.zero_()
        if lse is not None:
            lse.fill_(-math.inf)
    return (o, lse) if return_lse else o


def backward_window(
    do: torch.Tensor,
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    o: torch.Tensor,
    lse: torch.Tensor,
    window: int,
    sinks: int = 0,
    softmax_scale: float | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """(dQ, dK, dV) for the gradient `do` of O, from forward_window(..., return_lse=True)'s O and
    LSE and the same window, sinks and scale. dK and dV are summed over the query heads that share
    a key/value head. Bitwise deterministic: no atomics."""
    _check(q, k, v)
    for t in (do, o):
        if t.shape != q.shape or t.dtype != q.dtype or t.device != q.device:
            raise RuntimeError("do and o must be tensors like q")
    if lse.shape != q.shape[:3] or lse.dtype != torch.float32 or lse.device != q.device or not lse.is_contiguous():
        raise RuntimeError("lse must be a contiguous float32 [B, H, Nq] tensor on q's device")
    dq, dk, dv = (torch.empty_like(t, memory_format=torch.contiguous_format) for t in (q, k, v))
    if q.numel() > 0 and k.numel() > 0:
        strides = (*_tensor_strides(do), *_tensor_strides(dq), *_tensor_strides(dk), *_tensor_strides(dv))
        grads = (do.data_ptr(), dq.data_ptr(), dk.data_ptr(), dv.data_ptr())
        params = _pack(q, k, v, o, lse, grads, strides, window, sinks, softmax_scale)
        _on_device(q.get_device(), _run_bwd, params, q.device)
    else:
        for t in (dq, dk, dv):
            t.zero_()
    return dq, dk, dv


def _loadable(t: torch.Tensor) -> torch.Tensor:
    """`t` itself when the kernels can read it, else a contiguous copy (autograd hands over
    gradients of any layout, an expanded one among them)."""
    ok = t.stride(3) == 1 and t.data_ptr() % 16 == 0
    ok = ok and all(n == 1 or (s > 0 and s % 8 == 0) for s, n in zip(t.stride()[:3], t.shape[:3]))
    return t if ok else t.contiguous()


class _Once(torch.autograd.Function):
    """Gradients as they are, whose own gradient is an error (and not, silently, nothing)."""

    @staticmethod
    def forward(ctx, q, k, v, *grads):
        return tuple(g.view_as(g) for g in grads)

    @staticmethod
    def backward(ctx, *_):
        raise RuntimeError("window_attention can be differentiated once")


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sinks, softmax_scale):
        o, lse = forward_window(q, k, v, window, sinks, softmax_scale, return_lse=True)
        ctx.save_for_backward(q, k, v, o, lse)
        ctx.how = (window, sinks, softmax_scale)
        return o

    @staticmethod
    def backward(ctx, do):
        q, k, v, o, lse = ctx.saved_tensors
        with torch.no_grad():
            grads = backward_window(_loadable(do), q, k, v, o, lse, *ctx.how)
        if torch.is_grad_enabled():  # create_graph, for whatever part of the model
            grads = _Once.apply(q, k, v, *grads)
        return (*grads, None, None, None)


def window_attention(
    q: torch.Tensor,
    k: torch.Tensor,
    v: torch.Tensor,
    window: int,
    sinks: int = 0,
    softmax_scale: float | None = None,
) -> torch.Tensor:
    """forward_window with a gradient: O [B, H, Nq, D], differentiable (once) in q, k and v."""
    return _WindowAttention.apply(q, k, v, window, sinks, softmax_scale)
