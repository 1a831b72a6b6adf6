"""Causal attention over a sliding window and a few first tokens (sinks), forward and backward.

Query i of q [B, H, Nq, D] is at position p = Nk - Nq + i of the keys k, v [B, Hkv, Nk, D] and
sees key j when 0 <= j <= p and (window == 0, or p - j < window, or j < sinks). H is a multiple of
Hkv: query head h reads key/value head h // (H // Hkv). A query that sees nothing gives O = 0.
float16 or bfloat16, D in {64, 128}; the last dim is contiguous, the other strides are multiples
of 8 elements (a [B, N, H, D] tensor's transpose(1, 2) is fine). Not in the reference, whose
attention is over all keys or all keys up to the query's own, and forward only.
"""

from __future__ import annotations

import ctypes
import math
import struct

import torch

from fa import _C

# FaWindowParams (include/fa_b200.h): 9 pointers, 8 x 3 strides, 8 ints, the scale, the dtype.
_PARAMS = struct.Struct("@9P24q8ifB3x")


def _tensor_strides(t: torch.Tensor) -> tuple[int, int, int]:
    """{batch, head, row} strides; 0 for a dim of one element, whose stride means nothing."""
    (s0, s1, s2, s3), (n0, n1, n2, n3) = t.stride(), t.shape
    if s3 != 1 and n3 > 1:
        raise RuntimeError("tensors must have a contiguous last dimension")
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


def _run(entry, size_entry, q, k, v, o, lse, do, dq, dk, dv, window, sinks, scale) -> None:
    """Packs FaWindowParams and calls `entry` on the current stream of q's device, with a
    workspace from torch of the size that `size_entry` (or None) names."""
    device = q.device
    zero = (0, 0, 0)
    grads = (do, dq, dk, dv)
    params = _PARAMS.pack(
        q.data_ptr(), k.data_ptr(), v.data_ptr(), o.data_ptr(), 0 if lse is None else lse.data_ptr(),
        *(0 if t is None else t.data_ptr() for t in grads),
        *_tensor_strides(q), *_tensor_strides(k), *_tensor_strides(v), *_tensor_strides(o),
        *(s for t in grads for s in (zero if t is None else _tensor_strides(t))),
        q.shape[0], q.shape[1], k.shape[1], q.shape[2], k.shape[2], q.shape[3], window, sinks, scale, _C.DTYPES[q.dtype])
    with torch.cuda.device(device):
        stream = torch.cuda.current_stream(device).cuda_stream
        if size_entry is None:
            rc = entry(params, stream)
        else:
            nbytes = ctypes.c_uint64(0)
            rc = size_entry(params, ctypes.byref(nbytes))
            if rc == _C.FA_OK:
                ws = torch.empty(nbytes.value, dtype=torch.uint8, device=device)
                rc = entry(params, ws.data_ptr(), nbytes.value, stream)
    if rc != _C.FA_OK:
        _C._raise(rc)


def _scale(softmax_scale: float | None, q: torch.Tensor) -> float:
    return 1.0 / math.sqrt(q.shape[3]) if softmax_scale is None else float(softmax_scale)


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
    o = torch.empty(q.shape, dtype=q.dtype, device=q.device)
    lse = torch.empty(q.shape[:3], dtype=torch.float32, device=q.device) if return_lse else None
    if q.numel() > 0 and k.shape[2] > 0:
        _run(_C.lib.fa_window_fwd, None, q, k, v, o, lse, None, None, None, None, window, sinks, _scale(softmax_scale, q))
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
    dq, dk, dv = (torch.empty(t.shape, dtype=t.dtype, device=t.device) for t in (q, k, v))
    if q.numel() > 0 and k.numel() > 0:
        _run(_C.lib.fa_window_bwd, _C.lib.fa_window_bwd_workspace_size, q, k, v, o, lse, do, dq, dk, dv, window, sinks,
             _scale(softmax_scale, q))
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


class _WindowAttention(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, v, window, sinks, softmax_scale):
        o, lse = forward_window(q, k, v, window, sinks, softmax_scale, return_lse=True)
        ctx.save_for_backward(q, k, v, o, lse)
        ctx.how = (window, sinks, softmax_scale)
        return o

    @staticmethod
    @torch.autograd.function.once_differentiable
    def backward(ctx, do):
        return (*backward_window(_loadable(do), *ctx.saved_tensors, *ctx.how), None, None, None)


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
