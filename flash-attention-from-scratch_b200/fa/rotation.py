"""Rotation of queries and keys by positions on one or several axes, forward and backward.

    q, k = fa.rotary(q, k, positions, cos, sin, axes=[0] * 16 + [1] * 24 + [2] * 24)    # time, height, width

Pair i of a row (the dims i and i + R / 2, or 2 i and 2 i + 1 when interleaved) turns by column i of the
tables cos, sin [rows, R / 2] at the row that positions[axes[i], b, t] names; dims from R on stay as they
are. append_kv turns by the slots' own numbers, in order; this is for positions that are others: patches of
images and frames, and the nodes of a tree of drafted tokens, whose position is their depth. Not in the
reference, which has no rotation.
"""

from __future__ import annotations

import struct
from collections.abc import Sequence

import torch

from fa import _C
from fa.window import _NO_STRIDES, _loadable, _on_device, _tensor_strides

# FaRotaryParams (include/fa_b200.h): 7 pointers, 3 x 3 strides, 8 ints, an axis for every pair, 3 flags.
_PARAMS = struct.Struct("@7P9q8i64s3B5x")


def _run(q, k, positions, cos, sin, axes, interleaved, inverse):
    dtype, device = q.dtype, q.device
    for t in (q,) if k is None else (q, k):
        if not t.is_cuda:
            raise RuntimeError("q, k must be CUDA tensors")
        if t.dtype not in _C.DTYPES:
            raise RuntimeError("q, k must be float16 (or bfloat16)")
        if t.dtype != dtype:
            raise RuntimeError("q, k must have the same dtype")
        if t.dim() != 4:
            raise RuntimeError("q, k must have shape [B, H, T, D]")
        if t.device != device:
            raise RuntimeError("q, k must be on the same device")
    batch, heads, tokens, dim = q.shape
    kv_heads = 0
    if k is not None:
        kv_heads = k.shape[1]
        if k.shape != (batch, kv_heads, tokens, dim):
            raise RuntimeError("k must have q's batch, tokens and head dim")
    for t in (cos, sin):
        if t.dtype != torch.float32 or t.dim() != 2 or t.device != device or not t.is_contiguous():
            raise RuntimeError("cos and sin must be contiguous float32 [rows, R / 2] tensors on q's device")
    if cos.shape != sin.shape:
        raise RuntimeError("cos and sin must have the same shape")
    if positions.dim() == 2:
        positions = positions[None]
    if positions.dtype != torch.int32 or positions.dim() != 3 or positions.device != device or positions.shape[1:] != (batch, tokens):
        raise RuntimeError("positions must be an int32 [axes, B, T] (or [B, T]) tensor on q's device")
    rows, half = cos.shape
    if axes is None:
        axes = b""
    else:
        if len(axes) != half:
            raise RuntimeError("axes must name an axis for each of the R / 2 pairs")
        axes = bytes(axes)
    out = torch.empty_like(q, memory_format=torch.contiguous_format)
    k_out = None if k is None else torch.empty_like(k, memory_format=torch.contiguous_format)
    if batch == 0 or tokens == 0:
        return out, k_out
    keys = (0, 0) if k is None else (k.data_ptr(), k_out.data_ptr())
    params = _PARAMS.pack(
        q.data_ptr(), keys[0], out.data_ptr(), keys[1], positions.data_ptr(), cos.data_ptr(), sin.data_ptr(),
        *_tensor_strides(q), *(_NO_STRIDES if k is None else _tensor_strides(k)), *positions.stride(),
        batch, heads, kv_heads, tokens, dim, 2 * half, rows, positions.shape[0], axes, interleaved, inverse, _C.DTYPES[dtype])
    _on_device(q.get_device(), _C.lib.fa_rotary, params)
    return out, k_out


def forward_rotary(
    q: torch.Tensor,
    k: torch.Tensor | None,
    positions: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    axes: Sequence[int] | None = None,
    interleaved: bool = False,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """(q, k) turned: q [B, H, T, D], k [B, Hkv, T, D] (or None), float16 or bfloat16, D in {64, 128}.

    positions: int32 [A, B, T] (or [B, T] for one axis; expanded dims are fine), A up to 4. axes: the
    axis of each of the R / 2 pairs, all 0 without. A token with a negative position on any axis is padding:
    zeros. One with a position beyond the tables is zeros, too, and sets bit 5 (32) of
    fa._C.device_status. The rotation is in float32 and rounded once, to the bit what append_kv makes
    of the same angles. The result carries no gradient: rotary does."""
    return _run(q, k, positions, cos, sin, axes, interleaved, False)


def backward_rotary(
    dq: torch.Tensor,
    dk: torch.Tensor | None,
    positions: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    axes: Sequence[int] | None = None,
    interleaved: bool = False,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """The gradients of forward_rotary's inputs from those of its results: turned back."""
    return _run(dq, dk, positions, cos, sin, axes, interleaved, True)


class _Rotary(torch.autograd.Function):
    @staticmethod
    def forward(ctx, q, k, positions, cos, sin, axes, interleaved, inverse):
        ctx.set_materialize_grads(False)
        ctx.save_for_backward(positions, cos, sin)
        ctx.how = (axes, interleaved, not inverse)
        return _run(q, k, positions, cos, sin, axes, interleaved, inverse)

    @staticmethod
    def backward(ctx, dq, dk):
        # A gradient of the gradients asked for (create_graph): they are results of a rotation like any other.
        turn = _Rotary.apply if torch.is_grad_enabled() else _run
        dk = None if dk is None else _loadable(dk)
        if dq is None:
            grads = (None, None) if dk is None else turn(dk, None, *ctx.saved_tensors, *ctx.how)[::-1]
        else:
            grads = turn(_loadable(dq), dk, *ctx.saved_tensors, *ctx.how)
        return (*grads, None, None, None, None, None, None)


def rotary(
    q: torch.Tensor,
    k: torch.Tensor | None,
    positions: torch.Tensor,
    cos: torch.Tensor,
    sin: torch.Tensor,
    axes: Sequence[int] | None = None,
    interleaved: bool = False,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """forward_rotary with a gradient in q and k (any number of times: a gradient is a rotation itself).

    A step captured in a CUDA graph may hold it as any operation of autograd: warmed up on a side stream, and with no
    graph of the same leaves left from before the capture, which torch does not survive. forward_rotary and
    backward_rotary have no such condition."""
    # As bytes: the gradients turn by what is in the sequence now, whatever becomes of it.
    return _Rotary.apply(q, k, positions, cos, sin, None if axes is None else bytes(tuple(axes)), interleaved, False)
