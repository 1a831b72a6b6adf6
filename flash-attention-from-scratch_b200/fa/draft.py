"""Drafted tokens over a paged cache: attention of a tree of them, and the accepted path kept.

    lengths += nodes                                                       # the tree's nodes behind the context
    q, k = fa.forward_rotary(q, k, context + depth, cos, sin)              # positions are depths, not slots
    fa.append_kv(cache, k, v, table, lengths)
    o = fa.forward_tree(q, cache, table, lengths, parents)
    ...                                                                    # the model accepts a path from a root
    lengths = fa.keep_tokens(cache, table, lengths, path, nodes)

Not in the reference, which has no cache. Serving only: no call carries a gradient. Lengths, counts,
parents, paths and the table stay on the device, so that a step can be captured in a CUDA graph.
"""

from __future__ import annotations

import ctypes
import math
import struct

import torch

from fa import _C
from fa.cache import _CACHE, PagedKVCache, _check_tokens
from fa.window import _on_device, _packed, _tensor_strides

# FaCache, then FaTreeParams' and FaKeepParams' own fields (include/fa_b200.h).
_TREE = struct.Struct("@" + _CACHE + "3P4q3ifB7x")
_KEEP = struct.Struct("@" + _CACHE + "2Pqi4x")


def _run_tree(params: bytes, device: torch.device, stream: int) -> int:
    """fa_tree_attention with a workspace from torch."""
    nbytes = ctypes.c_uint64(0)
    rc = _C.lib.fa_tree_workspace_size(params, ctypes.byref(nbytes))
    if rc == _C.FA_OK:
        need = nbytes.value
        ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        rc = _C.lib.fa_tree_attention(params, ws.data_ptr() if need else 0, need, stream)
    return rc


def _rows(t: torch.Tensor, name: str, batch: int, device: torch.device) -> int:
    """The stride of an int32 [B, n] tensor's rows, which may be one row for all."""
    if t.dtype != torch.int32 or t.dim() != 2 or t.device != device or t.shape[0] != batch or (t.stride(1) != 1 and t.shape[1] > 1):
        raise RuntimeError(f"{name} must be an int32 [B, n] tensor with contiguous rows on the cache's device")
    return t.stride(0) if batch > 1 else 0


def forward_tree(
    q: torch.Tensor,
    cache: PagedKVCache,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    parents: torch.Tensor,
    counts: torch.Tensor | None = None,
    window: int = 0,
    sinks: int = 0,
    softmax_scale: float | None = None,
) -> torch.Tensor:
    """O [B, H, T, D] of a tree of up to 256 drafted tokens, q [B, H, T, D] their queries.

    lengths and counts as in append_kv: the nodes are the counts[b] newest of lengths[b] tokens, and
    what is before them is the context. parents [B, T] int32 (expanded rows are fine): the index of each
    node's parent, below the node's own, or -1 for one that hangs on the context. Node t is at position
    p = context + (number of its ancestors); it sees the context's position j when window == 0, or p - j <
    window, or j < sinks, and of the nodes its ancestors and itself. window is 0 or at least T. Padding
    nodes (from counts[b] on) give zeros. With every parent the node before (a chain) this is
    forward_cached. Scores, softmax and sums are in float32; what a node does not see has no part in its
    output, infinities and NaN among it. The result carries no gradient."""
    _check_tokens(cache, q)
    batch, heads, tokens, dim = q.shape
    o = torch.empty_like(q, memory_format=torch.contiguous_format)
    fields = cache._fields(page_table, lengths, counts, batch, tokens)
    stride = _rows(parents, "parents", batch, cache._device)
    if parents.shape[1] != tokens:
        raise RuntimeError("parents must have an entry for every node")
    if q.numel() == 0:
        return o
    scale = 1.0 / math.sqrt(dim) if softmax_scale is None else float(softmax_scale)
    params = _packed(
        _TREE, *fields, q.data_ptr(), o.data_ptr(), parents.data_ptr(), *_tensor_strides(q), stride, heads, window, sinks,
        scale, _C.DTYPES[q.dtype])
    _on_device(cache._index, _run_tree, params, cache._device)
    return o


def keep_tokens(
    cache: PagedKVCache,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    kept: torch.Tensor,
    tokens: int,
    counts: torch.Tensor | None = None,
) -> torch.Tensor:
    """Moves the kept ones of the newest tokens together in the cache, and returns the new lengths.

    The counts[b] (or `tokens`, at most 256) newest of lengths[b] tokens are those to keep from; kept [B, n]
    int32 names them in ascending order (a path's nodes, from the root), as indices among the newest, up to
    the first -1 or the row's end. Token kept[b, j] goes to where token j was. The returned lengths count the
    context and the kept tokens. An entry that does not ascend or is no token's ends its row and sets
    bit 5 (32) of fa._C.device_status.

    An e4m3 page's scale becomes the largest of its own and of those that come in; where it grows the page's
    other tokens follow. What lies behind the new lengths is left as it is, but for that. The pages of the kept tokens
    have to be their sequence's own (reserve_pages)."""
    cache._look()
    if lengths.dim() != 1:
        raise RuntimeError("lengths must be an int32 [B] tensor")
    batch = lengths.shape[0]
    fields = cache._fields(page_table, lengths, counts, batch, tokens)
    stride = _rows(kept, "kept", batch, cache._device)
    if not 0 <= tokens <= 256:
        raise ValueError("keep_tokens: tokens must be at most 256")
    most = min(kept.shape[1], tokens)
    if batch == 0 or most == 0:
        return lengths.clamp(min=0) - (tokens if counts is None else counts.clamp(0, tokens))
    out = torch.empty_like(lengths)
    params = _KEEP.pack(*fields, kept.data_ptr(), out.data_ptr(), stride, most)
    _on_device(cache._index, _C.lib.fa_keep_tokens, params)
    return out
