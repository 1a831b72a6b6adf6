"""The pages of a cache: who holds which, forks of sequences, room for new tokens, copies.

    refs = torch.zeros(num_pages, dtype=torch.int32, device="cuda")           # how many entries hold each page
    table = torch.full((batch, width), -1, dtype=torch.int32, device="cuda")  # no pages yet
    granted, src, dst = fa.reserve_pages(refs, table, lengths, new, page_size)
    fa.copy_pages(cache, src, dst)                                            # for the cache of every layer
    beams = fa.fork_pages(refs, table, rows)                                  # shares all pages
    fa.free_pages(refs, table)

A sequence that is forked shares its pages until one of them gets new tokens: reserve_pages then gives it a
page of its own, and says which page has to be copied to it. Everything stays on the device, and for the
same state the same pages are taken, so that steps can be captured in CUDA graphs and repeated. Not in the
reference, which has no cache.
"""

from __future__ import annotations

import ctypes
import struct

import torch

from fa import _C
from fa.cache import _CACHE, PagedKVCache
from fa.window import _on_device

# FaCache and FaCopyParams' own fields; FaPages (include/fa_b200.h).
_COPY = struct.Struct("@" + _CACHE + "2Pi4x")
_PAGES = struct.Struct("@10P2q6i")


def copy_pages(cache: PagedKVCache, src: torch.Tensor, dst: torch.Tensor) -> None:
    """Copies pages src[i] to dst[i] ([n] int32), all heads of k and v with their scales.

    A pair with a negative page is skipped; one with a page outside the pool too, and sets bit 5 (32) of
    fa._C.device_status. No page may be the target of two pairs, nor target of one and source of another."""
    cache._look()
    for t in (src, dst):
        if t.dtype != torch.int32 or t.dim() != 1 or t.device != cache._device or not t.is_contiguous() or t.shape != src.shape:
            raise RuntimeError("src and dst must be contiguous int32 [n] tensors on the cache's device")
    if src.numel() == 0 or cache._k.numel() == 0:
        return
    params = _COPY.pack(*cache._pointers, 0, 0, 0, *cache._strides, 0, *cache._pool, 0, *cache._heads, 0, 0, cache._dtype,
                        src.data_ptr(), dst.data_ptr(), src.shape[0])
    _on_device(cache._index, _C.lib.fa_copy_pages, params)


def _check(refs: torch.Tensor, *tables: torch.Tensor) -> None:
    if not refs.is_cuda or refs.dtype != torch.int32 or refs.dim() != 1 or not refs.is_contiguous():
        raise RuntimeError("refs must be a contiguous int32 [pages] CUDA tensor")
    for t in tables:
        if t.dtype != torch.int32 or t.dim() != 2 or t.device != refs.device or (t.stride(1) != 1 and t.shape[1] > 1):
            raise RuntimeError("page_table must be an int32 [B, pages] tensor with contiguous rows on refs' device")


def _check_rows(refs: torch.Tensor, name: str, batch: int | None, *tensors: torch.Tensor | None) -> None:
    for t in tensors:
        if t is not None and (t.dtype != torch.int32 or t.dim() != 1 or t.device != refs.device or not t.is_contiguous()
                              or (batch is not None and t.shape[0] != batch)):
            raise RuntimeError(f"{name} must be contiguous int32 [B] tensors on refs' device")


def _stride(t: torch.Tensor) -> int:
    return t.stride(0) if t.shape[0] > 1 else t.shape[1]


def _pointer(t: torch.Tensor | None) -> int:
    return 0 if t is None else t.data_ptr()


def fork_pages(refs: torch.Tensor, page_table: torch.Tensor, rows: torch.Tensor) -> torch.Tensor:
    """A new table [n, width] whose row i holds the pages of row rows[i] ([n] int32), each counted once more
    in refs. rows[i] = -1 gives a row without pages. Entries of -1 hold none; entries outside the pool and rows outside
    the table are taken for -1 and set bit 5 (32) of fa._C.device_status."""
    _check(refs, page_table)
    _check_rows(refs, "rows", None, rows)
    (batch, width), n = page_table.shape, rows.shape[0]
    out = page_table.new_empty((n, width))
    if out.numel() == 0:
        return out
    if batch == 0 or refs.numel() == 0:
        raise ValueError("fork_pages: the table and the pool must not be empty")
    params = _PAGES.pack(refs.data_ptr(), out.data_ptr(), page_table.data_ptr(), rows.data_ptr(), 0, 0, 0, 0, 0, 0, width,
                         _stride(page_table), refs.shape[0], n, width, batch, 0, 0)
    _on_device(refs.get_device(), _C.lib.fa_fork_pages, params)
    return out


def free_pages(refs: torch.Tensor, page_table: torch.Tensor, keep: torch.Tensor | None = None) -> None:
    """Gives back the pages of entries from keep[b] ([B] int32; without it: all) on: they count one less in
    refs, the entries become -1. A page with no count left, or outside the pool, sets bit 5 (32) of fa._C.device_status."""
    _check(refs, page_table)
    batch, width = page_table.shape
    _check_rows(refs, "keep", batch, keep)
    if batch == 0 or width == 0:
        return
    params = _PAGES.pack(refs.data_ptr(), page_table.data_ptr(), 0, 0, _pointer(keep), 0, 0, 0, 0, 0, _stride(page_table), 0,
                         refs.shape[0], batch, width, 0, 0, 0)
    _on_device(refs.get_device(), _C.lib.fa_free_pages, params)


def _run_reserve(params: bytes, device: torch.device, stream: int) -> int:
    """fa_reserve_pages with a workspace from torch."""
    nbytes = ctypes.c_uint64(0)
    rc = _C.lib.fa_reserve_workspace_size(params, ctypes.byref(nbytes))
    if rc == _C.FA_OK:
        ws = torch.empty(nbytes.value, dtype=torch.uint8, device=device)
        rc = _C.lib.fa_reserve_pages(params, ws.data_ptr(), nbytes.value, stream)
    return rc


def reserve_pages(
    refs: torch.Tensor,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    tokens: int,
    page_size: int,
    counts: torch.Tensor | None = None,
) -> tuple[torch.Tensor, torch.Tensor, torch.Tensor]:
    """Room for new tokens, in place in page_table and refs: (granted, src, dst).

    lengths [B] int32 counts the new tokens, of which a row has counts[b] (or `tokens`), as in append_kv.
    Every entry that gets some of them holds a page of its own afterwards: a missing page, or one that
    other entries hold too, is replaced by a free one (refs 0), lowest number first, rows in order, entries in order. Where the
    first of them held older tokens, src[b] and dst[b] ([B] int32, else -1) are the pages to copy
    (copy_pages) before anything is appended or reserved again. Free and shared is what the call finds so.

    granted [B] bool: whether the row has its pages. A row is denied, and stays as it was, when the rows up
    to it need more pages than there are: do not append to it. A row whose positions do not fit
    the table is denied, too, and sets bit 5 (32) of fa._C.device_status."""
    _check(refs, page_table)
    batch, width = page_table.shape
    _check_rows(refs, "lengths and counts", batch, lengths, counts)
    src, dst = torch.empty_like(lengths), torch.empty_like(lengths)
    granted = torch.empty(batch, dtype=torch.bool, device=refs.device)
    if batch == 0:
        return granted, src, dst
    if tokens == 0:
        return granted.fill_(True), src.fill_(-1), dst.fill_(-1)
    try:
        params = _PAGES.pack(refs.data_ptr(), page_table.data_ptr(), 0, 0, 0, lengths.data_ptr(), _pointer(counts), granted.data_ptr(),
                             src.data_ptr(), dst.data_ptr(), _stride(page_table), 0, refs.shape[0], batch, width, 0, tokens, page_size)
    except struct.error as e:
        raise ValueError(f"tokens and page_size must be 32-bit integers: {e}") from None
    _on_device(refs.get_device(), _run_reserve, params, refs.device)
    return granted, src, dst
