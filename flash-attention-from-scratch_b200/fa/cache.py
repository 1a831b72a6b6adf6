"""A paged key/value cache: appending to it (with the rotation by position) and attention over it.

    cache = fa.PagedKVCache.empty(num_pages, page_size, kv_heads, head_dim)      # e4m3 with scales
    lengths += new                                                              # tokens, the new ones included
    q = fa.append_kv(cache, k, v, table, lengths, cos=cos, sin=sin, q=q)         # store k, v; rotate q
    o = fa.forward_cached(q, cache, table, lengths, window=4096, sinks=4)

Position j of sequence b is in slot j % page_size of page table[b, j // page_size]. Not in the
reference, which has no cache (its q, k and v have one length).

Serving only: neither call carries a gradient (to k, v or q, or into the cache).

lengths, counts and the table stay on the device and are not read by the host, so a call can be
captured in a CUDA graph and replayed as they change. Positions outside the table and pages outside
the pool are skipped by the kernels and set bit 5 (32) of fa._C.device_status.
"""

from __future__ import annotations

import ctypes
import math
import operator
import struct

import torch

from fa import _C
from fa.window import _NO_STRIDES, _on_device, _packed, _tensor_strides

# FaCache, then FaAppendParams' and FaCachedParams' own fields (include/fa_b200.h).
_CACHE = "7P5q7iB3x"
_APPEND = struct.Struct("@" + _CACHE + "6P9q3iBB2x")
_CACHED = struct.Struct("@" + _CACHE + "2P3q3ifB3x4x")


def _tensor(name: str) -> property:
    """One of a cache's tensors. Another one in its place is looked at by the next call."""

    def put(self, t):
        setattr(self, name, t)
        self._pointers = None

    return property(operator.attrgetter(name), put)


class PagedKVCache:
    """The pool of pages: k, v [num_pages, kv_heads, page_size, head_dim] (the last two dims
    contiguous), float8_e4m3fn with k_scale, v_scale [num_pages, kv_heads] float32 (a value is its
    code times its page's and head's scale), or float16 / bfloat16 without scales.

    The four may be replaced (a pool grows by cache.k = torch.cat([cache.k, more]), and so on for the
    others): the next call checks them and uses them. A captured graph keeps those it was captured with."""

    k, v, k_scale, v_scale = (_tensor(name) for name in ("_k", "_v", "_k_scale", "_v_scale"))
    num_pages = property(lambda self: self._k.shape[0])
    kv_heads = property(lambda self: self._k.shape[1])
    page_size = property(lambda self: self._k.shape[2])
    head_dim = property(lambda self: self._k.shape[3])
    device = property(lambda self: self._k.device)

    def __init__(self, k: torch.Tensor, v: torch.Tensor, k_scale: torch.Tensor | None = None,
                 v_scale: torch.Tensor | None = None) -> None:
        self._k, self._v, self._k_scale, self._v_scale = k, v, k_scale, v_scale
        self._lay_out()

    def _addresses(self) -> tuple[int, int, int, int]:
        ks, vs = self._k_scale, self._v_scale
        return (self._k.data_ptr(), self._v.data_ptr(), 0 if ks is None else ks.data_ptr(), 0 if vs is None else vs.data_ptr())

    def _lay_out(self) -> None:
        """Checks the tensors and takes down the parts of FaCache that stay as they are with them."""
        k, v, k_scale, v_scale = self._k, self._v, self._k_scale, self._v_scale
        for t in (k, v):
            if not t.is_cuda:
                raise RuntimeError("the cache's k and v must be CUDA tensors")
            if t.dtype not in _C.DTYPES and t.dtype != torch.float8_e4m3fn:
                raise RuntimeError("the cache's k and v must be float8_e4m3fn, float16 or bfloat16")
            if t.dim() != 4:
                raise RuntimeError("the cache's k and v must have shape [pages, kv_heads, page_size, head_dim]")
            if t.numel() > 0 and (t.stride(3) != 1 or t.stride(2) != t.shape[3]):
                raise RuntimeError("a page's tokens must be contiguous for every head")
        if k.shape != v.shape or k.dtype != v.dtype or k.device != v.device:
            raise RuntimeError("the cache's k and v must have the same shape, dtype and device")
        e4m3 = k.dtype == torch.float8_e4m3fn
        for s in (k_scale, v_scale):
            if (s is not None) != e4m3:
                raise RuntimeError("a float8_e4m3fn cache needs k_scale and v_scale, a 16-bit one has none")
            if s is not None and (s.shape != k.shape[:2] or s.dtype != torch.float32 or s.device != k.device
                                  or not s.is_contiguous()):
                raise RuntimeError("k_scale and v_scale must be contiguous float32 [pages, kv_heads] on k's device")
        (pages, heads, page_size, head_dim), (k0, k1, _, _), (v0, v1, _, _) = k.shape, k.stride(), v.stride()
        self._strides = (k0 * (pages > 1), k1 * (heads > 1), v0 * (pages > 1), v1 * (heads > 1))
        self._pool = (pages, page_size)
        self._heads = (heads, head_dim)
        self._dtype = _C.DTYPES.get(k.dtype, _C.FA_DTYPE_FLOAT8_E4M3)
        self._tokens_as = None if e4m3 else k.dtype
        self._device, self._index = k.device, k.get_device()
        self._pointers = self._addresses()

    def _look(self) -> None:
        """Memory that was replaced, or moved under a tensor that was not, is never reached by its old address."""
        if self._addresses() != self._pointers:
            self._lay_out()

    @classmethod
    def empty(cls, num_pages: int, page_size: int, kv_heads: int, head_dim: int,
              dtype: torch.dtype = torch.float8_e4m3fn, device: torch.device | str = "cuda") -> PagedKVCache:
        """A pool of zeroed pages."""
        shape = (num_pages, kv_heads, page_size, head_dim)
        k, v = (torch.zeros(shape, dtype=torch.uint8 if dtype == torch.float8_e4m3fn else dtype, device=device).view(dtype)
                for _ in "kv")
        scales = (None, None)
        if dtype == torch.float8_e4m3fn:
            scales = tuple(torch.ones(shape[:2], dtype=torch.float32, device=device) for _ in "kv")
        return cls(k, v, *scales)

    def _fields(self, table: torch.Tensor, lengths: torch.Tensor, counts: torch.Tensor | None, batch: int, tokens: int):
        """FaCache's fields for these sequences, checked."""
        device = self._device
        if table.dtype != torch.int32 or table.dim() != 2 or table.device != device:
            raise RuntimeError("page_table must be an int32 [B, pages] tensor on the cache's device")
        (rows, width), (stride, unit) = table.shape, table.stride()
        if rows != batch or (unit != 1 and width > 1):
            raise RuntimeError("page_table must be an int32 [B, pages] tensor with contiguous rows")
        for t in (lengths,) if counts is None else (lengths, counts):
            if t.dtype != torch.int32 or t.shape != (batch,) or t.device != device or not t.is_contiguous():
                raise RuntimeError("lengths and counts must be contiguous int32 [B] tensors on the cache's device")
        return (*self._pointers, table.data_ptr(), lengths.data_ptr(), 0 if counts is None else counts.data_ptr(),
                *self._strides, stride if batch > 1 else width, *self._pool, width, *self._heads, batch, tokens, self._dtype)


def _check_tokens(cache: PagedKVCache, *tensors: torch.Tensor) -> None:
    cache._look()
    only, device, dim = cache._tokens_as, cache._device, cache._heads[1]
    dtype, want = tensors[0].dtype, None
    for t in tensors:
        if not t.is_cuda:
            raise RuntimeError("q, k, v must be CUDA tensors")
        if t.dtype not in _C.DTYPES:
            raise RuntimeError("q, k, v must be float16 (or bfloat16)")
        if t.dtype != dtype or (only is not None and dtype != only):
            raise RuntimeError("q, k, v must have the same dtype, that of a 16-bit cache")
        if t.dim() != 4:
            raise RuntimeError("q, k, v must have shape [B, H, T, D]")
        if t.device != device:
            raise RuntimeError("q, k, v must be on the cache's device")
        b, _, n, d = t.shape
        if (b, n) != (want or (b, n)) or d != dim:
            raise RuntimeError("q, k, v must have the same batch and tokens, and the cache's head dim")
        want = (b, n)


def append_kv(
    cache: PagedKVCache,
    k: torch.Tensor,
    v: torch.Tensor,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    counts: torch.Tensor | None = None,
    cos: torch.Tensor | None = None,
    sin: torch.Tensor | None = None,
    q: torch.Tensor | None = None,
    interleaved: bool = False,
) -> torch.Tensor | None:
    """Stores k, v [B, Hkv, T, D] into the cache and returns q [B, H, T, D] rotated (None without q).

    lengths [B] int32 counts every sequence's tokens with the new ones; of the T new ones the first
    counts[b] (all without counts) are real, at positions lengths[b] - counts[b] onwards, and the
    rest is padding: not stored, zeros in the returned q. cos, sin [rows, R / 2] float32 turn the
    first R dims (a multiple of 16) of q and k in pairs (i, i + R / 2), or (2 i, 2 i + 1) when
    interleaved; without them nothing is turned. The rotation is in float32 and rounded once.

    An e4m3 page's scale is the smallest power of two (2^-60 or more) that brings its values within
    448. It grows while the page fills (older tokens are rescaled, exactly but for subnormal codes)
    and starts anew with the page's first slot. No two sequences may append to one page. The returned q
    carries no gradient."""
    tensors = (k, v) if q is None else (k, v, q)
    _check_tokens(cache, *tensors)
    if k.shape != v.shape or k.shape[1] != cache._heads[0]:
        raise RuntimeError("k and v must have shape [B, kv_heads, T, D]")
    batch, _, tokens, dim = k.shape
    rows = half = 0
    if (cos is None) != (sin is None):
        raise RuntimeError("cos and sin go together")
    if cos is not None:
        for t in (cos, sin):
            if t.dtype != torch.float32 or t.dim() != 2 or t.device != k.device or not t.is_contiguous():
                raise RuntimeError("cos and sin must be contiguous float32 [rows, R / 2] tensors on k's device")
        if cos.shape != sin.shape:
            raise RuntimeError("cos and sin must have the same shape")
        rows, half = cos.shape
    out = None if q is None else torch.empty_like(q, memory_format=torch.contiguous_format)
    fields = cache._fields(page_table, lengths, counts, batch, tokens)
    if batch == 0 or tokens == 0:
        return out
    tables = (0, 0) if cos is None else (cos.data_ptr(), sin.data_ptr())
    query = (0, 0) if q is None else (q.data_ptr(), out.data_ptr())
    params = _APPEND.pack(
        *fields, k.data_ptr(), v.data_ptr(), *query, *tables, *_tensor_strides(k), *_tensor_strides(v),
        *(_NO_STRIDES if q is None else _tensor_strides(q)), 0 if q is None else q.shape[1], rows, 2 * half,
        interleaved, _C.DTYPES[k.dtype])
    _on_device(cache._index, _C.lib.fa_append_kv, params)
    return out


def _run_cached(params: bytes, device: torch.device, stream: int) -> int:
    """fa_cached_attention with a workspace from torch."""
    nbytes = ctypes.c_uint64(0)
    rc = _C.lib.fa_cached_workspace_size(params, ctypes.byref(nbytes))
    if rc == _C.FA_OK:
        need = nbytes.value
        ws = torch.empty(need, dtype=torch.uint8, device=device) if need else None
        rc = _C.lib.fa_cached_attention(params, ws.data_ptr() if need else 0, need, stream)
    return rc


def forward_cached(
    q: torch.Tensor,
    cache: PagedKVCache,
    page_table: torch.Tensor,
    lengths: torch.Tensor,
    counts: torch.Tensor | None = None,
    window: int = 0,
    sinks: int = 0,
    softmax_scale: float | None = None,
) -> torch.Tensor:
    """O [B, H, T, D] of the newest tokens' queries q [B, H, T, D] over the cache.

    lengths and counts as in append_kv: query t of sequence b is at position p = lengths[b] -
    counts[b] + t and sees position j when 0 <= j <= p and (window == 0, or p - j < window, or
    j < sinks); a row that sees nothing, padding among them, is zeros. H is a multiple of the
    cache's heads, grouped as in forward_window. Scores, softmax and sums are in float32. The result
    carries no gradient."""
    _check_tokens(cache, q)
    batch, heads, tokens, dim = q.shape
    o = torch.empty_like(q, memory_format=torch.contiguous_format)
    fields = cache._fields(page_table, lengths, counts, batch, tokens)
    if q.numel() == 0:
        return o
    scale = 1.0 / math.sqrt(dim) if softmax_scale is None else float(softmax_scale)
    params = _packed(
        _CACHED, *fields, q.data_ptr(), o.data_ptr(), *_tensor_strides(q), heads, window, sinks, scale,
        _C.DTYPES[q.dtype])
    _on_device(cache._index, _run_cached, params, cache._device)
    return o
