"""The paged cache on the GPU: appending (bit for bit against the definition in float32, and
against 64 bits within e4m3's rounding) and attention over it (against the 64-bit definition; the
bounds are derived in stream_oracle)."""

import math

import pytest
import torch

import fa
import stream_oracle as oracle
from fa import _C

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
HALF, BF, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


def _ints(*x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _rand(gen, shape, dtype):
    return torch.randn(shape, generator=gen, device=DEV).to(dtype)


def _tables(d, rows, rotary=None, seed=3):
    gen = torch.Generator(DEV).manual_seed(seed)
    a = torch.rand(rows, (rotary or d) // 2, generator=gen, device=DEV) * 6.28
    return a.cos(), a.sin()


def _cache(gen, batch, most, page, heads, d, dtype, spare=2):
    """A cache filled with values, and a table of its pages in random order."""
    per = -(-most // page)
    pages = batch * per + spare
    table = torch.randperm(pages, generator=gen, device=DEV)[: batch * per].to(torch.int32).view(batch, per)
    x = [_rand(gen, (pages, heads, page, d), HALF) for _ in "kv"]
    if dtype != E4M3:
        return fa.PagedKVCache(*(t.to(dtype) for t in x)), table
    # Any positive scales, not powers of two alone.
    scales = [torch.rand(pages, heads, generator=gen, device=DEV) * 0.05 + 0.004 for _ in "kv"]
    codes = [(t.float() / s[..., None, None]).clamp(-448, 448).to(E4M3) for t, s in zip(x, scales)]
    return fa.PagedKVCache(*codes, *scales), table


# --------------------------------------------------------------------------------------- append


def _check_append(cache, k, v, table, lengths, counts, cos, sin, q, interleaved=False):
    t = k.shape[2]
    every = torch.full_like(lengths, t) if counts is None else counts
    step = torch.arange(t, device=DEV)
    real = step < every[:, None]
    pos = torch.where(real, (lengths - every)[:, None] + step, 0).long()
    want = [oracle.append(p, s, oracle.turned(x, pos, c, n, interleaved, torch.float32), table, lengths, every)
            for p, s, x, c, n in ((cache.k, cache.k_scale, k, cos, sin), (cache.v, cache.v_scale, v, None, None))]
    out = fa.append_kv(cache, k, v, table, lengths, counts=counts, cos=cos, sin=sin, q=q, interleaved=interleaved)
    for (pool, scale), got, got_scale in zip(want, (cache.k, cache.v), (cache.k_scale, cache.v_scale)):
        bits = (lambda x: x.view(torch.uint8)) if scale is not None else (lambda x: x.view(torch.int16))
        assert torch.equal(bits(got), bits(pool))
        assert scale is None or torch.equal(got_scale, scale)
    if q is None:
        assert out is None
    else:
        exact = torch.where(real[:, None, :, None], oracle.turned(q, pos, cos, sin, interleaved), 0.0)
        oracle.check(out, exact, oracle.unit(q.dtype) * exact.abs() + 2.0**-21 * q.double().abs().max(), "q")
        plain = torch.where(real[:, None, :, None], oracle.turned(q, pos, cos, sin, interleaved, torch.float32), 0.0)
        assert torch.equal(out, plain.to(q.dtype))
    # What is stored stands for the values to e4m3's half ulp (2^-4, or 2^-10 of the scale below
    # its normal range), or the 16-bit type's.
    k64 = oracle.turned(k, pos, cos, sin, interleaved)
    stored = oracle.dense(cache.k, cache.k_scale, table)
    for b in range(k.shape[0]):
        n, length = int(every[b]), int(lengths[b])
        exact, got = k64[b, :, :n], stored[b, :, length - n : length]
        if cache.k_scale is None:
            bound = oracle.unit(k.dtype) * exact.abs() + 2.0**-21 * k.double().abs().max()
        else:
            pages = table[b].long()[torch.arange(length - n, length, device=DEV) // cache.page_size]
            bound = 2.0**-4 * exact.abs() + 2.0**-10 * cache.k_scale[pages].double().T[..., None] + 1e-5
        assert ((got - exact).abs() <= bound).all()
    assert _C.device_status(0) == 0


@pytest.mark.parametrize("page", [8, 16, 64, 128, 256])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype,cache_dtype", [(BF, E4M3), (HALF, E4M3), (BF, BF), (HALF, HALF)])
def test_append_ragged(page, d, dtype, cache_dtype):
    gen = torch.Generator(DEV).manual_seed(page + d)
    cache, table = _cache(gen, 5, 420, page, 2, d, cache_dtype)
    k, v, q = (_rand(gen, (5, h, 300, d), dtype) for h in (2, 2, 6))
    # a whole count, none, one, a page's edge, an odd one; starts at 0, mid-page and at an edge
    counts = _ints(300, 0, 1, page, 177)
    lengths = _ints(300, 40, 1, 2 * page if page < 200 else page + 3, 177 + 33)
    cos, sin = _tables(d, 512)
    _check_append(cache, k, v, table, lengths, counts, cos, sin, q)


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("d,rotary", [(64, 16), (64, 64), (128, 48), (128, 96), (128, 128)])
def test_append_rotary_dims(interleaved, d, rotary):
    gen = torch.Generator(DEV).manual_seed(rotary)
    cache, table = _cache(gen, 3, 100, 16, 2, d, E4M3)
    k, v, q = (_rand(gen, (3, h, 9, d), BF) for h in (2, 2, 2))
    cos, sin = _tables(d, 100, rotary)
    _check_append(cache, k, v, table, _ints(9, 50, 100), None, cos, sin, q, interleaved)


@pytest.mark.parametrize("dtype,cache_dtype", [(BF, E4M3), (HALF, HALF)])
def test_append_tokens_one_by_one(dtype, cache_dtype):
    """A decode step at a time, values growing and shrinking, so that scales grow mid-page."""
    gen = torch.Generator(DEV).manual_seed(1)
    cache, table = _cache(gen, 2, 80, 32, 3, 64, cache_dtype)
    cos, sin = _tables(64, 80)
    for step in range(40):
        k, v, q = (_rand(gen, (2, h, 1, 64), dtype) * 2.0 ** (step % 7 - 3) for h in (3, 3, 3))
        _check_append(cache, k, v, table, _ints(step + 1, step + 31), None, cos, sin, q)


def test_append_in_parts_is_append_at_once():
    """Scales are powers of two that only grow, so the split of a prompt into calls shows in
    nothing but codes that were rounded as subnormals before a scale grew."""
    gen = torch.Generator(DEV).manual_seed(2)
    k, v = (_rand(gen, (1, 2, 150, 128), BF) for _ in "kv")
    whole, table = _cache(gen, 1, 150, 64, 2, 128, E4M3)
    parts = fa.PagedKVCache(whole.k.clone(), whole.v.clone(), whole.k_scale.clone(), whole.v_scale.clone())
    fa.append_kv(whole, k, v, table, _ints(150))
    at = 0
    for n in (1, 5, 63, 64, 17):
        fa.append_kv(parts, k[:, :, at : at + n], v[:, :, at : at + n], table, _ints(at + n))
        at += n
    used = table[0].long()
    assert torch.equal(whole.k_scale[used], parts.k_scale[used]) and torch.equal(whole.v_scale[used], parts.v_scale[used])
    a, b = (oracle.dense(c.k, c.k_scale, table)[0, :, :150] for c in (whole, parts))
    # two roundings to the coarser grid's subnormals: at most one of its steps apart
    assert ((a - b).abs() <= 2.0**-9 * float(whole.k_scale[used].max())).all()
    assert (a == b).double().mean() > 0.9


def test_append_extreme_values():
    gen = torch.Generator(DEV).manual_seed(4)
    cache, table = _cache(gen, 1, 64, 16, 1, 64, E4M3)
    k = torch.zeros(1, 1, 48, 64, dtype=BF, device=DEV)  # page 0: zeros
    k[0, 0, 16, 0], k[0, 0, 17, 1] = 448.0, -3e-30       # page 1: the range's end and far below it
    k[0, 0, 32, :4] = torch.tensor([math.inf, -math.inf, math.nan, 3e38], device=DEV)
    fa.append_kv(cache, k, k, table, _ints(48))
    scale = cache.k_scale[table[0].long(), 0].double()
    assert scale[:2].tolist() == [2.0**-60, 1.0] and scale[2] == oracle.power_of_two(float(k[0, 0, 32, 3]))
    got = oracle.dense(cache.k, cache.k_scale, table)[0, 0]
    assert not got[:16].any() and got[16, 0] == 448.0 and got[17, 1] == 0
    assert got[32, 0] == 448 * scale[2] and got[32, 1] == -448 * scale[2] and got[32, 2].isnan()
    # 449 needs the next power of two
    k[0, 0, 16, 0] = 450.0
    fa.append_kv(cache, k, k, table, _ints(48))
    assert cache.k_scale[int(table[0, 1]), 0] == 2.0


def test_append_strides_pools_and_streams():
    """Packed projections, a pool that interleaves layers, and another stream."""
    gen = torch.Generator(DEV).manual_seed(5)
    qkv = _rand(gen, (2, 21, 4 + 2 + 2, 64), HALF)
    q, k, v = (t.transpose(1, 2) for t in qkv.split([4, 2, 2], 2))
    pool = torch.zeros(6, 3, 2, 2, 16, 64, dtype=HALF, device=DEV)  # pages, layers, k/v, heads, slots, dims
    cache = fa.PagedKVCache(pool[:, 1, 0], pool[:, 1, 1])
    table = _ints(4, 0, 5, 2).view(2, 2)
    cos, sin = _tables(64, 64)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _check_append(cache, k, v, table, _ints(21, 30), None, cos, sin, q)
    torch.cuda.synchronize()
    assert not pool[:, 0].any() and not pool[:, 2].any()


def test_append_outside_the_table_is_skipped_and_reported():
    gen = torch.Generator(DEV).manual_seed(6)
    k = _rand(gen, (1, 1, 20, 64), HALF)
    for table, lengths, rows in ((_ints(0, 7), 32, None), (_ints(0, -1), 32, None), (_ints(0), 32, None), (_ints(0, 1), 10, None),
                                 (_ints(0, 1), 32, 20)):
        pool = [torch.zeros(3, 1, 16, 64, dtype=HALF, device=DEV) for _ in "kv"]
        cos, sin = (None, None) if rows is None else _tables(64, rows)
        q = fa.append_kv(fa.PagedKVCache(*pool), k, k, table.view(1, -1), _ints(lengths), cos=cos, sin=sin, q=k)
        assert _C.device_status(0) == 32 and _C.device_status(0) == 0
        assert not pool[0][1:, :, 4:].any() and not pool[1][2].any() and torch.isfinite(q).all()


def test_append_refusals():
    gen = torch.Generator(DEV).manual_seed(7)
    cache, table = _cache(gen, 2, 64, 16, 2, 64, E4M3)
    k = _rand(gen, (2, 2, 4, 64), HALF)
    n = _ints(4, 4)
    cos, sin = _tables(64, 64)
    for error, match, call in (
        (RuntimeError, "head dim", lambda: fa.append_kv(cache, k[..., :32], k[..., :32], table, n)),
        (RuntimeError, "kv_heads", lambda: fa.append_kv(cache, k[:, :1], k[:, :1], table, n)),
        (RuntimeError, "go together", lambda: fa.append_kv(cache, k, k, table, n, cos=cos)),
        (RuntimeError, "float32", lambda: fa.append_kv(cache, k, k, table, n, cos=cos.half(), sin=sin.half())),
        (RuntimeError, "int32", lambda: fa.append_kv(cache, k, k, table.long(), n)),
        (RuntimeError, "int32", lambda: fa.append_kv(cache, k, k, table, n[:1])),
        (RuntimeError, "same dtype", lambda: fa.append_kv(cache, k, k.bfloat16(), table, n)),
        (RuntimeError, "CUDA", lambda: fa.append_kv(cache, k.cpu(), k.cpu(), table, n)),
        (ValueError, "rotary_dim", lambda: fa.append_kv(cache, k, k, table, n, cos=cos[:, :4].contiguous(), sin=sin[:, :4].contiguous())),
        (ValueError, "multiples of 8", lambda: fa.append_kv(cache, torch.zeros(2, 2, 4, 68, dtype=HALF, device=DEV)[..., :64], k, table, n)),
        (RuntimeError, "needs k_scale", lambda: fa.PagedKVCache(cache.k, cache.v)),
        (RuntimeError, "has none", lambda: fa.PagedKVCache(k, k, n, n)),
        (ValueError, "power of two", lambda: fa.append_kv(fa.PagedKVCache.empty(4, 24, 2, 64), k, k, table, n)),
        (ValueError, "multiple of kv_heads", lambda: fa.append_kv(cache, k, k, table, n, q=k[:, :1])),
    ):
        with pytest.raises(error, match=match):
            call()


# ------------------------------------------------------------------------------ attention over it


def _check_cached(q, cache, table, lengths, counts=None, window=0, sinks=0, scale=None):
    got = fa.forward_cached(q, cache, table, lengths, counts=counts, window=window, sinks=sinks, softmax_scale=scale)
    want, vmax = oracle.cached(q, cache, table, lengths, counts, window, sinks, scale)
    # P is float16 over an e4m3 cache, else of the tensors' type.
    u_p = oracle.unit(HALF if cache.k_scale is not None else q.dtype)
    oracle.check(got, want, oracle.forward_bound(want, vmax, u_p, oracle.unit(q.dtype)), "O")
    assert torch.equal(got, fa.forward_cached(q, cache, table, lengths, counts=counts, window=window, sinks=sinks, softmax_scale=scale))
    assert _C.device_status(0) == 0
    return got


TYPES = [(BF, E4M3), (HALF, E4M3), (BF, BF), (HALF, HALF)]


@pytest.mark.parametrize("h,hk,t", [(1, 1, 1), (8, 2, 1), (8, 1, 1), (4, 4, 3), (8, 2, 4), (32, 2, 1), (16, 1, 5), (3, 1, 17)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype,cache_dtype", TYPES)
def test_cached_matches_definition(h, hk, t, d, dtype, cache_dtype):
    gen = torch.Generator(DEV).manual_seed(h + t + d)
    cache, table = _cache(gen, 4, 700, 32, hk, d, cache_dtype)
    q = _rand(gen, (4, h, t, d), dtype)
    lengths = _ints(max(t, 1), 333, 700, t + 64)
    _check_cached(q, cache, table, lengths)
    _check_cached(q, cache, table, lengths, window=100, sinks=5)


@pytest.mark.parametrize("page", [8, 16, 64, 256])
@pytest.mark.parametrize("window,sinks", [(0, 0), (1, 0), (33, 1), (64, 70), (500, 4), (4096, 3)])
@pytest.mark.parametrize("cache_dtype", [E4M3, BF])
def test_cached_windows_and_pages(page, window, sinks, cache_dtype):
    gen = torch.Generator(DEV).manual_seed(page + window)
    cache, table = _cache(gen, 6, 1500, page, 2, 64, cache_dtype)
    q = _rand(gen, (6, 4, 2, 64), BF)
    _check_cached(q, cache, table, _ints(2, 31, 64, 65, 1024, 1500), window=window, sinks=sinks)


@pytest.mark.parametrize("cache_dtype", [E4M3, HALF])
def test_cached_ragged_tokens_and_empty_rows(cache_dtype):
    """Padding tokens, a sequence of no tokens, and one whose queries start before position 0."""
    gen = torch.Generator(DEV).manual_seed(8)
    cache, table = _cache(gen, 5, 300, 16, 2, 128, cache_dtype)
    q = _rand(gen, (5, 4, 6, 128), HALF)
    got = _check_cached(q, cache, table, _ints(300, 100, 0, 3, 6), _ints(6, 2, 0, 6, 1), window=50, sinks=2)
    assert not got[1, :, 2:].any() and not got[2].any() and not got[3, :, :3].any() and got[3, :, 3:].any()


@pytest.mark.parametrize("cache_dtype", [E4M3, BF])
def test_cached_many_sequences_and_one_long(cache_dtype):
    """Unequal work over the whole GPU: one sequence of many splits among short ones."""
    gen = torch.Generator(DEV).manual_seed(9)
    cache, table = _cache(gen, 1, 20000, 64, 2, 128, cache_dtype)
    q = _rand(gen, (1, 8, 1, 128), BF)
    _check_cached(q, cache, table, _ints(19999))
    cache, table = _cache(gen, 200, 300, 64, 2, 64, cache_dtype)
    q = _rand(gen, (200, 4, 1, 64), BF)
    lengths = torch.randint(1, 301, (200,), generator=gen, device=DEV, dtype=torch.int32)
    _check_cached(q, cache, table, lengths)


def test_cached_long_chunk_of_tokens():
    gen = torch.Generator(DEV).manual_seed(10)
    cache, table = _cache(gen, 2, 400, 32, 2, 64, E4M3)
    q = _rand(gen, (2, 8, 150, 64), BF)
    _check_cached(q, cache, table, _ints(400, 222), _ints(150, 101), window=120, sinks=3)


def test_cached_shared_pages_and_other_scales():
    """Two sequences that share their first pages; negative and zero softmax scales."""
    gen = torch.Generator(DEV).manual_seed(11)
    cache, _ = _cache(gen, 1, 64, 16, 2, 64, E4M3, spare=4)
    table = _ints(0, 1, 2, 3, 0, 1, 5, 6).view(2, 4)
    q = _rand(gen, (2, 4, 1, 64), HALF)
    for scale in (-0.3, 0.0, 1.0):
        _check_cached(q, cache, table, _ints(60, 64), scale=scale)


def test_cached_scales_far_apart():
    """Values whose pages' scales differ by many powers of two, down to 2^-60, and a scale of 0: the
    rounding of P must not drop what a row of small values attends to."""
    gen = torch.Generator(DEV).manual_seed(12)
    cache, table = _cache(gen, 1, 128, 16, 1, 64, E4M3, spare=0)
    cache.v_scale[table[0].long(), 0] = torch.tensor([2.0**-60, 2.0**-30, 2.0**-12, 1e-5, 1.0, 64.0, 2.0**-40, 0.0], device=DEV)
    q = _rand(gen, (1, 1, 1, 64), HALF)
    for length in range(16, 129, 16):
        one = _ints(length)
        want, _ = oracle.cached(q, cache, table, one)
        got = fa.forward_cached(q, cache, table, one)
        # relative to the row's own weighted values, not to the largest value in the cache
        k, v = oracle.dense(cache.k, cache.k_scale, table)[0, 0], oracle.dense(cache.v, cache.v_scale, table)[0, 0]
        p = torch.softmax(q[0, 0, 0].double() @ k[:length].T / 8, -1)
        size = (p[:, None] * v[:length].abs()).sum(0)
        bound = (4 * 2.0**-11 + 2 * oracle.POLY) * size + 2.0**-11 * want.abs() + 2.0**-25
        oracle.check(got, want, bound.expand_as(want), f"O at {length}")


def test_cached_hidden_slots_may_hold_anything():
    gen = torch.Generator(DEV).manual_seed(13)
    for dtype in (E4M3, HALF):
        cache, table = _cache(gen, 1, 256, 32, 1, 64, dtype)
        q = _rand(gen, (1, 2, 1, 64), HALF)
        got = fa.forward_cached(q, cache, table, _ints(200), window=50, sinks=3)
        flat = table[0].long()
        for x in (cache.k, cache.v):
            raw = x.view(torch.uint8) if dtype == E4M3 else x.view(torch.int16)
            nan = 0x7F if dtype == E4M3 else 0x7E00
            for j in [*range(3, 150), *range(200, 256)]:
                raw[flat[j // 32], :, j % 32] = nan
        assert torch.equal(got, fa.forward_cached(q, cache, table, _ints(200), window=50, sinks=3))


def test_cached_infinite_scores_and_nan_stay_in_their_rows():
    gen = torch.Generator(DEV).manual_seed(14)
    cache, table = _cache(gen, 1, 64, 16, 2, 64, HALF)
    q = _rand(gen, (1, 2, 1, 64), HALF)
    q[0, 1] = math.nan
    got = fa.forward_cached(q, cache, table, _ints(64))
    assert torch.isfinite(got[0, 0]).all() and got[0, 1].isnan().all()


def test_cached_strided_queries_pools_and_streams():
    gen = torch.Generator(DEV).manual_seed(15)
    pool = _rand(gen, (9, 3, 2, 2, 16, 64), HALF)
    cache = fa.PagedKVCache(pool[:, 1, 0], pool[:, 2, 1])
    table = torch.randperm(9, generator=gen, device=DEV)[:8].to(torch.int32).view(2, 4)
    qkv = _rand(gen, (2, 3, 8, 64), HALF)
    q = qkv[:, :, :4].transpose(1, 2)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        _check_cached(q, cache, table, _ints(50, 64))
    torch.cuda.synchronize()


def test_cached_pages_beyond_32_bit_offsets():
    """A pool of more than 2^31 elements, its last page read."""
    pages = (1 << 31) // (64 * 128) + 64
    pool = [torch.zeros(pages, 1, 64, 128, dtype=torch.uint8, device=DEV).view(E4M3) for _ in "kv"]
    cache = fa.PagedKVCache(*pool, *(torch.ones(pages, 1, device=DEV) for _ in "kv"))
    gen = torch.Generator(DEV).manual_seed(16)
    k, v, q = (_rand(gen, (1, h, 64, 128), BF) for h in (1, 1, 2))
    table = _ints(pages - 1).view(1, 1)
    fa.append_kv(cache, k, v, table, _ints(64))
    _check_cached(q[:, :, -2:], cache, table, _ints(64))


def test_cached_outside_the_table_is_reported():
    gen = torch.Generator(DEV).manual_seed(17)
    cache, table = _cache(gen, 1, 64, 16, 1, 64, E4M3, spare=0)
    q = _rand(gen, (1, 1, 1, 64), HALF)
    bad = table.clone()
    bad[0, 1] = 99
    got = fa.forward_cached(q, cache, bad, _ints(64))
    assert _C.device_status(0) == 32 and torch.isfinite(got).all()
    got = fa.forward_cached(q, cache, table, _ints(100))  # longer than the table
    assert _C.device_status(0) == 32 and torch.isfinite(got).all()
    assert _C.device_status(0) == 0


def test_cached_in_a_graph_follows_the_lengths():
    gen = torch.Generator(DEV).manual_seed(18)
    cache, table = _cache(gen, 2, 512, 64, 2, 64, E4M3)
    q, lengths = _rand(gen, (2, 4, 1, 64), BF), _ints(1, 1)
    fa.forward_cached(q, cache, table, lengths)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = fa.forward_cached(q, cache, table, lengths)
    for a, b in ((3, 512), (400, 17)):
        lengths.copy_(_ints(a, b))
        graph.replay()
        assert torch.equal(out, fa.forward_cached(q, cache, table, lengths))


def test_append_then_attend_is_window_attention():
    """The two ways to the same numbers: a prompt appended and attended to over a 16-bit cache, and
    dense window attention."""
    gen = torch.Generator(DEV).manual_seed(19)
    q, k, v = (_rand(gen, (2, h, 90, 64), BF) for h in (4, 2, 2))
    cache, table = _cache(gen, 2, 90, 16, 2, 64, BF)
    cos, sin = _tables(64, 90)
    lengths = _ints(90, 90)
    turned = fa.append_kv(cache, k, v, table, lengths, cos=cos, sin=sin, q=q)
    kt = fa.append_kv(cache, k, v, table, lengths, cos=cos, sin=sin, q=k)
    got = fa.forward_cached(turned, cache, table, lengths, window=30, sinks=2)
    want = fa.forward_window(turned, kt, v, 30, 2)
    u = oracle.unit(BF)
    bound = 2 * oracle.forward_bound(want.double(), v.double().abs().max(), u, u)
    oracle.check(got, want.double(), bound, "O")


def test_cached_refusals():
    gen = torch.Generator(DEV).manual_seed(20)
    cache, table = _cache(gen, 2, 64, 16, 2, 64, E4M3)
    q, n = _rand(gen, (2, 4, 1, 64), HALF), _ints(5, 6)
    for error, match, call in (
        (ValueError, "multiple of kv_heads", lambda: fa.forward_cached(q[:, :3], cache, table, n)),
        (ValueError, "must not be negative", lambda: fa.forward_cached(q, cache, table, n, window=-1)),
        (ValueError, "finite", lambda: fa.forward_cached(q, cache, table, n, softmax_scale=math.inf)),
        (RuntimeError, "head dim", lambda: fa.forward_cached(q[..., :32], cache, table, n)),
        (RuntimeError, "float16", lambda: fa.forward_cached(q.float(), cache, table, n)),
        (RuntimeError, "int32", lambda: fa.forward_cached(q, cache, table[:1], n)),
        (RuntimeError, "16-bit cache", lambda: fa.forward_cached(q, fa.PagedKVCache.empty(4, 16, 2, 64, BF), table, n)),
        (ValueError, "power of two", lambda: fa.forward_cached(q, fa.PagedKVCache.empty(4, 512, 2, 64), table, n)),
    ):
        with pytest.raises(error, match=match):
            call()
