"""The streaming operators at the edges of their contracts: a cache whose tensors are replaced, and
what else a caller may do or bring that the ordinary cases do not show."""

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


def _rand(gen, shape, dtype, scale=1.0):
    return (torch.randn(shape, generator=gen, device=DEV) * scale).to(dtype)


def _bytes(t):
    return t.view(torch.uint8)


# ------------------------------------------------------------------------------------ the cache


def _grown(t, more):
    """t with `more` pages of zeros after its own."""
    new = torch.cat([_bytes(t), torch.zeros((more, *_bytes(t).shape[1:]), dtype=torch.uint8, device=DEV)])
    return new.view(t.dtype)


@pytest.mark.parametrize("dtype", [E4M3, HALF])
def test_cache_follows_tensors_that_are_replaced(dtype):
    """A pool that grows, one that is moved to other memory under the same tensor: what was there is
    neither read nor written any more. (The old tensors stay alive here.)"""
    gen = torch.Generator(DEV).manual_seed(1)
    cache = fa.PagedKVCache.empty(2, 16, 2, 64, dtype=dtype, device=DEV)
    k, v, q = (_rand(gen, (1, h, 40, 64), HALF) for h in (2, 2, 4))
    fa.append_kv(cache, k[:, :, :32], v[:, :, :32], _ints(1, 0).view(1, 2), _ints(32))
    old = [t for t in (cache.k, cache.v, cache.k_scale, cache.v_scale) if t is not None]
    was = [_bytes(t).clone() for t in old]

    cache.k = _grown(cache.k, 1)
    assert cache.num_pages == 3
    with pytest.raises(RuntimeError, match="same shape"):  # v has not followed yet
        fa.append_kv(cache, k[:, :, 32:], v[:, :, 32:], _ints(1, 0, 2).view(1, 3), _ints(40))
    cache.v = _grown(cache.v, 1)
    if dtype == E4M3:
        cache.k_scale, cache.v_scale = (torch.cat([s, torch.ones(1, 2, device=DEV)]) for s in (cache.k_scale, cache.v_scale))
    table = _ints(1, 0, 2).view(1, 3)
    fa.append_kv(cache, k[:, :, 32:], v[:, :, 32:], table, _ints(40))
    whole = fa.PagedKVCache.empty(3, 16, 2, 64, dtype=dtype, device=DEV)
    fa.append_kv(whole, k, v, table, _ints(40))
    assert torch.equal(_bytes(cache.k), _bytes(whole.k)) and torch.equal(_bytes(cache.v), _bytes(whole.v))
    assert torch.equal(fa.forward_cached(q[:, :, -1:], cache, table, _ints(40)), fa.forward_cached(q[:, :, -1:], whole, table, _ints(40)))
    assert all(torch.equal(_bytes(t), w) for t, w in zip(old, was))

    moved = cache.k.data
    was = _bytes(moved).clone()
    cache.k.data = _bytes(cache.k).clone().view(dtype)
    fa.append_kv(cache, -k[:, :, :8], v[:, :, :8], table, _ints(8))
    fa.append_kv(whole, -k[:, :, :8], v[:, :, :8], table, _ints(8))
    assert torch.equal(_bytes(moved), was) and torch.equal(_bytes(cache.k), _bytes(whole.k))
    assert _C.device_status(0) == 0


def _filled(gen, batch, pages, page, heads, d, dtype):
    """A cache of values near 1 and a table of all its pages, in random order."""
    table = torch.randperm(batch * pages, generator=gen, device=DEV).to(torch.int32).view(batch, pages)
    k, v = (_rand(gen, (batch * pages, heads, page, d), HALF).to(dtype) for _ in "kv")
    scales = (torch.ones(batch * pages, heads, device=DEV) for _ in "kv") if dtype == E4M3 else (None, None)
    return fa.PagedKVCache(k, v, *scales), table


@pytest.mark.parametrize("dtype", [E4M3, HALF])
@pytest.mark.parametrize("page,pages", [(8, 3), (16, 4), (64, 20)])
@pytest.mark.parametrize("window,sinks", [(0, 0), (30, 0), (30, 5), (5000, 40)])
def test_lengths_beyond_the_table_end_with_it(page, pages, window, sinks, dtype):
    """A length that the table has no place for costs no more than the table's own, and what the table has of
    its view is attended to; the other sequences are as they would be."""
    gen = torch.Generator(DEV).manual_seed(2)
    cache, table = _filled(gen, 6, pages, page, 2, 64, dtype)
    most = page * pages
    q = _rand(gen, (6, 4, 2, 64), HALF)
    lengths = _ints(most, most + 1, most + 20, 2**31 - 1, -(2**31), 7)
    got = fa.forward_cached(q, cache, table, lengths, window=window, sinks=sinks)
    assert _C.device_status(0, clear=True) == 32
    lengths = lengths.clamp(min=0)
    want, vmax = oracle.cached(q, cache, table, lengths, None, window, sinks)
    oracle.check(got, want, oracle.forward_bound(want, vmax, oracle.unit(HALF), oracle.unit(HALF)), "O")


@pytest.mark.parametrize("length", [2**31 - 1, 2**31 - 17, -(2**31), -1])
@pytest.mark.parametrize("page", [8, 64])
def test_append_at_the_ends_of_the_integers_is_skipped_and_reported(length, page):
    """Lengths that no table has a place for, at the ends of their type: nothing is stored for them, the bit is set,
    and the other sequence is as it would be."""
    gen = torch.Generator(DEV).manual_seed(3)
    cache = fa.PagedKVCache(*(torch.zeros(6, 1, page, 64, dtype=HALF, device=DEV) for _ in "kv"))
    k = _rand(gen, (2, 1, 20, 64), HALF)
    table = _ints(0, 1, 2, 3, 4, 5).view(2, 3)
    fa.append_kv(cache, k, k, table, _ints(length, 20))
    assert _C.device_status(0, clear=True) == 32
    for pool in (cache.k, cache.v):
        assert not pool[:3].any() and torch.equal(oracle.dense(pool, None, table)[1, :, :20], k[1].double())


# ------------------------------------------------------------------------------ window attention


def _dense(b, h, hk, nq, nk, d, dtype, seed):
    gen = torch.Generator(DEV).manual_seed(seed)
    return tuple(_rand(gen, s, dtype) for s in ((b, h, nq, d), (b, hk, nk, d), (b, hk, nk, d), (b, h, nq, d)))


def _step(q, k, v, do, window, sinks):
    o, lse = fa.forward_window(q, k, v, window, sinks, return_lse=True)
    return (o, lse, *fa.backward_window(do, q, k, v, o, lse, window, sinks))


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("big", [3e38, -3e38])
def test_bf16_hidden_values_weigh_nothing(d, big):
    """Later keys, and keys before the window, that share a tile with visible ones: values at the end of
    bfloat16's range do not move a row that does not see them by a bit."""
    q, k, v, _ = _dense(1, 2, 2, 400, 400, d, BF, seed=3)
    for window, sinks in ((40, 0), (40, 3), (0, 0)):
        o, lse = fa.forward_window(q, k, v, window, sinks, return_lse=True)
        later, k2 = v.clone(), k.clone()
        later[:, :, 200:], k2[:, :, 200:] = big, 1e30
        o2, lse2 = fa.forward_window(q, k2, later, window, sinks, return_lse=True)
        assert torch.equal(o[:, :, :200], o2[:, :, :200]) and torch.equal(lse[:, :, :200], lse2[:, :, :200])
        if window:
            before = v.clone()
            before[:, :, sinks:200] = big
            assert torch.equal(o[:, :, 239:], fa.forward_window(q, k, before, window, sinks)[:, :, 239:])


@pytest.mark.parametrize("d", [64, 128])
def test_bf16_gradients_of_hidden_pairs_are_zero(d):
    """Hidden values of 1e36 (their products with dO stay finite) leave the gradients of rows and keys that have no
    part in them as they are; keys that no query sees, and rows that see nothing, have gradients of 0."""
    q, k, v, do = _dense(1, 2, 1, 400, 400, d, BF, seed=4)
    plain = _step(q, k, v, do, 40, 0)
    v2 = v.clone()
    v2[:, :, 200:] = 1e36
    other = _step(q, k, v2, do, 40, 0)
    assert torch.equal(plain[2][:, :, :200], other[2][:, :, :200])  # dQ
    assert torch.equal(plain[3][:, :, :161], other[3][:, :, :161])  # dK: key 160 is seen up to row 199
    assert torch.equal(plain[4][:, :, :161], other[4][:, :, :161])  # dV

    q, k, v, do = _dense(1, 2, 1, 100, 700, d, BF, seed=5)
    _, _, _, dk, dv = _step(q, k, v, do, 64, 4)
    assert not dk[:, :, 4:537].any() and not dv[:, :, 4:537].any() and dk[:, :, 537:].any()

    q, k, v, do = _dense(1, 2, 1, 500, 100, d, BF, seed=6)  # rows up to 399 see nothing
    o, lse, dq, dk, dv = _step(q, k, v, do, 50, 0)
    assert not o[:, :, :400].any() and (lse[:, :, :400] == -math.inf).all() and not dq[:, :, :400].any()
    do[:, :, :400] = 1e36
    again = fa.backward_window(do, q, k, v, o, lse, 50, 0)
    assert torch.equal(again[1], dk) and torch.equal(again[2], dv) and not again[0][:, :, :400].any()


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [HALF, BF])
def test_nan_in_a_key_reaches_every_row_that_sees_it(d, dtype):
    """Whatever column of a tile the key is in: 2^x is computed in two ways, by columns."""
    q, k, v, do = _dense(1, 2, 1, 300, 300, d, dtype, seed=7)
    window = 100
    plain = _step(q, k, v, do, window, 0)
    for key in range(130, 146):
        bad = k.clone()
        bad[0, 0, key, 5] = math.nan
        o, lse, dq, dk, dv = _step(q, bad, v, do, window, 0)
        sees = slice(key, key + window)
        assert o[:, :, sees].isnan().all() and lse[:, :, sees].isnan().all(), key
        for x, y in ((o, plain[0]), (lse, plain[1])):
            assert torch.equal(x[:, :, :key], y[:, :, :key]) and torch.equal(x[:, :, key + window :], y[:, :, key + window :])
        assert dq[:, :, sees].isnan().all(), key
        # Their keys: those rows' P is NaN.
        keys = slice(key - window + 1, key + window)
        assert dk[:, :, keys].isnan().all() and dv[:, :, keys].isnan().all(), key


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [HALF, BF])
def test_nan_in_a_key_of_the_dense_forward(d, dtype):
    q, k, v, _ = _dense(1, 2, 2, 600, 600, d, dtype, seed=8)
    plain = fa.forward(q, k, v, causal=True)
    for key in (*range(260, 276), 599):
        bad = k.clone()
        bad[0, :, key, 3] = math.nan
        o = fa.forward(q, bad, v, causal=True)
        assert o[:, :, key:].isnan().all() and torch.equal(o[:, :, :key], plain[:, :, :key]), key
        assert fa.forward(q, bad, v).isnan().all(), key
        assert fa.forward_splitkv(q, bad, v, num_splits=3).isnan().all(), key
        if dtype == HALF:
            for variant in ("baseline", "fp16acc"):
                assert fa.forward_variant(q, bad, v, variant=variant).isnan().all(), (variant, key)


def test_a_graph_of_the_gradients_may_be_asked_for():
    """create_graph for another part's sake: the gradients are the same, and only differentiating them again
    through the attention is refused."""
    q, k, v, do = _dense(1, 2, 1, 64, 64, 64, HALF, seed=9)
    for t in (q, k, v):
        t.requires_grad_(True)
    o = fa.window_attention(q, k, v, 20)
    plain = torch.autograd.grad(o, (q, k, v), do, retain_graph=True)
    again = torch.autograd.grad(o, (q, k, v), do, create_graph=True)
    assert all(torch.equal(a, b) for a, b in zip(plain, again))
    other = torch.ones(3, device=DEV, requires_grad=True)  # a penalty on another part's gradient
    slope = torch.autograd.grad((o.float().sum() * 0 + (other**3).sum()), (q, other), create_graph=True)[1]
    assert torch.equal(torch.autograd.grad(slope.sum(), other)[0], 6 * other.detach())
    with pytest.raises(RuntimeError, match="differentiated once"):
        again[0].sum().backward()


# ------------------------------------------------------------------------- several tokens at once


@pytest.mark.parametrize("dtype,cache_dtype", [(BF, E4M3), (HALF, E4M3), (BF, BF), (HALF, HALF)])
@pytest.mark.parametrize("h,hk,t,page", [(4, 4, 4, 64), (16, 2, 4, 16), (8, 2, 3, 8), (2, 1, 20, 32), (3, 1, 37, 64)])
@pytest.mark.parametrize("d", [64, 128])
def test_values_that_are_not_finite_stay_with_the_rows_that_see_them(dtype, cache_dtype, h, hk, t, page, d):
    """Of a later drafted token, and of a key that only the first tokens' windows still hold: an infinite or
    NaN value makes its own column infinite or NaN in the rows that see it, and changes nothing else."""
    gen = torch.Generator(DEV).manual_seed(10 + t)
    pages = -(-150 // page)
    cache, table = _filled(gen, 2, pages, page, hk, d, cache_dtype)
    q = _rand(gen, (2, h, t, d), dtype)
    lengths = _ints(150, 90 + t)
    first = (lengths - t).tolist()
    raw = cache.v.view(torch.uint8 if cache_dtype == E4M3 else torch.int16)
    codes = {E4M3: (0x7F, 0xFF), HALF: (0x7E00, 0x7C00), BF: (0x7FC0, 0x7F80)}[cache_dtype]
    for window, sinks in ((0, 0), (40, 3)):
        plain = fa.forward_cached(q, cache, table, lengths, window=window, sinks=sinks)
        assert torch.isfinite(plain).all()
        for which, offset in enumerate((t - 1, 1, 1 - window) if window else (t - 1, 1)):
            keys = [f + offset for f in first]
            where = [(int(table[b, k // page]), k % page) for b, k in enumerate(keys)]
            column = 5 + 16 * which
            was = [raw[at, :, slot, column].clone() for at, slot in where]
            for (at, slot) in where:
                raw[at, :, slot, column] = codes[which % 2]
            got = fa.forward_cached(q, cache, table, lengths, window=window, sinks=sinks)
            want = plain.clone()
            for b, k in enumerate(keys):
                pos = first[b] + torch.arange(t, device=DEV)
                sees = (k <= pos) & ((pos - k < window) if window else torch.ones_like(pos, dtype=torch.bool))
                assert sees.any() and not sees.all()
                bad = ~torch.isfinite(got[b, :, sees, column])
                assert bad.all()
                want[b, :, sees, column] = got[b, :, sees, column]
            same = (got == want) | (got.isnan() & want.isnan())
            assert same.all(), (window, which)
            for (at, slot), x in zip(where, was):
                raw[at, :, slot, column] = x
    assert _C.device_status(0) == 0


def test_scores_of_a_later_token_that_are_nan_stay_with_it():
    gen = torch.Generator(DEV).manual_seed(11)
    cache, table = _filled(gen, 1, 3, 64, 2, 128, E4M3)
    q = _rand(gen, (1, 8, 4, 128), BF)
    plain = fa.forward_cached(q, cache, table, _ints(130))
    cache.k.view(torch.uint8)[int(table[0, 2]), :, 1, 9] = 0x7F  # position 129, the last token's
    got = fa.forward_cached(q, cache, table, _ints(130))
    assert torch.equal(got[:, :, :3], plain[:, :, :3]) and got[:, :, 3].isnan().all()


# ------------------------------------------------------------------------- bfloat16 queries, e4m3 keys


@pytest.mark.parametrize("d", [64, 128])
def test_bf16_queries_of_mixed_size_over_e4m3(d):
    """A row whose values are up to 2^30 apart, the small ones meeting large keys: they are in the scores in full.
    From 2^-38 on they are not there, and nothing else happens."""
    gen = torch.Generator(DEV).manual_seed(12)
    k = (torch.randn(2, 1, 64, d, generator=gen, device=DEV) * 64).to(E4M3)
    k[..., 0] = 0
    v = _rand(gen, (2, 1, 64, d), HALF).to(E4M3)
    table, lengths = _ints(0, 1).view(1, 2), _ints(100)
    for power, exact in ((-20, True), (-29, True), (-30, True), (-40, False)):
        # the small queries' scores are of the order of 1 whatever their size
        scale = torch.full((2, 1), 2.0 ** (-power - 6), device=DEV)
        cache = fa.PagedKVCache(k, v, scale, torch.ones(2, 1, device=DEV))
        q = torch.zeros(1, 2, 1, d, dtype=BF, device=DEV)
        q[..., 0] = 1.0
        q[:, 0, :, 1:9] = 1.9921875 * 2.0**power
        q[:, 1, :, 1:9] = -1.0078125 * 2.0**power
        got = fa.forward_cached(q, cache, table, lengths)
        want, vmax = oracle.cached(q if exact else torch.zeros_like(q), cache, table, lengths)
        oracle.check(got, want, oracle.forward_bound(want, vmax, oracle.unit(HALF), oracle.unit(BF)), f"O at 2^{power}")


# ------------------------------------------------------------------------------------ arguments


@pytest.mark.parametrize("change", [{"window": 1 << 31}, {"sinks": 1 << 40}, {"window": 2.5}])
def test_arguments_beyond_their_types_are_refused(change):
    """In the library's manner: an error that says what is wrong with which argument."""
    q, k, v, do = _dense(1, 2, 1, 16, 16, 64, HALF, seed=13)
    cache = fa.PagedKVCache.empty(1, 16, 1, 64, device=DEV)
    args = {"window": 4, "sinks": 1} | change
    o, lse = fa.forward_window(q, k, v, 4, return_lse=True)
    for call in (lambda: fa.forward_window(q, k, v, **args), lambda: fa.backward_window(do, q, k, v, o, lse, **args),
                 lambda: fa.forward_cached(q[:, :, :1], cache, _ints(0).view(1, 1), _ints(5), **args)):
        with pytest.raises(ValueError, match="32-bit"):
            call()
