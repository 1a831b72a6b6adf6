"""Attention of trees of drafted tokens against the 64-bit definition; the bounds are derived in draft_oracle."""

import math
import random
import sys

import pytest
import torch

import draft_oracle as oracle
import fa
import stream_oracle
from fa import _C

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
HALF, BF, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _parents(batch, tokens, span, seed):
    rng = random.Random(seed)
    return _ints([[max(-1, i - rng.randint(1, span)) for i in range(tokens)] for _ in range(batch)])


ROOM = 0  # tokens that tables have places for behind the pages that they hold


@pytest.fixture(params=[0, 4200], ids=["short", "long"])
def room(request, monkeypatch):
    """What a table could hold decides how a call is cut and whether its rows come 128 or 256 at a time."""
    monkeypatch.setattr(sys.modules[__name__], "ROOM", request.param)


def _cache(gen, batch, most, page, heads, d, dtype, spare=2, low=0.004):
    per = max(1, -(-most // page))
    pages = batch * per + spare
    table = torch.randperm(pages, generator=gen, device=DEV)[: batch * per].to(torch.int32).view(batch, per)
    table = torch.cat((table, table.new_full((batch, ROOM // page), -1)), dim=1)
    x = [torch.randn(pages, heads, page, d, generator=gen, device=DEV).to(HALF) for _ in "kv"]
    if dtype != E4M3:
        return fa.PagedKVCache(*(t.to(dtype) for t in x)), table
    # Any positive scales, not powers of two alone.
    scales = [torch.rand(pages, heads, generator=gen, device=DEV) * 0.05 + low for _ in "kv"]
    codes = [(t.float() / s[..., None, None]).clamp(-448, 448).to(E4M3) for t, s in zip(x, scales)]
    return fa.PagedKVCache(*codes, *scales), table


def _check(q, cache, table, lengths, parents, status=0, **how):
    want, bound = oracle.tree(q, cache, table, lengths, parents, **how)
    kw = {("softmax_scale" if k == "scale" else k): v for k, v in how.items()}
    out = fa.forward_tree(q, cache, table, lengths, parents, **kw)
    assert out.is_contiguous() and out.dtype == q.dtype
    stream_oracle.check(out, want, bound, "o")
    assert _C.device_status(0, clear=True) == status
    return out


KINDS = [(HALF, HALF), (BF, BF), (HALF, E4M3), (BF, E4M3)]


@pytest.mark.usefixtures("room")
@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("group,hk,d,tokens,page,lengths,counts", [
    (1, 1, 64, 1, 16, [1, 2, 200], None),
    (4, 2, 128, 8, 64, [8, 9, 135, 136, 137, 1000], None),
    (3, 2, 64, 5, 8, [700, 5, 64, 333], [5, 0, 3, 1]),
    (4, 1, 128, 33, 32, [33, 160, 161, 2000], [33, 1, 33, 20]),
    (8, 2, 128, 64, 64, [64, 200, 3000], None),
    (2, 1, 64, 256, 256, [256, 300, 1500], [256, 255, 129]),
    (5, 1, 128, 100, 16, [99, 1000], [98, 100]),
    (16, 1, 64, 61, 128, [5000], None),
    (1, 3, 128, 129, 64, [129, 258], None),
])
def test_trees(group, hk, d, tokens, page, lengths, counts, dtype, kind):
    gen = torch.Generator(DEV).manual_seed(tokens)
    cache, table = _cache(gen, len(lengths), max(lengths), page, hk, d, kind)
    q = torch.randn(len(lengths), group * hk, tokens, d, generator=gen, device=DEV).to(dtype)
    for span in (1, 4, 300):
        parents = _parents(len(lengths), tokens, span, span)
        _check(q, cache, table, _ints(lengths), parents, counts=None if counts is None else _ints(counts))


@pytest.mark.usefixtures("room")
@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("group,tokens,window,sinks,lengths", [
    (4, 7, 7, 0, [7, 20, 300, 1000]), (4, 32, 130, 4, [40, 129, 600, 3000]), (1, 20, 20, 300, [100, 700, 320]), (2, 128, 1000, 1, [1128, 4000, 128]),
    (4, 64, 64, 17, [64, 65, 500, 81]), (2, 3, 1 << 30, 5, [800, 3]), (3, 70, 2300, 130, [2500, 70, 4100, 2400]),
])
def test_windows(group, tokens, window, sinks, lengths, dtype, kind):
    gen = torch.Generator(DEV).manual_seed(window)
    cache, table = _cache(gen, len(lengths), max(lengths), 32, 2, 128, kind)
    q = torch.randn(len(lengths), 2 * group, tokens, 128, generator=gen, device=DEV).to(dtype)
    _check(q, cache, table, _ints(lengths), _parents(len(lengths), tokens, 3, 1), window=window, sinks=sinks)


@pytest.mark.parametrize("dtype,kind", KINDS)
def test_a_long_context(dtype, kind):
    gen = torch.Generator(DEV).manual_seed(2)
    cache, table = _cache(gen, 2, 40001, 64, 1, 128, kind)
    for tokens in (2, 24, 77):
        q = torch.randn(2, 4, tokens, 128, generator=gen, device=DEV).to(dtype)
        _check(q, cache, table, _ints([40001, 29]), _parents(2, tokens, 5, 1), counts=_ints([tokens, min(tokens, 29)]))


@pytest.mark.usefixtures("room")
@pytest.mark.parametrize("dtype,kind", KINDS)
def test_many_short_sequences(dtype, kind):
    gen = torch.Generator(DEV).manual_seed(3)
    lengths = [12 + 37 * i % 190 for i in range(200)]
    cache, table = _cache(gen, 200, max(lengths), 16, 2, 64, kind)
    q = torch.randn(200, 4, 12, 64, generator=gen, device=DEV).to(dtype)
    _check(q, cache, table, _ints(lengths), _parents(200, 12, 4, 1))


@pytest.mark.parametrize("kind", [BF, E4M3])
def test_chains_are_cached_attention(kind):
    gen = torch.Generator(DEV).manual_seed(4)
    cache, table = _cache(gen, 2, 900, 32, 2, 64, kind)
    q = torch.randn(2, 8, 6, 64, generator=gen, device=DEV).to(BF)
    lengths, counts, chain = _ints([900, 411]), _ints([6, 4]), torch.arange(-1, 5, device=DEV, dtype=torch.int32)[None].expand(2, 6)
    out = _check(q, cache, table, lengths, chain, counts=counts)
    same = fa.forward_cached(q, cache, table, lengths, counts=counts)
    _, bound = oracle.tree(q, cache, table, lengths, chain, counts=counts)
    stream_oracle.check(out, same.double(), 2 * bound, "chain")
    assert not out[1, :, 4:].any()


def test_strides_scales_and_one_tree_for_all():
    gen = torch.Generator(DEV).manual_seed(5)
    both = torch.randn(12, 2, 2, 16, 64, generator=gen, device=DEV).to(BF)
    cache = fa.PagedKVCache(both[:, 0], both[:, 1])
    table = _ints([[3, 1, 4, 11, 5], [9, 2, 6, 0, 7]])[:, :4]
    qkv = torch.randn(2, 9, 10, 64, generator=gen, device=DEV).to(BF)
    q = qkv[:, :, 1:5].transpose(1, 2)
    parents = _parents(1, 9, 2, 0).expand(2, 9)
    for scale in (None, 0.0, -0.3, 2.0):
        _check(q, cache, table, _ints([64, 33]), parents, scale=scale)


@pytest.mark.usefixtures("room")
@pytest.mark.parametrize("tokens", [3, 40])
def test_scales_far_from_one(tokens):
    """Values' scales from 2^-100 to 2^60 in one sequence; the scores' stay where the softmax has a say."""
    gen = torch.Generator(DEV).manual_seed(6)
    cache, table = _cache(gen, 1, 600, 16, 1, 64, E4M3)
    q = torch.randn(1, 4, tokens, 64, generator=gen, device=DEV).to(BF)
    for low, high in ((-100, -70), (-66, -50), (-20, 60)):
        cache.v_scale = 2.0 ** torch.linspace(low, high, cache.num_pages, device=DEV)[:, None].contiguous()
        # bfloat16 holds 2^-126 and up; P and sums below 2^-126 of the largest vanish. (1e-6 less 1e-6 is no 1e-23.)
        least = 2.0**-120 * (1 + 2.0 ** (high + 8))
        want, bound = oracle.tree(q, cache, table, _ints([600]), _parents(1, tokens, 3, 0), least=least)
        out = fa.forward_tree(q, cache, table, _ints([600]), _parents(1, tokens, 3, 0))
        stream_oracle.check(out, want, bound, f"o {low}")


@pytest.mark.parametrize("dtype,kind", KINDS)
def test_large_scores(dtype, kind):
    gen = torch.Generator(DEV).manual_seed(7)
    cache, table = _cache(gen, 2, 500, 32, 1, 128, kind)
    q = 30 * torch.randn(2, 4, 20, 128, generator=gen, device=DEV).to(dtype)
    _check(q, cache, table, _ints([500, 77]), _parents(2, 20, 4, 0))


@pytest.mark.usefixtures("room")
@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("tokens,window", [(2, 0), (9, 16), (50, 0), (70, 128)])
def test_hidden_values_have_no_part(dtype, kind, tokens, window):
    """NaN and infinities in slots behind the sequences, before the window, in pages of nobody, and in nodes that
    others do not see: only the rows that see them show them."""
    gen = torch.Generator(DEV).manual_seed(8)
    lengths = [333, 200]
    cache, table = _cache(gen, 2, 400, 16, 2, 64, kind)
    q = torch.randn(2, 8, tokens, 64, generator=gen, device=DEV).to(dtype)
    parents = _parents(2, tokens, 6, 3)
    clean = fa.forward_tree(q, cache, table, _ints(lengths), parents, window=window)
    poison = [math.nan] if kind == E4M3 else [math.nan, math.inf, -math.inf]

    def put(b, position, value, head, dim):
        for x in (cache.k, cache.v):
            bits = x.view(torch.uint8) if kind == E4M3 else x
            bits[int(table[b, position // 16]), head, position % 16, dim] = 0x7F if kind == E4M3 else value

    for b, length in enumerate(lengths):
        for position in range(length, 400):
            put(b, position, poison[position % len(poison)], 0, position % 64)
        for position in range(0, max(0, length - tokens - window) if window else 0):
            put(b, position, poison[position % len(poison)], 1, slice(None))
    out = _check(q, cache, table, _ints(lengths), parents, window=window)
    assert torch.equal(out, clean)
    # In values of nodes (keys' would make rows NaN through their scores), one and several of a dim.
    nodes = sorted({tokens // 2, tokens - 1, 0 if tokens < 9 else 5})
    for n, node in enumerate(nodes):
        value = poison[n % len(poison)]
        bits = cache.v.view(torch.uint8) if kind == E4M3 else cache.v
        position = lengths[0] - tokens + node
        bits[int(table[0, position // 16]), 0, position % 16, 7 + (n > 1)] = 0x7F if kind == E4M3 else value
    want, bound = oracle.tree(q, cache, table, _ints(lengths), parents, window=window)
    out = fa.forward_tree(q, cache, table, _ints(lengths), parents, window=window)
    odd = ~torch.isfinite(want)
    assert odd.any() and not odd[1].any() and not odd[0, 4:].any()
    assert torch.equal(out[odd].nan_to_num(7.0), want[odd].to(dtype).nan_to_num(7.0))
    stream_oracle.check(torch.where(odd, 0.0, out.double()), torch.where(odd, 0.0, want), torch.where(odd, 1.0, bound), "beside")


@pytest.mark.usefixtures("room")
def test_infinite_and_nan_queries_stay_in_their_rows():
    gen = torch.Generator(DEV).manual_seed(9)
    for tokens in (3, 60):
        cache, table = _cache(gen, 1, 300, 16, 2, 64, BF)
        q = torch.randn(1, 4, tokens, 64, generator=gen, device=DEV).to(BF)
        parents = _parents(1, tokens, 6, 3)
        clean = fa.forward_tree(q, cache, table, _ints([300]), parents)
        q[0, 1, 2, 5] = math.nan
        q[0, 3, 1, 5] = math.inf
        out = fa.forward_tree(q, cache, table, _ints([300]), parents)
        assert torch.isnan(out[0, 1, 2]).all() and torch.isnan(out[0, 3, 1]).all()
        out[0, 1, 2] = clean[0, 1, 2]
        out[0, 3, 1] = clean[0, 3, 1]
        assert torch.equal(out, clean)


@pytest.mark.usefixtures("room")
@pytest.mark.parametrize("dtype", [HALF, BF])
@pytest.mark.parametrize("tokens", [3, 20, 60])
def test_infinite_queries_over_an_e4m3_cache(tokens, dtype):
    """e4m3 has no infinity: a row with one is NaN, as it is where the products are taken in 16 bits, and alone."""
    gen = torch.Generator(DEV).manual_seed(9)
    cache, table = _cache(gen, 1, 300, 16, 2, 128, E4M3)
    q = torch.randn(1, 8, tokens, 128, generator=gen, device=DEV).to(dtype)
    parents = _parents(1, tokens, 6, 3)
    clean = fa.forward_tree(q, cache, table, _ints([300]), parents)
    q[0, 1, 2, 5], q[0, 6, 1, 100], q[0, 7, 0, 0] = math.inf, -math.inf, math.nan
    out = fa.forward_tree(q, cache, table, _ints([300]), parents)
    for h, t in ((1, 2), (6, 1), (7, 0)):
        assert torch.isnan(out[0, h, t]).all()
        out[0, h, t] = clean[0, h, t]
    assert torch.equal(out, clean)


@pytest.mark.usefixtures("room")
@pytest.mark.parametrize("dtype,kind", KINDS)
def test_tiny_and_zero_queries_and_scales(dtype, kind):
    """Rows of zeros and of values at the small end of their type weigh what they see alike, or as little apart."""
    gen = torch.Generator(DEV).manual_seed(10)
    cache, table = _cache(gen, 1, 300, 32, 1, 64, kind)
    for tokens in (4, 40):
        q = torch.randn(1, 4, tokens, 64, generator=gen, device=DEV).to(dtype)
        q[0, 0], q[0, 1, 0], q[0, 2] = 0.0, torch.finfo(dtype).tiny, q[0, 2] * 2.0**-12
        if kind == E4M3:
            cache.v_scale[int(table[0, 2])] = 0.0
            cache.k_scale[int(table[0, 4])] = 0.0
        _check(q, cache, table, _ints([300]), _parents(1, tokens, 3, 0))


@pytest.mark.parametrize("tokens", [4, 50])
def test_bad_parents_pages_and_lengths(tokens):
    gen = torch.Generator(DEV).manual_seed(10)
    cache, table = _cache(gen, 3, 320, 16, 2, 64, E4M3)
    q = torch.randn(3, 8, tokens, 64, generator=gen, device=DEV).to(BF)
    parents = _parents(3, tokens, 3, 0)
    parents[1, 2], parents[2, 3], parents[2, 1] = 2, 2**31 - 1, -(2**31)
    _check(q, cache, table, _ints([300, 200, 100]), parents, status=32)
    # What is behind counts[b] is not looked at.
    _check(q, cache, table, _ints([300, 200, 100]), parents, counts=_ints([tokens, 2, 1]))
    good = _parents(3, tokens, 3, 0)
    table[0, 3], table[1, 0], table[2, 2] = -1, cache.num_pages, 2**31 - 1
    _check(q, cache, table, _ints([300, 200, 100]), good, status=32)
    # More tokens than the table has places, more nodes than tokens, lengths at the ends of their type.
    cache, table = _cache(gen, 3, 320, 16, 2, 64, E4M3)
    _check(q, cache, table, _ints([320 + tokens // 2, 400 + tokens, 2]), good, status=32)
    out = fa.forward_tree(q, cache, table, _ints([2**31 - 1, -(2**31), 0]), good, window=300)
    assert torch.isfinite(out).all() and not out[1:].any() and _C.device_status(0, clear=True) == 32


def test_pages_beyond_32_bits():
    """A pool whose last pages begin beyond 2^31 elements."""
    pages = (1 << 31) // (256 * 64) + 40
    k = torch.zeros(pages, 1, 256, 64, dtype=torch.uint8, device=DEV).view(E4M3)
    v = torch.zeros(pages, 1, 256, 64, dtype=torch.uint8, device=DEV).view(E4M3)
    gen = torch.Generator(DEV).manual_seed(11)
    for x in (k, v):
        x[-4:] = torch.randn(4, 1, 256, 64, generator=gen, device=DEV).to(E4M3)
    ones = torch.ones(pages, 1, device=DEV)
    cache, table = fa.PagedKVCache(k, v, ones, ones), _ints([[pages - 1, pages - 3, pages - 4]])
    small = fa.PagedKVCache(k[-4:], v[-4:], ones[-4:], ones[-4:])
    q = torch.randn(1, 4, 30, 64, generator=gen, device=DEV).to(HALF)
    parents = _parents(1, 30, 4, 0)
    out = fa.forward_tree(q, cache, table, _ints([700]), parents)
    assert torch.equal(out, fa.forward_tree(q, small, table - (pages - 4), _ints([700]), parents))
    _check(q, small, table - (pages - 4), _ints([700]), parents)
    fa.copy_pages(cache, _ints([pages - 1]), _ints([5]))
    assert torch.equal(k[5].view(torch.uint8), k[-1].view(torch.uint8))
    fa.keep_tokens(cache, table, _ints([700]), _ints([[3, 7]]), 30)
    fa.keep_tokens(small, table - (pages - 4), _ints([700]), _ints([[3, 7]]), 30)
    assert _C.device_status(0, clear=True) == 0


def test_same_bits_every_time_and_in_a_graph():
    gen = torch.Generator(DEV).manual_seed(12)
    for tokens, kind in ((4, E4M3), (48, E4M3), (48, BF), (90, BF)):
        cache, table = _cache(gen, 3, 3000, 64, 2, 128, kind)
        q = torch.randn(3, 8, tokens, 128, generator=gen, device=DEV).to(BF)
        lengths, parents = _ints([3000, 100, 1700]), _parents(3, tokens, 5, 0)
        first = fa.forward_tree(q, cache, table, lengths, parents, window=1000, sinks=4)
        for _ in range(3):
            assert torch.equal(first, fa.forward_tree(q, cache, table, lengths, parents, window=1000, sinks=4))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            out = fa.forward_tree(q, cache, table, lengths, parents, window=1000, sinks=4)
        graph.replay()
        assert torch.equal(out, first)
        lengths.copy_(_ints([200, 2999, 95]))
        parents.copy_(_parents(3, tokens, 2, 7))
        graph.replay()
        want, bound = oracle.tree(q, cache, table, lengths, parents, window=1000, sinks=4)
        stream_oracle.check(out, want, bound, "replayed")
        # Two streams at once, each with its workspace.
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        here = [fa.forward_tree(q, cache, table, lengths, parents, window=1000, sinks=4) for _ in range(4)]
        with torch.cuda.stream(side):
            there = [fa.forward_tree(q, cache, table, lengths, parents, window=1000, sinks=4) for _ in range(4)]
        torch.cuda.synchronize()
        assert all(torch.equal(x, out) for x in here + there)


def test_empty_and_refused():
    cache, table = _cache(torch.Generator(DEV).manual_seed(0), 1, 32, 16, 2, 64, BF)
    q, lengths, parents = torch.zeros(1, 4, 3, 64, device=DEV, dtype=BF), _ints([20]), _ints([[-1, 0, 1]])
    assert fa.forward_tree(q[:, :, :0], cache, table, lengths, parents[:, :0]).shape == (1, 4, 0, 64)
    for bad, match in ((lambda: fa.forward_tree(q, cache, table, lengths, parents[:, :2]), "every node"), (lambda: fa.forward_tree(q, cache, table, lengths, parents.long()), "parents"),
                       (lambda: fa.forward_tree(q, cache, table, lengths, parents.cpu()), "parents"), (lambda: fa.forward_tree(q, cache, table, lengths, _ints([[0], [1], [2]]).mT.repeat(1, 2)[:, ::2]), "contiguous rows"),
                       (lambda: fa.forward_tree(q.half(), cache, table, lengths, parents), "same dtype"), (lambda: fa.forward_tree(q, cache, table, lengths.long(), parents), "lengths")):
        with pytest.raises(RuntimeError, match=match):
            bad()
    wide = fa.PagedKVCache(cache.k[:1].expand(3, 2, 16, 64), cache.v[:1].expand(3, 2, 16, 64))
    for bad, match in ((lambda: fa.forward_tree(q, wide, table, lengths, parents), "strides must be positive"),
                       (lambda: fa.forward_tree(q, cache, table, lengths, parents, window=2), "at least the number"), (lambda: fa.forward_tree(q[:, :3], cache, table, lengths, parents), "multiple of kv_heads"),
                       (lambda: fa.forward_tree(q, cache, table, lengths, parents, sinks=-1), "negative"), (lambda: fa.forward_tree(q, cache, table, lengths, parents, window=2**40), "32-bit"),
                       (lambda: fa.forward_tree(q.repeat(1, 1, 100, 1), cache, table, lengths, parents.repeat(1, 100)), "at most 256"),
                       (lambda: fa.forward_tree(q, cache, table, lengths, parents, softmax_scale=math.nan), "finite")):
        with pytest.raises(ValueError, match=match):
            bad()
