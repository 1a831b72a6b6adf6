"""Tree and cached attention against 64 bits within the bound that tree_bound derives from what the kernels round."""

import math
import random

import pytest
import torch

import draft_oracle
import fa
import stream_oracle
import tree_bound
from fa import _C

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
HALF, BF, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn
KINDS = [(HALF, HALF), (BF, BF), (HALF, E4M3), (BF, E4M3)]
# Query rows of a kv head of 4 query heads: the cached attention's kernel, one row tile, two.
NODES = [3, 20, 70]


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


def _parents(batch, tokens, span, seed):
    rng = random.Random(seed)
    return _ints([[max(-1, i - rng.randint(1, span)) for i in range(tokens)] for _ in range(batch)])


def _cache(gen, batch, most, page, heads, d, dtype, room=0):
    """Unit normals; `room` places of a table behind the pages that it holds. Every second page of the pool is used."""
    per = -(-most // page)
    table = (2 * torch.randperm(batch * per, generator=gen, device=DEV)).to(torch.int32).view(batch, per)
    table = torch.cat((table, table.new_full((batch, room // page), -1)), dim=1)
    x = [torch.randn(2 * batch * per, heads, page, d, generator=gen, device=DEV) for _ in "kv"]
    if dtype != E4M3:
        return fa.PagedKVCache(*(t.to(dtype) for t in x)), table
    scales = [torch.rand(t.shape[:2], generator=gen, device=DEV) * 0.05 + 0.004 for t in x]
    codes = [(t / s[..., None, None]).clamp(-448, 448).to(E4M3) for t, s in zip(x, scales)]
    return fa.PagedKVCache(*codes, *scales), table


def _check(q, cache, table, lengths, parents, what="o", **how):
    held = -(-int(lengths.max()) // cache.page_size)
    want, bound = tree_bound.tree(q, cache, table[:, :held], lengths, parents, **how)
    kw = {("softmax_scale" if k == "scale" else k): v for k, v in how.items()}
    out = fa.forward_tree(q, cache, table, lengths, parents, **kw)
    stream_oracle.check(out, want, bound, what)
    assert _C.device_status(0, clear=True) == 0
    return out


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("room", [0, 131072], ids=["narrow", "wide"])
@pytest.mark.parametrize("tokens", NODES)
@pytest.mark.parametrize("page,d", [(8, 64), (16, 128), (64, 128)])
def test_trees(page, d, tokens, room, dtype, kind):
    gen = torch.Generator(DEV).manual_seed(page + tokens)
    lengths, parents = [1000, tokens, 333], _parents(3, tokens, 4, tokens)
    cache, table = _cache(gen, 3, 1000, page, 2, d, kind, room)
    q = torch.randn(3, 8, tokens, d, generator=gen, device=DEV).to(dtype)
    for window, sinks in ((0, 0), (100, 9)):
        _check(q, cache, table, _ints(lengths), parents, window=window, sinks=sinks)


MANY = 320  # sequences with the same pages: so many that most of them are not cut, and a maximum stays theirs throughout


def _check_many(q, cache, table, length, parents, scale):
    """One sequence's answer from 64 bits, MANY from the kernels."""
    want, bound = tree_bound.tree(q, cache, table, _ints([length]), parents, scale=scale)
    of_all = [x.repeat(MANY, *[1] * (x.dim() - 1)) for x in (q, table, _ints([length]), parents)]
    out = fa.forward_tree(of_all[0], cache, *of_all[1:], softmax_scale=scale)
    for b in range(MANY):
        stream_oracle.check(out[b : b + 1], want, bound, f"sequence {b}")
    tokens = q.shape[2]
    if tokens <= 4:
        chain = torch.arange(-1, tokens - 1, device=DEV, dtype=torch.int32)[None]
        want, bound = tree_bound.tree(q, cache, table, _ints([length]), chain, scale=scale)
        out = fa.forward_cached(of_all[0], cache, *of_all[1:3], softmax_scale=scale)
        for b in range(MANY):
            stream_oracle.check(out[b : b + 1], want, bound, f"cached, sequence {b}")
    assert _C.device_status(0, clear=True) == 0
    return want


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("tokens", [1, 2] + NODES[1:])
def test_a_long_tail_beside_a_sink(tokens, dtype, kind):
    """One key, whose value is 0, outweighs every other by 14 to 17 nats; 33000 of those together are the answer."""
    gen = torch.Generator(DEV).manual_seed(2)
    cache, table = _cache(gen, 1, 33000, 64, 1, 64, kind)
    values = torch.randint(4, 13, cache.v.shape, generator=gen, device=DEV) / 8
    if kind == E4M3:
        cache.k_scale.fill_(1.0)
        cache.v_scale.fill_(1.0)
    bits = (lambda x: x.view(torch.uint8)) if kind == E4M3 else (lambda x: x)
    bits(cache.k).zero_()
    bits(cache.v).copy_(bits(values.to(kind)))
    first = int(table[0, 0])
    bits(cache.k)[first, 0, 0] = bits(torch.ones(64, device=DEV).to(kind))
    bits(cache.v)[first, 0, 0] = 0
    # Row (h, t) puts the sink 14 + h + (t % 4) / 16 nats above the others: 64 q_d k_d / 64.
    h, t = torch.arange(4, device=DEV)[:, None, None], torch.arange(tokens, device=DEV)[:, None] % 4
    q = (14.0 + h + t / 16.0).expand(4, tokens, 64)[None].to(dtype)
    want = _check_many(q, cache, table, 33000, _parents(1, tokens, 3, 0), 1 / 64)
    assert (want > 4e-4).all() and (want < 0.1).all()


@pytest.mark.parametrize("tokens", NODES)
def test_a_tail_of_other_scales(tokens):
    """The same where the tail's pages have smaller and larger value scales than the sink's."""
    gen = torch.Generator(DEV).manual_seed(3)
    cache, table = _cache(gen, 1, 20000, 32, 1, 128, E4M3)
    cache.v_scale = 2.0 ** torch.randint(-6, 3, cache.v_scale.shape, generator=gen, device=DEV).float()
    cache.k.view(torch.uint8).zero_()
    cache.k_scale.fill_(1.0)
    first = int(table[0, 0])
    cache.k.view(torch.uint8)[first, 0, 0] = torch.ones(128, device=DEV).to(E4M3).view(torch.uint8)
    cache.v.view(torch.uint8)[first, 0, 0] = 0
    q = torch.linspace(13, 17, 4 * tokens, device=DEV).view(1, 4, tokens, 1).expand(1, 4, tokens, 128).to(BF)
    _check_many(q, cache, table, 20000, _parents(1, tokens, 3, 0), 1 / 128)


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("tokens", NODES)
def test_scores_beyond_whole_numbers(tokens, dtype, kind):
    """Scores of 2^14 to 2^26, whose own steps reach 2: a key that is far above the others is all of the answer."""
    gen = torch.Generator(DEV).manual_seed(8)
    cache, table = _cache(gen, 2, 700, 16, 1, 64, kind)
    lengths, parents = _ints([700, 300]), _parents(2, tokens, 3, 0)
    q = torch.randn(2, 4, tokens, 64, generator=gen, device=DEV).to(dtype)
    k, v = (stream_oracle.dense(x, s, table)[:, :, None] for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    seen = draft_oracle.tree_mask(parents.cpu(), [700, 300], [tokens, tokens], k.shape[3], 0, 0).to(DEV)
    s = torch.where(seen[:, None, None], q.double()[:, None] @ k.mT, -math.inf)
    # Scores are off by less than D 2^-23 of |q||k|, 30 nats are nothing beside the largest: a gap of 2^-10 |q||k| stands.
    top, at = s.topk(2, -1)
    clear = (top[..., 0] - top[..., 1] > 2.0**-10 * q.double().norm(dim=-1)[:, None] * k.norm(dim=-1).max())[:, 0]
    assert clear.double().mean() > 0.8
    want = v[:, 0, 0].gather(1, at[:, 0, ..., 0].reshape(2, -1, 1).expand(-1, -1, 64)).view(2, 4, tokens, 64)
    for power in range(10, 23):
        out = fa.forward_tree(q, cache, table, lengths, parents, softmax_scale=2.0**power)
        stream_oracle.check(out[clear], want[clear], 2.0**-7 * want[clear].abs() + 1e-6, f"2^{power}")


@pytest.mark.parametrize("kind", [BF, E4M3])
@pytest.mark.parametrize("tokens", [1] + NODES)
def test_bfloat16_queries_far_beyond_float16(tokens, kind):
    """Largest elements from 2^100 to 2^121 in rows whose scores are about 1: the others are beside them as they are."""
    gen = torch.Generator(DEV).manual_seed(4)
    cache, table = _cache(gen, 1, 500, 16, 1, 64, kind)
    x = torch.randn(1, 4, tokens, 64, generator=gen, device=DEV).clamp(-3.9, 3.9)
    for power in (100, 108, 112, 119):
        q = (x * 2.0**power).to(BF)
        q[..., ::7] *= 2.0**-8
        _check(q, cache, table, _ints([500]), _parents(1, tokens, 3, 0), f"2^{power}", scale=2.0 ** (-power - 2))
        if tokens < 20:
            chain = torch.arange(-1, tokens - 1, device=DEV, dtype=torch.int32)[None]
            want, bound = tree_bound.tree(q, cache, table, _ints([500]), chain, scale=2.0 ** (-power - 2))
            out = fa.forward_cached(q, cache, table, _ints([500]), softmax_scale=2.0 ** (-power - 2))
            stream_oracle.check(out, want, bound, f"cached 2^{power}")


@pytest.mark.parametrize("tokens", NODES)
def test_large_values_of_bfloat16(tokens):
    """Values of 2^117, the later ones 2^7 times as heavy as the first: a sum of weights up to 1 times them is in range."""
    gen = torch.Generator(DEV).manual_seed(7)
    cache, table = _cache(gen, 1, 400, 16, 1, 64, BF)
    cache.k.fill_(0.0)
    for i in range(25):
        cache.k[int(table[0, i]), ..., 0] = 1.0 if i >= 8 else 0.0
    cache.v.copy_(2.0**117 * (1 + torch.rand(cache.v.shape, generator=gen, device=DEV)))
    q = torch.zeros(1, 4, tokens, 64, device=DEV, dtype=BF)
    q[..., 0] = 7 * math.log(2)
    _check(q, cache, table, _ints([400]), _parents(1, tokens, 3, 0), scale=1.0)


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("tokens", NODES)
def test_queries_with_one_large_channel(tokens, dtype, kind):
    """One channel 2^3 to 2^10 times the others, where the keys have next to nothing."""
    gen = torch.Generator(DEV).manual_seed(5)
    cache, table = _cache(gen, 2, 400, 32, 1, 128, kind)
    if kind == E4M3:
        cache.k.view(torch.uint8)[..., 77] &= 0x87  # subnormal codes
    else:
        cache.k[..., 77] *= 2.0**-8
    q = torch.randn(2, 4, tokens, 128, generator=gen, device=DEV)
    for power in (3, 6, 9):
        q[..., 77] = 2.0**power * (1 + torch.rand(2, 4, tokens, generator=gen, device=DEV))
        _check(q.to(dtype), cache, table, _ints([400, 111]), _parents(2, tokens, 3, 0), f"2^{power}", scale=0.02)


@pytest.mark.parametrize("dtype,kind", KINDS)
@pytest.mark.parametrize("tokens", NODES)
def test_scales_of_any_sign_and_strided_pools(tokens, dtype, kind):
    gen = torch.Generator(DEV).manual_seed(6)
    plain, table = _cache(gen, 2, 300, 16, 2, 64, kind)
    # [pages][k, v][slots][heads] of another pool's pages: page and head strides of their own.
    raw = torch.uint8 if kind == E4M3 else kind
    both = torch.zeros(plain.num_pages, 3, 2, 16, 64, device=DEV, dtype=raw)
    both[:, 0], both[:, 2] = plain.k.view(raw), plain.v.view(raw)
    cache = fa.PagedKVCache(both[:, 0].view(kind), both[:, 2].view(kind), plain.k_scale, plain.v_scale)
    q = torch.randn(2, tokens, 8, 64, generator=gen, device=DEV).to(dtype).transpose(1, 2)
    for scale in (0.0, -0.125, -0.4, 0.3):
        out = _check(q, cache, table, _ints([300, 200]), _parents(2, tokens, 3, 0), f"scale {scale}", scale=scale)
        assert torch.equal(out, fa.forward_tree(q, plain, table, _ints([300, 200]), _parents(2, tokens, 3, 0), softmax_scale=scale))
