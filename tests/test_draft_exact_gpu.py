"""A server's steps with drafted trees again: every answer against attention over what the cache holds, within the bound
that the kernels' roundings leave, which wrong ancestors exceed; and kept tokens in pages beyond 32 bits."""

import random

import pytest
import torch

import draft_oracle as oracle
import fa
import stream_oracle
import tree_bound
from fa import _C

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
HALF, BF, E4M3 = torch.float16, torch.bfloat16, torch.float8_e4m3fn
HK, D, PAGE, WIDTH, TEXT = 2, 64, 16, 14, 200


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("dtype,kind", [(HALF, HALF), (BF, BF), (HALF, E4M3), (BF, E4M3)])
@pytest.mark.parametrize("group,nodes_most", [(2, 6), (2, 12), (8, 20)])
def test_answers_of_a_server(group, nodes_most, dtype, kind):
    rng, gen, heads = random.Random(nodes_most), torch.Generator(DEV).manual_seed(0), group * HK
    rows = torch.randn(TEXT, heads + 2 * HK, D, generator=gen, device=DEV).to(dtype)
    cos, sin = (f(torch.arange(300, device=DEV)[:, None] * 10000.0 ** (-torch.arange(D // 2, device=DEV) * 2 / D)).contiguous()
                for f in (torch.cos, torch.sin))
    cache = fa.PagedKVCache.empty(80, PAGE, HK, D, dtype=kind)
    refs = torch.zeros(80, dtype=torch.int32, device=DEV)

    def split(tokens):
        x = rows[torch.tensor(tokens, device=DEV)].transpose(1, 2)
        return x[:, :heads], x[:, heads : heads + HK], x[:, heads + HK :]

    texts = [[rng.randrange(TEXT) for _ in range(n)] for n in (33, 5)]
    lengths = _ints([len(t) for t in texts])
    table = torch.full((2, WIDTH), -1, dtype=torch.int32, device=DEV)
    fa.reserve_pages(refs, table, lengths, 33, PAGE, counts=lengths)
    _, k, v = split([t + [0] * (33 - len(t)) for t in texts])
    fa.append_kv(cache, k, v, table, lengths, counts=lengths.clone(), cos=cos, sin=sin)
    for step in range(5):
        if step == 1:
            parents = [0, 1, 0, 0]
            new = fa.fork_pages(refs, table, _ints(parents))
            fa.free_pages(refs, table)
            table, texts, lengths = new, [list(texts[p]) for p in parents], lengths[_ints(parents).long()]
        batch = len(texts)
        hang = [[max(-1, i - rng.randint(1, 4)) for i in range(nodes_most)] for _ in range(batch)]
        drafts = [[rng.randrange(TEXT) for _ in range(nodes_most)] for _ in range(batch)]
        nodes = [rng.randint(2, nodes_most) for _ in range(batch)]
        for h in hang:
            h[1] = 0  # every tree has a path
        lengths = lengths + _ints(nodes)
        granted, src, dst = fa.reserve_pages(refs, table, lengths, nodes_most, PAGE, counts=_ints(nodes))
        assert granted.all()
        fa.copy_pages(cache, src, dst)
        q, k, v = split(drafts)
        sees = [oracle.ancestors(h, n) for h, n in zip(hang, nodes)]
        depth = [[int(s[i].sum()) - 1 if i < n else -10**6 for i in range(nodes_most)] for s, n in zip(sees, nodes)]
        q, k = fa.forward_rotary(q, k, (lengths - _ints(nodes))[:, None] + _ints(depth), cos, sin)
        fa.append_kv(cache, k, v, table, lengths, counts=_ints(nodes))
        out = fa.forward_tree(q, cache, table, lengths, _ints(hang), counts=_ints(nodes))
        want, bound = tree_bound.tree(q, cache, table, lengths, _ints(hang), counts=_ints(nodes))
        stream_oracle.check(out, want, bound, f"step {step}")
        # The bound tells other trees apart: nobody's ancestors, and every earlier node's.
        alone, _ = tree_bound.tree(q, cache, table, lengths, torch.full_like(_ints(hang), -1), counts=_ints(nodes))
        chain = torch.arange(-1, nodes_most - 1, device=DEV, dtype=torch.int32).expand(batch, nodes_most)
        every, _ = tree_bound.tree(q, cache, table, lengths, chain, counts=_ints(nodes))
        for b in range(batch):
            for i in range(nodes[b]):
                n = int(sees[b][i].sum())
                for other, differs in ((alone, n > 1), (every, n < i + 1)):
                    over = ((other - want).abs() / bound)[b, :, i].max()
                    assert (over > 2) == differs, (step, b, i, float(over))
        kept = []
        for b in range(batch):
            path = sees[b][rng.randrange(nodes[b])].nonzero()[:, 0].tolist()
            path = path[: rng.randint(0, len(path))]
            kept.append(path + [-1] * (nodes_most - len(path)))
            texts[b] += [drafts[b][i] for i in path]
        lengths = fa.keep_tokens(cache, table, lengths, _ints(kept), nodes_most, counts=_ints(nodes))
        assert lengths.tolist() == [len(t) for t in texts]
        fa.free_pages(refs, table, (lengths + PAGE - 1) // PAGE)
    fa.free_pages(refs, table)
    assert not refs.any() and _C.device_status(0, clear=True) == 0


def test_kept_tokens_and_copies_beyond_32_bits():
    """The last pages of a pool, which begin beyond 2^31 elements, beside the same pages in a pool of their own."""
    pages = (1 << 31) // (256 * 64) + 40
    gen = torch.Generator(DEV).manual_seed(11)
    k, v = (torch.zeros(pages, 1, 256, 64, dtype=torch.uint8, device=DEV) for _ in "kv")
    ks, vs = (2.0 ** torch.randint(-5, 5, (pages, 1), generator=gen, device=DEV).float() for _ in "kv")
    for x in (k, v):
        x[-4:] = (30 * torch.randn(4, 1, 256, 64, generator=gen, device=DEV)).to(E4M3).view(torch.uint8)
    cache = fa.PagedKVCache(k.view(E4M3), v.view(E4M3), ks, vs)
    small = fa.PagedKVCache(*(x[-4:].clone().view(E4M3) for x in (k, v)), *(x[-4:].clone() for x in (ks, vs)))
    table, path = _ints([[pages - 1, pages - 3, pages - 4]]), _ints([[3, 7, 200, 249]])
    before = small.k.view(torch.uint8).clone()
    new = fa.keep_tokens(cache, table, _ints([700]), path, 250)
    assert torch.equal(new, fa.keep_tokens(small, table - (pages - 4), _ints([700]), path, 250)) and new.tolist() == [454]
    assert not torch.equal(small.k.view(torch.uint8), before)
    for big, little in ((cache.k, small.k), (cache.v, small.v)):
        big = big.view(torch.uint8)
        assert torch.equal(big[-4:], little.view(torch.uint8)) and not big[:-4].any()
    assert torch.equal(cache.k_scale[-4:], small.k_scale) and torch.equal(cache.v_scale[-4:], small.v_scale)
    fa.copy_pages(cache, _ints([pages - 1, pages - 4]), _ints([5, pages - 9]))
    for x, s in ((k, ks), (v, vs)):
        for src, dst in ((pages - 1, 5), (pages - 4, pages - 9)):
            assert x[src].any() and torch.equal(x[dst], x[src]) and torch.equal(s[dst], s[src])
        assert not x[:5].any() and not x[6 : pages - 9].any() and not x[pages - 8 : pages - 4].any()
    assert _C.device_status(0, clear=True) == 0
