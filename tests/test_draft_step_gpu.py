"""The operators for drafted tokens as a server runs them together: sequences are forked, drafted on as trees,
checked, the accepted paths kept, pages given back; against whole rows of the tokens that every sequence holds."""

import math
import random

import pytest
import torch

import draft_oracle as oracle
import fa
import stream_oracle
from fa import _C

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
BF, E4M3 = torch.bfloat16, torch.float8_e4m3fn
H, HK, D, PAGE, NODES, WIDTH = 4, 2, 64, 16, 12, 12


def _ints(x):
    return torch.tensor(x, dtype=torch.int32, device=DEV)


@pytest.mark.parametrize("kind", [BF, E4M3])
def test_serving_with_drafts(kind):
    rng, gen = random.Random(0), torch.Generator(DEV).manual_seed(0)
    # A token's row of queries, keys and values, before it is turned.
    rows = torch.randn(200, H + 2 * HK, D, generator=gen, device=DEV).to(BF)
    cos, sin = (f(torch.arange(300, device=DEV)[:, None] * 10000.0 ** (-torch.arange(D // 2, device=DEV) * 2 / D)).contiguous()
                for f in (torch.cos, torch.sin))
    num_pages = 60
    cache = fa.PagedKVCache.empty(num_pages, PAGE, HK, D, dtype=kind)
    refs = torch.zeros(num_pages, dtype=torch.int32, device=DEV)

    def split(tokens):  # [B][T] token numbers -> q, k, v
        x = rows[torch.tensor(tokens, device=DEV)].transpose(1, 2)
        return x[:, :H], x[:, H : H + HK], x[:, H + HK :]

    # Prompts of unequal length, padded.
    texts = [[rng.randrange(200) for _ in range(n)] for n in (33, 5)]
    counts = _ints([len(t) for t in texts])
    table = torch.full((2, WIDTH), -1, dtype=torch.int32, device=DEV)
    lengths = counts.clone()
    granted, _, _ = fa.reserve_pages(refs, table, lengths, 33, PAGE, counts=counts)
    assert granted.all()
    _, k, v = split([t + [0] * (33 - len(t)) for t in texts])
    fa.append_kv(cache, k, v, table, lengths, counts=counts, cos=cos, sin=sin)
    for step in range(6):
        if step == 1:  # three answers from the first prompt, one from the second
            parents = [0, 1, 0, 0]
            new = fa.fork_pages(refs, table, _ints(parents))
            fa.free_pages(refs, table)
            table, texts, lengths = new, [list(texts[p]) for p in parents], lengths[_ints(parents).long()]
        batch = len(texts)
        hang = [[max(-1, i - rng.randint(1, 4)) for i in range(NODES)] for _ in range(batch)]
        drafts = [[rng.randrange(200) for _ in range(NODES)] for _ in range(batch)]
        nodes = [rng.randint(1, NODES) for _ in range(batch)]
        lengths = lengths + _ints(nodes)
        granted, src, dst = fa.reserve_pages(refs, table, lengths, NODES, PAGE, counts=_ints(nodes))
        assert granted.all() and (step == 1) == bool((src >= 0).any())
        fa.copy_pages(cache, src, dst)
        q, k, v = split(drafts)
        sees = [oracle.ancestors(h, n) for h, n in zip(hang, nodes)]
        depth = [[int(s[i].sum()) - 1 if i < n else -10**6 for i in range(NODES)] for s, n in zip(sees, nodes)]
        at = (lengths - _ints(nodes))[:, None] + _ints(depth)
        q, k = fa.forward_rotary(q, k, at, cos, sin)
        fa.append_kv(cache, k, v, table, lengths, counts=_ints(nodes))
        out = fa.forward_tree(q, cache, table, lengths, _ints(hang), counts=_ints(nodes))
        # Every node's answer is attention over its text and path, each token turned by its place in them.
        for b, text in enumerate(texts):
            assert not out[b, :, nodes[b] :].any()
            for i in range(nodes[b]):
                line = text + [drafts[b][a] for a in sees[b][i].nonzero()[:, 0].tolist()]
                lq, lk, lv = (x.double() for x in split([line]))
                place = torch.arange(len(line), device=DEV, dtype=torch.int32)[None]
                lq, lk = (oracle.rotary(x, place, cos, sin) for x in (lq, lk))
                p = (lq[0, :, -1:].view(HK, H // HK, D) @ lk[0].mT / math.sqrt(D)).softmax(-1)
                want = (p @ lv[0]).view(H, D)
                # Queries and keys are rounded: to u of a rotated pair's size (norms of 64 and below 12), which moves a
                # score by 2 u |q||k| / 8; an e4m3 cache rounds keys and values to 2^-4 of each (2^-10 of a page's largest), errors without a
                # common sign: the norm over 64 dims of a key's makes 2^-4 |q| max|k| / 8.
                u = 2.0**-8
                move = 2 * u * 12 * 12 / 8 if kind == BF else 2 * u * 12 * 12 / 8 + 2.0**-4 * 4.2 * 12 / 8 * 1.0
                value = 0.0 if kind == BF else 2.0**-4 * lv.abs().max().item()
                bound = (math.expm1(min(2 * move, 3.0)) + 3 * u) * lv.abs().max() + value
                stream_oracle.check(out[b, :, i], want, bound.expand(H, D), f"step {step} node {i}")
        # Each keeps a path of its tree, some of it.
        kept = []
        for b in range(batch):
            path = sees[b][rng.randrange(nodes[b])].nonzero()[:, 0].tolist()
            path = path[: rng.randint(0, len(path))]
            kept.append(path + [-1] * (NODES - len(path)))
            texts[b] += [drafts[b][i] for i in path]
        lengths = fa.keep_tokens(cache, table, lengths, _ints(kept), NODES, counts=_ints(nodes))
        assert lengths.tolist() == [len(t) for t in texts]
        fa.free_pages(refs, table, (lengths + PAGE - 1) // PAGE)
        held = [int((row >= 0).sum()) for row in table]
        assert held == [-(-len(t) // PAGE) for t in texts]
        # The cache holds every sequence's tokens, turned by their places: as a plain prompt of them would be.
        for b, text in enumerate(texts):
            _, k, v = split([text])
            place = torch.arange(len(text), device=DEV, dtype=torch.int32)[None]
            k = oracle.rotary(k, place, cos, sin)
            for x, pool, scale in ((k, cache.k, cache.k_scale), (v.double(), cache.v, cache.v_scale)):
                got = stream_oracle.dense(pool, scale, table[b : b + 1].clamp(min=0))[:, :, : len(text)]
                bound = 2.0**-8 * x.abs() + 2.0**-20 if kind == BF else (2.0**-4 + 2.0**-7) * x.abs() + 2.0**-9 * x.abs().max()
                stream_oracle.check(got, x, bound, "cache")
    fa.free_pages(refs, table)
    assert not refs.any() and (table == -1).all() and _C.device_status(0, clear=True) == 0
