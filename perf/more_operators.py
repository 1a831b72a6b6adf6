"""Cases of the operators with which a model drafts, checks and keeps tokens, with their plain forms.

Four operators, next to the paged cache and the attention over it:

  turn   rotation of queries and keys by positions on one or several axes (time, height, width),
         forward ("fwd") or a training step's forward and backward ("train")
  tree   attention of a tree of drafted tokens over the cache: a node sees the context and its ancestors
  keep   the accepted path's tokens moved together behind the context, in the cache
  fork   sequences forked (last step's forks given back, pages shared, the pages that get new
         tokens made their own and copied)

``own`` False computes the plain form in 32-bit torch operations; ``own`` True calls the
framework's entry points.
"""

import math
import os
import sys

import torch

own = False

TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}


def _fa():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash-attention-from-scratch_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import fa

    return fa


# ------------------------------------------------------------------------------------ the cases


def _turn(name, mode, batch, tokens, heads, kv_heads, dim, dtype, rotary, axes, interleaved, token_major, padded):
    return dict(name=name, op="turn", mode=mode, batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim,
                dtype=dtype, rotary=rotary, axes=axes, interleaved=interleaved, token_major=token_major, padded=padded)


def _tree(name, batch, tokens, span, heads, kv_heads, dim, dtype, cache, page, length, spread, window, sinks, ragged):
    return dict(name=name, op="tree", batch=batch, tokens=tokens, span=span, heads=heads, kv_heads=kv_heads, dim=dim,
                dtype=dtype, cache=cache, page=page, length=length, spread=spread, window=window, sinks=sinks,
                ragged=ragged)


def _keep(name, batch, tokens, kept, kv_heads, dim, cache, page, length, ragged):
    return dict(name=name, op="keep", batch=batch, tokens=tokens, kept=kept, kv_heads=kv_heads, dim=dim, cache=cache,
                page=page, length=length, ragged=ragged)


def _fork(name, parents, children, tokens, kv_heads, dim, cache, page, length):
    return dict(name=name, op="fork", parents=parents, children=children, tokens=tokens, kv_heads=kv_heads, dim=dim,
                cache=cache, page=page, length=length)


def listed():
    return [
        # One user, one new token: nothing but the latency of a call.
        _turn("turn one token", "fwd", 1, 1, 16, 16, 64, "f16", 64, 1, False, False, False),
        # A prompt of images and text, as the projections leave it: heads next to each other, an odd length.
        _turn("turn an image prompt", "fwd", 2, 4999, 32, 8, 128, "bf16", 128, 3, False, True, True),
        # A training step on long video rows, half of the dims turned.
        _turn("turn in training", "train", 1, 16384, 16, 4, 128, "bf16", 64, 3, True, True, False),
        # One user, a small tree over a short context in 16 bits.
        _tree("tree of one user", 1, 16, 6, 16, 16, 64, "f16", "f16", 16, 777, 0.0, 0, 0, False),
        # A served batch of unequal contexts, eight drafted tokens each, 8-bit cache.
        _tree("small trees", 32, 8, 4, 32, 8, 128, "bf16", "e4m3", 64, 8192, 0.5, 0, 0, False),
        # The same batch with trees of up to 64 nodes.
        _tree("trees of a batch", 32, 64, 16, 32, 8, 128, "bf16", "e4m3", 64, 8192, 0.5, 0, 0, True),
        # Few users with very long documents.
        _tree("trees on long documents", 4, 32, 8, 32, 8, 128, "bf16", "e4m3", 64, 131000, 0.1, 0, 0, False),
        # A 16-bit cache with small pages, a window and sinks, an odd tree.
        _tree("trees in a window", 16, 61, 12, 32, 8, 128, "bf16", "bf16", 32, 20000, 0.5, 4096, 4, False),
        # One user's accepted path.
        _keep("keep one path", 1, 16, 4, 16, 64, "f16", 16, 777, False),
        # The accepted paths of a served batch, 8-bit cache.
        _keep("keep paths of a batch", 128, 64, 9, 8, 128, "e4m3", 64, 1500, True),
        # One answer sampled four times from one prompt.
        _fork("fork one sample", 1, 4, 1, 16, 64, "f16", 16, 777),
        # A large batch of beams, long pages of 16 bits.
        _fork("fork a batch of beams", 64, 256, 1, 8, 128, "bf16", 128, 1100),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["turn", "turn", "tree", "tree", "tree", "keep", "fork"])
    dim = rng.choice([64, 128])
    dtype = rng.choice(["f16", "bf16"])
    cache = rng.choice([dtype, "e4m3", "e4m3"])
    page = rng.choice([16, 32, 64, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    if op == "turn":
        heads = kv_heads * rng.choice([1, 2, 4])
        budget = 60_000_000 // (heads * dim)  # tokens in all
        batch = _log(rng, 1, 64)
        tokens = 1 if rng.random() < 0.2 else max(1, min(_log(rng, 2, 16384), budget // batch))
        return dict(op=op, mode=rng.choice(["fwd", "train"]), batch=batch, tokens=tokens, heads=heads,
                    kv_heads=kv_heads, dim=dim, dtype=dtype, rotary=rng.choice([dim, dim, dim // 2, 48]),
                    axes=rng.choice([1, 2, 3, 3]), interleaved=rng.random() < 0.5, token_major=rng.random() < 0.5,
                    padded=rng.random() < 0.3)
    if op == "tree":
        group = rng.choice([1, 2, 4, 8])
        tokens = 1 if rng.random() < 0.1 else _log(rng, 2, 256)
        batch = _log(rng, 1, 64)
        budget = 500_000_000 // (kv_heads * dim * (1 if cache == "e4m3" else 2) * batch)
        budget = min(budget, 400_000_000 // (kv_heads * group * tokens * batch))
        length = max(tokens, min(tokens + _log(rng, 1, 131000) - 1, budget))
        window = rng.choice([0, 0, max(tokens, _log(rng, 16, 4096))])
        return dict(op=op, batch=batch, tokens=tokens, span=rng.choice([1, 3, 8, 300]), heads=kv_heads * group,
                    kv_heads=kv_heads, dim=dim, dtype=dtype, cache=cache, page=page, length=length,
                    spread=rng.choice([0.0, 0.3, 0.8]), window=window, sinks=rng.choice([0, 1, 4, 17]) if window else 0,
                    ragged=rng.random() < 0.5)
    if op == "keep":
        tokens = _log(rng, 2, 256)
        return dict(op=op, batch=_log(rng, 1, 128), tokens=tokens, kept=rng.randint(1, tokens // 2), kv_heads=kv_heads,
                    dim=dim, cache=cache, page=page, length=tokens + _log(rng, 1, 1000) - 1, ragged=rng.random() < 0.5)
    parents = _log(rng, 1, 64)
    return dict(op=op, parents=parents, children=parents * rng.choice([1, 2, 3, 4]), tokens=rng.choice([1, 1, 2, 5]),
                kv_heads=kv_heads, dim=dim, cache=cache, page=page, length=_log(rng, 1, 1100))


# --------------------------------------------------------------------------------------- inputs


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _fraction(i):
    return math.modf((i + 1) * 0.6180339887)[0]


def _spread(case):
    """Lengths of the sequences, given by the case alone: the longest down to `spread` of it less."""
    longest, share = case["length"], case.get("spread", 0.0)
    return [max(case["tokens"], int(longest * (1 - share * _fraction(b) * (case["batch"] > 1)))) for b in range(case["batch"])]


def _counts(case):
    """Drafted tokens of every sequence: all of them, or (ragged) between a quarter and all."""
    t = case["tokens"]
    if not case["ragged"]:
        return [t] * case["batch"]
    return [max(1, int(t * (1 - 0.75 * _fraction(b)))) for b in range(case["batch"])]


def _pages(gen, batch, most, page):
    """A table of pages in random order, and how many pages the pool has."""
    per = -(-most // page)
    table = torch.randperm(batch * per + 3, generator=gen, device="cuda")[: batch * per]
    return table.to(torch.int32).view(batch, per), batch * per + 3


def _power_of_two(amax):
    """2^k with the smallest k >= -60 for which amax <= 448 * 2^k."""
    m, e = torch.frexp(amax)
    k = torch.where(amax > 0, torch.where(m <= 0.875, e - 9, e - 8), -60).clamp(min=-60)
    return torch.ldexp(torch.ones_like(amax), k)


def _filled(gen, pages, case, first=None):
    """A cache's pages as earlier tokens left them: values of unit scale with a few large channels, some pages'
    smaller (`first`: those, the others on one scale)."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    x = torch.empty(shape, device="cuda", dtype=torch.float16).normal_(generator=gen)
    x[..., ::32] *= 4
    small = torch.arange(pages, device="cuda") % 3 == 0 if first is None else torch.zeros(pages, dtype=torch.bool, device="cuda")
    if first is not None:
        small[first] = True
    x[small] *= 0.25
    if case["cache"] != "e4m3":
        return x.to(TYPES[case["cache"]]), None
    scale = _power_of_two(x.abs().amax(dim=(2, 3)).float())
    if first is not None:
        scale = torch.where(small, 2.0**-6, 2.0**-4)[:, None].expand_as(scale).contiguous()
    return (x.float() / scale[:, :, None, None]).to(TYPES["e4m3"]), scale


def _axis_of_pair(case):
    """Which axis turns each pair of dims: runs of pairs, the first axis a quarter of what is shared."""
    pairs, axes = case["rotary"] // 2, case["axes"]
    first = pairs if axes == 1 else max(1, pairs // (2 * axes - 1))
    rest = pairs - first
    return [0] * first + [1 + min(i * (axes - 1) // max(rest, 1), axes - 2) for i in range(rest)]


def _prepare_turn(s, gen):
    c = s["case"]
    b, t, d, dt = c["batch"], c["tokens"], c["dim"], TYPES[c["dtype"]]

    def normal(heads):
        if c["token_major"]:
            return torch.empty((b, t, heads, d), device="cuda", dtype=dt).normal_(generator=gen).transpose(1, 2)
        return torch.empty((b, heads, t, d), device="cuda", dtype=dt).normal_(generator=gen)

    s |= {"q": normal(c["heads"]), "k": normal(c["kv_heads"])}
    if c["mode"] == "train":
        s |= {"dq": normal(c["heads"]), "dk": normal(c["kv_heads"])}
        s["q"].requires_grad_(True)
        s["k"].requires_grad_(True)
    # Frames of 12 x 20 patches after a text of some tokens, as positions on every axis.
    text = int(torch.randint(0, 60, (1,), generator=gen, device="cuda"))
    at = torch.arange(t, device="cuda")
    patch = (at - text).clamp(min=0)
    grid = torch.stack([patch // 240, patch // 20 % 12, patch % 20])[: c["axes"]] + text
    rows = t + 64
    positions = torch.where(at < text, at, at if c["axes"] == 1 else grid)
    positions = positions.expand(c["axes"], t)[:, None].repeat(1, b, 1).to(torch.int32)
    if c["padded"]:  # rows of unequal length: no positions behind the last token
        for i in range(b):
            positions[:, i, max(1, int(t * (1 - 0.5 * _fraction(i)))):] = -1
    s["positions"] = positions
    half = c["rotary"] // 2
    turn = torch.arange(rows, device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
        -torch.arange(half, device="cuda", dtype=torch.float64) / half)
    s |= {"cos": turn.cos().float(), "sin": turn.sin().float(), "axes": _axis_of_pair(c)}


def _prepare_fork(s, gen):
    c = s["case"]
    page, parents, children, t = c["page"], c["parents"], c["children"], c["tokens"]
    lengths = [max(1, int(c["length"] * (1 - 0.5 * _fraction(i) * (parents > 1)))) for i in range(parents)]
    width = -(-(max(lengths) + t) // page)
    held = [-(-n // page) for n in lengths]
    pages = sum(held) + children * (t // page + 2) + 5
    order = torch.randperm(pages, generator=gen, device="cuda").to(torch.int32)
    table = torch.full((parents, width), -1, dtype=torch.int32, device="cuda")
    used = 0
    for i, n in enumerate(held):
        table[i, :n] = order[used : used + n]
        used += n
    refs = torch.zeros(pages, dtype=torch.int32, device="cuda")
    refs[order[:used].long()] = 1
    rows = torch.randint(0, parents, (children,), generator=gen, device="cuda").to(torch.int32)
    s |= {"table": table, "refs": refs, "rows": rows, "lengths": _ints(lengths)[rows.long()] + t,
          "kids": torch.full((children, width), -1, dtype=torch.int32, device="cuda")}
    return pages


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    s = {"case": dict(case)}
    if case["op"] == "turn":
        _prepare_turn(s, gen)
        return s
    b, t = case.get("batch"), case["tokens"]
    if case["op"] == "fork":
        pages = _prepare_fork(s, gen)
    else:
        lengths, counts = _spread(case), _counts(case)
        s["lengths"] = _ints(lengths)
        s["counts"] = _ints(counts) if case["ragged"] else None
        s["table"], pages = _pages(gen, b, max(lengths), case["page"])
        if case["op"] == "tree":
            s["q"] = torch.empty((b, case["heads"], t, case["dim"]), device="cuda",
                                 dtype=TYPES[case["dtype"]]).normal_(generator=gen)
            # A node hangs on one of the `span` nodes before it, or on the context.
            at = torch.arange(t, device="cuda")
            back = torch.rand((b, t), generator=gen, device="cuda") * (at + 1).clamp(max=case["span"])
            s["parents"] = (at - 1 - back.long()).clamp(min=-1).to(torch.int32)
        else:
            # Paths that start behind where they go, so that a pass can be taken again.
            kept = []
            scores = torch.rand((b, t), generator=gen, device="cuda").cpu()
            for i, n in enumerate(counts):
                m = min(case["kept"], n // 2)
                path = (scores[i, m:n].argsort()[:m] + m).sort().values.tolist()
                kept.append(path + [-1] * (case["kept"] - m))
            s["kept"] = _ints(kept)
    first = None
    if case["op"] == "keep":
        # The page in which the drafted tokens begin holds smaller values: it grows with those that come in, and only it.
        first = torch.tensor([row[(n - m) // case["page"]] for row, n, m in zip(s["table"].tolist(), lengths, counts)],
                             device="cuda")
    (s["k"], s["ks"]), (s["v"], s["vs"]) = (_filled(gen, pages, case, first) for _ in "kv")
    if own:
        s["cache"] = _fa().PagedKVCache(s["k"], s["v"], s["ks"], s["vs"])
    return s


# ---------------------------------------------------------------------------------- plain forms


def _turned(x, cos, sin, interleaved, real):
    r = 2 * cos.shape[-1]
    y, rest = x[..., :r].float(), x[..., r:].float()
    a, b = (y[..., ::2], y[..., 1::2]) if interleaved else y.chunk(2, -1)
    a, b = a * cos - b * sin, b * cos + a * sin
    y = torch.stack([a, b], -1).flatten(-2) if interleaved else torch.cat([a, b], -1)
    return torch.where(real, torch.cat([y, rest], -1), 0.0).to(x.dtype)


def _plain_turn(s):
    c = s["case"]
    axes = torch.tensor(s["axes"], device="cuda")
    at = s["positions"].long()[axes].movedim(0, -1)  # [b, t, pairs]
    real = (s["positions"] >= 0).all(0)[:, None, :, None]
    cos, sin = (s[x].gather(0, at.clamp(min=0).flatten(0, 1)).view(at.shape)[:, None] for x in ("cos", "sin"))
    out = [_turned(s[x].detach(), cos, sin, c["interleaved"], real) for x in "qk"]
    if c["mode"] == "train":
        out += [_turned(s[x], cos, -sin, c["interleaved"], real) for x in ("dq", "dk")]
    return tuple(out)


def _dense(pool, scales, table, wide=torch.float32):
    """A cache's pages side by side: [batch, heads, positions, dim]."""
    x = pool[table].to(wide)
    if scales is not None:
        x = x * scales[table].to(wide)[..., None, None]
    b, p, h, n, d = x.shape
    return x.transpose(1, 2).reshape(b, h, p * n, d)


def _plain_tree(s):
    c = s["case"]
    b, hk, t, d = c["batch"], c["kv_heads"], c["tokens"], c["dim"]
    g = c["heads"] // hk
    table, lengths = s["table"].long(), s["lengths"].long()
    counts = s["counts"].long() if s["counts"] is not None else torch.full_like(lengths, t)
    context = lengths - counts
    node = torch.arange(t, device="cuda")
    # Ancestors and itself, by squaring the relation "itself or its parent".
    up = ((s["parents"][:, :, None] == node) | (node[:, None] == node)).float()
    for _ in range(max(1, (t - 1).bit_length())):
        up = (up @ up).clamp(max=1)
    k, v = _dense(s["k"], s["ks"], table), _dense(s["v"], s["vs"], table)
    key = torch.arange(k.shape[2], device="cuda")
    at = key - context[:, None]  # a key's place in the tree
    seen = up.bool().gather(2, at.clamp(0, t - 1)[:, None].expand(b, t, -1)) & (at >= 0)[:, None] & (at < counts[:, None])[:, None]
    if c["window"]:
        position = context[:, None] + up.sum(2).long() - 1
        near = (position[:, :, None] - key < c["window"]) | (key < c["sinks"])
    else:
        near = torch.ones_like(seen)
    seen = (seen | (near & (at < 0)[:, None])) & (node < counts[:, None])[:, :, None]
    scores = (s["q"].float().view(b, hk, g * t, d) @ k.transpose(-1, -2)).mul_(1 / math.sqrt(d)).view(b, hk, g, t, -1)
    scores.masked_fill_(~seen[:, None, None], -math.inf)
    top = scores.amax(-1, keepdim=True)
    scores.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    scores.div_(scores.sum(-1, keepdim=True).clamp(min=1e-37))
    return (scores.view(b, hk, g * t, -1) @ v).view(b, hk * g, t, d).to(s["q"].dtype)


def _plain_keep(s):
    c = s["case"]
    page, table = c["page"], s["table"].long()
    lengths = s["lengths"].long()
    counts = s["counts"].long() if s["counts"] is not None else torch.full_like(lengths, c["tokens"])
    context = lengths - counts
    kept = s["kept"].long()
    real = kept >= 0
    j = torch.arange(kept.shape[1], device="cuda").expand_as(kept)
    to, of = context[:, None] + j, context[:, None] + kept.clamp(min=0)
    last = table.shape[1] * page - 1
    to_page, of_page = (table.gather(1, x.clamp(max=last) // page) for x in (to, of))
    bb, jj = real.nonzero(as_tuple=True)
    new = s["lengths"] - counts.int() + real.sum(1, dtype=torch.int32)
    out = [new]
    for pool, scales in ((s["k"], s["ks"]), (s["v"], s["vs"])):
        moved = pool.view(torch.uint8 if scales is not None else pool.dtype)[of_page[bb, jj], :, of[bb, jj] % page]
        if scales is None:
            pool[to_page[bb, jj], :, to[bb, jj] % page] = moved
            out.append(pool)
            continue
        # A page's scale: the largest of its own and those that come in. Where it grows the page's tokens follow.
        before = scales.clone()
        after = before.scatter_reduce(0, to_page[bb, jj][:, None].expand(-1, scales.shape[1]), before[of_page[bb, jj]], "amax")
        filled = torch.zeros(pool.shape[0], dtype=torch.long, device="cuda")
        filled[table] = (lengths[:, None] - torch.arange(table.shape[1], device="cuda") * page).clamp(0, page)
        grown = (after > before).any(1).nonzero()[:, 0]
        codes = pool[grown]
        again = (codes.float() * (before[grown] / after[grown])[:, :, None, None]).to(pool.dtype)
        there = (torch.arange(page, device="cuda") < filled[grown][:, None])[:, None, :, None]
        pool.view(torch.uint8)[grown] = torch.where(there, again.view(torch.uint8), codes.view(torch.uint8))
        ratio = (before[of_page[bb, jj]] / after[to_page[bb, jj]])[..., None]
        moved = (moved.view(pool.dtype).float() * ratio).to(pool.dtype)
        pool.view(torch.uint8)[to_page[bb, jj], :, to[bb, jj] % page] = moved.view(torch.uint8)
        scales.copy_(after)
        out += [pool, scales]
    return tuple(out)


def _plain_fork(s):
    c = s["case"]
    page, refs, pages = c["page"], s["refs"], s["refs"].shape[0]
    # Last step's forks are given back.
    old = s["kids"].flatten().long()
    refs.index_add_(0, old.clamp(min=0), -(old >= 0).int())
    # The new ones share their parents' pages.
    kids = s["table"][s["rows"].long()]
    now = kids.flatten().long()
    refs.index_add_(0, now.clamp(min=0), (now >= 0).int())
    # Pages that get new tokens: those that are missing or shared are taken from the free ones.
    lengths = s["lengths"].long()
    start = lengths - c["tokens"]
    index = torch.arange(kids.shape[1], device="cuda")
    want = (index >= (start // page)[:, None]) & (index < ((lengths + page - 1) // page)[:, None])
    shared = (kids >= 0) & (refs[kids.long().clamp(min=0)] > 1)
    need = want & ((kids < 0) | shared)
    each = need.sum(1)
    free = (refs == 0).long()
    rank = free.cumsum(0)
    granted = (each == 0) | (each.cumsum(0) <= rank[-1])
    take = need & granted[:, None]
    which = torch.where(take, (each.cumsum(0) - each)[:, None] + need.cumsum(1) - 1, 0)
    nth = torch.zeros(pages + 1, dtype=torch.long, device="cuda")
    nth[torch.where(free > 0, rank - 1, pages)] = torch.arange(pages, device="cuda")
    page_of = nth[which]
    copies = take & shared & (index == (start // page)[:, None]) & (start % page > 0)[:, None]
    src = torch.where(copies, kids, -1).amax(1)
    dst = torch.where(copies, page_of.int(), -1).amax(1)
    gone = torch.where(take & shared, kids, -1).flatten().long()
    refs.index_add_(0, gone.clamp(min=0), -(gone >= 0).int())
    refs.index_add_(0, page_of.flatten(), take.flatten().int())
    kids = torch.where(take, page_of.int(), kids)
    s["kids"] = kids
    a, z = src.long().clamp(min=0), torch.where(dst >= 0, dst.long(), pages)
    some = (dst >= 0).nonzero()[:, 0]
    out = [kids, refs, granted, src, dst]
    for pool, scales in ((s["k"], s["ks"]), (s["v"], s["vs"])):
        raw = pool.view(torch.uint8) if scales is not None else pool
        raw[z[some]] = raw[a[some]]
        out.append(pool)
        if scales is not None:
            scales[z[some]] = scales[a[some]]
            out.append(scales)
    return tuple(out)


def run(state):
    s, c = state, state["case"]
    if not own:
        return {"turn": _plain_turn, "tree": _plain_tree, "keep": _plain_keep, "fork": _plain_fork}[c["op"]](s)
    fa = _fa()
    if c["op"] == "turn":
        how = (s["positions"], s["cos"], s["sin"])
        if c["mode"] == "fwd":
            return fa.forward_rotary(s["q"], s["k"], *how, axes=s["axes"], interleaved=c["interleaved"])
        q, k = fa.rotary(s["q"], s["k"], *how, axes=s["axes"], interleaved=c["interleaved"])
        return (q.detach(), k.detach(), *torch.autograd.grad((q, k), (s["q"], s["k"]), (s["dq"], s["dk"])))
    if c["op"] == "tree":
        return fa.forward_tree(s["q"], s["cache"], s["table"], s["lengths"], s["parents"], counts=s["counts"],
                               window=c["window"], sinks=c["sinks"])
    pools = (s["k"], s["v"]) if s["ks"] is None else (s["k"], s["ks"], s["v"], s["vs"])
    if c["op"] == "keep":
        return (fa.keep_tokens(s["cache"], s["table"], s["lengths"], s["kept"], c["tokens"], counts=s["counts"]), *pools)
    fa.free_pages(s["refs"], s["kids"])
    s["kids"] = fa.fork_pages(s["refs"], s["table"], s["rows"])
    granted, src, dst = fa.reserve_pages(s["refs"], s["kids"], s["lengths"], c["tokens"], c["page"])
    fa.copy_pages(s["cache"], src, dst)
    return (s["kids"], s["refs"], granted, src, dst, *pools)


# --------------------------------------------------------------------------------- 64-bit values


def _exact_turn(s):
    c = s["case"]
    half = c["rotary"] // 2

    def turn(x, sign):
        x = x.detach().double()
        y = x.clone()
        for i, axis in enumerate(s["axes"]):
            at = s["positions"][axis].long().clamp(min=0)
            cos, sin = s["cos"][at, i].double()[:, None], s["sin"][at, i].double()[:, None] * sign
            lo, hi = (2 * i, 2 * i + 1) if c["interleaved"] else (i, i + half)
            y[..., lo] = cos * x[..., lo] - sin * x[..., hi]
            y[..., hi] = sin * x[..., lo] + cos * x[..., hi]
        return y * (s["positions"].amin(0) >= 0)[:, None, :, None]

    out = [turn(s["q"], 1), turn(s["k"], 1)]
    if c["mode"] == "train":
        out += [turn(s["dq"], -1), turn(s["dk"], -1)]
    return tuple(out)


def _exact_tree(s):
    c = s["case"]
    t, d, g = c["tokens"], c["dim"], c["heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    counts = s["counts"].tolist() if s["counts"] is not None else [t] * c["batch"]
    for b, (length, count) in enumerate(zip(s["lengths"].tolist(), counts)):
        ids = s["table"][b : b + 1].long()
        k, v = (_dense(s[x], s[y], ids, torch.float64)[0, :, :length] for x, y in (("k", "ks"), ("v", "vs")))
        context, parents = length - count, s["parents"][b].tolist()
        sees = torch.zeros((count, length), dtype=torch.bool)
        for i in range(count):
            line, at = [], i
            while at >= 0:
                line.append(context + at)
                at = parents[at]
            position = context + len(line) - 1
            first = max(0, position - c["window"] + 1) if c["window"] else 0
            sees[i, first:context] = True
            sees[i, : min(c["sinks"], context)] = True
            sees[i, line] = True
        hidden = ~sees.to("cuda")
        for h in range(c["heads"]):
            score = (s["q"][b, h, :count].double() @ k[h // g].T / math.sqrt(d)).masked_fill_(hidden, -math.inf)
            out[b, h, :count] = torch.softmax(score, -1) @ v[h // g]
    return out


def _exact_keep(s):
    """Token by token; codes stay unrounded (what they stand for, over the scale)."""
    c = s["case"]
    page = c["page"]
    counts = s["counts"].tolist() if s["counts"] is not None else [c["tokens"]] * c["batch"]
    pools = [s["k"].double(), s["v"].double()]
    scales = [x.double() if x is not None else None for x in (s["ks"], s["vs"])]
    table, new = s["table"].tolist(), []
    for b, (length, count, kept) in enumerate(zip(s["lengths"].tolist(), counts, s["kept"].tolist())):
        kept = [x for x in kept if x >= 0]
        start = length - count
        new.append(start + len(kept))
        for pool, scale in zip(pools, scales):
            at = [divmod(start + x, page) for x in kept]
            values = [pool[table[b][p], :, i].clone() for p, i in at]
            units = [scale[table[b][p]].clone() if scale is not None else None for p, i in at]
            for nth in range(start // page, (new[b] - 1) // page + 1):
                to = table[b][nth]
                mine = [j for j in range(len(kept)) if (start + j) // page == nth]
                if scale is not None and mine:
                    top = torch.stack([units[j] for j in mine] + [scale[to]]).amax(0)
                    pool[to, :, : min(page, length - nth * page)] *= (scale[to] / top)[:, None, None]
                    scale[to] = top
                for j in mine:
                    pool[to, :, (start + j) % page] = values[j] if scale is None else values[j] * (units[j] / scale[to])[:, None]
    new = torch.tensor(new, dtype=torch.int32)
    if scales[0] is None:
        return new, pools[0], pools[1]
    return new, pools[0], scales[0], pools[1], scales[1]


def _exact_fork(s):
    """Page by page, on lists."""
    c = s["case"]
    page, refs = c["page"], s["refs"].tolist()
    table, rows, lengths = s["table"].tolist(), s["rows"].tolist(), s["lengths"].tolist()
    kids = [list(table[r]) for r in rows]
    for row in kids:
        for p in row:
            if p >= 0:
                refs[p] += 1
    free, was = [p for p, n in enumerate(refs) if n == 0], list(refs)
    granted, src, dst, asked = [], [], [], 0
    for row, length in zip(kids, lengths):
        start = length - c["tokens"]
        need = [i for i in range(start // page, -(-length // page)) if row[i] < 0 or was[row[i]] > 1]
        asked += len(need)
        granted.append(not need or asked <= len(free))
        src.append(-1)
        dst.append(-1)
        for n, i in enumerate(need if granted[-1] else []):
            new = free[asked - len(need) + n]
            if row[i] >= 0:
                refs[row[i]] -= 1
                if i == start // page and start % page:
                    src[-1], dst[-1] = row[i], new
            refs[new] += 1
            row[i] = new
    pools = [s[x].double() if s[x] is not None else None for x in ("k", "ks", "v", "vs")]
    for a, z in zip(src, dst):
        for x in pools:
            if z >= 0 and x is not None:
                x[z] = x[a]
    out = [torch.tensor(x, dtype=torch.int32) for x in (kids, refs)] + [torch.tensor(granted)]
    return (*out, torch.tensor(src, dtype=torch.int32), torch.tensor(dst, dtype=torch.int32), *(x for x in pools if x is not None))


def exact(case, seed):
    s = prepare(case, seed)
    return {"turn": _exact_turn, "tree": _exact_tree, "keep": _exact_keep, "fork": _exact_fork}[case["op"]](s)


# ----------------------------------------------------------------------------------------- work


def work(case):
    hk, d, t = case["kv_heads"], case["dim"], case["tokens"]
    if case["op"] == "turn":
        tokens = case["batch"] * t
        rows = tokens * (case["heads"] + hk) * (2 if case["mode"] == "train" else 1)
        return {"bytes": rows * d * 4 + tokens * 4 * case["axes"] + (t + 64) * case["rotary"] * 4, "flops": rows * case["rotary"] * 3}
    size = 1 if case["cache"] == "e4m3" else 2
    if case["op"] == "keep":
        tokens = sum(min(case["kept"], n // 2) for n in _counts(case))
        return {"bytes": tokens * hk * 2 * (2 * d * size + (8 if size == 1 else 0)) + tokens * 12, "flops": 0}
    if case["op"] == "fork":
        whole = hk * 2 * (case["page"] * d * size + (4 if size == 1 else 0))
        # as many pages as children copied, their tables read and written
        return {"bytes": case["children"] * (2 * whole + 8 * (case["length"] // case["page"] + 1)), "flops": 0}
    w, g = case["window"], case["heads"] // hk
    tokens = pairs = 0
    for n, count in zip(_spread(case), _counts(case)):
        context = n - count
        shown = min(context, w + min(case["sinks"], context - w)) if w and context > w else context
        tokens += shown + count
        pairs += count * (shown + min(count, 2 + int(math.log2(count))))
    return {"bytes": tokens * hk * 2 * (d * size + (4 / case["page"] if size == 1 else 0)) + case["batch"] * hk * g * t * d * 4,
            "flops": 4 * d * hk * g * pairs}
