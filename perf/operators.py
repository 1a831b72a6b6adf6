"""Cases of the attention layer's streaming operators, with their plain forms.

Three operators, as a model that attends over a sliding window and a few first tokens (sinks)
trains and serves with them:

  append   rotation of new queries and keys by their positions, keys and values stored into a
           paged cache (16 bits, or e4m3 with a power-of-two scale for every page and head)
  cached   attention of the newest tokens of every sequence over that cache
  window   causal attention with a window and sinks over dense tensors, forward ("fwd") or a
           training step's forward and backward ("train")

``own`` False computes the plain form in 32-bit torch operations; ``own`` True calls the
framework's entry points.
"""

import math
import os
import sys

import torch

own = False

E4M3_MAX = 448.0
MIN_EXP = -60  # smallest exponent of a block scale
TYPES = {"f16": torch.float16, "bf16": torch.bfloat16, "e4m3": torch.float8_e4m3fn}


def _fa():
    here = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "flash-attention-from-scratch_b200")
    if here not in sys.path:
        sys.path.insert(0, here)
    import fa

    return fa


# ------------------------------------------------------------------------------------ the cases


def _append(name, batch, tokens, heads, kv_heads, dim, dtype, cache, page, before, ragged):
    return dict(name=name, op="append", batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim,
                dtype=dtype, cache=cache, page=page, before=before, ragged=ragged)


def _cached(name, batch, tokens, heads, kv_heads, dim, dtype, cache, page, length, spread, window, sinks):
    return dict(name=name, op="cached", batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim,
                dtype=dtype, cache=cache, page=page, length=length, spread=spread, window=window, sinks=sinks)


def _window(name, mode, batch, heads, kv_heads, n, dim, dtype, window, sinks):
    return dict(name=name, op="window", mode=mode, batch=batch, heads=heads, kv_heads=kv_heads, n=n, dim=dim,
                dtype=dtype, window=window, sinks=sinks)


def listed():
    return [
        # One user, one new token: nothing but the latency of a call.
        _append("append one token", 1, 1, 16, 16, 64, "f16", "f16", 16, 500, False),
        # One decoding step of a served batch, grouped heads, 8-bit cache.
        _append("append a decode step", 128, 1, 32, 8, 128, "bf16", "e4m3", 64, 3000, False),
        # Prompts of unequal length entering the cache.
        _append("append prompts", 4, 4000, 32, 8, 128, "bf16", "e4m3", 64, 0, True),
        # One user, one token over a short context in 16 bits.
        _cached("decode one short", 1, 1, 16, 16, 64, "f16", "f16", 16, 777, 0.0, 0, 0),
        # A served batch of unequal contexts, 8-bit cache, one token each.
        _cached("decode a batch", 32, 1, 32, 8, 128, "bf16", "e4m3", 64, 8192, 0.5, 0, 0),
        # Few users with very long documents.
        _cached("decode long documents", 4, 1, 32, 8, 128, "bf16", "e4m3", 64, 131000, 0.1, 0, 0),
        # Four drafted tokens checked at once, window and sinks.
        _cached("check drafted tokens", 64, 4, 32, 8, 128, "bf16", "e4m3", 64, 16384, 0.5, 4096, 4),
        # The smallest forward: a short prompt in a small model.
        _window("window forward, short", "fwd", 1, 4, 4, 512, 64, "f16", 128, 4),
        # A prompt batch, the framework's 4 x 16 heads x 4096 x 128 configuration.
        _window("window forward", "fwd", 4, 16, 16, 4096, 128, "bf16", 1024, 4),
        # A training step on short odd rows, head dim 64, grouped heads.
        _window("window training, short", "train", 2, 8, 2, 1000, 64, "f16", 256, 1),
        # A training step on long rows that end inside a tile.
        _window("window training", "train", 1, 16, 4, 8191, 128, "bf16", 1024, 4),
        # The longest training rows, a wide window.
        _window("window training, long", "train", 1, 8, 2, 16384, 128, "bf16", 4096, 4),
    ]


def _log(rng, low, high):
    return int(round(math.exp(rng.uniform(math.log(low), math.log(high)))))


def draw(rng):
    op = rng.choice(["append", "cached", "window", "window"])
    dim = rng.choice([64, 128])
    dtype = rng.choice(["f16", "bf16"])
    cache = rng.choice([dtype, "e4m3", "e4m3"])
    page = rng.choice([16, 32, 64, 128])
    kv_heads = rng.choice([1, 2, 4, 8, 16])
    if op == "append":
        heads = kv_heads * rng.choice([1, 2, 4])
        budget = 60_000_000 // (heads * dim)  # tokens in all
        batch = _log(rng, 1, 128)
        tokens = 1 if rng.random() < 0.4 else max(1, min(_log(rng, 2, 4000), budget // batch))
        return dict(op=op, batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype,
                    cache=cache, page=page, before=_log(rng, 1, 3001) - 1, ragged=rng.random() < 0.5)
    if op == "cached":
        heads = kv_heads * rng.choice([1, 2, 4, 8])
        tokens = 1 if rng.random() < 0.6 else rng.randint(2, 8)
        batch = _log(rng, 1, 64)
        budget = 500_000_000 // (kv_heads * dim * (1 if cache == "e4m3" else 2) * batch)
        length = max(tokens, min(_log(rng, 20, 131000), budget))
        window = rng.choice([0, 0, _log(rng, 16, 4096)])
        return dict(op=op, batch=batch, tokens=tokens, heads=heads, kv_heads=kv_heads, dim=dim, dtype=dtype,
                    cache=cache, page=page, length=length, spread=rng.choice([0.0, 0.3, 0.8]), window=window,
                    sinks=rng.choice([0, 1, 4, 17]) if window else 0)
    kv_heads = rng.choice([1, 2, 4])
    heads = kv_heads * rng.choice([1, 2, 4])
    n = _log(rng, 30, 8192)
    batch = rng.choice([1, 2, 3]) if n < 4096 else 1
    return dict(op=op, mode=rng.choice(["fwd", "train"]), batch=batch, heads=heads, kv_heads=kv_heads, n=n, dim=dim,
                dtype=dtype, window=_log(rng, 16, 4096), sinks=rng.choice([0, 1, 4, 17, 130]))


# --------------------------------------------------------------------------------------- inputs


def _spread(case):
    """Lengths of the sequences, given by the case alone: the longest down to `spread` of it less."""
    longest, share = case["length"], case["spread"]
    return [max(case["tokens"], int(longest * (1 - share * math.modf((b + 1) * 0.6180339887)[0] * (case["batch"] > 1))))
            for b in range(case["batch"])]


def _counts(case):
    """New tokens of every sequence: all of them, or (ragged) between a quarter and all."""
    t = case["tokens"]
    if not case["ragged"]:
        return [t] * case["batch"]
    return [max(1, int(t * (1 - 0.75 * math.modf(b * 0.6180339887)[0]))) for b in range(case["batch"])]


def _ints(values):
    return torch.tensor(values, dtype=torch.int32, device="cuda")


def _pages(gen, batch, most, page):
    """A table of pages in random order, and how many pages the pool has."""
    per = -(-most // page)
    table = torch.randperm(batch * per + 3, generator=gen, device="cuda")[: batch * per]
    return table.to(torch.int32).view(batch, per), batch * per + 3


def _power_of_two(amax):
    """2^k with the smallest k >= MIN_EXP for which amax <= 448 * 2^k."""
    m, e = torch.frexp(amax)
    k = torch.where(amax > 0, torch.where(m <= 0.875, e - 9, e - 8), MIN_EXP).clamp(min=MIN_EXP)
    return torch.ldexp(torch.ones_like(amax), k)


def _filled(gen, pages, case):
    """A cache's pages as earlier tokens left them: values of unit scale with a few large channels."""
    shape = (pages, case["kv_heads"], case["page"], case["dim"])
    x = torch.empty(shape, device="cuda", dtype=torch.float16).normal_(generator=gen)
    x[..., :: 32] *= 4
    if case["cache"] != "e4m3":
        return x.to(TYPES[case["cache"]]), None
    scale = _power_of_two(x.abs().amax(dim=(2, 3)).float())
    return (x.float() / scale[:, :, None, None]).to(TYPES["e4m3"]), scale


def prepare(case, seed):
    gen = torch.Generator("cuda").manual_seed(seed)
    b, d = case["batch"], case["dim"]
    hq, hk = case["heads"], case["kv_heads"]
    dt = TYPES[case["dtype"]]

    def normal(*shape):
        return torch.empty(shape, device="cuda", dtype=dt).normal_(generator=gen)

    s = {"case": dict(case)}
    if case["op"] == "window":
        n = case["n"]
        s |= {"q": normal(b, hq, n, d), "k": normal(b, hk, n, d), "v": normal(b, hk, n, d)}
        if case["mode"] == "train":
            s["do"] = normal(b, hq, n, d)
            for x in ("q", "k", "v"):
                s[x].requires_grad_(True)
        return s
    t = case["tokens"]
    if case["op"] == "append":
        before, counts = case["before"], _counts(case)
        lengths = [before + (7 * i) % 64 + c for i, c in enumerate(counts)]
        s |= {"k_new": normal(b, hk, t, d), "v_new": normal(b, hk, t, d)}
        s["counts"] = _ints(counts) if case["ragged"] else None
        turn = torch.arange(max(lengths), device="cuda", dtype=torch.float64)[:, None] * 10000.0 ** (
            -torch.arange(d // 2, device="cuda", dtype=torch.float64) * 2 / d)
        s |= {"cos": turn.cos().float(), "sin": turn.sin().float()}
    else:
        lengths, s["counts"] = _spread(case), None
    s["q"] = normal(b, hq, t, d)
    s["lengths"] = _ints(lengths)
    s["table"], pages = _pages(gen, b, max(lengths), case["page"])
    (s["k"], s["ks"]), (s["v"], s["vs"]) = (_filled(gen, pages, case) for _ in "kv")
    if own:
        s["cache"] = _fa().PagedKVCache(s["k"], s["v"], s["ks"], s["vs"])
    return s


# ---------------------------------------------------------------------------------- plain forms


def _visible(pos, keys, window, sinks):
    """Truth values [..., queries, keys]: which key positions a query at `pos` sees."""
    gap = pos[..., :, None] - keys
    seen = gap >= 0
    return seen & ((gap < window) | (keys < sinks)) if window else seen


def _softmax(s, seen):
    """Probabilities of masked scores; zeros in a row that sees nothing. Works on `s` in place."""
    s.masked_fill_(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    s.sub_(torch.where(top == -math.inf, 0.0, top)).exp_()
    return s.div_(s.sum(-1, keepdim=True).clamp(min=1e-37))


def _rotate(x, cos, sin):
    a, b = x.chunk(2, -1)
    return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)


def _plain_append(s):
    c = s["case"]
    t, page = c["tokens"], c["page"]
    b, table = c["batch"], s["table"].long()
    lengths = s["lengths"].long()
    counts = s["counts"].long() if s["counts"] is not None else torch.full_like(lengths, t)
    start = lengths - counts
    pos = start[:, None] + torch.arange(t, device="cuda")
    real = torch.arange(t, device="cuda") < counts[:, None]
    at = pos.clamp(max=s["cos"].shape[0] - 1)
    cos, sin = s["cos"][at][:, None], s["sin"][at][:, None]
    q = torch.where(real[:, None, :, None], _rotate(s["q"].float(), cos, sin), 0.0).to(s["q"].dtype)
    k, v = _rotate(s["k_new"].float(), cos, sin), s["v_new"].float()
    if c["cache"] != "e4m3":
        slot = torch.where(real, table.gather(1, pos.clamp(max=table.shape[1] * page - 1) // page), 0)
        bb, tt = real.nonzero(as_tuple=True)
        for pool, new in ((s["k"], k), (s["v"], v)):
            pool[slot[bb, tt], :, pos[bb, tt] % page] = new[bb, :, tt].to(pool.dtype)
        return q, s["k"], s["v"]
    # Every page that gets a token, as a whole: older tokens keep their place, new ones join them.
    first = start // page
    span = (t + page - 2) // page + 1
    which = first[:, None] + torch.arange(span, device="cuda")
    touched = which * page < lengths[:, None]
    ids = table.gather(1, which.clamp(max=table.shape[1] - 1))
    where = which[..., None] * page + torch.arange(page, device="cuda")  # [b, span, page] positions
    new = (where >= start[:, None, None]) & (where < lengths[:, None, None])
    old = where < start[:, None, None]
    src = (where - start[:, None, None]).clamp(0, t - 1)
    out = [q]
    for pool, scales, x in ((s["k"], s["ks"], k), (s["v"], s["vs"], v)):
        h, d = x.shape[1], x.shape[3]
        fresh = x.transpose(1, 2).gather(1, src.view(b, -1, 1, 1).expand(-1, -1, h, d))
        fresh = fresh.view(b, span, page, h, d).transpose(2, 3)
        amax = torch.where(new[:, :, None, :, None], fresh.abs(), 0.0).amax((3, 4))
        before = torch.where(old.any(-1)[..., None], scales[ids], 0.0)
        scale = torch.maximum(_power_of_two(amax), before)
        codes = pool[ids]
        grown = (codes.float() * (before / scale)[..., None, None]).to(pool.dtype)
        coded = (fresh / scale[..., None, None]).to(pool.dtype)
        codes = torch.where(new[:, :, None, :, None], coded.float(), torch.where(old[:, :, None, :, None], grown.float(), codes.float()))
        bb, pp = touched.nonzero(as_tuple=True)
        pool.view(torch.uint8)[ids[bb, pp]] = codes.to(pool.dtype)[bb, pp].view(torch.uint8)
        scales[ids[bb, pp]] = scale[bb, pp]
        out += [pool, scales]
    return tuple(out)


def _dense(pool, scales, table, wide=torch.float32):
    """A cache's pages side by side: [batch, heads, positions, dim]."""
    x = pool[table].to(wide)
    if scales is not None:
        x = x * scales[table].to(wide)[..., None, None]
    b, p, h, n, d = x.shape
    return x.transpose(1, 2).reshape(b, h, p * n, d)


def _plain_cached(s):
    c = s["case"]
    b, hk, t, d = c["batch"], c["kv_heads"], c["tokens"], c["dim"]
    g = c["heads"] // hk
    table = s["table"].long()
    k, v = _dense(s["k"], s["ks"], table), _dense(s["v"], s["vs"], table)
    q = s["q"].float().view(b, hk, g * t, d)
    scores = (q @ k.transpose(-1, -2)).mul_(1 / math.sqrt(d))
    pos = s["lengths"].long()[:, None] - t + torch.arange(t, device="cuda")
    seen = _visible(pos, torch.arange(k.shape[2], device="cuda"), c["window"], c["sinks"])
    p = _softmax(scores.view(b, hk, g, t, -1), seen[:, None, None])
    return (p.view(b, hk, g * t, -1) @ v).view(b, hk * g, t, d).to(s["q"].dtype)


def _plain_window(s):
    c = s["case"]
    b, hk, n, d = c["batch"], c["kv_heads"], c["n"], c["dim"]
    g, scale = c["heads"] // hk, 1 / math.sqrt(d)
    q, k, v = s["q"].detach().float().view(b, hk, g, n, d), s["k"].detach().float()[:, :, None], s["v"].detach().float()[:, :, None]
    at = torch.arange(n, device="cuda")
    seen = _visible(at, at, c["window"], c["sinks"])
    p = _softmax((q @ k.transpose(-1, -2)).mul_(scale), seen)
    o = p @ v
    out = o.view(b, hk * g, n, d).to(s["q"].dtype)
    if c["mode"] == "fwd":
        return out
    do = s["do"].float().view(b, hk, g, n, d)
    dv = (p.transpose(-1, -2) @ do).sum(2)
    ds = (do @ v.transpose(-1, -2)).sub_((do * o).sum(-1, keepdim=True)).mul_(p).mul_(scale)
    dq = (ds @ k).view(b, hk * g, n, d)
    dk = (ds.transpose(-1, -2) @ q).sum(2)
    return out, dq.to(out.dtype), dk.to(out.dtype), dv.to(out.dtype)


def run(state):
    c = state["case"]
    if not own:
        return {"append": _plain_append, "cached": _plain_cached, "window": _plain_window}[c["op"]](state)
    fa = _fa()
    if c["op"] == "append":
        q = fa.append_kv(state["cache"], state["k_new"], state["v_new"], state["table"], state["lengths"],
                         counts=state["counts"], cos=state["cos"], sin=state["sin"], q=state["q"])
        if c["cache"] != "e4m3":
            return q, state["k"], state["v"]
        return q, state["k"], state["ks"], state["v"], state["vs"]
    if c["op"] == "cached":
        return fa.forward_cached(state["q"], state["cache"], state["table"], state["lengths"],
                                 window=c["window"], sinks=c["sinks"])
    if c["mode"] == "fwd":
        return fa.forward_window(state["q"], state["k"], state["v"], c["window"], sinks=c["sinks"])
    o = fa.window_attention(state["q"], state["k"], state["v"], c["window"], sinks=c["sinks"])
    return (o.detach(), *torch.autograd.grad(o, (state["q"], state["k"], state["v"]), state["do"]))


# --------------------------------------------------------------------------------- 64-bit values


def _exact_append(s):
    """The definition token by token in 64 bits; codes stay unrounded (what they stand for, over the scale)."""
    c = s["case"]
    page, half = c["page"], c["dim"] // 2
    counts = s["counts"].tolist() if s["counts"] is not None else [c["tokens"]] * c["batch"]
    q = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    pools = [s["k"].double(), s["v"].double()]
    scales = [x.double() if x is not None else None for x in (s["ks"], s["vs"])]
    for b, (length, count) in enumerate(zip(s["lengths"].tolist(), counts)):
        start = length - count
        cos, sin = (s[x][start:length].double() for x in ("cos", "sin"))

        def turned(x):
            x = x[b, :, :count].double()
            y = torch.empty_like(x)
            y[..., :half] = x[..., :half] * cos - x[..., half:] * sin
            y[..., half:] = x[..., half:] * cos + x[..., :half] * sin
            return y

        q[b, :, :count] = turned(s["q"])
        for i, x in enumerate((turned(s["k_new"]), s["v_new"][b, :, :count].double())):
            for nth in range(start // page, -(-length // page)):
                lo, hi = max(start, nth * page), min(length, (nth + 1) * page)
                new, at = x[:, lo - start : hi - start], int(s["table"][b, nth])
                if scales[i] is not None:
                    need = 2.0 ** torch.ceil(torch.log2(new.abs().amax((1, 2)).clamp(min=1e-300) / E4M3_MAX)).clamp(min=MIN_EXP)
                    have = scales[i][at] if lo > nth * page else torch.zeros_like(need)
                    scale = torch.maximum(need, have)
                    pools[i][at, :, : lo - nth * page] *= (have / scale)[:, None, None]
                    new, scales[i][at] = new / scale[:, None, None], scale
                pools[i][at, :, lo - nth * page : hi - nth * page] = new
    if scales[0] is None:
        return q, pools[0], pools[1]
    return q, pools[0], scales[0], pools[1], scales[1]


def _exact_cached(s):
    c = s["case"]
    t, d, g = c["tokens"], c["dim"], c["heads"] // c["kv_heads"]
    out = torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda")
    for b, length in enumerate(s["lengths"].tolist()):
        ids = s["table"][b : b + 1].long()
        k, v = (_dense(s[x], s[y], ids, torch.float64)[0, :, :length] for x, y in (("k", "ks"), ("v", "vs")))
        key = torch.arange(length, device="cuda")
        for i in range(t):
            p = length - t + i
            mask = key <= p
            if c["window"]:
                mask &= (key > p - c["window"]) | (key < c["sinks"])
            for h in range(c["kv_heads"]):
                w = torch.softmax((s["q"][b, h * g : (h + 1) * g, i].double() @ k[h].T / math.sqrt(d)).masked_fill(~mask, -math.inf), -1)
                out[b, h * g : (h + 1) * g, i] = w @ v[h]
    return out


def _exact_window(s):
    c = s["case"]
    n, d, g = c["n"], c["dim"], c["heads"] // c["kv_heads"]
    i = torch.arange(n, device="cuda")
    hidden = (i > i[:, None]) | ((i <= i[:, None] - c["window"]) & (i >= c["sinks"]))
    o, dq = (torch.zeros(s["q"].shape, dtype=torch.float64, device="cuda") for _ in "ab")
    dk, dv = (torch.zeros(s["k"].shape, dtype=torch.float64, device="cuda") for _ in "ab")
    for b in range(c["batch"]):
        for h in range(c["heads"]):
            q, k, v = s["q"][b, h].detach().double(), s["k"][b, h // g].detach().double(), s["v"][b, h // g].detach().double()
            w = torch.softmax((q @ k.T / math.sqrt(d)).masked_fill_(hidden, -math.inf), -1)
            o[b, h] = w @ v
            if c["mode"] == "fwd":
                continue
            do = s["do"][b, h].double()
            dv[b, h // g] += w.T @ do
            dw = do @ v.T
            w *= dw - (w * dw).sum(-1, keepdim=True)
            dq[b, h] = w @ k / math.sqrt(d)
            dk[b, h // g] += w.T @ q / math.sqrt(d)
    return o if c["mode"] == "fwd" else (o, dq, dk, dv)


def exact(case, seed):
    s = prepare(case, seed)
    return {"append": _exact_append, "cached": _exact_cached, "window": _exact_window}[case["op"]](s)


# ----------------------------------------------------------------------------------------- work


def _seen(pos, window, sinks):
    """How many keys a query at position `pos` sees."""
    if not window or pos < window:
        return pos + 1
    return window + min(sinks, pos + 1 - window)


def work(case):
    hq, hk, d = case["heads"], case["kv_heads"], case["dim"]
    if case["op"] == "window":
        b, n, w, z = case["batch"], case["n"], case["window"], case["sinks"]
        pairs = sum(_seen(p, w, z) for p in range(n)) * b * hq
        rows = b * n * d * 2
        if case["mode"] == "fwd":
            return {"bytes": rows * (2 * hq + 2 * hk), "flops": 4 * d * pairs}
        return {"bytes": rows * (4 * hq + 4 * hk), "flops": 14 * d * pairs}
    size = 1 if case["cache"] == "e4m3" else 2
    if case["op"] == "append":
        tokens = sum(_counts(case))
        pages = tokens // case["page"] + 1
        # queries in and out, keys and values in and into the cache, scales, the tables' rows
        return {"bytes": tokens * d * (4 * hq + 2 * hk * (2 + size)) + (8 * hk * pages if size == 1 else 0) + tokens * d * 4,
                "flops": tokens * d * 3 * (hq + hk)}
    t, tokens, pairs = case["tokens"], 0, 0
    for n in _spread(case):
        first = max(0, n - t)
        lo = max(0, first - case["window"] + 1) if case["window"] else 0
        tokens += n - lo + min(case["sinks"], lo)
        pairs += sum(_seen(p, case["window"], case["sinks"]) for p in range(first, n))
    return {"bytes": tokens * hk * 2 * (d * size + (4 / case["page"] if size == 1 else 0)) + case["batch"] * hq * t * d * 4,
            "flops": 4 * d * hq * pairs}
