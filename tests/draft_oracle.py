"""64-bit definitions of the operators for drafted tokens, an error bound for tree attention, and the
pages' bookkeeping on lists.

The tree kernel rounds P to 16 bits for the matrix instruction (a relative error u_p each: 2^-11 in
float16, which it takes over an e4m3 cache, else the tensors' unit), normalises by the sum of P as it
rounded it or before (another u_p at most), and takes 2^x to 2^-22 (a degree-3 polynomial for some columns:
1.0e-4). A score is a float32 sum of D products: off by at most D 2^-24 of the sum of their sizes, which is
below 2^-17 |q||k| scale for D = 128, and by as much again for float16 queries made of bfloat16 ones. So P is off by e = 2 u_p + 3e-4 + 2^-16 max|q||k|scale, relative to
its value, and O = sum P v / sum P by e (sum P |v| + |O|), rounded once more."""

import math

import torch

import stream_oracle

POLY = 3e-4


def ancestors(parents, count):
    """[T, T] truth values: node t sees node a (itself and its ancestors); nothing from `count` on."""
    t = len(parents)
    sees = torch.zeros(t, t, dtype=torch.bool)
    for i in range(count):
        at = i
        while True:
            sees[i, at] = True
            up = int(parents[at])
            if up < 0 or up >= at:  # a parent that is none hangs the node on the context
                break
            at = up
    return sees


def tree_mask(parents, lengths, counts, keys, window, sinks):
    """[B, T, keys] truth values."""
    b, t = parents.shape
    out = torch.zeros(b, t, keys, dtype=torch.bool)
    j = torch.arange(keys)
    for i in range(b):
        count = min(max(int(counts[i]), 0), t)
        context = max(int(lengths[i]), 0) - count
        sees = ancestors(parents[i].tolist(), count)
        for n in range(count):
            position = context + int(sees[n].sum()) - 1
            row = j < context
            if window:
                row &= (position - j < window) | (j < sinks)
            at = context + sees[n].nonzero()[:, 0]
            row[at[(at >= 0) & (at < keys)]] = True
            out[i, n] = row
    return out


def tree(q, cache, table, lengths, parents, counts=None, window=0, sinks=0, scale=None, least=1e-6):
    """(O, bound on what the kernel makes of it, at least `least`) in float64. Pages outside the pool are not seen."""
    (b, h, t, d), hk = q.shape, cache.kv_heads
    scale = 1 / math.sqrt(d) if scale is None else scale
    counts = torch.full_like(lengths, t) if counts is None else counts
    there = ((table >= 0) & (table < cache.num_pages)).repeat_interleave(cache.page_size, 1)
    safe = torch.where((table >= 0) & (table < cache.num_pages), table, 0)
    k, v = (stream_oracle.dense(x, s, safe) for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    seen = tree_mask(parents.cpu().expand(b, t), lengths.tolist(), counts.tolist(), k.shape[2], window, sinks).to(q.device)
    seen = (seen & there[:, None])[:, None, None]
    s = q.double().reshape(b, hk, h // hk, t, d) @ k.transpose(-1, -2)[:, :, None] * scale
    p, _ = stream_oracle.softmax(s, seen)
    # 0 times what is hidden, infinities and NaN among it, is 0; what every row hides is left out, the rest row by row.
    o = torch.zeros(b, hk, h // hk, t, d, dtype=torch.float64, device=q.device)
    size = torch.zeros_like(o)
    odd = ~torch.isfinite(v).all(-1)  # [b, hk, keys]
    clean = torch.where(odd[..., None], 0.0, v)
    o += p @ clean[:, :, None]
    size += p @ clean.abs()[:, :, None]
    for i, j, key in odd.nonzero().tolist():
        w = p[i, j, :, :, key][..., None]
        o[i, j] += torch.where(seen[i, :, 0, :, key, None], w * v[i, j, key], 0.0)
    finite = lambda x: torch.where(torch.isfinite(x), x, 0.0)  # noqa: E731
    big = (finite(q.double()).norm(dim=-1).max() * finite(k).norm(dim=-1).max() * abs(scale)).item()
    u = stream_oracle.unit(q.dtype)
    u_p = 2.0**-11 if cache.k.dtype == torch.float8_e4m3fn else u
    e = 2 * u_p + POLY + 2.0**-16 * big
    bound = e * (size + o.abs()) + u * o.abs() + least
    return o.reshape(b, h, t, d), bound.reshape(b, h, t, d)


def rotary(x, positions, cos, sin, axes=None, interleaved=False, inverse=False, wide=torch.float64):
    """x [B, H, T, D] turned, from the formula, in `wide`."""
    if positions.dim() == 2:
        positions = positions[None]
    rows, half = cos.shape
    axes = [0] * half if axes is None else axes
    y = x.to(wide).clone()
    for i in range(half):
        at = positions[axes[i]].long().clamp(0, rows - 1)
        c, s = cos[at, i].to(wide)[:, None], sin[at, i].to(wide)[:, None]
        s = -s if inverse else s
        lo, hi = (2 * i, 2 * i + 1) if interleaved else (i, i + half)
        a, b = x[..., lo].to(wide), x[..., hi].to(wide)
        y[..., lo] = a * c - b * s
        y[..., hi] = b * c + a * s
    real = ((positions >= 0) & (positions < rows)).all(0)
    return torch.where(real[:, None, :, None], y, 0.0)


def keep(pool, scale, table, lengths, kept, counts, tokens):
    """A pool (and scales) after the kept tokens moved, with float32's products, and the new lengths."""
    pool = pool.clone()
    scale = None if scale is None else scale.clone()
    pages, heads, page, _ = pool.shape
    new = []
    for b, row in enumerate(kept.tolist()):
        count = tokens if counts is None else min(max(int(counts[b]), 0), tokens)
        length = max(int(lengths[b]), 0)
        start = length - count
        path = []
        for x in row[:tokens]:
            if x <= (path[-1] if path else -1) or x >= count:
                break
            path.append(x)
        new.append(start + len(path))

        def place(token):
            position = start + token
            if position < 0 or position // page >= table.shape[1]:
                return None
            at = int(table[b, position // page])
            return (at, position % page) if 0 <= at < pages else None

        moves = [(place(x), place(j)) for j, x in enumerate(path)]
        moves = [m for m in moves if None not in m]
        rows = [pool[f[0], :, f[1]].clone() for f, _ in moves]
        if scale is not None:
            before = scale.clone()
            for f, to in moves:
                scale[to[0]] = torch.maximum(scale[to[0]], before[f[0]])
            for i in range(max(start, 0) // page, -(-length // page)):
                at = int(table[b, i]) if i < table.shape[1] else -1
                if not 0 <= at < pages:
                    continue
                grown = scale[at] > before[at]
                n = min(page, length - i * page)
                again = (pool[at, :, :n].float() * (before[at] / scale[at])[:, None, None]).to(pool.dtype)
                pool.view(torch.uint8)[at, :, :n] = torch.where(grown[:, None, None], again.view(torch.uint8), pool.view(torch.uint8)[at, :, :n])
            rows = [(x.float() * (before[f[0]] / scale[to[0]])[:, None]).to(pool.dtype) for x, (f, to) in zip(rows, moves)]
        raw = pool.view(torch.uint8) if scale is not None else pool
        for x, (_, to) in zip(rows, moves):
            raw[to[0], :, to[1]] = x.view(raw.dtype)
    return pool, scale, new


class Pages:
    """The bookkeeping on lists."""

    def __init__(self, refs):
        self.refs = list(refs)

    def inside(self, p):
        return 0 <= p < len(self.refs)

    def fork(self, table, rows):
        out = [[p if self.inside(p) else -1 for p in table[r]] if 0 <= r < len(table) else [-1] * len(table[0]) for r in rows]
        for p in sum(out, []):
            if p >= 0:
                self.refs[p] += 1
        return out

    def free(self, table, keep=None):
        for b, row in enumerate(table):
            for i in range(0 if keep is None else max(keep[b], 0), len(row)):
                if self.inside(row[i]):
                    self.refs[row[i]] = max(self.refs[row[i]] - 1, 0)
                row[i] = -1

    def reserve(self, table, lengths, tokens, page, counts=None):
        was, free = list(self.refs), [p for p, n in enumerate(self.refs) if n == 0]
        granted, src, dst, asked = [], [], [], 0
        for b, row in enumerate(table):
            count = tokens if counts is None else min(max(counts[b], 0), tokens)
            start = lengths[b] - count
            fits = start >= 0 and lengths[b] <= len(row) * page
            need = []
            if fits and count:
                need = [i for i in range(start // page, -(-lengths[b] // page)) if not self.inside(row[i]) or was[row[i]] > 1]
            asked += len(need)
            granted.append(fits and (not need or asked <= len(free)))
            src.append(-1)
            dst.append(-1)
            for n, i in enumerate(need if granted[-1] else []):
                new = free[asked - len(need) + n]
                if self.inside(row[i]):
                    self.refs[row[i]] -= 1
                    if i == start // page and start % page:
                        src[-1], dst[-1] = row[i], new
                self.refs[new] += 1
                row[i] = new
        return granted, src, dst
