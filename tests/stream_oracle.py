"""64-bit definitions of the streaming operators, and error bounds of the kernels against them.

u is the unit roundoff of the tensors' type (2^-11 float16, 2^-8 bfloat16). The kernels round P and
dS to 16 bits for the matrix instructions (relative u each), sum in float32 (relative errors of
about 2^-20, below the slack), may take 2^x by a degree-3 polynomial (1.0e-4) and divide by the sum
of the rounded P, which makes P relative to its exact value at most e = 2 u + 3e-4 off."""

import math

import torch

POLY = 3e-4


def unit(dtype):
    return 2.0**-11 if dtype == torch.float16 else 2.0**-8


def visible(pos, keys, window, sinks):
    """[..., queries, keys] for query positions `pos`."""
    j = torch.arange(keys, device=pos.device)
    gap = pos[..., :, None] - j
    seen = gap >= 0
    return seen & ((gap < window) | (j < sinks)) if window else seen


def softmax(s, seen):
    s = s.masked_fill(~seen, -math.inf)
    top = s.amax(-1, keepdim=True)
    w = (s - torch.where(top == -math.inf, 0.0, top)).exp()
    w = torch.where(seen, w, 0.0)
    total = w.sum(-1, keepdim=True)
    p = w / torch.where(total > 0, total, 1.0)
    lse = torch.where(total > 0, top + total.log(), -math.inf)[..., 0]
    return p, lse


def window_forward(q, k, v, window, sinks, scale=None):
    """(O, LSE, P) in float64; P [B, Hkv, G, Nq, Nk]."""
    (b, h, n, d), hk = q.shape, k.shape[1]
    scale = 1 / math.sqrt(d) if scale is None else scale
    qd, kd, vd = q.double().reshape(b, hk, h // hk, n, d), k.double()[:, :, None], v.double()[:, :, None]
    pos = k.shape[2] - n + torch.arange(n, device=q.device)
    p, lse = softmax(qd @ kd.transpose(-1, -2) * scale, visible(pos, k.shape[2], window, sinks))
    return (p @ vd).reshape(b, h, n, d), lse.reshape(b, h, n), p


def window_backward(do, q, k, v, window, sinks, scale=None):
    """(dQ, dK, dV) in float64 by the formulas, and dS and P they are made of."""
    (b, h, n, d), hk = q.shape, k.shape[1]
    scale = 1 / math.sqrt(d) if scale is None else scale
    o, _, p = window_forward(q, k, v, window, sinks, scale)
    split = lambda t: t.double().reshape(b, hk, h // hk, n, d)  # noqa: E731
    kd, vd = k.double()[:, :, None], v.double()[:, :, None]
    delta = (split(do) * split(o)).sum(-1, keepdim=True)
    ds = p * (split(do) @ vd.transpose(-1, -2) - delta) * scale
    dq = (ds @ kd).reshape(b, h, n, d)
    dk = (ds.transpose(-1, -2) @ split(q)).sum(2)
    dv = (p.transpose(-1, -2) @ split(do)).sum(2)
    return dq, dk, dv, ds, p


def forward_bound(o, vmax, u_p, u_out):
    """|O - exact| elementwise: P's errors move O by at most (their size) * 2 max|v|; O is rounded
    once."""
    return (2 * u_p + POLY) * 2 * vmax + u_out * o.abs() + 1e-6


def backward_bounds(do, q, k, v, window, sinks, scale=None):
    """Elementwise bounds of (dQ, dK, dV). P is off by e relative; delta = dO.O by |dO| times O's
    own bound; dS by (e + u)|dS| + p scale |its delta's error|; sums add these up."""
    (b, h, n, d), hk = q.shape, k.shape[1]
    scale = abs(1 / math.sqrt(d) if scale is None else scale)
    u = unit(q.dtype)
    e = 2 * u + POLY
    o, _, _ = window_forward(q, k, v, window, sinks, scale)
    dq, dk, dv, ds, p = window_backward(do, q, k, v, window, sinks, scale)
    split = lambda t: t.double().reshape(b, hk, h // hk, n, d).abs()  # noqa: E731
    o_err = forward_bound(o, v.double().abs().max(), u, u)
    delta_err = (split(do) * o_err.reshape(b, hk, h // hk, n, d)).sum(-1, keepdim=True)
    ds_err = (e + u) * ds.abs() + p * scale * delta_err
    q_err = (ds_err @ k.double().abs()[:, :, None]).reshape(b, h, n, d) + u * dq.abs() + 1e-6
    k_err = (ds_err.transpose(-1, -2) @ split(q)).sum(2) + u * dk.abs() + 1e-6
    v_err = ((e + u) * p.transpose(-1, -2) @ split(do)).sum(2) + u * dv.abs() + 1e-6
    return q_err, k_err, v_err


def check(got, want, bound, what):
    got = got.double()
    assert got.shape == want.shape, (what, got.shape, want.shape)
    assert torch.isfinite(got).all(), f"{what}: not finite"
    over = ((got - want).abs() / bound).max().item() if want.numel() else 0.0
    assert over <= 1.0, f"{what}: error is {over:.3g} of its bound"


# ------------------------------------------------------------------------------------ the cache


def dense(pool, scale, table):
    """A cache's pages side by side in float64: [B, Hkv, positions, D]."""
    x = pool[table.long()].double()
    if scale is not None:
        x = x * scale[table.long()].double()[..., None, None]
    b, p, h, n, d = x.shape
    return x.transpose(1, 2).reshape(b, h, p * n, d)


def cached(q, cache, table, lengths, counts=None, window=0, sinks=0, scale=None):
    (b, h, t, d), hk = q.shape, cache.kv_heads
    scale = 1 / math.sqrt(d) if scale is None else scale
    k, v = dense(cache.k, cache.k_scale, table), dense(cache.v, cache.v_scale, table)
    counts = torch.full_like(lengths, t) if counts is None else counts
    step = torch.arange(t, device=q.device)
    pos = torch.where(step < counts[:, None], (lengths - counts)[:, None] + step, -1)
    seen = visible(pos, k.shape[2], window, sinks)[:, None, None]
    s = q.double().reshape(b, hk, h // hk, t, d) @ k.transpose(-1, -2)[:, :, None] * scale
    p, _ = softmax(s, seen)
    # Positions that no query sees may hold anything, NaN among it.
    v = torch.where(seen.any(-2).any(2)[..., None], v, 0.0)
    return (p @ v[:, :, None]).reshape(b, h, t, d), v.abs().max()


def turned(x, pos, cos, sin, interleaved=False, wide=torch.float64):
    """x [..., T, D] rotated at positions [B, T]; float32 gives the kernels' own roundings."""
    x = x.to(wide)
    if cos is None:
        return x
    c, s = cos[pos].to(wide)[:, None], sin[pos].to(wide)[:, None]
    r = 2 * cos.shape[1]
    y = x.clone()
    if interleaved:
        a, b = x[..., 0:r:2], x[..., 1:r:2]
        y[..., 0:r:2], y[..., 1:r:2] = a * c - b * s, b * c + a * s
    else:
        a, b = x[..., : r // 2], x[..., r // 2 : r]
        y[..., : r // 2], y[..., r // 2 : r] = a * c - b * s, b * c + a * s
    return y


def power_of_two(amax):
    """The e4m3 block scale of a largest value (a Python float)."""
    if amax == 0:
        return 2.0**-60
    m, e = math.frexp(amax)
    return 2.0 ** max(-60, e - 9 if m <= 0.875 else e - 8)


def append(pool, scale, new, table, lengths, counts):
    """Stores new [B, Hkv, T, D] (float32, rotated) into copies of (pool, scale), token by token of
    the definition; returns (pool, scale)."""
    pool = pool.clone()
    scale = None if scale is None else scale.clone()
    page = pool.shape[2]
    raw = pool.view(torch.uint8) if scale is not None else pool
    for b in range(new.shape[0]):
        length, count = int(lengths[b]), int(counts[b])
        start = length - count
        if count == 0:
            continue
        for nth in range(start // page, -(-length // page)):
            lo, hi = max(start, nth * page), min(length, (nth + 1) * page)
            at = int(table[b, nth])
            for h in range(new.shape[1]):
                x = new[b, h, lo - start : hi - start]
                if scale is None:
                    pool[at, h, lo - nth * page : hi - nth * page] = x.to(pool.dtype)
                    continue
                fine = torch.where(torch.isfinite(x), x.abs(), 0.0)
                s = power_of_two(float(fine.max()))
                if lo > nth * page:
                    before = float(scale[at, h])
                    s = max(s, before)
                    old = pool[at, h, : lo - nth * page].float() * (before / s)
                    raw[at, h, : lo - nth * page] = old.to(pool.dtype).view(torch.uint8)
                y = torch.where(x.isnan(), x, (x / s).clamp(-448, 448))
                raw[at, h, lo - nth * page : hi - nth * page] = y.to(pool.dtype).view(torch.uint8)
                scale[at, h] = s
    return pool, scale
