"""What tree attention (and, for chains, the cached attention) may be off by, term by term, in float64.

O_t = sum p_j v_j, p = softmax(s). With a row's relative errors e_j of the weights w_j = e^(s_j) (which are in its O and in
its sum alike), u_p of P as a matrix operand and the output's unit u, to first order

    |O - exact| <= sum p_j |v_j| (e_j + u_p + a_o) + |O| (sum p_j e_j + a_l) + tail + u |O|

u_p: 2^-11 where P is float16 (float16 and e4m3 caches), 2^-8 where it is bfloat16.

e_j: a score is a float32 sum of D exact products, whose additions may truncate: D 2^-23 sum_d |q_d k_d| scale. The factor and
the exponent's argument are rounded to 2^-24 of their sizes, at most M (the largest |s| and |log2 of a V scale| that the row
sees, and the 16 that P may be shifted by): 2^-21 M with log2's 3 units. 2^x and 1 / scale are good to 2^-21.
Over an e4m3 cache more than 16 rows of a kv head are sums of e4m3 terms beside a largest element of 2^8 or more: what is
below 2^-10 (bfloat16, 2 terms of 4 bits) or 2^-7 (float16, 3) of it is rounded to steps of 2^-9, so to 2^-18 of the largest.
bfloat16 rows up to 16 are float16 there, the largest at least 2^13: 2^-38 of it.

a_o: the products' sums, 16 keys at a time over n keys, truncated: (n / 16 + 8) 2^-23. a_l: (n / 32 + 16) 2^-23 for the sum.

tail: float16's steps end at 2^-24, and P is 2^7 times a weight relative to a maximum that is at most the row's largest w_j
(times its V scale): 2^-32 of that for every key whose P may be below float16's normal 2^-14, times what P multiplies.

The second order is below a 50th of it as long as e_j is, which is asserted."""

import math

import torch

import draft_oracle
import stream_oracle


def tree(q, cache, table, lengths, parents, counts=None, window=0, sinks=0, scale=None):
    """(O, bound)."""
    (b, h, t, d), hk = q.shape, cache.kv_heads
    scale = 1 / math.sqrt(d) if scale is None else scale
    counts = torch.full_like(lengths, t) if counts is None else counts
    e4m3, half = cache.k.dtype == torch.float8_e4m3fn, q.dtype == torch.float16
    there = ((table >= 0) & (table < cache.num_pages)).repeat_interleave(cache.page_size, 1)
    safe = torch.where((table >= 0) & (table < cache.num_pages), table, 0)
    k, v = (stream_oracle.dense(x, s, safe)[:, :, None] for x, s in ((cache.k, cache.k_scale), (cache.v, cache.v_scale)))
    keys = k.shape[3]
    seen = draft_oracle.tree_mask(parents.cpu().expand(b, t), lengths.tolist(), counts.tolist(), keys, window, sinks).to(q.device)
    seen = (seen & there[:, None])[:, None, None]
    q = q.double().reshape(b, hk, h // hk, t, d)
    k, v = (torch.where(seen.any(-2)[..., None], x, 0.0) for x in (k, v))  # what no row sees may hold anything
    s = q @ k.mT * scale
    p, _ = stream_oracle.softmax(s, seen)
    o = p @ v
    most = q.abs().amax(-1, keepdim=True)
    off = q.abs() @ k.abs().mT * (abs(scale) * d * 2.0**-23)
    if e4m3 and h // hk * t > 16:
        rounded = q.abs() < most * 2.0 ** (-7 if half else -10)
        off += (rounded.double() * most) @ k.abs().mT * (abs(scale) * 2.0**-18)
    elif e4m3 and not half:
        off += most * k.abs().sum(-1)[..., None, :] * (abs(scale) * 2.0**-38)
    # The V scale of every position, 1 where there is none.
    vs = torch.ones(b, 1, 1, 1, keys, dtype=torch.float64, device=q.device)
    if e4m3:
        vs = cache.v_scale[safe.long()].double().transpose(1, 2).repeat_interleave(cache.page_size, 2)[:, :, None, None]
    sizes = torch.where(seen, torch.maximum(s.abs(), vs.log2().abs()), 0.0).amax(-1, keepdim=True) * 1.5 + 16
    e = torch.where(seen, off + 2.0**-21 * sizes + 2.0**-21, 0.0)
    assert e.max() < 0.02
    u = 2.0**-11 if half else 2.0**-8
    u_p = 2.0**-11 if e4m3 or half else 2.0**-8
    n = seen.sum(-1, keepdim=True)
    a_o, a_l = (n / 16 + 8) * 2.0**-23, (n / 32 + 16) * 2.0**-23
    bound = (p * (e + u_p + a_o)) @ v.abs() + o.abs() * ((p * e).sum(-1, keepdim=True) + a_l + u)
    if u_p == 2.0**-11:
        w = p * vs
        low = seen & (w < 2.0**-20 * w.amax(-1, keepdim=True))
        bound += 2.0**-32 * w.amax(-1, keepdim=True) * (low.double() @ (v / vs.transpose(-1, -2)).abs())
    bound = bound * 1.04 + (2.0**-25 if half else 2.0**-130)
    return o.reshape(b, h, t, d), bound.reshape(b, h, t, d)
