"""How far the window kernels' results spread around the 64-bit definition, as root mean squares.

stream_oracle's bounds add up worst cases, element by element, and let errors through that are far above what
rounding makes. Here roundings are what they are, independent of one another: a rounding to a type of unit
roundoff u is off by u/sqrt(3) of the value in root mean square at most (half that for a uniform mantissa), so
variances add. The norm of the error over a head's block of 128 rows is then held to LIMIT times its own root
mean square. LIMIT is 4: within a row several errors are common to all elements (those of the normaliser and
of delta), so a block of one row is as good as one normal variable, beyond 4 deviations once in 16000; a block
of 128 rows is far from it.

What enters, for a pair of query i and key j (p, ds: the definition's; s: |softmax scale|):
  P V, P^T dO      P rounded to 16 bits: u p, independent
  normaliser       the sum of the rounded P, and 2^x by a polynomial of 1.0e-4: e_i = u sqrt(sum_j p^2) / sqrt(3) + 1.2e-4, common to
                   a row, in O, in the LSE and so in the P of the backward
  O                the above and its own rounding; delta_i = dO_i . O_i has sum_d dO^2 var(O) of it
  dP, delta        float32 sums: 2^-20 of the sum of their terms' sizes
  dS               rounded once: u ds
  results          rounded once; in float16 by 2^-25 at least, half of its least step
"""

import math

import torch

import stream_oracle as oracle

LIMIT = 4.0
ROW_BLOCK = 128


def _rounding(x, dtype):
    """Variance of rounding x to `dtype`."""
    step = oracle.unit(dtype) * x.abs()
    if dtype == torch.float16:
        step = step.clamp(min=2.0**-25)
    return step.square() / 3


def backward(do, q, k, v, window, sinks, scale=None):
    """((dQ, dK, dV), their variances) in float64."""
    (b, h, n, d), hk = q.shape, k.shape[1]
    s = abs(1 / math.sqrt(d) if scale is None else scale)
    u2 = oracle.unit(q.dtype) ** 2 / 3
    dq, dk, dv, ds, p = oracle.window_backward(do, q, k, v, window, sinks, scale)
    split = lambda t: t.double().reshape(b, hk, h // hk, n, d)  # noqa: E731
    qd, dod, kd, vd = split(q), split(do), k.double()[:, :, None], v.double()[:, :, None]
    p_var = p.square() * u2
    if q.dtype == torch.float16:
        p_var = torch.where(p > 0, p_var.clamp(min=2.0**-50 / 3), p_var)
    e2 = (u2**0.5 * p.square().sum(-1, keepdim=True).sqrt() + 1.2e-4).square()
    o = p @ vd
    o_var = p_var @ vd.square() + e2 * o.square() + _rounding(o, q.dtype)
    delta_var = (dod.square() * o_var).sum(-1, keepdim=True)
    fine = 2.0**-20 * (dod.abs() @ vd.abs().transpose(-1, -2) + (dod * o).abs().sum(-1, keepdim=True))
    ds_var = ds.square() * u2
    common = ds.square() * e2 + (p * s).square() * (delta_var + fine.square())
    dq_var = ds_var @ kd.square() + e2 * split(dq).square() + delta_var * (s * (p @ kd)).square()
    dq_var = dq_var + ((p * s * fine) @ kd.abs()).square()
    dk_var = ((ds_var + common).transpose(-1, -2) @ qd.square()).sum(2)
    dv_var = ((p_var + p.square() * e2).transpose(-1, -2) @ dod.square()).sum(2)
    out = (dq, dq_var.reshape(b, h, n, d)), (dk, dk_var), (dv, dv_var)
    return (dq, dk, dv), tuple(var + _rounding(x, q.dtype) for x, var in out)


def worst(got, want, var):
    """The largest ratio, over heads and blocks of 128 rows, of the error's norm and its root mean square."""
    err, var = (got.double() - want).square().sum(-1), var.sum(-1)
    pad = -err.shape[-1] % ROW_BLOCK
    blocks = lambda t: torch.nn.functional.pad(t, (0, pad)).unflatten(-1, (-1, ROW_BLOCK)).sum(-1)  # noqa: E731
    err, var = blocks(err), blocks(var)
    # Where nothing can be off (no query sees a block's keys), nothing may be.
    ratio = torch.where(var > 0, err / var.clamp(min=1e-300), torch.where(err > 0, math.inf, 0.0))
    return ratio.max().sqrt().item() if ratio.numel() else 0.0


def check(got, want, var, what):
    assert torch.isfinite(got).all(), f"{what}: not finite"
    r = worst(got, want, var)
    assert r <= LIMIT, f"{what}: the error's norm is {r:.3g} of its root mean square"
