"""The norm check of the window gradients rejects what it is there to reject: gradients of a window that is one
off, without delta, without one streamed tile, without one head of a group, zeros; in both types."""

import math

import pytest
import torch

import stream_oracle as oracle
import stream_spread as spread


def _inputs(b, h, hk, nq, nk, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    return tuple(torch.randn(s, generator=g).to(dtype) for s in ((b, h, nq, d), (b, hk, nk, d), (b, hk, nk, d), (b, h, nq, d)))


def _gradients(do, q, k, v, window, sinks, wrong=None):
    """The definition's in float64, with one thing wrong."""
    (b, h, n, d), hk = q.shape, k.shape[1]
    if wrong == "window":
        window += 1
    _, _, _, ds, p = oracle.window_backward(do, q, k, v, window, sinks)
    split = lambda t: t.double().reshape(b, hk, h // hk, n, d)  # noqa: E731
    if wrong == "delta":
        ds = p * (split(do) @ v.double()[:, :, None].transpose(-1, -2)) / math.sqrt(d)
    if wrong == "tile":  # the last query tile's pairs with the tile of keys before its own
        rows, last = slice((n - 1) // 128 * 128, n), (k.shape[2] - 1) // 128
        cols = slice((last - 1) * 128, last * 128)
        p, ds = p.clone(), ds.clone()
        p[..., rows, cols] = ds[..., rows, cols] = 0
    keep = slice(1, None) if wrong == "head" else slice(None)
    dq = (ds @ k.double()[:, :, None]).reshape(b, h, n, d)
    dk = (ds.transpose(-1, -2) @ split(q))[:, :, keep].sum(2)
    dv = (p.transpose(-1, -2) @ split(do))[:, :, keep].sum(2)
    return dq, dk, dv


SHAPES = [  # b, h, hk, nq, nk, window, sinks
    (1, 2, 2, 129, 129, 64, 4),
    (1, 4, 1, 300, 300, 100, 130),
    (1, 4, 2, 1000, 1000, 256, 1),
    (1, 2, 2, 777, 777, 0, 0),
    (1, 2, 1, 100, 900, 200, 4),
    (1, 2, 1, 1, 700, 300, 2),
]


@pytest.mark.parametrize("b,h,hk,nq,nk,window,sinks", SHAPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_wrong_gradients_are_rejected(b, h, hk, nq, nk, window, sinks, d, dtype):
    q, k, v, do = _inputs(b, h, hk, nq, nk, d, dtype, seed=nq)
    want, var = spread.backward(do, q, k, v, window, sinks)
    ratios = lambda got: [spread.worst(g, w, x) for g, w, x in zip(got, want, var)]  # noqa: E731
    assert max(ratios([w.to(dtype) for w in want])) <= 1.01  # rounding alone: u/sqrt(3) is its most
    assert max(ratios(_gradients(do, q, k, v, window, sinks))) <= 1e-6
    assert min(ratios([torch.zeros_like(w) for w in want])) > spread.LIMIT
    if window:
        assert min(ratios(_gradients(do, q, k, v, window, sinks, "window"))) > spread.LIMIT
    assert min(ratios(_gradients(do, q, k, v, window, sinks, "delta"))[:2]) > spread.LIMIT
    if nk > 256 and nq > 128:
        assert min(ratios(_gradients(do, q, k, v, window, sinks, "tile"))) > spread.LIMIT
    if h > hk:
        assert min(ratios(_gradients(do, q, k, v, window, sinks, "head"))[1:]) > spread.LIMIT
