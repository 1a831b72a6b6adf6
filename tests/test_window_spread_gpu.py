"""Window gradients by norms, a head's 128 rows at a time: errors of the size that rounding makes, and no more
(stream_spread; test_window_spread_cpu shows what this rejects)."""

import pytest
import torch

import fa
import stream_spread as spread
from fa import _C

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
HALF, BF = torch.float16, torch.bfloat16


def _inputs(b, h, hk, nq, nk, d, dtype, seed):
    g = torch.Generator(DEV).manual_seed(seed)
    return tuple(torch.randn(s, generator=g, device=DEV).to(dtype) for s in ((b, h, nq, d), (b, hk, nk, d), (b, hk, nk, d), (b, h, nq, d)))


def _check(q, k, v, do, window, sinks, scale=None, heads=None):
    """`heads`: the kv heads to look at, one at a time (all at once without)."""
    o, lse = fa.forward_window(q, k, v, window, sinks, scale, return_lse=True)
    got = fa.backward_window(do, q, k, v, o, lse, window, sinks, scale)
    g = q.shape[1] // k.shape[1]
    for j in [None] if heads is None else heads:
        one = (lambda t: t) if j is None else (lambda t: t[:, j : j + 1])  # noqa: E731, B023
        own = (lambda t: t) if j is None else (lambda t: t[:, j * g : (j + 1) * g])  # noqa: E731, B023
        want, var = spread.backward(own(do), own(q), one(k), one(v), window, sinks, scale)
        for name, x, w, s in zip(("dQ", "dK", "dV"), (own(got[0]), one(got[1]), one(got[2])), want, var):
            spread.check(x, w, s, name)
    assert _C.device_status(0) == 0


@pytest.mark.parametrize("b,h,hk,nq,nk,window,sinks", [
    (1, 1, 1, 1, 1, 1, 0), (2, 2, 1, 17, 17, 5, 1), (1, 4, 2, 128, 128, 128, 0), (1, 2, 2, 129, 129, 64, 4), (2, 3, 3, 257, 257, 1, 0),
    (1, 4, 1, 300, 300, 100, 130), (1, 2, 1, 640, 640, 129, 3), (1, 8, 2, 1000, 1000, 256, 1), (1, 2, 2, 777, 777, 0, 0),
    (1, 2, 2, 500, 500, 5000, 9), (1, 2, 1, 513, 513, 255, 513), (1, 2, 1, 100, 900, 200, 4), (1, 2, 1, 1, 700, 300, 2),
    (1, 2, 1, 700, 100, 50, 2), (1, 2, 1, 385, 129, 64, 0), (3, 32, 8, 300, 300, 70, 2), (1, 2, 1, 4097, 4097, 200, 5),
])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [HALF, BF])
def test_gradients_by_norms(b, h, hk, nq, nk, window, sinks, d, dtype):
    q, k, v, do = _inputs(b, h, hk, nq, nk, d, dtype, seed=100 + nq + window)
    _check(q, k, v, do, window, sinks)


@pytest.mark.parametrize("b,h,hk,n,d,window,sinks", [(1, 16, 4, 8191, 128, 1024, 4), (1, 6, 2, 9000, 64, 3000, 130), (1, 4, 1, 6000, 128, 0, 0)])
@pytest.mark.parametrize("dtype", [HALF, BF])
def test_gradients_of_long_rows_by_norms(b, h, hk, n, d, window, sinks, dtype):
    q, k, v, do = _inputs(b, h, hk, n, n, d, dtype, seed=n)
    _check(q, k, v, do, window, sinks, heads=range(hk))


@pytest.mark.parametrize("scale", [0.0, -0.1, 0.5])
@pytest.mark.parametrize("dtype", [HALF, BF])
def test_gradients_of_other_scales_by_norms(scale, dtype):
    q, k, v, do = _inputs(1, 4, 2, 300, 300, 64, dtype, seed=107)
    _check(q, k, v, do, 100, 3, scale)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("size", [1e-3, 1e-4, 1e-5])
def test_float16_gradients_of_small_do(d, size):
    """dS of dO like a mean loss's: P / window of it is far below float16's normal range."""
    q, k, v, do = _inputs(1, 4, 2, 3000, 3000, d, HALF, seed=200)
    _check(q, k, v, (do.float() * size).to(HALF), 1500, 4)


@pytest.mark.parametrize("d", [64, 128])
def test_float16_gradients_of_large_do(d):
    """dP beyond float16's range, with gradients within it."""
    q, k, v, do = _inputs(1, 2, 2, 500, 500, d, HALF, seed=201)
    _check(q * 0.25, k * 0.25, v * 30, do * 1000, 0, 0)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("h,hk", [(4, 2), (4, 4)])
def test_float16_gradients_of_uneven_do(d, h, hk):
    """Rows, heads and sequences whose dO are up to 10^4 apart, rows of zeros and a head of zeros among them; keys
    seen from one end of a row alone."""
    q, k, v, do = _inputs(3, h, hk, 700, 700, d, HALF, seed=202)
    size = 10.0 ** (torch.arange(700, device=DEV) % 5 - 4.0)[:, None]
    size[::7] = 0
    do = (do.float() * size).to(HALF)
    do[1] *= 1e-3
    do[2, 1] = 0
    v[2] *= 100
    _check(q, k, v, do, 200, 3)
