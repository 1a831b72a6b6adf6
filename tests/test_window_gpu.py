"""Window attention with sinks on the GPU, forward and backward, against the 64-bit definition at
the sizes and masks where tiles, windows and groups end unevenly. The bounds are derived in
stream_oracle."""

import math

import pytest
import torch

import fa
import stream_oracle as oracle
from fa import _C

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
HALF, BF = torch.float16, torch.bfloat16


def _inputs(b, h, hk, nq, nk, d, dtype, seed=0, scale=1.0):
    g = torch.Generator(DEV).manual_seed(seed)
    new = lambda *s: (torch.randn(s, generator=g, device=DEV) * scale).to(dtype)  # noqa: E731
    return new(b, h, nq, d), new(b, hk, nk, d), new(b, hk, nk, d), new(b, h, nq, d)


def _check_forward(q, k, v, window, sinks, scale=None):
    o, lse = fa.forward_window(q, k, v, window, sinks, scale, return_lse=True)
    want, want_lse, _ = oracle.window_forward(q, k, v, window, sinks, scale)
    u = oracle.unit(q.dtype)
    oracle.check(o, want, oracle.forward_bound(want, v.double().abs().max(), u, u), "O")
    empty = want_lse == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    assert not o[empty].any()
    # A relative error e of the sum moves its logarithm by about e.
    assert (lse.double() - want_lse)[~empty].abs().max().item() <= 2 * (u + oracle.POLY) if (~empty).any() else True
    assert torch.equal(o, fa.forward_window(q, k, v, window, sinks, scale))
    return o, lse


def _check_backward(do, q, k, v, window, sinks, scale=None):
    o, lse = fa.forward_window(q, k, v, window, sinks, scale, return_lse=True)
    got = fa.backward_window(do, q, k, v, o, lse, window, sinks, scale)
    want = oracle.window_backward(do, q, k, v, window, sinks, scale)[:3]
    for name, g, w, e in zip(("dQ", "dK", "dV"), got, want, oracle.backward_bounds(do, q, k, v, window, sinks, scale)):
        oracle.check(g, w, e, name)
    return got


SHAPES = [  # b, h, hk, nq, nk, window, sinks
    (1, 1, 1, 1, 1, 1, 0),
    (2, 2, 1, 17, 17, 5, 1),
    (1, 4, 2, 128, 128, 128, 0),
    (1, 2, 2, 129, 129, 64, 4),
    (2, 3, 3, 257, 257, 1, 0),
    (1, 4, 1, 300, 300, 100, 130),
    (1, 2, 1, 640, 640, 129, 3),
    (1, 8, 2, 1000, 1000, 256, 1),
    (1, 2, 2, 777, 777, 0, 0),       # no window
    (1, 2, 2, 500, 500, 5000, 9),    # a window beyond the row
    (1, 2, 1, 513, 513, 255, 513),   # everything a sink
    (1, 2, 1, 100, 900, 200, 4),     # queries at the end of longer keys
    (1, 2, 1, 1, 700, 300, 2),
    (1, 2, 1, 700, 100, 50, 2),      # rows before the first key see nothing
    (1, 2, 1, 385, 129, 64, 0),
]


@pytest.mark.parametrize("b,h,hk,nq,nk,window,sinks", SHAPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [HALF, BF])
def test_forward_matches_definition(b, h, hk, nq, nk, window, sinks, d, dtype):
    q, k, v, _ = _inputs(b, h, hk, nq, nk, d, dtype, seed=nq + window)
    _check_forward(q, k, v, window, sinks)
    assert _C.device_status(0) == 0


@pytest.mark.parametrize("b,h,hk,nq,nk,window,sinks", SHAPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("dtype", [HALF, BF])
def test_backward_matches_formula(b, h, hk, nq, nk, window, sinks, d, dtype):
    q, k, v, do = _inputs(b, h, hk, nq, nk, d, dtype, seed=nq + window)
    _check_backward(do, q, k, v, window, sinks)
    assert _C.device_status(0) == 0


@pytest.mark.parametrize("d", [64, 128])
def test_long_rows_small_window_and_far_sinks(d):
    """Many tiles between the sinks and the window, a long list of queries for the sinks' keys."""
    q, k, v, do = _inputs(1, 2, 1, 4097, 4097, d, BF, seed=5)
    _check_forward(q, k, v, 200, 5)
    _check_backward(do, q, k, v, 200, 5)


@pytest.mark.parametrize("b,h,hk,n,d,window,sinks", [(1, 16, 4, 8191, 128, 1024, 4), (1, 6, 2, 9000, 64, 3000, 130)])
def test_last_wave_of_single_query_tiles(b, h, hk, n, d, window, sinks):
    """More row blocks than SMs and a short last wave, whose query tiles go one to a CTA: every row's O and
    LSE are its own, and so are the gradients made of them."""
    q, k, v, do = _inputs(b, h, hk, n, n, d, BF, seed=n)
    o, lse = fa.forward_window(q, k, v, window, sinks, return_lse=True)
    got = fa.backward_window(do, q, k, v, o, lse, window, sinks)
    u, g = oracle.unit(BF), h // hk
    for j in range(hk):
        one = lambda t: t[:, j : j + 1]  # noqa: E731
        own = lambda t: t[:, j * g : (j + 1) * g]  # noqa: E731
        args = (own(q), one(k), one(v), window, sinks)
        want, want_lse, _ = oracle.window_forward(*args)
        oracle.check(own(o), want, oracle.forward_bound(want, v.double().abs().max(), u, u), "O")
        assert (own(lse).double() - want_lse).abs().max().item() <= 2 * (u + oracle.POLY)
        grads = oracle.window_backward(own(do), *args)[:3]
        for name, x, w, e in zip(("dQ", "dK", "dV"), (own(got[0]), one(got[1]), one(got[2])), grads,
                                 oracle.backward_bounds(own(do), *args)):
            oracle.check(x, w, e, name)


def test_many_heads_walk_a_persistent_grid():
    q, k, v, do = _inputs(3, 32, 8, 300, 300, 64, HALF, seed=6)
    _check_forward(q, k, v, 70, 2)
    _check_backward(do, q, k, v, 70, 2)


@pytest.mark.parametrize("scale", [0.0, -0.1, 0.5])
def test_other_scales(scale):
    q, k, v, do = _inputs(1, 2, 1, 300, 300, 64, HALF, seed=7)
    _check_forward(q, k, v, 100, 3, scale)
    _check_backward(do, q, k, v, 100, 3, scale)


def test_large_scores_stay_finite():
    q, k, v, do = _inputs(1, 2, 1, 400, 400, 128, BF, seed=8, scale=8.0)
    o, lse = fa.forward_window(q, k, v, 130, 2, return_lse=True)
    got = fa.backward_window(do, q, k, v, o, lse, 130, 2)
    assert all(torch.isfinite(t.float()).all() for t in (o, lse, *got))


def test_hidden_keys_may_hold_anything():
    """Keys outside a query's view do not touch it, infinities among them."""
    q, k, v, _ = _inputs(1, 2, 2, 400, 400, 64, HALF, seed=9)
    o = fa.forward_window(q, k, v, 40, 0)
    k2, v2 = k.clone(), v.clone()
    k2[:, :, 200:], v2[:, :, 200:] = 60000.0, -60000.0
    o2 = fa.forward_window(q, k2, v2, 40, 0)
    assert torch.equal(o[:, :, :200], o2[:, :, :200])


def test_transposed_and_sliced_tensors():
    g = torch.Generator(DEV).manual_seed(10)
    packed = torch.randn(2, 333, 4 + 2 + 2, 64, generator=g, device=DEV).to(BF)
    q, k, v = (t.transpose(1, 2) for t in packed.split([4, 2, 2], 2))
    wide = torch.randn(2, 4, 333, 64 + 64, generator=g, device=DEV).to(BF)
    do = wide[..., 64:]
    o, lse = fa.forward_window(q, k, v, 90, 3, return_lse=True)
    oc, lsec = fa.forward_window(q.contiguous(), k.contiguous(), v.contiguous(), 90, 3, return_lse=True)
    assert torch.equal(o, oc) and torch.equal(lse, lsec)
    got = fa.backward_window(do, q, k, v, o, lse, 90, 3)
    want = fa.backward_window(do.contiguous(), q.contiguous(), k.contiguous(), v.contiguous(), o, lse, 90, 3)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_same_bits_every_time_and_on_another_stream():
    q, k, v, do = _inputs(2, 8, 2, 1000, 1000, 128, BF, seed=11)
    o, lse = fa.forward_window(q, k, v, 256, 4, return_lse=True)
    first = fa.backward_window(do, q, k, v, o, lse, 256, 4)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        o2, lse2 = fa.forward_window(q, k, v, 256, 4, return_lse=True)
        again = fa.backward_window(do, q, k, v, o2, lse2, 256, 4)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(o, o2) and all(torch.equal(a, b) for a, b in zip(first, again))


def test_step_in_a_graph_follows_its_inputs():
    """Forward and backward captured once and replayed on other values."""
    q, k, v, do = _inputs(1, 8, 2, 1500, 1500, 64, BF, seed=21)
    def step():
        o, lse = fa.forward_window(q, k, v, 300, 4, return_lse=True)
        return (o, lse, *fa.backward_window(do, q, k, v, o, lse, 300, 4))

    step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for seed in (22, 23):
        for t, x in zip((q, k, v, do), _inputs(1, 8, 2, 1500, 1500, 64, BF, seed=seed)):
            t.copy_(x)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, step()))


def test_matches_plain_causal_forward_without_a_window():
    q, k, v, _ = _inputs(1, 4, 4, 900, 900, 128, BF, seed=12)
    u = oracle.unit(BF)
    want = fa.forward(q, k, v, causal=True).double()
    bound = 2 * oracle.forward_bound(want, v.double().abs().max(), u, u)
    oracle.check(fa.forward_window(q, k, v, 0), want, bound, "O")


def test_gradient_against_differences():
    """The gradient along a direction against a difference of forwards: exact in v (O is linear in
    it) but for roundings, and within the truncation that the definition's own difference shows
    in q and k."""
    q, k, v, do = _inputs(1, 4, 2, 200, 200, 64, HALF, seed=13, scale=0.5)
    window, sinks, h = 60, 2, 0.125
    o, lse = fa.forward_window(q, k, v, window, sinks, return_lse=True)
    grads = fa.backward_window(do, q, k, v, o, lse, window, sinks)
    u = oracle.unit(HALF)
    bounds = oracle.backward_bounds(do, q, k, v, window, sinks)
    for i in range(3):
        args = [q, k, v]
        step = (torch.randn(args[i].shape, generator=torch.Generator(DEV).manual_seed(i), device=DEV).sign() * h).to(HALF)
        # The two points as float16 holds them, and the step between them.
        up, down = args[i] + step, args[i] - step
        step = (up.double() - down.double()) / 2
        ends, exact = [], []
        noise = 0.0
        for t in (up, down):
            args[i] = t
            out = fa.forward_window(*args, window, sinks)
            want, _, _ = oracle.window_forward(*args, window, sinks)
            ends.append((out.double() * do.double()).sum())
            exact.append((want * do.double()).sum())
            err = oracle.forward_bound(want, args[2].double().abs().max(), u, u)
            # Roundings of single outputs are independent: their sum is within 6 deviations.
            noise += 6 * (err * do.double()).square().sum().sqrt()
        truth = sum((w * s).sum() for w, s in zip(oracle.window_backward(do, q, k, v, window, sinks)[i : i + 1], [step]))
        truncation = abs((exact[0] - exact[1]) / 2 - truth)
        slack = 6 * (bounds[i] * step).square().sum().sqrt()
        got = (grads[i].double() * step).sum()
        assert abs((ends[0] - ends[1]) / 2 - got) <= noise / 2 + truncation + slack, ("qkv"[i], float(got))


def test_autograd_sums_over_shared_heads():
    q, k, v, do = _inputs(1, 4, 1, 150, 150, 64, BF, seed=14)
    for t in (q, k, v):
        t.requires_grad_(True)
    o = fa.window_attention(q, k, v, 40, 2)
    o.backward(do)
    plain, lse = fa.forward_window(q.detach(), k.detach(), v.detach(), 40, 2, return_lse=True)
    want = fa.backward_window(do, q.detach(), k.detach(), v.detach(), plain, lse, 40, 2)
    assert torch.equal(o, plain)
    assert all(torch.equal(t.grad, w) for t, w in zip((q, k, v), want))
    # An expanded gradient (a sum's).
    k.grad = None
    fa.window_attention(q, k, v, 40, 2).sum().backward()
    ones = torch.ones_like(do)
    assert torch.equal(k.grad, fa.backward_window(ones, q.detach(), k.detach(), v.detach(), plain, lse, 40, 2)[1])


def test_empty_tensors():
    q, k, v, do = _inputs(1, 2, 1, 5, 5, 64, HALF)
    o, lse = fa.forward_window(q, k[:, :, :0], v[:, :, :0], 4, return_lse=True)
    assert not o.any() and (lse == -math.inf).all()
    dq, dk, dv = fa.backward_window(do, q, k[:, :, :0], v[:, :, :0], o, lse, 4)
    assert not dq.any() and dk.shape == (1, 1, 0, 64)
    o, lse = fa.forward_window(q[:, :, :0], k, v, 4, return_lse=True)
    assert o.shape == (1, 2, 0, 64)
    assert not fa.backward_window(do[:, :, :0], q[:, :, :0], k, v, o, lse, 4)[1].any()


def test_refusals():
    q, k, v, do = _inputs(1, 4, 2, 64, 64, 64, HALF)
    o, lse = fa.forward_window(q, k, v, 16, return_lse=True)
    with pytest.raises(ValueError, match="multiple of kv_heads"):
        fa.forward_window(q[:, :3], k, v, 16)
    with pytest.raises(ValueError, match="must not be negative"):
        fa.forward_window(q, k, v, -1)
    with pytest.raises(ValueError, match="must not be negative"):
        fa.forward_window(q, k, v, 16, sinks=-2)
    with pytest.raises(ValueError, match="finite"):
        fa.forward_window(q, k, v, 16, softmax_scale=math.nan)
    with pytest.raises(ValueError, match="head_dim"):
        fa.forward_window(*(t[..., :32].contiguous() for t in (q, k, v)), 16)
    with pytest.raises(ValueError, match="16-byte aligned"):
        odd = torch.zeros(q.numel() + 1, dtype=HALF, device=DEV)[1:].view(q.shape)
        fa.forward_window(odd, k, v, 16)
    with pytest.raises(ValueError, match="multiples of 8"):
        fa.forward_window(torch.zeros(1, 4, 64, 68, dtype=HALF, device=DEV)[..., :64], k, v, 16)
    with pytest.raises(ValueError, match="positive strides"):
        fa.forward_window(q, k[:, :1].expand(1, 2, 64, 64), v, 16)
    with pytest.raises(RuntimeError, match="contiguous last"):
        fa.forward_window(q.transpose(2, 3), k, v, 16)
    with pytest.raises(RuntimeError, match="same dtype"):
        fa.forward_window(q, k.bfloat16(), v, 16)
    with pytest.raises(RuntimeError, match="shape"):
        fa.forward_window(q, k, v[:, :, :32], 16)
    with pytest.raises(RuntimeError, match="lse must be"):
        fa.backward_window(do, q, k, v, o, lse.double(), 16)
    with pytest.raises(RuntimeError, match="like q"):
        fa.backward_window(do[:, :2], q, k, v, o, lse, 16)
