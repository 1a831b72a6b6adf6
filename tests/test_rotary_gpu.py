"""Rotation by positions on several axes, forward and backward, against the formula: to the bit in float32
(the kernel's products and sum are rounded one by one, as torch's are), within one rounding of 64 bits."""

import pytest
import torch

import draft_oracle as oracle
import fa
import stream_oracle
from fa import _C

pytestmark = pytest.mark.gpu

DEV = "cuda:0"
HALF, BF = torch.float16, torch.bfloat16


def _tables(rows, half, seed=3):
    gen = torch.Generator(DEV).manual_seed(seed)
    a = torch.rand(rows, half, generator=gen, device=DEV) * 6.28
    return a.cos(), a.sin()


def _check(out, x, *how, **kw):
    exact = oracle.rotary(x, *how, **kw)
    # One rounding to the type, and float32's three (2^-24 of |x1| + |x2| each).
    bound = stream_oracle.unit(x.dtype) * exact.abs() + 2.0**-21 * x.double().abs().max() + 2.0**-25
    stream_oracle.check(out, exact, bound, "rotary")
    assert torch.equal(out, oracle.rotary(x, *how, **kw, wide=torch.float32).to(x.dtype))


@pytest.mark.parametrize("interleaved", [False, True])
@pytest.mark.parametrize("b,h,hk,t,d,r,axes,dtype", [
    (1, 1, 1, 1, 64, 64, 1, HALF), (2, 3, 1, 5, 64, 48, 2, BF), (3, 8, 2, 33, 128, 128, 3, BF), (1, 5, 5, 77, 128, 16, 4, HALF),
    (4, 32, 8, 1, 128, 96, 3, BF), (2, 2, 0, 130, 64, 32, 2, HALF), (1, 40, 8, 700, 128, 128, 3, BF), (70, 2, 1, 2, 64, 64, 1, HALF),
])
def test_forward_and_backward(b, h, hk, t, d, r, axes, dtype, interleaved):
    gen = torch.Generator(DEV).manual_seed(b + t)
    q = torch.randn(b, h, t, d, generator=gen, device=DEV).to(dtype)
    k = torch.randn(b, hk, t, d, generator=gen, device=DEV).to(dtype) if hk else None
    positions = torch.randint(0, 50, (axes, b, t), generator=gen, device=DEV, dtype=torch.int32)
    cos, sin = _tables(50, r // 2)
    names = [int(x) for x in torch.randint(0, axes, (r // 2,), generator=torch.Generator().manual_seed(t))]
    if axes == 1 and t == 1:
        names, positions = None, positions[0]
    oq, ok = fa.forward_rotary(q, k, positions, cos, sin, axes=names, interleaved=interleaved)
    _check(oq, q, positions, cos, sin, names, interleaved)
    if k is None:
        assert ok is None
    else:
        _check(ok, k, positions, cos, sin, names, interleaved)
    # The gradient is the rotation back: against the formula.
    dq, dk = fa.backward_rotary(q, k, positions, cos, sin, axes=names, interleaved=interleaved)
    _check(dq, q, positions, cos, sin, names, interleaved, inverse=True)
    assert dk is None or k is not None and _check(dk, k, positions, cos, sin, names, interleaved, inverse=True) is None
    assert _C.device_status(0, clear=True) == 0


def test_strides_and_shared_positions():
    gen = torch.Generator(DEV).manual_seed(0)
    b, t, h, hk, d = 2, 19, 6, 2, 128
    qkv = torch.randn(b, t, h + 2 * hk, d, generator=gen, device=DEV).to(BF)
    q, k, _ = (x.transpose(1, 2) for x in qkv.split([h, hk, hk], 2))
    cos, sin = _tables(40, 32)
    one = torch.randint(0, 40, (2, 1, t), generator=gen, device=DEV, dtype=torch.int32)
    axes = [0, 1] * 16
    out = fa.forward_rotary(q, k, one.expand(2, b, t), cos, sin, axes=axes)
    want = fa.forward_rotary(q.contiguous(), k.contiguous(), one.repeat(1, b, 1), cos, sin, axes=axes)
    assert all(torch.equal(x, y) for x, y in zip(out, want))
    _check(out[1], k, one.expand(2, b, t), cos, sin, axes)
    same = fa.forward_rotary(q, k, one[0, 0, 3].expand(b, t), cos, sin)
    _check(same[0], q, one[0, 0, 3].expand(b, t), cos, sin)


def test_padding_and_positions_beyond_the_tables():
    gen = torch.Generator(DEV).manual_seed(0)
    q = torch.randn(2, 4, 9, 64, generator=gen, device=DEV).to(HALF)
    cos, sin = _tables(16, 32)
    positions = torch.randint(0, 16, (2, 2, 9), generator=gen, device=DEV, dtype=torch.int32)
    positions[0, 0, 3] = -1
    positions[1, 1, 8] = -(2**31)
    q[0, :, 3] = float("nan")
    axes = [0] * 20 + [1] * 12
    out, _ = fa.forward_rotary(q, None, positions, cos, sin, axes=axes)
    assert not out[0, :, 3].any() and not out[1, :, 8].any() and _C.device_status(0, clear=True) == 0
    _check(out[1:], q[1:], positions[:, 1:], cos, sin, axes)
    positions[1, 1, 2] = 16
    positions[0, 1, 4] = 2**31 - 1
    out, _ = fa.forward_rotary(q, None, positions, cos, sin, axes=axes)
    assert not out[1, :, 2].any() and not out[1, :, 4].any() and out[1, :, 3].any()
    assert _C.device_status(0, clear=True) == 32


def test_same_bits_as_the_cache_gets():
    """append_kv turns by the slots' numbers: the same rotation to the bit."""
    gen = torch.Generator(DEV).manual_seed(5)
    q, k = (torch.randn(1, n, 20, 64, generator=gen, device=DEV).to(HALF) for n in (4, 2))
    cos, sin = _tables(30, 32)
    for interleaved in (False, True):
        cache = fa.PagedKVCache.empty(3, 16, 2, 64, dtype=HALF)
        table, lengths = torch.tensor([[1, 0]], dtype=torch.int32, device=DEV), torch.tensor([20], dtype=torch.int32, device=DEV)
        want = fa.append_kv(cache, k, k, table, lengths, cos=cos, sin=sin, q=q, interleaved=interleaved)
        at = torch.arange(20, device=DEV, dtype=torch.int32)[None]
        oq, ok = fa.forward_rotary(q, k, at, cos, sin, interleaved=interleaved)
        assert torch.equal(oq, want)
        assert torch.equal(ok[0], cache.k[[1, 0]].transpose(0, 1).reshape(2, 32, 64)[:, :20])


def test_gradients_through_autograd():
    gen = torch.Generator(DEV).manual_seed(6)
    q, k = (torch.randn(2, n, 7, 64, generator=gen, device=DEV).to(BF).requires_grad_() for n in (4, 1))
    positions = torch.randint(-1, 9, (3, 2, 7), generator=gen, device=DEV, dtype=torch.int32)
    cos, sin = _tables(9, 32)
    axes = [i % 3 for i in range(32)]
    oq, ok = fa.rotary(q, k, positions, cos, sin, axes=axes, interleaved=True)
    assert torch.equal(oq, fa.forward_rotary(q, k, positions, cos, sin, axes=axes, interleaved=True)[0])
    # A gradient of any layout, an expanded one among them.
    dq, dk = torch.randn(2, 7, 4, 64, generator=gen, device=DEV).to(BF).transpose(1, 2), torch.ones(64, device=DEV, dtype=BF).expand(2, 1, 7, 64)
    got = torch.autograd.grad((oq, ok), (q, k), (dq, dk), retain_graph=True)
    _check(got[0], dq, positions, cos, sin, axes, True, inverse=True)
    _check(got[1], dk, positions, cos, sin, axes, True, inverse=True)
    # One result alone, and the gradient of a gradient: forward again.
    only = torch.autograd.grad(ok, (q, k), dk, retain_graph=True, allow_unused=True)
    assert only[0] is None and torch.equal(only[1], got[1])
    w = torch.randn(2, 4, 7, 64, generator=gen, device=DEV).to(BF).requires_grad_()
    first, = torch.autograd.grad(oq, q, w, create_graph=True)
    second, = torch.autograd.grad(first, w, dq)
    _check(second, dq, positions, cos, sin, axes, True)


def test_gradient_against_differences():
    """In float16 the rotation is linear up to its rounding: a step of x moves the result by the rotated step."""
    gen = torch.Generator(DEV).manual_seed(7)
    x = torch.randn(1, 2, 33, 128, generator=gen, device=DEV).to(HALF).requires_grad_()
    step, dy = (torch.randn(1, 2, 33, 128, generator=gen, device=DEV).to(HALF) for _ in "ab")
    at = torch.randint(0, 9, (1, 33), generator=gen, device=DEV, dtype=torch.int32)
    cos, sin = _tables(9, 64)
    y, _ = fa.rotary(x, None, at, cos, sin)
    grad, = torch.autograd.grad(y, x, dy)
    with torch.no_grad():
        value = lambda s: (fa.forward_rotary((x + s * step), None, at, cos, sin)[0].double() * dy.double()).sum()  # noqa: E731
        differences = value(1) - value(-1)
        change = ((x + step).double() - (x - step).double())  # the steps as they were rounded
        # Two results and a gradient (times a change of 2 steps) are each off by 2^-11 of their sizes, which are about 1 to 6; the
        # errors of 33 * 256 products with |dy| have no common sign: 6 times the norm of 18 2^-11 |dy|, far more than they reach.
        got = (grad.double() * change).sum()
        noise = 2.0**-11 * 18.0 * dy.double().norm()
    assert abs(differences - got) < 6 * noise


def test_graph_and_streams():
    gen = torch.Generator(DEV).manual_seed(8)
    q = torch.randn(2, 4, 3, 64, generator=gen, device=DEV).to(HALF)
    at = torch.zeros(2, 3, device=DEV, dtype=torch.int32)
    cos, sin = _tables(100, 32)
    graph = torch.cuda.CUDAGraph()
    fa.forward_rotary(q, q, at, cos, sin)
    with torch.cuda.graph(graph):
        oq, ok = fa.forward_rotary(q, q, at, cos, sin)
    for i in (5, 90):
        at.fill_(i)
        graph.replay()
        _check(oq, q, at, cos, sin)
        assert torch.equal(oq, ok)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        out, _ = fa.forward_rotary(q, None, at, cos, sin)
    side.synchronize()
    assert torch.equal(out, oq)


def test_a_training_step_in_a_graph():
    """Forward and gradients captured, by the pair of calls and by autograd, and replayed on other values."""
    gen = torch.Generator(DEV).manual_seed(9)
    q, dq = (torch.randn(2, 4, 33, 128, generator=gen, device=DEV).to(BF) for _ in range(2))
    k, dk = (torch.randn(2, 2, 33, 128, generator=gen, device=DEV).to(BF) for _ in range(2))
    at = torch.randint(0, 50, (2, 33), generator=gen, device=DEV).to(torch.int32)
    cos, sin = _tables(50, 32)

    def step(q, k):
        turned = fa.rotary(q, k, at, cos, sin)
        return *turned, *torch.autograd.grad(turned, (q, k), (dq, dk))

    def pair(q, k):
        return *fa.forward_rotary(q, k, at, cos, sin), *fa.backward_rotary(dq, dk, at, cos, sin)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    q, k = q.requires_grad_(), k.requires_grad_()
    with torch.cuda.stream(side):
        step(q, k)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(q, k)
        same = pair(q.detach(), k.detach())
    for seed in (1, 2):
        with torch.no_grad():
            for t in (q, k, dq, dk):
                t.copy_(torch.randn(t.shape, generator=gen, device=DEV))
        at.copy_(torch.randint(0, 50, at.shape, generator=gen, device=DEV))
        graph.replay()
        for x, y, z in zip(out, same, pair(q.detach(), k.detach())):
            assert torch.equal(x, z) and torch.equal(y, z)


def test_empty_and_refused():
    cos, sin = _tables(9, 32)
    at = torch.zeros(0, 3, device=DEV, dtype=torch.int32)
    q = torch.zeros(0, 4, 3, 64, device=DEV, dtype=HALF)
    assert fa.forward_rotary(q, q, at, cos, sin)[1].shape == q.shape
    q, at = torch.zeros(2, 4, 3, 64, device=DEV, dtype=HALF), torch.zeros(2, 3, device=DEV, dtype=torch.int32)
    for bad, match in ((lambda: fa.forward_rotary(q, q.to(BF), at, cos, sin), "same dtype"), (lambda: fa.forward_rotary(q.float(), None, at, cos, sin), "float16"),
                       (lambda: fa.forward_rotary(q, q[:, :, :2], at, cos, sin), "batch, tokens"), (lambda: fa.forward_rotary(q, None, at.long(), cos, sin), "int32"),
                       (lambda: fa.forward_rotary(q, None, at[:1], cos, sin), "positions"), (lambda: fa.forward_rotary(q, None, at, cos, sin, axes=[0] * 31), "each of the"),
                       (lambda: fa.forward_rotary(q, None, at, cos, sin[:3]), "same shape"), (lambda: fa.forward_rotary(q, None, at, cos.half(), sin), "float32"),
                       (lambda: fa.forward_rotary(q.mT.contiguous().mT, None, at, cos, sin), "contiguous last")):
        with pytest.raises(RuntimeError, match=match):
            bad()
    for bad, match in ((lambda: fa.forward_rotary(q, None, at, cos, sin, axes=[1] * 32), "axis_of_pair"), (lambda: fa.forward_rotary(q, None, at, cos, sin, axes=[-1] * 32), "range"),
                       (lambda: fa.forward_rotary(q[..., :48], None, at, cos, sin), "head_dim"), (lambda: fa.forward_rotary(q, None, at, *_tables(9, 20)), "rotary_dim"),
                       (lambda: fa.forward_rotary(torch.zeros(2, 4, 3, 68, device=DEV, dtype=HALF)[..., :64], None, at, cos, sin), "multiples of 8")):
        with pytest.raises(ValueError, match=match):
            bad()


def test_axes_edited_between_forward_and_backward():
    """The gradient turns by the axes that the forward turned by, whatever becomes of the caller's list."""
    gen = torch.Generator(DEV).manual_seed(10)
    q, k = (torch.randn(2, n, 7, 64, generator=gen, device=DEV).to(BF).requires_grad_() for n in (4, 1))
    positions = torch.randint(0, 9, (2, 2, 7), generator=gen, device=DEV, dtype=torch.int32)
    cos, sin = _tables(9, 32)
    axes = [i % 2 for i in range(32)]
    turned = fa.rotary(q, k, positions, cos, sin, axes=axes)
    dq, dk = (torch.randn(t.shape, generator=gen, device=DEV).to(BF) for t in turned)
    want = fa.backward_rotary(dq, dk, positions, cos, sin, axes=axes)
    axes[:] = [0] * 32
    got = torch.autograd.grad(turned, (q, k), (dq, dk))
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
