"""Rotary positions against their definition in 64 bits."""
import pytest
import torch

import layer_reference as ref
from rnn_train_ring_attractor_b200.rotary import rotary, rotary_frequencies

pytestmark = pytest.mark.gpu

FP32, BF16, FP16 = torch.float32, torch.bfloat16, torch.float16


def _bound(x, want, amplitude=1.0):
    """Two products and a sum, the cosine and the sine (their argument in half turns rounded once, 2^-24 of at most pi, then at most
    two steps of each), and the amplitude: 10 * 2^-24 of |x1| + |x2|, that is at most 20 * 2^-24 of the largest; then the rounding to the type."""
    top = x.double().abs().amax(dim=-1, keepdim=True)
    return 20 * 2.0 ** -24 * top * abs(amplitude) + ref.U[x.dtype] * (want.abs() + 20 * 2.0 ** -24 * top * abs(amplitude)) + ref.TINY[x.dtype]


def _randn(*shape, dtype, seed=0):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


CASES = [  # dtype, B, T, Hq, Hk, D, R
    (BF16, 1, 1, 1, 1, 2, 2), (BF16, 3, 1, 16, 4, 128, 128), (BF16, 2, 70, 5, 1, 96, 64), (BF16, 2, 33, 3, 3, 100, 36), (BF16, 1, 50, 2, 2, 66, 22),
    (FP16, 2, 40, 4, 2, 64, 64), (FP32, 2, 129, 3, 1, 96, 96), (FP32, 1, 17, 7, 7, 10, 6), (FP32, 2, 5, 40, 8, 72, 8), (BF16, 2, 300, 9, 2, 256, 16),
    (FP16, 1, 7, 1, 1, 7, 2)]


@pytest.mark.parametrize("dtype,B,T,Hq,Hk,D,R", CASES)
@pytest.mark.parametrize("interleaved", [False, True])
def test_forward_and_gradients(dtype, B, T, Hq, Hk, D, R, interleaved, achieved):
    f = rotary_frequencies(R, 1e4)
    q, k = _randn(B, T, Hq, D, dtype=dtype, seed=1), _randn(B, T, Hk, D, dtype=dtype, seed=2)
    d_q, d_k = _randn(B, T, Hq, D, dtype=dtype, seed=3), _randn(B, T, Hk, D, dtype=dtype, seed=4)
    pos = torch.randint(-5, 1 << 20, (B, T), device="cuda", generator=torch.Generator(device="cuda").manual_seed(5))
    worst = 0.0
    for p in (pos, pos.int(), pos[:, :1].expand(B, T)):
        q.requires_grad_(), k.requires_grad_()
        got = rotary(q, k, f, p, interleaved=interleaved, amplitude=0.7)
        grads = torch.autograd.grad(got, (q, k), (d_q, d_k))
        for x, y in zip((q, k), got):
            want = ref.turn(x.detach(), p, f, interleaved, 0.7)
            worst = max(worst, ref.worst(y.detach(), want, _bound(x.detach(), want)))
            assert torch.equal(y[..., R:], x[..., R:])
        for x, y in zip((d_q, d_k), grads):
            want = ref.turn(x, p, f, interleaved, 0.7, inverse=True)
            worst = max(worst, ref.worst(y, want, _bound(x, want)))
    assert worst <= 1.0
    achieved(f"rotary {str(dtype)[6:]} {B}x{T} {Hq}+{Hk} {D}/{R} (of the bound)", worst=worst)


def test_first_position_and_one_tensor_alone():
    f = rotary_frequencies(64)
    q, k = _randn(2, 30, 3, 64, dtype=BF16, seed=1), _randn(2, 30, 2, 64, dtype=BF16, seed=2)
    pos = (1 << 33) + torch.arange(30, device="cuda")
    a, b = rotary(q, k, f, 1 << 33)
    c, d = rotary(q, k, f, pos.expand(2, 30))
    e, none = rotary(q, None, f, 1 << 33)
    assert torch.equal(a, c) and torch.equal(b, d) and torch.equal(a, e) and none is None
    # one gradient of two, and a key's alone
    k.requires_grad_()
    g, = torch.autograd.grad(rotary(q, k, f, 7)[1], k, k.detach())
    want = ref.turn(k.detach(), (7 + torch.arange(30, device="cuda")).expand(2, 30), f, False, inverse=True)
    assert ref.worst(g, want, _bound(k.detach(), want)) <= 1.0


def test_distance_is_all_that_matters():
    """A query's product with a key depends on the difference of their positions, also a million positions on: the bound is
    that of the two tensors' elements, summed over the head."""
    f = rotary_frequencies(128, 1e6)
    q, k = _randn(1, 1, 1, 128, dtype=FP32, seed=1), _randn(1, 1, 1, 128, dtype=FP32, seed=2)
    near = (rotary(q, None, f, 25)[0].double() * rotary(k, None, f, 5)[0].double()).sum()
    far = (rotary(q, None, f, 10 ** 6 + 20)[0].double() * rotary(k, None, f, 10 ** 6)[0].double()).sum()
    room = 2 * 128 * 2 * 21 * 2.0 ** -24 * float(q.abs().max() * k.abs().max()) * 2
    assert abs(float(near - far)) <= room


def test_strides():
    B, T, Hq, Hk, D = 2, 20, 4, 2, 64
    f = rotary_frequencies(48)
    q, k = _randn(B, T, Hq, D, dtype=BF16, seed=1), _randn(B, T, Hk, D, dtype=BF16, seed=2)
    want = rotary(q, k, f, 3)
    wide = torch.cat((q, k), dim=2)
    odd = torch.full((B, T, Hq + Hk, D + 3), float("nan"), device="cuda", dtype=BF16)
    odd[..., 1:1 + D] = wide
    for w in (wide, wide.transpose(1, 2).contiguous().transpose(1, 2), odd[..., 1:1 + D], wide.transpose(2, 3).contiguous().transpose(2, 3)):
        for a, b in zip(rotary(w[:, :, :Hq], w[:, :, Hq:], f, 3), want):
            assert torch.equal(a, b)
    shared = k[:, :, :1].clone().requires_grad_()
    _, y = rotary(q, shared.expand(B, T, 3, D), f, 3)
    y.sum().backward()
    ones = torch.ones(B, T, 3, D, device="cuda", dtype=BF16)
    assert torch.equal(shared.grad, torch.autograd.grad(rotary(q, shared.expand(B, T, 3, D), f, 3)[1], shared, ones)[0])


def test_nothing_is_written_beyond_the_outputs():
    import ctypes as C
    from rnn_train_ring_attractor_b200 import _lib
    for dtype, code, D, R in ((BF16, 1, 100, 36), (FP32, 0, 10, 6), (BF16, 1, 128, 64), (FP16, 2, 7, 2)):
        B, T, Hq, Hk = 2, 3, 5, 2
        f = rotary_frequencies(R)
        q, k = _randn(B, T, Hq, D, dtype=dtype, seed=1), _randn(B, T, Hk, D, dtype=dtype, seed=2)
        pad = 64
        qo, ko = (torch.full((x.numel() + 2 * pad,), 77.0, device="cuda", dtype=dtype) for x in (q, k))
        sd = lambda t: _lib.Strided(t.data_ptr(), *t.stride()[:3])  # noqa: E731
        p = _lib.Rotary(B, T, Hq, Hk, D, R, code, 0, 0, 1.0, sd(q), sd(k), f.data_ptr(), None, 0, 0, 0, 9, qo[pad:].data_ptr(), ko[pad:].data_ptr())
        assert _lib.lib().ringrnn_rotary(C.byref(p), None) == 0
        torch.cuda.synchronize()
        for t, x in zip((qo, ko), rotary(q, k, f, 9)):
            assert bool((t[:pad] == 77).all()) and bool((t[-pad:] == 77).all()) and torch.equal(t[pad:-pad].view_as(x), x)


def test_captured_and_replayed_on_new_positions():
    f = rotary_frequencies(64)
    q, k = _randn(4, 1, 6, 64, dtype=BF16, seed=1), _randn(4, 1, 2, 64, dtype=BF16, seed=2)
    pos = torch.zeros(4, 1, device="cuda", dtype=torch.int64)
    rotary(q, k, f, pos)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = rotary(q, k, f, pos)
    for at in (3, 4000):
        pos.fill_(at)
        graph.replay()
        torch.cuda.synchronize()
        for a, b in zip(held, rotary(q, k, f, at)):
            assert torch.equal(a, b)


def test_refusals_and_empty_calls():
    f = rotary_frequencies(8)
    q, k = _randn(2, 3, 2, 8, dtype=BF16), _randn(2, 3, 1, 8, dtype=BF16)
    for bad in ((q[0], None, f), (q, k[:, :2], f), (q, k.float(), f), (q, k, f.float()), (q, k, f.cpu()), (q, k, rotary_frequencies(10)),
                (q, k, f[:0]), (q, k, f, torch.zeros(2, 3, device="cuda")), (q, k, f, torch.zeros(3, device="cuda", dtype=torch.int64)),
                (q, k[:, :, :0], f), (q[:, :, :0], k, f), (q.double(), None, f)):
        with pytest.raises(RuntimeError):
            rotary(*bad)
    a, b = rotary(q[:, :0], k[:, :0], f)
    assert a.shape == (2, 0, 2, 8) and b.shape == (2, 0, 1, 8)


def test_frequencies_that_ask_for_a_gradient_are_refused():
    q = torch.randn(1, 3, 2, 8, device="cuda")
    f = rotary_frequencies(8).requires_grad_()
    with pytest.raises(RuntimeError, match="frequencies have no gradient"):
        rotary(q, None, f)
    with torch.no_grad():
        assert torch.equal(rotary(q, None, f)[0], rotary(q, None, f.detach())[0])
