"""Linear attention in fp16: how exact a result is goes by the numbers' bits and not by their size.

Norms are of all elements.  Roundings of random numbers have either sign, so what n of them leave is the root of the sum of their
squares, which for sums of random products is at most half a step (u = 2^-11) of the sums' own norm.  1.1: a norm of thousands of
random terms stands within a few percent of what is expected of it.
"""
import pytest
import torch

import layer_reference as ref
from rnn_train_ring_attractor_b200.linear_attention import linear_attention

pytestmark = pytest.mark.gpu

FP16, U = torch.float16, 2.0 ** -11


def _randn(*shape, seed, size=1.0, to=FP16):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return (torch.randn(*shape, device="cuda", generator=g) * size).to(to)


def _decays(H):
    steps = torch.tensor([50.3, 700.9, 7.3, 3000.0] * ((H + 3) // 4), device="cuda", dtype=torch.float64)[:H]
    return torch.log1p(-1.0 / steps).float()


def _off(got, want):
    return float((got.double() - want).norm() / want.norm())


def _room(want):
    """the output's own rounding, and one of what goes into each product of its sum"""
    rounded = (want.to(FP16).double() - want).norm()
    return 1.1 * float(torch.sqrt(rounded ** 2 + (U * want.norm()) ** 2) / want.norm())


# Keys with their weights as two numbers keep 22 bits: 2^-22 of a product.  A chunk's 128 products are added by eight instructions for each of
# the two, which may cut off a step of fp32 (2^-23) each; a few more for the chunks' sum.
STATE_ROOM = 2.0 ** -22 + 20 * 2.0 ** -23


@pytest.mark.parametrize("B,T,H,dk,dv", [(1, 512, 2, 64, 64), (1, 400, 2, 128, 128), (1, 5003, 1, 128, 64), (1, 5003, 2, 64, 64), (40, 300, 4, 64, 128)])
@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-3, 1e-4, 1e-6])
def test_states_of_small_keys(B, T, H, dk, dv, size, achieved):
    q, k, v = _randn(B, T, H, dk, seed=1), _randn(B, T, H, dk, seed=2, size=size), _randn(B, T, H, dv, seed=3)
    l = _decays(H)
    out, final = linear_attention(q, k, v, l, scale=1.0)
    want, want_s = ref.attend(q, k, v, l, 1.0)
    e = [_off(final[:, h], want_s[:, h]) for h in range(H)]
    achieved(f"fp16 state of keys of {size:g} {B}x{T}x{H} {dk}/{dv}", worst=max(e), room=STATE_ROOM)
    assert max(e) <= STATE_ROOM, e
    assert _off(out, want) <= _room(want)


@pytest.mark.parametrize("B,T,H,state", [(1, 1024, 2, False), (1, 700, 2, True), (1, 6007, 1, True), (4, 300, 16, False), (16, 200, 12, True)])
@pytest.mark.parametrize("size", [1.0, 1e-2, 1e-4, 1e-5])
def test_small_gradients(B, T, H, state, size, achieved):
    """One sequence for itself, with states, in segments, and batches whose gradients of keys and values go in pairs."""
    dk, dv = 128, 128
    q, k, v = (_randn(B, T, H, 128, seed=s).requires_grad_() for s in (1, 2, 3))
    d_out = _randn(B, T, H, dv, seed=4, size=size)
    s, d_final = (_randn(B, H, dk, dv, seed=5, to=torch.float32).requires_grad_(), _randn(B, H, dk, dv, seed=6, size=size, to=torch.float32)) if state else (None, None)
    l = _decays(H)
    scale = dk ** -0.5
    out, final = linear_attention(q, k, v, l, scale=scale, initial_state=s)
    leaves = [q, k, v] + ([s] if state else [])
    got = torch.autograd.grad((out, final) if state else out, leaves, (d_out, d_final) if state else d_out)
    want = ref.attend_grads(q, k, v, l, scale, s, None, d_out, d_final)
    e = [_off(a, b) for a, b in zip(got, want)]
    achieved(f"fp16 gradients of {size:g} {B}x{T}x{H} (of the bound)", **{n: x / _room(y) for n, x, y in zip(("dq", "dk", "dv"), e, want)})
    for x, y in zip(e[:3], want):
        assert x <= _room(y), (e, [_room(y) for y in want[:3]])
    if state:
        assert e[3] <= STATE_ROOM, e


@pytest.mark.parametrize("B,H", [(1, 2), (4, 16)])
@pytest.mark.parametrize("scale", [1e-6, 1.0, 300.0, -0.25])
def test_any_scale(B, H, scale):
    """A scale takes part in scores and in gradients' keys; here its place is taken by the values' (and the gradients') size."""
    T, d = 300, 64
    size = min(1.0, 0.1 / abs(scale))
    q, k, v = (_randn(B, T, H, d, seed=s, size=f).requires_grad_() for s, f in ((1, 1.0), (2, 1.0), (3, min(1.0, 10 * size))))
    d_out = _randn(B, T, H, d, seed=4, size=min(1.0, 10 * size))
    l = _decays(H)
    out, _ = linear_attention(q, k, v, l, scale=scale)
    want = [ref.attend(q, k, v, l, scale)[0].detach(), *ref.attend_grads(q, k, v, l, scale, None, None, d_out, None)[:3]]
    for a, b in zip((out.detach(), *torch.autograd.grad(out, (q, k, v), d_out)), want):
        assert bool(torch.isfinite(a).all()) and _off(a, b) <= _room(b), (_off(a, b), _room(b))


def test_scores_beyond_the_types_range():
    """Products of queries and keys of 10^6 and more, values small enough for the outputs to fit."""
    T, H, d = 300, 2, 64
    q, k, v = _randn(1, T, H, d, seed=1, size=400.0), _randn(1, T, H, d, seed=2, size=400.0), _randn(1, T, H, d, seed=3, size=2.0 ** -11)
    l = _decays(H)
    out, final = linear_attention(q, k, v, l, scale=1.0)
    want, want_s = ref.attend(q, k, v, l, 1.0)
    assert float(want.abs().max()) < 65504 and float((q.float().transpose(1, 2) @ k.float().permute(0, 2, 3, 1)).abs().max()) > 1e6
    assert bool(torch.isfinite(out).all()) and _off(out, want) <= _room(want) and _off(final, want_s) <= STATE_ROOM


def _last(x, T):
    """sum over the 127 tokens before and the token itself: more than a chunk's"""
    c = torch.nn.functional.pad(x.cumsum(1), (0, 0, 0, 0, 128, 0))
    return c[:, 128:] - c[:, :T]


@pytest.mark.parametrize("B,H", [(1, 2), (6, 20)])
@pytest.mark.parametrize("lengths", [None, 131])
def test_tokens_of_very_different_sizes(B, H, lengths):
    """Sizes from 1 down to 2^-12 in turn: elementwise, with what a chunk's largest numbers leave others.

    Scores are brought below 2^15, but their bound (width times the largest query's and key's element) not below 2^14, so half a step of
    the smallest numbers, 2^-25, is 2^-39 of the bound.  Weighted keys are two numbers, 2^-38 of the chunk's largest; the state likewise."""
    T, d = 300, 64
    sizes = 2.0 ** -(torch.arange(T, device="cuda") * 5 % 13).double()[None, :, None, None]
    q, k, v = ((_randn(B, T, H, d, seed=s).double() * (sizes if s < 3 else sizes.flip(1))).to(FP16) for s in (1, 2, 3))
    n = None if lengths is None else torch.full((B,), lengths, device="cuda", dtype=torch.int32)
    l, scale = _decays(H), 0.25
    if n is not None:  # what stands behind has no part in a chunk's largest number either
        q[:, lengths:], k[:, lengths:], v[:, lengths:] = 60000.0, float("inf"), float("nan")
    out, final = linear_attention(q, k, v, l, scale=scale, lengths=n)
    want, want_s = ref.attend(q, k, v, l, scale, None, n)
    live = torch.ones(T, device="cuda", dtype=torch.bool) if n is None else torch.arange(T, device="cuda") < lengths
    qa, ka, va = (torch.where(live[:, None, None], x.double().abs(), 0.0) for x in (q, k, v))
    top, top_s = ref.attend(qa, ka, va, l, scale, None, n)
    f_out, f_state = ref.attend_bounds(FP16, T, d, True)
    state = top_s.amax((2, 3))[:, None, :, None]
    small = 2.0 ** -39 * d * qa.amax() * ka.amax() * scale * _last(va, T) + scale * qa.sum(-1, keepdim=True) * (2.0 ** -38 * state + 2.0 ** -37 * ka.amax() * va.sum(1, keepdim=True).amax())
    room = f_out * top + small
    assert ref.worst(out, want, room + U * (want.abs() + room) + ref.TINY[FP16]) <= 1.0
    assert ref.worst(final, want_s, f_state * top_s + 2.0 ** -37 * ka.amax() * va.sum(1)[:, :, None, :]) <= 1.0


@pytest.mark.parametrize("B,T,H", [(1, 300, 2), (1, 5003, 1), (6, 300, 20)])
def test_zeros(B, T, H):
    """Nothing to scale by: a scale of zero, zero keys, zero queries, and a state that goes on beside them."""
    q, k, v = (_randn(B, T, H, 64, seed=s) for s in (1, 2, 3))
    s = _randn(B, H, 64, 64, seed=4, to=torch.float32)
    l = _decays(H)
    for scale, a, b in ((0.0, q, k), (1.0, q, torch.zeros_like(k)), (1.0, torch.zeros_like(q), k)):
        leaves = [x.clone().requires_grad_() for x in (a, b, v)]
        out, final = linear_attention(*leaves, l, scale=scale, initial_state=s)
        want, want_s = ref.attend(a, b, v, l, scale, s)
        if bool(want.any()):
            assert _off(out, want) <= _room(want)
        else:
            assert not out.any()
        # A state that has decayed below 2^-126 is a multiple of 2^-149 (e^-99, in the middle case): each of at most 40 chunks, and of as many
        # segments, multiplies it by two numbers and rounds to one, by 2^-150 at most each time, and later factors are below one.
        assert float((final.double() - want_s).norm()) <= STATE_ROOM * float(want_s.norm()) + 160 * 2.0 ** -150 * final.numel() ** 0.5
        grads = ref.attend_grads(a, b, v, l, scale, s, None, v, None)
        for x, y in zip(torch.autograd.grad(out, leaves, v), grads):
            assert _off(x, y) <= _room(y) if bool(y.any()) else not x.any()


@pytest.mark.parametrize("B,T,H", [(1, 300, 2), (1, 5003, 1), (6, 300, 20)])
def test_two_streams_and_a_captured_call(B, T, H):
    sets = [[_randn(B, T, H, 128, seed=10 * i + s, size=10.0 ** -i) for s in range(4)] for i in range(2)]
    l = _decays(H)

    def run(q, k, v, d):
        leaves = [x.detach().requires_grad_() for x in (q, k, v)]
        out, final = linear_attention(*leaves, l, scale=0.1)
        return (out.detach(), final.detach(), *torch.autograd.grad(out, leaves, d))

    want = [run(*x) for x in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (x, st) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(st):
                got[i].append(run(*x))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for one in g:
            assert all(torch.equal(a, b) for a, b in zip(one, w))
    held = [x.clone() for x in sets[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = run(*held)
    for x, w in zip(sets[::-1], want[::-1]):
        for a, b in zip(held, x):
            a.copy_(b)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(got, w))
