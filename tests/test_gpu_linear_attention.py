"""Linear attention with decay against its definition in 64 bits: sequences, gradients, single tokens, refusals."""
import ctypes as C

import pytest
import torch

import layer_reference as ref
from rnn_train_ring_attractor_b200 import _lib
from rnn_train_ring_attractor_b200.linear_attention import linear_attention, linear_attention_step

pytestmark = pytest.mark.gpu

FP32, BF16, FP16 = torch.float32, torch.bfloat16, torch.float16


def _gen(seed):
    return torch.Generator(device="cuda").manual_seed(seed)


def _inputs(dtype, B, T, H, dk, dv, seed=0, state=True, lengths=None):
    g = _gen(seed)
    r = lambda *s, to=dtype: torch.randn(*s, device="cuda", generator=g).to(to)  # noqa: E731
    q, k, v, d_out = r(B, T, H, dk), r(B, T, H, dk), r(B, T, H, dv), r(B, T, H, dv)
    s, d_final = (r(B, H, dk, dv, to=FP32), r(B, H, dk, dv, to=FP32)) if state else (None, None)
    # memories from none to long ones; the first head keeps everything
    l = -torch.logspace(-4, 0.5, max(H, 2), device="cuda")[:H].clone()
    l[0] = 0.0
    n = None if lengths is None else torch.tensor(lengths, device="cuda", dtype=torch.int32)
    return q, k, v, l, s, n, d_out, d_final


def _on_tensor_cores(dtype, dk, dv):
    return dtype is not FP32 and dk <= 128 and dv <= 128


def _masked(x, n):
    return x if n is None else torch.where((torch.arange(x.shape[1], device="cuda") < n[:, None])[:, :, None, None], x, 0)


def _floors(q, k, v, scale, n, d_out=None):
    """The types' smallest numbers: additions to the bounds of (out, state) or of (dq, dk, dv, dstate)."""
    if not _on_tensor_cores(q.dtype, q.shape[-1], v.shape[-1]):
        return (ref.single_floor(q.shape[1], max(q.shape[-1], v.shape[-1]), q, k, v, d_out),) * 4
    if q.dtype is BF16:
        return (0.0,) * 4
    q, k, v = (_masked(x, n) for x in (q, k, v))
    if d_out is None:
        return ref.half_floor(q, k, v, scale, n), ref.half_floor_state(k, v)
    d_out = _masked(d_out, n)
    return (ref.half_floor(d_out, v, k, scale, n), ref.half_floor(v, d_out, q, scale, n, True), ref.half_floor(k, q, d_out, scale, n, True),
            ref.half_floor_state(q, d_out, scale) + ref.half_floor_state(d_out, q, scale).transpose(-1, -2))


def _abs(*ts):
    return [None if t is None else t.double().abs() for t in ts]


def _check_forward(got, q, k, v, l, scale, s, n):
    dtype, T = q.dtype, q.shape[1]
    dk, dv = q.shape[-1], v.shape[-1]
    f_out, f_state = ref.attend_bounds(dtype, T, max(dk, dv), _on_tensor_cores(dtype, dk, dv))
    want, want_s = ref.attend(q, k, v, l, scale, s, n)
    top, top_s = ref.attend(*_abs(q, k, v), l, scale, *_abs(s), n)
    more, more_s = _floors(q, k, v, scale, n)[:2]
    room = f_out * top + more
    e = ref.worst(got[0], want, room + ref.U[dtype] * (want.abs() + room) + ref.TINY[dtype])
    es = ref.worst(got[1], want_s, f_state * top_s + more_s + ref.TINY[FP32])
    assert e <= 1.0 and es <= 1.0, (e, es)
    return e, es


def _check_grads(got, q, k, v, l, scale, s, n, d_out, d_final):
    dtype, T = q.dtype, q.shape[1]
    dk, dv = q.shape[-1], v.shape[-1]
    f_out, f_state = ref.attend_bounds(dtype, T, max(dk, dv), _on_tensor_cores(dtype, dk, dv))
    want = ref.attend_grads(q, k, v, l, scale, s, n, d_out, d_final)
    top = ref.attend_grads(*_abs(q, k, v), l, scale, *_abs(s), n, *_abs(d_out, d_final))
    worst = []
    more = _floors(q, k, v, scale, n, d_out)
    for x, y, m, add in zip(got[:3], want, top, more):
        room = f_out * m + add
        worst.append(ref.worst(x, y, room + ref.U[dtype] * (y.abs() + room) + ref.TINY[dtype]))
    if s is not None:
        worst.append(ref.worst(got[3], want[3], f_state * top[3] + more[3] + ref.TINY[FP32]))
    assert max(worst) <= 1.0, worst
    return worst


def _run(q, k, v, l, scale, s, n, d_out, d_final):
    leaves = [x.detach().requires_grad_() for x in (q, k, v)] + ([] if s is None else [s.detach().requires_grad_()])
    out, final = linear_attention(*leaves[:3], l, scale=scale, initial_state=None if s is None else leaves[3], lengths=n)
    outs, grads = ((out,), (d_out,)) if d_final is None else ((out, final), (d_out, d_final))
    return (out.detach(), final.detach()), torch.autograd.grad(outs, leaves, grads)


CASES = [  # dtype, B, T, H, dk, dv
    (FP32, 1, 1, 1, 1, 1), (FP32, 2, 31, 3, 16, 24), (FP32, 2, 33, 2, 48, 64), (FP32, 1, 129, 2, 7, 130), (FP32, 1, 70, 2, 256, 256),
    (FP16, 2, 65, 2, 64, 64), (FP16, 1, 40, 3, 33, 100), (BF16, 1, 37, 2, 160, 192), (BF16, 1, 20, 1, 256, 3),
    (BF16, 1, 1, 1, 64, 64), (BF16, 2, 2, 3, 128, 128), (BF16, 2, 127, 2, 64, 128), (BF16, 1, 128, 3, 128, 64),
    (BF16, 2, 129, 2, 128, 128), (BF16, 3, 257, 2, 72, 104), (BF16, 1, 511, 1, 8, 16), (BF16, 2, 300, 2, 13, 99), (BF16, 1, 1000, 2, 64, 64),
    (BF16, 1, 130, 2, 1, 1), (BF16, 1, 384, 2, 127, 65),
    (FP16, 1, 1, 2, 128, 64), (FP16, 2, 129, 2, 128, 128), (FP16, 1, 300, 3, 64, 64), (FP16, 1, 257, 2, 17, 120), (FP16, 1, 200, 1, 150, 40)]


@pytest.mark.parametrize("dtype,B,T,H,dk,dv", CASES)
@pytest.mark.parametrize("state", [False, True])
def test_forward_and_gradients(dtype, B, T, H, dk, dv, state, achieved):
    q, k, v, l, s, n, d_out, d_final = _inputs(dtype, B, T, H, dk, dv, seed=T + dk, state=state)
    scale = dk ** -0.5
    got, grads = _run(q, k, v, l, scale, s, n, d_out, d_final)
    e, es = _check_forward(got, q, k, v, l, scale, s, n)
    w = _check_grads(grads, q, k, v, l, scale, s, n, d_out, d_final)
    achieved(f"linear attention {str(dtype)[6:]} {B}x{T}x{H} {dk}/{dv} (of the bound)", out=e, state=es, grads=max(w))


@pytest.mark.parametrize("dtype,T,dk,dv", [(FP32, 90, 24, 40), (BF16, 300, 64, 128), (BF16, 300, 128, 72), (BF16, 70, 200, 20),
                                           (FP16, 300, 64, 128)])
def test_padded_batches_ignore_what_stands_behind_a_sequence(dtype, T, dk, dv):
    lengths = [T, 0, 1, T - 1, 128 if T > 128 else 32, T // 2]
    q, k, v, l, s, n, d_out, d_final = _inputs(dtype, len(lengths), T, 2, dk, dv, seed=5, lengths=lengths)
    clean, clean_grads = _run(q, k, v, l, 0.2, s, n, d_out, d_final)
    _check_forward(clean, q, k, v, l, 0.2, s, n)
    _check_grads(clean_grads, q, k, v, l, 0.2, s, n, d_out, d_final)
    for bad in (float("nan"), float("inf"), torch.finfo(dtype).min):
        for x in (q, k, v, d_out):
            for b, m in enumerate(lengths):
                x[b, m:] = bad
        got, grads = _run(q, k, v, l, 0.2, s, n, d_out, d_final)
        for a, b in zip((*got, *grads), (*clean, *clean_grads)):
            assert torch.equal(a, b)
    for b, m in enumerate(lengths):
        assert not clean[0][b, m:].any() and not any(x[b, m:].any() for x in clean_grads[:3])
    assert torch.equal(clean[1][1], s[1]) and torch.equal(clean_grads[3][1], d_final[1])
    # lengths outside 0..T count as the nearest of them
    wild = torch.tensor([T + 9, -3, 1, T - 1, lengths[4], T // 2], device="cuda", dtype=torch.int32)
    for a, b in zip(linear_attention(q, k, v, l, scale=0.2, initial_state=s, lengths=wild), clean):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype,T,dk,dv", [(BF16, 300, 64, 64), (BF16, 385, 128, 72), (BF16, 140, 40, 128), (BF16, 1000, 128, 128),
                                           (BF16, 257, 13, 99), (FP16, 300, 128, 128), (FP16, 513, 64, 128)])
def test_more_sequences_than_processors(dtype, T, dk, dv):
    """Where the gradients of keys and values of a sequence are one block's work; padding with NaN behind the sequences as well."""
    lengths, H = [T, 0, 1, T - 1, 128, T // 2, T, T], 19
    q, k, v, l, s, n, d_out, d_final = _inputs(dtype, len(lengths), T, H, dk, dv, seed=12, lengths=lengths)
    clean, clean_grads = _run(q, k, v, l, 0.2, s, n, d_out, d_final)
    _check_forward(clean, q, k, v, l, 0.2, s, n)
    _check_grads(clean_grads, q, k, v, l, 0.2, s, n, d_out, d_final)
    for x in (q, k, v, d_out):
        for b, m in enumerate(lengths):
            x[b, m:] = float("nan")
    got, grads = _run(q, k, v, l, 0.2, s, n, d_out, d_final)
    for a, b in zip((*got, *grads), (*clean, *clean_grads)):
        assert torch.equal(a, b)


@pytest.mark.parametrize("dtype,B,T,H,dk,dv", [(FP32, 1, 2500, 1, 40, 24), (BF16, 1, 5003, 1, 128, 64), (BF16, 2, 4100, 1, 64, 128),
                                               (BF16, 1, 2600, 3, 20, 33), (FP16, 1, 3000, 1, 200, 64),
                                               (FP16, 1, 5003, 1, 64, 128)])
def test_long_sequences_of_few_heads(dtype, B, T, H, dk, dv):
    """Cut into segments that run at once: the same bounds, ends inside and before segments, and one call like two."""
    for lengths in (None, [T - 1001] + [7] * (B - 1)):
        q, k, v, l, s, n, d_out, d_final = _inputs(dtype, B, T, H, dk, dv, seed=2, lengths=lengths)
        l[0] = -1e-3
        p = _lib.LinearAttention(B, T, H, dk, dv, 0, 1.0)
        assert _lib.lib().ringrnn_linear_attention_bytes(C.byref(p), None) > 0
        got, grads = _run(q, k, v, l, 0.3, s, n, d_out, d_final)
        _check_forward(got, q, k, v, l, 0.3, s, n)
        _check_grads(grads, q, k, v, l, 0.3, s, n, d_out, d_final)
    at = 1777
    _, half = linear_attention(q[:, :at], k[:, :at], v[:, :at], l, scale=0.3, initial_state=s)
    out, final = linear_attention(q[:, at:], k[:, at:], v[:, at:], l, scale=0.3, initial_state=half)
    whole = torch.cat((linear_attention(q[:, :at], k[:, :at], v[:, :at], l, scale=0.3, initial_state=s)[0], out), dim=1)
    _check_forward((whole, final), q, k, v, l, 0.3, s, None)


@pytest.mark.parametrize("T,H,dk,dv", [(30011, 8, 128, 128), (20003, 20, 64, 64), (9000, 37, 64, 128)])
def test_many_chunks_in_a_segment(T, H, dk, dv):
    """Against the fp32 kernel on the same numbers (itself held to the definition above): what the two may differ by."""
    q, k, v, l, s, n, d_out, d_final = _inputs(BF16, 1, T, H, dk, dv, seed=15)
    l = l - 1e-3
    one = [x.float() for x in (q, k, v)]
    for _ in range(3):  # (the kernels' roles run ahead of each other by what the loads leave them)
        got, grads = _run(q, k, v, l, 0.1, s, n, d_out, d_final)
    want, want_g = _run(*one, l, 0.1, s, n, d_out.float(), d_final)
    top, top_g = _run(*(x.abs() for x in one), l, 0.1, s.abs(), n, d_out.float().abs(), d_final.abs())
    u = ref.U[BF16]
    # (the fp32 kernel gives the bound's own sums to a part in 2^10, which the factor 1.01 covers)
    for i, (a, b, t) in enumerate(zip((*got, *grads), (*want, *want_g), (*top, *top_g))):
        # a memory is at most a thousand steps long here: sums of 8192 terms at most count, in either kernel
        f = ref.attend_bounds(BF16, 8192, 128, True)[i in (1, 5)] + 2 * ref.attend_bounds(FP32, 8192, 128, False)[0]
        allowed = 1.01 * (f + (0 if i in (1, 5) else u * (1 + f))) * t.double() + ref.TINY[BF16]
        assert ref.worst(a, b.double(), allowed) <= 1.0, i


@pytest.mark.parametrize("decay", [0.0, -1e-5, -0.3, -5.0, -60.0, -3e38, float("-inf")])
@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
def test_decays_from_none_to_all(dtype, decay):
    q, k, v, l, s, n, d_out, d_final = _inputs(dtype, 1, 200, 2, 64, 64, seed=9)
    l[:] = decay
    got, grads = _run(q, k, v, l, 0.125, s, n, d_out, d_final)
    _check_forward(got, q, k, v, l, 0.125, s, n)
    _check_grads(grads, q, k, v, l, 0.125, s, n, d_out, d_final)


@pytest.mark.parametrize("dtype,dk,dv", [(BF16, 64, 64), (BF16, 128, 96), (BF16, 24, 50), (FP32, 20, 30)])
def test_strides(dtype, dk, dv):
    B, T, H = 2, 150, 3
    q, k, v, l, s, n, d_out, d_final = _inputs(dtype, B, T, H, dk, dv, seed=4)
    want = linear_attention(q, k, v, l, initial_state=s)
    # heads first, tokens first, inside a wider tensor at an odd offset, one tensor for q and k
    turned = [x.transpose(1, 2).contiguous().transpose(1, 2) for x in (q, k, v)]
    first = [x.transpose(0, 1).contiguous().transpose(0, 1) for x in (q, k, v)]
    inside = []
    for x in (q, k, v):
        wide = torch.full((B, T, H, x.shape[-1] + 7), float("nan"), device="cuda", dtype=dtype)
        wide[..., 3:3 + x.shape[-1]] = x
        inside.append(wide[..., 3:3 + x.shape[-1]])
    both = torch.cat((q, k), dim=-1)
    split = [both[..., :dk], both[..., dk:], v]
    last = [x.transpose(2, 3).contiguous().transpose(2, 3) for x in (q, k, v)]
    for xs in (turned, first, inside, split, last):
        for a, b in zip(linear_attention(*xs, l, initial_state=s), want):
            assert torch.equal(a, b)


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_gradients_of_shared_heads_and_sequences(dtype):
    """One key head and one value sequence for all, by expand: autograd sums what the kernel gives each."""
    B, T, H, d = 2, 140, 3, 64
    q, k, v, l, s, n, _, _ = _inputs(dtype, B, T, H, d, d, seed=6)
    k1, v1 = k[:, :, :1].clone().requires_grad_(), v[:1].clone().requires_grad_()
    ke, ve = k1.expand(B, T, H, d), v1.expand(B, T, H, d)
    out, final = linear_attention(q, ke, ve, l, scale=0.125)
    _check_forward((out.detach(), final.detach()), q, ke.detach(), ve.detach(), l, 0.125, None, None)
    out.sum().backward()  # a gradient without strides of its own
    d_out = torch.ones_like(out)
    want = ref.attend_grads(q, ke, ve, l, 0.125, None, None, d_out, None)
    top = ref.attend_grads(*_abs(q, ke.detach(), ve.detach()), l, 0.125, None, None, _abs(d_out)[0], None)
    f, _ = ref.attend_bounds(dtype, T, d, _on_tensor_cores(dtype, d, d))
    u = ref.U[dtype]
    for got, y, m, dim in ((k1.grad, want[1], top[1], 2), (v1.grad, want[2], top[2], 0)):
        # each part has its own rounding, the sum of up to three one for every addition
        y, m = y.sum(dim, keepdim=True), m.sum(dim, keepdim=True)
        assert ref.worst(got, y, (f + u * (1 + f)) * m + 3 * u * (1 + f) * m) <= 1.0


@pytest.mark.parametrize("size", [2.0 ** 9, 2.0 ** -9])
def test_range_of_half_states(size):
    """States far beyond fp16's range, or far below its step, read out as exactly as others."""
    q, k, v, l, s, n, d_out, d_final = _inputs(FP16, 1, 300, 2, 64, 128, seed=31)
    q = (q / size).to(FP16)
    k, v, s = (k * min(1.0, size)).to(FP16), (v * size).to(FP16), s * size ** 2
    out, final = linear_attention(q, k, v, l, scale=0.125, initial_state=s)
    assert bool(torch.isfinite(out).all())
    _check_forward((out, final), q, k, v, l, 0.125, s, n)


def test_offsets_beyond_32_bits():
    T, H, d = 130, 1, 64
    far = (1 << 32) + 8 * 1001
    store = torch.zeros(far + T * H * d, device="cuda", dtype=BF16)
    q, k, v, l, s, n, d_out, d_final = _inputs(BF16, 2, T, H, d, d, seed=8)
    wide = torch.as_strided(store, (2, T, H, d), (far, H * d, d, 1))
    wide.copy_(k)
    for a, b in zip(linear_attention(q, wide, v, l), linear_attention(q, k, v, l)):
        assert torch.equal(a, b)
    wide.copy_(v)
    for a, b in zip(linear_attention(q.float(), k.float(), wide.float(), l), linear_attention(q.float(), k.float(), v.float(), l)):
        assert torch.equal(a, b)


def test_gradients_against_differences():
    """The operator is linear in each input, so a difference quotient in fp32 has no error but rounding: the two evaluations'
    bounds over the step of 2."""
    q, k, v, l, s, n, d_out, d_final = _inputs(FP32, 1, 40, 2, 12, 20, seed=11)
    _, grads = _run(q, k, v, l, 0.3, s, n, d_out, d_final)
    g = _gen(12)
    f, fs = ref.attend_bounds(FP32, 40, 20, False)
    for i, x in enumerate((q, k, v, s)):
        way = torch.randn(x.shape, device="cuda", generator=g)
        ends, room = [], 0.0
        for sign in (1.0, -1.0):
            xs = [q, k, v, s]
            xs[i] = x + sign * way
            out, final = linear_attention(*xs[:3], l, scale=0.3, initial_state=xs[3])
            ends.append(float((out.double() * d_out).sum() + (final.double() * d_final).sum()))
            a, b = ref.attend(*_abs(*xs[:3]), l, 0.3, *_abs(xs[3]))
            room += float((a * d_out.abs()).sum() * (f + 2 * ref.U[FP32]) + (b * d_final.abs()).sum() * (fs + 2 * ref.U[FP32]))
        got = float((grads[i].double() * way).sum())
        top = ref.attend_grads(*_abs(q, k, v), l, 0.3, *_abs(s), n, *_abs(d_out, d_final))[i]
        room = room / 2 + float((top * way.abs()).sum()) * (f + ref.U[FP32])
        assert abs(got - (ends[0] - ends[1]) / 2) <= room


@pytest.mark.parametrize("dtype", [FP32, BF16])
def test_same_bits_twice_and_parts_of_gradients(dtype):
    q, k, v, l, s, n, d_out, d_final = _inputs(dtype, 2, 700, 2, 64, 128, seed=13)
    one, two = (_run(q, k, v, l, 0.1, s, n, d_out, d_final) for _ in range(2))
    for a, b in zip((*one[0], *one[1]), (*two[0], *two[1])):
        assert torch.equal(a, b)
    # one leaf at a time, and one output at a time
    for i in range(4):
        xs = [x.detach() for x in (q, k, v, s)]
        xs[i].requires_grad_()
        out, final = linear_attention(*xs[:3], l, scale=0.1, initial_state=xs[3])
        a, = torch.autograd.grad((out, final), xs[i], (d_out, d_final), retain_graph=True)
        assert torch.equal(a, one[1][i])
        if i != 0:
            b, = torch.autograd.grad(final, xs[i], d_final)
            want = ref.attend_grads(q, k, v, l, 0.1, s, n, torch.zeros_like(d_out), d_final)[i]
            top = ref.attend_grads(*_abs(q, k, v), l, 0.1, *_abs(s), n, torch.zeros_like(d_out), d_final.abs())[i]
            f = ref.attend_bounds(dtype, 700, 128, _on_tensor_cores(dtype, 64, 128))[0]
            floor = ref.single_floor(700, 128, q, k, v, s, d_final)
            assert ref.worst(b, want, (f + ref.U[dtype] * (1 + f)) * top + floor + ref.TINY[dtype]) <= 1.0
        xs[i].requires_grad_(False)


def test_empty_calls():
    l = torch.zeros(2, device="cuda")
    q = torch.zeros(3, 0, 2, 8, device="cuda", requires_grad=True)
    s = torch.randn(3, 2, 8, 8, device="cuda", requires_grad=True)
    out, final = linear_attention(q, q, q, l, initial_state=s)
    assert out.shape == (3, 0, 2, 8) and torch.equal(final, s)
    final.sum().backward()
    assert torch.equal(s.grad, torch.ones_like(s)) and q.grad.shape == q.shape
    out, final = linear_attention(q.detach(), q.detach(), q.detach(), l)
    assert not final.any()
    none = torch.zeros(0, 2, 8, device="cuda")
    assert linear_attention_step(none, none, none, torch.zeros(0, 2, 8, 8, device="cuda"), l).shape == (0, 2, 8)


# ---- one token -----------------------------------------------------------------------------------------------------------
@pytest.mark.parametrize("dtype,B,H,dk,dv", [(FP32, 1, 1, 1, 1), (BF16, 3, 2, 128, 128), (FP16, 2, 3, 64, 96), (BF16, 2, 2, 33, 50),
                                             (FP32, 2, 1, 1024, 36), (BF16, 1, 2, 200, 333), (BF16, 5, 1, 8, 2),
                                             # states enough to go row by row
                                             (BF16, 20, 17, 100, 100), (FP32, 30, 10, 33, 33), (FP16, 37, 8, 128, 50), (BF16, 300, 1, 5, 1),
                                             (BF16, 60, 5, 64, 1000), (FP32, 99, 3, 70, 256), (BF16, 75, 4, 3, 255)])
def test_step(dtype, B, H, dk, dv, achieved):
    q, k, v, l, s, _, _, _ = _inputs(dtype, B, 1, H, dk, dv, seed=dk)
    l = l - 0.01
    state = s.clone()
    before = state._version
    out = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], state, l, scale=0.3)
    assert state._version > before
    want, want_s = ref.attend_by_steps(q, k, v, l, 0.3, s)
    top, top_s = ref.attend_by_steps(*_abs(q, k, v), l, 0.3, *_abs(s))
    f = (dk + 16) * 2.0 ** -23
    e = ref.worst(out, want[:, 0], f * top[:, 0] + ref.U[dtype] * (want[:, 0].abs() + f * top[:, 0]) + ref.TINY[dtype])
    es = ref.worst(state, want_s, 16 * 2.0 ** -23 * top_s + ref.TINY[FP32])
    assert e <= 1.0 and es <= 1.0
    achieved(f"step {str(dtype)[6:]} {B}x{H} {dk}/{dv} (of the bound)", out=e, state=es)


def test_steps_continue_a_prompt_and_skip_what_is_not_active():
    B, T, H, d = 3, 70, 2, 64
    q, k, v, l, s, n, _, _ = _inputs(BF16, B, T + 5, H, d, d, seed=21)
    l[0] = -0.02
    _, state = linear_attention(q[:, :T], k[:, :T], v[:, :T], l, initial_state=s)
    outs = [linear_attention_step(q[:, T + i], k[:, T + i], v[:, T + i], state, l) for i in range(5)]
    whole, final = linear_attention(q, k, v, l, initial_state=s)
    both = torch.cat((linear_attention(q[:, :T], k[:, :T], v[:, :T], l, initial_state=s)[0], torch.stack(outs, dim=1)), dim=1)
    for got in ((both, state), (whole, final)):
        _check_forward(got, q, k, v, l, d ** -0.5, s, None)
    active = torch.tensor([True, False, True], device="cuda")
    held, k[1, 0] = state.clone(), float("nan")
    out = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], state, l, active=active)
    assert torch.equal(state[1], held[1]) and not out[1].any()
    alone = held[[0, 2]].contiguous()
    want = linear_attention_step(q[[0, 2], 0], k[[0, 2], 0], v[[0, 2], 0], alone, l)
    assert torch.equal(out[[0, 2]], want) and torch.equal(state[[0, 2]], alone)


def test_step_strides():
    B, H, dk, dv = 2, 3, 40, 24
    q, k, v, l, s, _, _, _ = _inputs(BF16, B, 4, H, dk, dv, seed=22)
    a, b = s.clone(), s.clone()
    want = linear_attention_step(q[:, 2].contiguous(), k[:, 2].contiguous(), v[:, 2].contiguous(), a, l)
    wide = torch.cat((q, k, v), dim=-1)[:, 2]
    got = linear_attention_step(wide[..., :dk], wide[..., dk:2 * dk], wide[..., 2 * dk:], b, l)
    assert torch.equal(got, want) and torch.equal(a, b)
    odd = torch.cat((torch.zeros(1, device="cuda"), s.flatten()))[1:].view_as(s)  # a state that no vector load may touch
    got = linear_attention_step(q[:, 2], k[:, 2], v[:, 2], odd, l)
    f = (dk + 16) * 2.0 ** -23
    top, _ = ref.attend_by_steps(*_abs(q[:, 2:3], k[:, 2:3], v[:, 2:3]), l, dk ** -0.5, *_abs(s))
    assert ref.worst(got, want.double(), 2 * f * top[:, 0] + 2 * ref.U[BF16] * (1 + f) * top[:, 0]) <= 1.0
    assert torch.equal(odd, a)


# ---- streams, graphs, refusals ----------------------------------------------------------------------------------------------
@pytest.mark.parametrize("B,H,dk,dv", [(300, 2, 12, 100), (150, 2, 20, 33)])
def test_step_of_many_narrow_states(B, H, dk, dv):
    """Row by row like column by column (a state that starts off a 16-byte boundary); inactive ones stay; nothing beside is written."""
    q, k, v, l, s, _, _, _ = _inputs(BF16, B, 1, H, dk, dv, seed=3)
    active = torch.rand(B, device="cuda", generator=_gen(4)) < 0.7
    one = s.clone()
    flat = torch.full((s.numel() + 9,), 7.0, device="cuda")
    two = flat[5:5 + s.numel()].view(s.shape)
    two.copy_(s)
    a, b = (linear_attention_step(q[:, 0], k[:, 0], v[:, 0], x, l, active=active) for x in (one, two))
    few = torch.cat([linear_attention_step(q[i:i + 10, 0], k[i:i + 10, 0], v[i:i + 10, 0], s[i:i + 10], l, active=active[i:i + 10]) for i in range(0, B, 10)])
    assert torch.equal(one, two) and torch.equal(one, s)
    assert not a[~active].any() and not b[~active].any() and not few[~active].any()
    room = dk * 2.0 ** -20 * (q[:, 0].float().abs().unsqueeze(-1) * s.abs()).sum(-2) + 2.0 ** -7 * few.float().abs() + 1e-30
    assert ((a.float() - few.float()).abs() <= room).all() and ((b.float() - few.float()).abs() <= room).all()
    assert (flat[:5] == 7.0).all() and (flat[5 + s.numel():] == 7.0).all()


@pytest.mark.parametrize("T,H", [(20, 2), (300, 2), (4100, 1), (300, 60)])
def test_two_streams_at_once(T, H):
    sets = [_inputs(BF16, 1, T, H, 64, 64, seed=i) for i in range(2)]
    want = [_run(*x[:4], 0.1, *x[4:]) for x in sets]
    streams = [torch.cuda.Stream() for _ in sets]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(5):
        for i, (x, st) in enumerate(zip(sets, streams)):
            with torch.cuda.stream(st):
                got[i].append(_run(*x[:4], 0.1, *x[4:]))
    torch.cuda.synchronize()
    for g, w in zip(got, want):
        for one in g:
            for a, b in zip((*one[0], *one[1]), (*w[0], *w[1])):
                assert torch.equal(a, b)


@pytest.mark.parametrize("T,H", [(20, 2), (300, 2), (4100, 1), (300, 60)])
def test_captured_and_replayed(T, H):
    q, k, v, l, s, n, d_out, d_final = _inputs(BF16, 1, T, H, 64, 64, seed=1, lengths=[T - 5])
    state = s.clone()
    leaves = [x.requires_grad_() for x in (q, k, v, s)]

    def work():
        out, final = linear_attention(q, k, v, l, scale=0.1, initial_state=s, lengths=n)
        grads = torch.autograd.grad((out, final), leaves, (d_out, d_final))
        with torch.no_grad():
            step = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], state, l)
        return (out, final, *grads, step, state)

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
    other = _inputs(BF16, 1, T, H, 64, 64, seed=2)
    with torch.no_grad():
        for a, b in zip((q, k, v, s, d_out, d_final), (*other[:3], other[4], *other[6:])):
            a.copy_(b)
        n.fill_(T - 77)
        state.copy_(s)
    graph.replay()
    torch.cuda.synchronize()
    got = [x.clone() for x in held]
    with torch.no_grad():
        state.copy_(s)
    for a, b in zip(got, work()):
        assert torch.equal(a, b)


def test_first_cuda_call_of_a_host_thread():
    """The library called from threads that have not touched the GPU before, as autograd's are."""
    import threading
    L = _lib.lib()
    q, k, v, l, s, n, _, _ = _inputs(BF16, 1, 70, 2, 64, 64)
    want, _ = linear_attention(q, k, v, l, scale=0.5)
    out = torch.empty_like(want)
    sd = lambda t: _lib.Strided(t.data_ptr(), *t.stride()[:3])  # noqa: E731
    p = _lib.LinearAttention(1, 70, 2, 64, 64, 1, 0.5, sd(q), sd(k), sd(v), l.data_ptr())
    torch.cuda.synchronize()
    got = []
    for _ in range(3):
        t = threading.Thread(target=lambda: got.append(L.ringrnn_linear_attention_fwd(C.byref(p), out.data_ptr(), None, None, 0, None)))
        t.start()
        t.join()
    torch.cuda.synchronize()
    assert got == [0, 0, 0] and torch.equal(out, want)


@pytest.mark.parametrize("pad", [64, 65, 66])
def test_nothing_is_written_beyond_the_outputs(pad):
    """Exact-size outputs inside a larger block, at any boundary, by the C entry points: what surrounds them stays."""
    L = _lib.lib()
    for dtype, code, B, T, H, dk, dv in ((BF16, 1, 2, 131, 2, 24, 40), (FP32, 0, 1, 45, 3, 7, 9), (BF16, 1, 1, 140, 1, 13, 99),
                                       (BF16, 1, 1, 200, 3, 64, 128), (BF16, 1, 2, 131, 1, 128, 127), (FP16, 2, 1, 140, 3, 30, 61),
                                       (BF16, 1, 4, 131, 17, 127, 128)):
        q, k, v, l, s, n, d_out, d_final = _inputs(dtype, B, T, H, dk, dv, seed=3)
        sd = lambda t: _lib.Strided(t.data_ptr(), *t.stride()[:3])  # noqa: E731
        p = _lib.LinearAttention(B, T, H, dk, dv, code, 0.2, sd(q), sd(k), sd(v), l.data_ptr(), None, s.data_ptr())

        def block(numel, dt):
            t = torch.full((numel + 2 * pad,), 77.0, device="cuda", dtype=dt)
            return t, t[pad:pad + numel].data_ptr()

        (o, po), (f, pf) = block(B * T * H * dv, dtype), block(B * H * dk * dv, FP32)
        (a, pa), (b, pb), (c, pc), (e, pe) = (block(B * T * H * dk, dtype), block(B * T * H * dk, dtype), block(B * T * H * dv, dtype),
                                             block(B * H * dk * dv, FP32))
        for backward in (0, 1):
            size = L.ringrnn_linear_attention_bytes(C.byref(p), C.byref(sd(d_out)) if backward else None)
            ws = torch.full((size + 512,), 85, device="cuda", dtype=torch.uint8)
            if backward:
                rc = L.ringrnn_linear_attention_bwd(C.byref(p), C.byref(sd(d_out)), d_final.data_ptr(), pa, pb, pc, pe, ws.data_ptr(), size, None)
            else:
                rc = L.ringrnn_linear_attention_fwd(C.byref(p), po, pf, ws.data_ptr(), size, None)
            torch.cuda.synchronize()
            assert rc == 0 and bool((ws[size:] == 85).all())
        for t in (o, f, a, b, c, e):
            assert bool((t[:pad] == 77).all()) and bool((t[-pad:] == 77).all())
        got, grads = _run(q, k, v, l, 0.2, s, n, d_out, d_final)
        for t, x in zip((o, f, a, b, c, e), (*got, *grads)):
            assert torch.equal(t[pad:-pad].view_as(x), x)


def test_refusals():
    q, k, v, l, s, n, _, _ = _inputs(BF16, 2, 8, 3, 16, 24)
    ok = dict(initial_state=s)
    for bad, match in (((q, k[:, :7], v, l), "k must have shape"), ((q, k, v[:1], l), "v must have shape"), ((q, k.float(), v, l), "k must be bfloat16"),
                       ((q[0], k[0], v[0], l), "4 dimensions"), ((q, k, v, l[:2]), "log_decay must have shape"), ((q, k, v, l.double()), "log_decay must be float32"),
                       ((q, k.cpu(), v, l), "k must be a CUDA tensor"), ((q.int(), k, v, l), "float32, bfloat16 or float16")):
        with pytest.raises(RuntimeError, match=match):
            linear_attention(*bad, **ok)
    with pytest.raises(RuntimeError, match="initial_state must be float32"):
        linear_attention(q, k, v, l, initial_state=s.to(BF16))
    with pytest.raises(RuntimeError, match="initial_state must be contiguous"):
        linear_attention(q, k, v, l, initial_state=s.transpose(2, 3).contiguous().transpose(2, 3))
    with pytest.raises(RuntimeError, match="lengths must be int32"):
        linear_attention(q, k, v, l, lengths=torch.tensor([1, 2], device="cuda"))
    with pytest.raises(RuntimeError, match="log_decay has no gradient"):
        linear_attention(q, k, v, l.clone().requires_grad_())
    wide = torch.zeros(1, 2, 1, 257, device="cuda")
    with pytest.raises(RuntimeError, match="between 1 and 256"):
        linear_attention(wide, wide, wide, l[:1])
    with pytest.raises(RuntimeError, match="no gradient"):
        linear_attention_step(q[:, 0].clone().requires_grad_(), k[:, 0], v[:, 0], s, l)
    with pytest.raises(RuntimeError, match="active must be bool"):
        linear_attention_step(q[:, 0], k[:, 0], v[:, 0], s, l, active=torch.ones(2, device="cuda"))
    with pytest.raises(RuntimeError, match="state must be contiguous"):
        linear_attention_step(q[:, 0], k[:, 0], v[:, 0], s.transpose(2, 3).contiguous().transpose(2, 3), l)
    x = q.clone().requires_grad_()
    out, _ = linear_attention(x, k, v, l)
    g, = torch.autograd.grad(out.float().square().sum(), x, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable"):
        g.float().sum().backward()
