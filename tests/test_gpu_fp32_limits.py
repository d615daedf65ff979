"""The fp32 kernel's products by themselves, and the largest numbers of the type."""
import pytest
import torch

import layer_reference as ref
from rnn_train_ring_attractor_b200.linear_attention import linear_attention

pytestmark = pytest.mark.gpu

FP32 = torch.float32
# A factor is taken as two numbers of eleven bits and is off by one unit of its last place at most (2^-23), and the product of the two
# second numbers (2^-12 of a factor each, and a little) is left out: 2 * 2^-23 + 2^-22 of a product, and parts in 2^-11 of that.
PRODUCT = 2.0 ** -21 * (1 + 2.0 ** -10)


def _full(*shape, seed, lo=1.0, hi=2.0):
    g = torch.Generator(device="cuda").manual_seed(seed)
    return torch.rand(*shape, device="cuda", generator=g) * (hi - lo) + lo


@pytest.mark.parametrize("lo,hi", [(1.0, 1.01), (1.0, 2.0), (-2.0, 2.0)])
def test_one_product(lo, hi, achieved):
    """One token of heads of one element: no sum that a product's error could hide in."""
    B, H = 4096, 64
    q, k, v = (_full(B, 1, H, 1, seed=s, lo=lo, hi=hi) for s in (1, 2, 3))
    l = torch.full((H,), -0.1, device="cuda")
    out, final = linear_attention(q, k, v, l, scale=1.0)
    want = q.double() * k.double() * v.double()
    want_s = (k.double() * v.double())[:, 0, :, :, None]
    e, es = float(((out.double() - want) / want).abs().max()), float(((final.double() - want_s) / want_s).abs().max())
    achieved(f"one fp32 product of {lo:g} to {hi:g}, in 2^-24", out=e * 2 ** 24, state=es * 2 ** 24)
    # sums of two parts, of zero and the product, the scale and the power: a rounding or a cut of 2^-23 each
    assert es <= PRODUCT + 4 * 2.0 ** -23
    assert e <= 2 * PRODUCT + 10 * 2.0 ** -23


@pytest.mark.parametrize("top", [torch.finfo(FP32).max, torch.finfo(FP32).min, 3.4e38, -(2.0 ** 128 - 2.0 ** 116)])
def test_largest_numbers_of_the_type(top):
    """Where what they are multiplied with leaves the result finite, it is right."""
    B, T, H, dk, dv = 1, 40, 2, 8, 8
    q, k, v = (_full(B, T, H, 8, seed=s, lo=-1.0, hi=1.0) for s in (1, 2, 3))
    l = torch.full((H,), -0.1, device="cuda")
    s = _full(B, H, dk, dv, seed=4, lo=-1.0, hi=1.0)
    # a key that is zero where a query is as large as can be, and the other way round
    q[..., 0], k[..., 0], s[:, :, 0] = top, 0.0, 0.0
    q[:, 5:9, :, 1], k[:, :9, :, 1], s[:, :, 1] = 0.0, top, 0.0
    q[:, 9:, :, 1] = 0.0
    q[:, :5, :, 1] = 0.0
    v = v * 2.0 ** -9
    out, final = linear_attention(q, k, v, l, scale=0.5, initial_state=s)
    want, want_s = ref.attend(q, k, v, l, 0.5, s)
    # (zeros times them are zero in the sums of absolute values too)
    top_o, top_s = ref.attend(*(x.double().abs() for x in (q, k, v)), l, 0.5, s.double().abs())
    f, fs = ref.attend_bounds(FP32, T, 8, False)
    floor = ref.single_floor(T, 8, q.clamp(-1, 1), k.clamp(-1, 1), v)
    assert bool(torch.isfinite(out).all()) and bool(torch.isfinite(final).all())
    assert ref.worst(out, want, (f + 2 * ref.U[FP32]) * top_o + floor + ref.TINY[FP32]) <= 1.0
    assert ref.worst(final, want_s, fs * top_s + floor + ref.TINY[FP32]) <= 1.0
    # values: outputs of a quarter of them
    one = torch.full((1, 1, 2, 1), 0.5, device="cuda")
    out, _ = linear_attention(one, one, torch.full((1, 1, 2, 3), top, device="cuda"), l, scale=1.0)
    assert ref.worst(out, torch.full((1, 1, 2, 3), top / 4, device="cuda", dtype=torch.float64), abs(top) / 4 * (f + 2 * ref.U[FP32])) <= 1.0
