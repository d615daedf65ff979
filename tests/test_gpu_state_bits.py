"""States of bf16 tensors that a caller sees: the third part of a weighted key counts."""
import pytest
import torch

import layer_reference as ref
from rnn_train_ring_attractor_b200.linear_attention import linear_attention

pytestmark = pytest.mark.gpu

BF16 = torch.bfloat16
# Three parts leave 2^-24 of a product; a chunk's sum is added up by 24 instructions that may cut off a step of fp32 (2^-23), half of one on
# average, of a running sum that is half of the whole on average: 24 * 2^-25 = 7e-7.  Two parts leave up to 2 * 2^-16 of a product, of a
# quarter of that on average: 2^-17 = 8e-6, of which half (3.8e-6) was measured.  In the middle, by ratio: 1.5e-6.
ROOM = 1.5e-6


@pytest.mark.parametrize("B,T,H,dk,dv", [(1, 700, 3, 128, 128), (1, 515, 2, 64, 64), (2, 300, 2, 72, 104), (1, 6007, 1, 128, 64), (1, 5003, 2, 64, 128),
                                         (10, 260, 16, 64, 64), (10, 260, 16, 128, 128)])
def test_states_keep_24_bits(B, T, H, dk, dv, achieved):
    """In one segment, in several, and with more blocks than processors."""
    g = torch.Generator(device="cuda").manual_seed(T)
    r = lambda *s, to=BF16: torch.randn(*s, device="cuda", generator=g).to(to)  # noqa: E731
    q, k, v, d_out, s, d_final = r(B, T, H, dk), r(B, T, H, dk), r(B, T, H, dv), r(B, T, H, dv), r(B, H, dk, dv, to=torch.float32), r(B, H, dk, dv, to=torch.float32)
    s.requires_grad_()
    steps = torch.tensor([37.3, 300.7, 1900.1, 90.9], device="cuda", dtype=torch.float64).repeat(4)[:H]
    l = torch.log1p(-1.0 / steps).float()
    out, final = linear_attention(q, k, v, l, scale=0.1, initial_state=s)
    d_initial, = torch.autograd.grad((out, final), s, (d_out, d_final))
    want = ref.attend(q, k, v, l, 0.1, s)[1]
    want_d = ref.attend_grads(q, k, v, l, 0.1, s, None, d_out, d_final)[3]
    off = lambda a, b: float(((a.double() - b).norm(dim=(2, 3)) / b.norm(dim=(2, 3))).max())  # noqa: E731
    got = dict(final=off(final.detach(), want.detach()), d_initial=off(d_initial, want_d))
    achieved(f"bf16 states {B}x{T}x{H} {dk}/{dv}", **got)
    assert max(got.values()) <= ROOM, got
