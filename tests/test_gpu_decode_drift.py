"""Thousands of single tokens: what a step does to a state has to be right on average, not only to a step's rounding."""
import pytest
import torch

from rnn_train_ring_attractor_b200.linear_attention import linear_attention, linear_attention_step

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,dv", [(torch.float32, 32), (torch.bfloat16, 32), (torch.bfloat16, 33)])
def test_a_long_memory_does_not_drift(dtype, dv, achieved):
    """Each token rounds an element of the state twice, to half a step (2^-24 of it) at most and with either sign.  What a memory of M
    tokens keeps of those is the root of the sum of their squares, g^2 a token: sqrt(M / 2) * 2^-23 of the state.  A factor that is off by d
    every time adds d M instead, 7e-5 of the state for a memory of 3000 with the factor in one float."""
    B, H, dk, N = 2, 4, 16, 9000
    steps = torch.tensor([8.0, 777.0, 1500.0, 3000.0], device="cuda", dtype=torch.float64)
    l = torch.log1p(-1.0 / steps).float()
    g = torch.Generator(device="cuda").manual_seed(3)
    q, k, v = (torch.randn(N, B, H, d, device="cuda", generator=g).to(dtype) for d in (dk, dk, dv))
    state = torch.randn(B, H, dk, dv, device="cuda", generator=g)
    _, by_sequence = linear_attention(q.transpose(0, 1), k.transpose(0, 1), v.transpose(0, 1), l, initial_state=state)
    decay = torch.exp(l.double())
    power = decay ** torch.arange(N - 1, -1, -1, device="cuda", dtype=torch.float64)[:, None]  # [N, H]
    want = torch.einsum("nh,nbha,nbhc->bhac", power, k.double(), v.double()) + (decay ** N)[None, :, None, None] * state.double()
    for i in range(N):
        out = linear_attention_step(q[i], k[i], v[i], state, l, scale=1.0)
    far = lambda x: ((x.double() - want).norm(dim=(2, 3)) / want.norm(dim=(2, 3))).amax(0)  # noqa: E731
    room = (steps / 2).sqrt() * 2.0 ** -23
    achieved(f"{N} tokens {str(dtype)[6:]} (of the bound)", step=float((far(state) / room).max()), sequence=float((far(by_sequence) / room).max()))
    assert bool((far(state) <= room).all()), far(state) / room
    want_out = torch.einsum("bha,bhac->bhc", q[-1].double(), want)
    # the output: the state's error, a sum of dk terms, and the rounding to the type
    u = torch.finfo(dtype).eps / 2
    error = (out.double() - want_out).norm(dim=2) / want_out.norm(dim=2)
    top = (q[-1].double().norm(dim=2) * want.norm(dim=(2, 3))) / want_out.norm(dim=2)
    assert bool((error <= u + top * (room + dk * 2.0 ** -24)).all())
