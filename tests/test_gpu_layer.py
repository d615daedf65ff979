"""The layer operators together, as a linear recurrent layer uses them: rotary queries and keys, linear attention with decay,
dropout onto the residual; a training step's gradients, and the same tokens one by one."""
import pytest
import torch

import layer_reference as ref
from rnn_train_ring_attractor_b200.dropout import dropout
from rnn_train_ring_attractor_b200.linear_attention import linear_attention, linear_attention_step
from rnn_train_ring_attractor_b200.rotary import rotary, rotary_frequencies

pytestmark = pytest.mark.gpu


def _layer(x, W, l, f, n, positions, p, seed):
    B, T, D = x.shape
    H = l.shape[0]
    q, k, v = (x @ W).view(B, T, H, -1).split(D // H, dim=-1)
    q, k = rotary(q, k, f, positions, interleaved=True)
    out, state = linear_attention(q, k, v, l, lengths=n)
    return dropout(out.reshape(B, T, D), p, seed, residual=x), state


def _layer_in_64_bits(x, W, l, f, n, positions, p, seed):
    B, T, D = x.shape
    H = l.shape[0]
    d = D // H
    q, k, v = (x @ W).view(B, T, H, -1).split(d, dim=-1)
    q, k = (ref.turn(y, positions, f, True) for y in (q, k))
    out, state = ref.attend(q, k, v, l, d ** -0.5, None, n)
    kept = ref.kept(B, T * D, p, seed, 0, 0).to(x.device).view(B, T, D)
    return torch.where(kept, out.reshape(B, T, D) / (1 - p), 0.0) + x, state


def _far(a, b):
    return float((a.double() - b).norm() / b.norm())


@pytest.mark.parametrize("dtype,T", [(torch.float32, 45), (torch.bfloat16, 140)])
def test_training_step_of_a_layer(dtype, T, achieved):
    B, H, D = 3, 4, 256
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn(B, T, D, device="cuda", generator=g).to(dtype).requires_grad_()
    W = (torch.randn(D, 3 * D, device="cuda", generator=g) * D ** -0.5).to(dtype).requires_grad_()
    d_y = torch.randn(B, T, D, device="cuda", generator=g).to(dtype)
    l = torch.log1p(-torch.tensor([0.5, 0.1, 0.02, 0.001], device="cuda"))
    f = rotary_frequencies(D // H)
    n = torch.tensor([T, T // 2, 1], device="cuda", dtype=torch.int32)
    positions = (100 + torch.arange(T, device="cuda")).expand(B, T)
    y, state = _layer(x, W, l, f, n, positions, 0.25, 7)
    dx, dW = torch.autograd.grad((y, state), (x, W), (d_y, torch.ones_like(state)))
    x64, W64 = (t.detach().double().requires_grad_() for t in (x, W))
    y64, s64 = _layer_in_64_bits(x64, W64, l, f, n, positions, 0.25, 7)
    want = torch.autograd.grad((y64, s64), (x64, W64), (d_y.double(), torch.ones_like(s64)))
    # Between the input and any output lie at most eight roundings to the tensors' type (the projection, the turn, the scores,
    # the attention's output, the sum; in the gradient the attention's, the turn's and the projection's again), each at most
    # half a step of values whose norms, for random signs, do not exceed four times the result's; in fp32 the sums of up to
    # 3 D terms (768 roundings) come on top.
    u = ref.U[dtype]
    room = 8 * 4 * u + (768 * 4 * 2.0 ** -23 if dtype is torch.float32 else 0.0)
    got = dict(y=_far(y.detach(), y64.detach()), state=_far(state.detach(), s64.detach()), dx=_far(dx, want[0]), dW=_far(dW, want[1]))
    achieved(f"layer {str(dtype)[6:]} T={T}", **got)
    assert max(got.values()) <= room, got


def test_serving_continues_a_prompt():
    """A prompt in one call, then token after token from its state, all in one captured graph: as one long sequence."""
    B, H, d, T, more = 2, 3, 64, 50, 4
    g = torch.Generator(device="cuda").manual_seed(2)
    q, k, v = (torch.randn(B, T + more, H, d, device="cuda", generator=g).to(torch.bfloat16) for _ in range(3))
    l = torch.tensor([-0.5, -0.05, -0.001], device="cuda")
    f = rotary_frequencies(d, 1e6, "ramp", 4.0, trained_length=4096)
    start = torch.tensor([[100], [70000]], device="cuda")
    qr, kr = rotary(q[:, :T], k[:, :T], f, start + torch.arange(T, device="cuda"))
    head, state = linear_attention(qr, kr, v[:, :T], l)
    tq, tk, tv = (x[:, T].clone() for x in (q, k, v))
    pos = start + T

    def token():
        a, b = rotary(tq[:, None], tk[:, None], f, pos)
        return linear_attention_step(a[:, 0], b[:, 0], tv, state, l)

    held = state.clone()
    token()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = token()
    state.copy_(held)
    tail = []
    for i in range(more):
        for a, b in zip((tq, tk, tv), (q, k, v)):
            a.copy_(b[:, T + i])
        pos.copy_(start + T + i)
        graph.replay()
        tail.append(out.clone())
    both = torch.cat((head, torch.stack(tail, dim=1)), dim=1)
    positions = start + torch.arange(T + more, device="cuda")
    a, b = rotary(q, k, f, positions)
    want, want_s = ref.attend(a, b, v, l, d ** -0.5)
    top, top_s = ref.attend(*(x.double().abs() for x in (a, b, v)), l, d ** -0.5)
    # (the turned tensors are the same bits either way)
    fo, fs = ref.attend_bounds(torch.bfloat16, T + more, d, True)
    u = ref.U[torch.bfloat16]
    assert ref.worst(both, want, (fo + u * (1 + fo)) * top) <= 1.0 and ref.worst(state, want_s, fs * top_s) <= 1.0
