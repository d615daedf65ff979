"""Rows behind the last token of a sequence that is far shorter than its tensor."""
import ctypes as C

import pytest
import torch

from rnn_train_ring_attractor_b200 import _lib

pytestmark = pytest.mark.gpu


def test_more_zeros_than_31_bits_count():
    """2^25 and more tokens of padding, 150 sequences that nobody cuts, and one output of 10 GB (the inputs are one token, shared by all)."""
    T, H, dk, n = (1 << 25) + 64, 150, 129, 3
    g = torch.Generator(device="cuda").manual_seed(1)
    q, k = (torch.randn(dk, device="cuda", generator=g).to(torch.bfloat16) for _ in range(2))
    v = torch.randn(1, device="cuda", generator=g).to(torch.bfloat16)
    l = torch.full((H,), -0.5, device="cuda")
    lengths = torch.tensor([n], device="cuda", dtype=torch.int32)
    shared = lambda t: _lib.Strided(t.data_ptr(), 0, 0, 0)  # noqa: E731
    p = _lib.LinearAttention(1, T, H, dk, 1, 1, 1.0, shared(q), shared(k), shared(v), l.data_ptr(), lengths.data_ptr(), None)
    assert _lib.lib().ringrnn_linear_attention_bytes(C.byref(p), None) == 0  # one segment each
    out = torch.full((T, H), 7.0, device="cuda", dtype=torch.bfloat16)
    assert _lib.lib().ringrnn_linear_attention_fwd(C.byref(p), out.data_ptr(), None, None, 0, None) == 0
    torch.cuda.synchronize()
    for rows in out[n:].split(1 << 22):
        assert not rows.any()
    score = float((q.double() * k.double()).sum()) * float(v)
    want = torch.tensor([score * sum(2.718281828459045 ** (-0.5 * i) for i in range(t + 1)) for t in range(n)], device="cuda")
    # one rounding to bf16; the sums of 129 products in fp32 arithmetic
    room = 2.0 ** -8 * want.abs() + 256 * 2.0 ** -23 * float((q.double() * k.double()).abs().sum()) * abs(float(v)) * 3
    assert bool(((out[:n].double() - want[:, None]).abs() <= room[:, None]).all())
