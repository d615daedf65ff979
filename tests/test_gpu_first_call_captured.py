"""The first call a process makes of an operator may be one that is captured."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))

PROGRAM = """
import torch
from rnn_train_ring_attractor_b200.dropout import dropout
from rnn_train_ring_attractor_b200.linear_attention import linear_attention, linear_attention_step
from rnn_train_ring_attractor_b200.rotary import rotary, rotary_frequencies

g = torch.Generator(device="cuda").manual_seed(1)
q, k, v, d = (torch.randn(2, 200, 3, 64, device="cuda", generator=g).to(torch.bfloat16) for _ in range(4))
l, f, numbers = torch.full((3,), -0.1, device="cuda"), rotary_frequencies(64), torch.tensor([5, 6], device="cuda")
q.requires_grad_()


def work():
    a, b = rotary(q, k, f, 3)
    out, state = linear_attention(a, b, v, l)
    y = dropout(out, 0.5, numbers)
    grad, = torch.autograd.grad(y, q, d)
    with torch.no_grad():
        step = linear_attention_step(q[:, 0], k[:, 0], v[:, 0], state, l)
    return y.detach(), grad, state.detach(), step


torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    held = work()
graph.replay()
torch.cuda.synchronize()
for a, b in zip(held, work()):
    assert torch.equal(a, b)
print("same")
"""


def test_without_a_call_before():
    got = subprocess.run([sys.executable, "-c", PROGRAM], capture_output=True, text=True, timeout=300, cwd=ROOT)
    assert got.returncode == 0 and "same" in got.stdout, got.stderr[-2000:]
