"""How far a NaN or an infinity inside a sequence reaches: its own sequence and head, what follows it, and what shares its chunk."""
import pytest
import torch

from rnn_train_ring_attractor_b200.linear_attention import linear_attention

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,chunk,B,T,H,d", [(torch.bfloat16, 128, 2, 700, 3, 64), (torch.float16, 128, 2, 700, 3, 64), (torch.float32, 32, 2, 300, 3, 64),
                                                 (torch.bfloat16, 128, 10, 400, 17, 128), (torch.float16, 128, 10, 400, 17, 64),
                                                 (torch.bfloat16, 128, 1, 5003, 2, 64)])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
@pytest.mark.parametrize("where", ["q", "k", "v", "d_out"])
def test_reach(dtype, chunk, B, T, H, d, bad, where):
    g = torch.Generator(device="cuda").manual_seed(7)
    x = {n: torch.randn(B, T, H, d, device="cuda", generator=g).to(dtype) for n in ("q", "k", "v", "d_out")}
    l = torch.full((H,), -0.02, device="cuda")

    def run():
        leaves = [x[n].detach().requires_grad_() for n in ("q", "k", "v")]
        out, final = linear_attention(*leaves, l, scale=0.1)
        return (out.detach(), final.detach(), *torch.autograd.grad(out, leaves, x["d_out"]))

    clean = run()
    b, t, h = B - 1, T // 2 + 3, 1
    x[where][b, t, h, 5] = bad
    got = run()
    for i, (a, c) in enumerate(zip(got, clean)):
        same = (a == c)
        (same[b, h] if i == 1 else same[b, :, h]).fill_(True)  # the one sequence and head
        assert bool(same.all()), i
    before, after = slice(0, t - chunk + 1), slice(t + chunk, None)
    # outputs and queries' gradients go forward in time, the others backward
    for i in (0, 2):
        assert torch.equal(got[i][b, before, h], clean[i][b, before, h]), i
    for i in (3, 4):
        assert torch.equal(got[i][b, after, h], clean[i][b, after, h]), i
