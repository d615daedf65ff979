"""Forward-mode derivatives: the operators have none, and say so instead of giving outputs without a tangent."""
import pytest
import torch
import torch.autograd.forward_ad as forward_ad

from rnn_train_ring_attractor_b200.dropout import dropout
from rnn_train_ring_attractor_b200.linear_attention import linear_attention, linear_attention_step
from rnn_train_ring_attractor_b200.rotary import rotary

ALL = ["cpu", pytest.param("cuda", marks=pytest.mark.gpu)]


def _calls(device):
    """(function, arguments by name); every floating-point one may carry a tangent"""
    r = lambda *s, **kw: torch.randn(*s, device=device, **kw)  # noqa: E731
    q, k, v, l, s = r(1, 5, 2, 8), r(1, 5, 2, 8), r(1, 5, 2, 8), -torch.rand(2, device=device), r(1, 2, 8, 8)
    return [(linear_attention, dict(q=q, k=k, v=v, log_decay=l, initial_state=s)),
            (linear_attention_step, dict(q=q[:, 0], k=k[:, 0], v=v[:, 0], state=s, log_decay=l)),
            (rotary, dict(q=q, k=k, frequencies=torch.rand(4, device=device, dtype=torch.float64))),
            (dropout, dict(x=v, p=0.5, seed=1, residual=k))]


@pytest.mark.parametrize("device", ALL)
@pytest.mark.parametrize("recording", [True, False])
def test_a_tangent_is_refused(device, recording):
    for f, args in _calls(device):
        for name, x in args.items():
            if not torch.is_tensor(x):
                continue
            before = x.clone()
            with forward_ad.dual_level(), torch.set_grad_enabled(recording):
                dual = forward_ad.make_dual(x, torch.ones_like(x))
                with pytest.raises(RuntimeError, match="forward-mode"):
                    f(**{**args, name: dual})
            assert torch.equal(x, before)


@pytest.mark.gpu
def test_no_tangent_is_no_hindrance():
    """Inside a level, without one of the arguments in it; and backward derivatives as ever."""
    for f, args in _calls("cuda"):
        want = f(**{n: x.clone() if torch.is_tensor(x) else x for n, x in args.items()})
        with forward_ad.dual_level():
            got = f(**args)
        for a, b in zip(*((x,) if torch.is_tensor(x) else x for x in (got, want))):
            assert torch.equal(a, b)
    f, args = _calls("cuda")[0]
    q = args["q"].requires_grad_()
    with forward_ad.dual_level():
        f(**args)[0].sum().backward()
    assert q.grad is not None


@pytest.mark.gpu
def test_a_tangent_of_a_gradient_is_refused():
    """Forward mode over the backward pass: the gradients of outputs carry the tangents."""
    for f, args in _calls("cuda"):
        if f is linear_attention_step:
            continue
        name = "x" if "x" in args else "q"
        x = args[name].requires_grad_()
        y = f(**args)
        y = y if torch.is_tensor(y) else y[0]
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(torch.ones_like(y), torch.ones_like(y))
            with pytest.raises(RuntimeError, match="forward-mode"):
                torch.autograd.grad(y, x, dual, retain_graph=True)
        assert torch.autograd.grad(y, x, torch.ones_like(y))[0].shape == x.shape
