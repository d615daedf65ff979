"""Linear attention with a decay for each head: whole sequences (training, prompts) and single tokens (serving).

    S_t = g_h S_{t-1} + k_t v_t^T          out_t = scale * S_t^T q_t          g_h = exp(log_decay[h])

The linear form of the ring recurrence (cpp/ring_rnn_cuda.py:18-52): a state that leaks by a fixed factor each step, is added
to, and is read out linearly.  With rotary queries and keys (``rotary``) the state also turns by a fixed angle each step.  The
reference has no counterpart; its comparison models are gated recurrent and softmax-attention networks (train/train_gru.py,
train/train_causal_transformer.py).
"""
import ctypes as C

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib
from .ring_rnn_cuda import _scratch, nvtx_range, on_device, stream_of

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_WIDTH = 256


def strided(t):
    """RingRnnStrided of a [B, T, H, d] tensor whose last dimension is contiguous."""
    b, n, h = t.stride()[:3]
    return _lib.Strided(t.data_ptr(), b, n, h)


def last_contiguous(t):
    return t if t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def _check(name, t, shape, device, dtype):
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor (the operator has no CPU path)")
    if t.device != device:
        raise RuntimeError(f"{name} must be on {device}, like q")
    if t.dtype != dtype:
        raise RuntimeError(f"{name} must be {str(dtype).replace('torch.', '')}")
    if tuple(t.shape) != shape:
        raise RuntimeError(f"{name} must have shape {shape}")


def _check_state(name, t, shape, device):
    _check(name, t, shape, device, torch.float32)
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")


def _check_qkv(q, k, v, log_decay, dims, widest):
    if q.dtype not in DTYPES:
        raise RuntimeError("q must be float32, bfloat16 or float16")
    if q.dim() != dims or k.dim() != dims or v.dim() != dims:
        raise RuntimeError(f"q, k and v must have {dims} dimensions")
    lead, dk, dv = tuple(q.shape[:-1]), q.shape[-1], v.shape[-1]
    _check("q", q, lead + (dk,), q.device, q.dtype)
    _check("k", k, lead + (dk,), q.device, q.dtype)
    _check("v", v, lead + (dv,), q.device, q.dtype)
    if not 1 <= dk <= widest or not 1 <= dv <= max(widest, MAX_WIDTH):
        raise RuntimeError(f"head widths must be between 1 and {widest}")
    _check("log_decay", log_decay, (lead[-1],), q.device, torch.float32)
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("log_decay has no gradient: the decays are constants of the layer (pass log_decay.detach())")
    return lead, dk, dv


def _problem(q, k, v, log_decay, scale, lengths, initial_state):
    B, T, H, dk = q.shape
    p = _lib.LinearAttention(B, T, H, dk, v.shape[-1], DTYPES[q.dtype], scale, strided(q), strided(k), strided(v),
                             log_decay.data_ptr())
    if lengths is not None:
        p.lengths = lengths.data_ptr()
    if initial_state is not None:
        p.initial_state = initial_state.data_ptr()
    return p


def _forward(q, k, v, log_decay, scale, lengths, initial_state):
    B, T, H, dk = q.shape
    dv, dev = v.shape[-1], q.device
    out = torch.empty(B, T, H, dv, device=dev, dtype=q.dtype)
    final = torch.empty(B, H, dk, dv, device=dev, dtype=torch.float32)
    if out.numel() == 0:  # no tokens or no sequences: the state is what it was
        return out, final.copy_(initial_state) if initial_state is not None else final.zero_()
    L = _lib.lib()
    with on_device(dev), nvtx_range("ringrnn_linear_attention_fwd"):
        p = _problem(q, k, v, log_decay, scale, lengths, initial_state)
        n = L.ringrnn_linear_attention_bytes(C.byref(p), None)
        if n == _lib.INVALID_BYTES:
            raise RuntimeError("linear_attention: batch, tokens or heads too large")
        ws = _scratch(n, dev)
        _lib.check(L.ringrnn_linear_attention_fwd(C.byref(p), out.data_ptr(), final.data_ptr(), ws.data_ptr(), n, stream_of(dev)))
    return out, final


class LinearAttentionFunc(Function):
    """apply(q, k, v, initial_state, log_decay, scale, lengths) -> (out, final_state)"""

    @staticmethod
    def forward(ctx, q, k, v, initial_state, log_decay, scale, lengths):
        ctx.save_for_backward(q, k, v, initial_state, log_decay, lengths)
        ctx.scale = scale
        ctx.set_materialize_grads(False)
        return _forward(q, k, v, log_decay, scale, lengths, initial_state)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_out, d_final):
        q, k, v, initial_state, log_decay, lengths = ctx.saved_tensors
        if d_out is None and d_final is None:
            return (None,) * 7
        dev = q.device
        d_out = torch.zeros_like(v) if d_out is None else last_contiguous(d_out)
        if d_final is not None:
            d_final = d_final.contiguous()
        # (all three come from one launch; what nobody asked for is dropped)
        dq, dk, dv = (torch.empty(t.shape, device=dev, dtype=t.dtype) for t in (q, k, v))
        d_initial = torch.empty(initial_state.shape, device=dev, dtype=torch.float32) if ctx.needs_input_grad[3] else None
        if dv.numel() == 0:
            if d_initial is not None:
                d_initial = d_initial.zero_() if d_final is None else d_initial.copy_(d_final)
            return dq, dk, dv, d_initial, None, None, None
        L = _lib.lib()
        with on_device(dev), nvtx_range("ringrnn_linear_attention_bwd"):
            p = _problem(q, k, v, log_decay, ctx.scale, lengths, initial_state)
            g = strided(d_out)
            n = L.ringrnn_linear_attention_bytes(C.byref(p), C.byref(g))
            ws = _scratch(n, dev)
            _lib.check(L.ringrnn_linear_attention_bwd(
                C.byref(p), C.byref(g), None if d_final is None else d_final.data_ptr(), dq.data_ptr(), dk.data_ptr(),
                dv.data_ptr(), None if d_initial is None else d_initial.data_ptr(), ws.data_ptr(), n, stream_of(dev)))
        need = ctx.needs_input_grad
        return (dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, d_initial, None, None, None)


def linear_attention(q, k, v, log_decay, scale=None, initial_state=None, lengths=None):
    """(out [B,T,H,dv] in q's type, final_state [B,H,dk,dv] fp32) of whole sequences.

    ``q``, ``k`` [B,T,H,dk], ``v`` [B,T,H,dv]: float32, bfloat16 or float16, widths up to 256; any strides (heads that share a
    tensor may be given with ``expand``).  ``log_decay`` [H] fp32, <= 0: the logarithm of the factor by which a head's state
    shrinks each step (``log(1 - alpha)`` for a leak of alpha); it has no gradient.  ``scale`` defaults to ``dk ** -0.5``.
    ``initial_state`` [B,H,dk,dv] fp32, or None for zero: pass the final state of one call to continue with the next.
    ``lengths`` [B] int32: sequences end after that many tokens (0 to T); outputs beyond are zero, and what q, k and v hold
    there has no influence.  A NaN or an infinity inside a sequence may reach up to 127 tokens before it.

    Sums and states are fp32.  float32 and float16 inputs are multiplied in fp32; bfloat16 ones of widths up to 128 on tensor
    cores, the state to sixteen bits and the scores of pairs rounded to bfloat16.
    Gradients: q, k, v and initial_state, from those of out and final_state.
    """
    lead, dk, dv = _check_qkv(q, k, v, log_decay, 4, MAX_WIDTH)
    B, T, H = lead
    dev = q.device
    if initial_state is not None:
        _check_state("initial_state", initial_state, (B, H, dk, dv), dev)
    if lengths is not None:
        _check("lengths", lengths, (B,), dev, torch.int32)
        lengths = lengths.contiguous()
    log_decay = log_decay.detach().contiguous()
    scale = dk ** -0.5 if scale is None else float(scale)
    q, k, v = last_contiguous(q), last_contiguous(k), last_contiguous(v)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad
                                    or (initial_state is not None and initial_state.requires_grad)):
        return LinearAttentionFunc.apply(q, k, v, initial_state, log_decay, scale, lengths)
    return _forward(q, k, v, log_decay, scale, lengths, initial_state)


def linear_attention_step(q, k, v, state, log_decay, scale=None, active=None):
    """out [B,H,dv] of one more token for each sequence; ``state`` [B,H,dk,dv] fp32 is updated IN PLACE.

    ``q``, ``k`` [B,H,dk], ``v`` [B,H,dv], any strides; widths of keys up to 1024.  ``active`` [B] bool: sequences that are False
    keep their state and get an output of zero (the unused rows of a batch of fixed size).  For inference: refused for tensors
    that require a gradient while gradients are recorded."""
    lead, dk, dv = _check_qkv(q, k, v, log_decay, 3, 1024)
    B, H = lead
    dev = q.device
    _check_state("state", state, (B, H, dk, dv), dev)
    if torch.is_grad_enabled() and (q.requires_grad or k.requires_grad or v.requires_grad or state.requires_grad):
        raise RuntimeError("linear_attention_step has no gradient: use linear_attention, or torch.no_grad()")
    if active is not None:
        _check("active", active, (B,), dev, torch.bool)
        active = active.contiguous()
    q, k, v, log_decay = last_contiguous(q), last_contiguous(k), last_contiguous(v), log_decay.contiguous()
    out = torch.empty(B, H, dv, device=dev, dtype=q.dtype)
    if out.numel() == 0:
        return out
    with on_device(dev):
        p = _lib.LinearAttention(B, 1, H, dk, dv, DTYPES[q.dtype], dk ** -0.5 if scale is None else float(scale),
                                 _lib.Strided(q.data_ptr(), q.stride(0), 0, q.stride(1)),
                                 _lib.Strided(k.data_ptr(), k.stride(0), 0, k.stride(1)),
                                 _lib.Strided(v.data_ptr(), v.stride(0), 0, v.stride(1)), log_decay.data_ptr())
        _lib.check(_lib.lib().ringrnn_linear_attention_step(C.byref(p), state.data_ptr(),
                                                            None if active is None else active.data_ptr(), out.data_ptr(),
                                                            stream_of(dev)))
    if not state.is_inference():
        torch.autograd.graph.increment_version(state)  # an in-place update that torch has to know of
    return out
