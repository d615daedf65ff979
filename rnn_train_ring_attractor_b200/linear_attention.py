"""Linear attention with a decay for each head: whole sequences (training, prompts) and single tokens (serving).

    S_t = g_h S_{t-1} + k_t v_t^T          out_t = scale * S_t^T q_t          g_h = exp(log_decay[h])

The linear form of the ring recurrence (cpp/ring_rnn_cuda.py:18-52): a state that leaks by a fixed factor each step, is added
to, and is read out linearly.  With rotary queries and keys (``rotary``) the state also turns by a fixed angle each step.  The
reference has no counterpart; its comparison models are gated recurrent and softmax-attention networks (train/train_gru.py,
train/train_causal_transformer.py).
"""
import torch
from torch._C import _cuda_getCurrentRawStream as raw_stream
from torch.autograd import Function, forward_ad
from torch.autograd.function import once_differentiable

from . import _lib
from .ring_rnn_cuda import on_device

DTYPES = {torch.float32: 0, torch.bfloat16: 1, torch.float16: 2}
MAX_WIDTH = 256


def last_contiguous(t):
    return t if t.is_contiguous() or t.stride(-1) == 1 or t.shape[-1] == 1 else t.contiguous()


def new(dev, dtype, a, b, c, d):
    """torch.empty(a, b, c, d), in two thirds of the time."""
    c_step = d or 1
    b_step = (c or 1) * c_step
    return torch.empty_strided((a, b, c, d), ((b or 1) * b_step, b_step, c_step, 1), device=dev, dtype=dtype)


def refuse_tangents(name, *tensors):
    """The kernels compute no forward-mode derivatives, and an output without a tangent would count as a constant."""
    if forward_ad._current_level >= 0 and any(t is not None and forward_ad.unpack_dual(t).tangent is not None for t in tensors):
        raise RuntimeError(f"{name} has no forward-mode derivative (an argument carries a tangent)")


def _check(name, t, shape, device, dtype):
    if t.is_cuda and t.device == device and t.dtype == dtype and t.shape == shape:
        return
    if not t.is_cuda:
        raise RuntimeError(f"{name} must be a CUDA tensor (the operator has no CPU path)")
    if t.device != device:
        raise RuntimeError(f"{name} must be on {device}, like q")
    if t.dtype != dtype:
        raise RuntimeError(f"{name} must be {str(dtype).replace('torch.', '')}")
    raise RuntimeError(f"{name} must have shape {tuple(shape)}")


def _check_state(name, t, shape, device):
    _check(name, t, shape, device, torch.float32)
    if not t.is_contiguous():
        raise RuntimeError(f"{name} must be contiguous")


def _check_qkv(q, k, v, log_decay, dims, widest):
    shape, dev, dtype = q.shape, q.device, q.dtype
    if (dtype in DTYPES and len(shape) == dims and v.dim() == dims and k.shape == shape and v.shape[:-1] == shape[:-1]
            and k.dtype is dtype and v.dtype is dtype and q.is_cuda and k.device == dev and v.device == dev
            and log_decay.dtype is torch.float32 and log_decay.device == dev and log_decay.shape == shape[-2:-1]
            and 1 <= shape[-1] <= widest and 1 <= v.shape[-1] <= max(widest, MAX_WIDTH) and not log_decay.requires_grad):
        return shape[:-1], shape[-1], v.shape[-1]
    # one of them is wrong: which
    if q.dtype not in DTYPES:
        raise RuntimeError("q must be float32, bfloat16 or float16")
    if q.dim() != dims or k.dim() != dims or v.dim() != dims:
        raise RuntimeError(f"q, k and v must have {dims} dimensions")
    lead, dk, dv, dev = q.shape[:-1], q.shape[-1], v.shape[-1], q.device
    _check("q", q, q.shape, dev, q.dtype)
    _check("k", k, q.shape, dev, q.dtype)
    _check("v", v, (*lead, dv), dev, q.dtype)
    if not 1 <= dk <= widest or not 1 <= dv <= max(widest, MAX_WIDTH):
        raise RuntimeError(f"head widths must be between 1 and {widest}")
    _check("log_decay", log_decay, (lead[-1],), dev, torch.float32)
    if log_decay.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("log_decay has no gradient: the decays are constants of the layer (pass log_decay.detach())")
    return lead, dk, dv


def _problem(q, k, v, log_decay, scale, lengths, initial_state):
    B, T, H, dk = q.shape
    qb, qt, qh, _ = q.stride()
    kb, kt, kh, _ = k.stride()
    vb, vt, vh, _ = v.stride()
    return _lib.LINEAR_ATTENTION.pack(B, T, H, dk, v.shape[3], DTYPES[q.dtype], scale, q.data_ptr(), qb, qt, qh, k.data_ptr(), kb,
                                      kt, kh, v.data_ptr(), vb, vt, vh, log_decay.data_ptr(),
                                      0 if lengths is None else lengths.data_ptr(),
                                      0 if initial_state is None else initial_state.data_ptr())


def _workspace(n, dev):
    """(tensor that owns n bytes, its address)"""
    if n == 0:
        return None, None
    if n == _lib.INVALID_BYTES:
        raise RuntimeError("linear_attention: batch, tokens or heads too large")
    ws = torch.empty(n, dtype=torch.uint8, device=dev)
    return ws, ws.data_ptr()


def _forward(q, k, v, log_decay, scale, lengths, initial_state):
    B, T, H, dk = q.shape
    dv, dev = v.shape[3], q.device
    out = new(dev, q.dtype, B, T, H, dv)
    final = new(dev, torch.float32, B, H, dk, dv)
    if out.numel() == 0:  # no tokens or no sequences: the state is what it was
        return out, final.copy_(initial_state) if initial_state is not None else final.zero_()
    L = _lib.lib()
    p = _problem(q, k, v, log_decay, scale, lengths, initial_state)
    with on_device(dev):
        n = L.ringrnn_linear_attention_bytes(p, None)
        ws, at = _workspace(n, dev)
        rc = L.ringrnn_linear_attention_fwd(p, out.data_ptr(), final.data_ptr(), at, n, raw_stream(dev.index))
        if rc:
            _lib.check(rc)
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
        refuse_tangents("the gradient of linear_attention", d_out, d_final)
        q, k, v, initial_state, log_decay, lengths = ctx.saved_tensors
        if d_out is None and d_final is None:
            return (None,) * 7
        dev = q.device
        d_out = torch.zeros_like(v) if d_out is None else last_contiguous(d_out)
        if d_final is not None:
            d_final = d_final.contiguous()
        # (all three come from one launch; what nobody asked for is dropped)
        B, T, H, width = q.shape
        dq, dk, dv = (new(dev, q.dtype, B, T, H, n) for n in (width, width, v.shape[3]))
        d_initial = torch.empty_like(initial_state) if ctx.needs_input_grad[3] else None
        if dv.numel() == 0:
            if d_initial is not None:
                d_initial = d_initial.zero_() if d_final is None else d_initial.copy_(d_final)
            return dq, dk, dv, d_initial, None, None, None
        L = _lib.lib()
        p = _problem(q, k, v, log_decay, ctx.scale, lengths, initial_state)
        g = _lib.STRIDED.pack(d_out.data_ptr(), *d_out.stride()[:3])
        with on_device(dev):
            n = L.ringrnn_linear_attention_bytes(p, g)
            ws, at = _workspace(n, dev)
            rc = L.ringrnn_linear_attention_bwd(p, g, None if d_final is None else d_final.data_ptr(), dq.data_ptr(),
                                                dk.data_ptr(), dv.data_ptr(), None if d_initial is None else d_initial.data_ptr(),
                                                at, n, raw_stream(dev.index))
            if rc:
                _lib.check(rc)
        need = ctx.needs_input_grad
        return (dq if need[0] else None, dk if need[1] else None, dv if need[2] else None, d_initial, None, None, None)


def linear_attention(q, k, v, log_decay, scale=None, initial_state=None, lengths=None):
    """(out [B,T,H,dv] in q's type, final_state [B,H,dk,dv] fp32) of whole sequences.

    ``q``, ``k`` [B,T,H,dk], ``v`` [B,T,H,dv]: float32, bfloat16 or float16, widths up to 256; any strides (heads that share a
    tensor may be given with ``expand``).  ``log_decay`` [H] fp32, <= 0 (what is above is not checked
    and not supported): the logarithm of the factor by which a head's state shrinks each step (``log(1 - alpha)`` for a leak of
    alpha); it has no gradient.  ``scale`` defaults to ``dk ** -0.5``.
    ``initial_state`` [B,H,dk,dv] fp32, or None for zero: pass the final state of one call to continue with the next.
    ``lengths`` [B] int32: sequences end after that many tokens (0 to T); outputs beyond are zero, and what q, k and v hold
    there has no influence.  A NaN or an infinity inside a sequence reaches, beside what follows it, up to 127 tokens before it
    (31 where the arithmetic is fp32), and in the gradients of k and v as many behind it; no other sequence or head.

    Sums and states are fp32.  bfloat16 and float16 of widths up to 128 are multiplied on tensor cores (but for batches of few
    sequences of up to 32 tokens, which are faster in fp32; the same sequence may so have other last bits in a larger batch):
    products of q and k, and the state where it goes into outputs, are rounded to that type (float16: multiplied by a power of
    two of each 128 tokens first), what is added to the state keeps 22 bits or more (float16: or 2^-38 of the largest of 128
    tokens).  Everything else is multiplied in fp32, products to 2^-21 of themselves or better; an infinity among the inputs may
    come out as NaN.
    Gradients: q, k, v and initial_state, from those of out and final_state.  Forward-mode derivatives are refused.
    """
    refuse_tangents("linear_attention", q, k, v, log_decay, initial_state)
    lead, dk, dv = _check_qkv(q, k, v, log_decay, 4, MAX_WIDTH)
    B, _, H = lead
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
    that require a gradient while gradients are recorded, or carry a forward-mode tangent."""
    refuse_tangents("linear_attention_step", q, k, v, state, log_decay)
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
    out = torch.empty_strided((B, H, dv), (H * dv, dv, 1), device=dev, dtype=q.dtype)
    if out.numel() == 0:
        return out
    (qb, qh, _), (kb, kh, _), (vb, vh, _) = q.stride(), k.stride(), v.stride()
    p = _lib.LINEAR_ATTENTION.pack(B, 1, H, dk, dv, DTYPES[q.dtype], dk ** -0.5 if scale is None else float(scale), q.data_ptr(),
                                   qb, 0, qh, k.data_ptr(), kb, 0, kh, v.data_ptr(), vb, 0, vh, log_decay.data_ptr(), 0, 0)
    with on_device(dev):
        rc = _lib.lib().ringrnn_linear_attention_step(p, state.data_ptr(), None if active is None else active.data_ptr(),
                                                      out.data_ptr(), raw_stream(dev.index))
        if rc:
            _lib.check(rc)
    if not state.is_inference():
        torch.autograd.graph.increment_version(state)  # an in-place update that torch has to know of
    return out
