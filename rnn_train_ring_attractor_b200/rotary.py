"""Rotary positions: pairs of a head's elements turned by an angle that grows with the token's position.

For the queries and keys of ``linear_attention`` (their products then depend on the distance of two tokens): the state of a
head turns by a fixed angle each step beside its decay, as the ring network's bump is shifted by its left and right matrices
(train/train_general_ring_no_gain.py:102-137).  The reference has no counterpart.
"""
import math
import operator

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib
from .linear_attention import DTYPES, last_contiguous, new, raw_stream, refuse_tangents
from .ring_rnn_cuda import on_device


def rotary_frequencies(dim, base=10000.0, scaling=None, factor=1.0, trained_length=None, low=1.0, high=32.0, device="cuda"):
    """[dim/2] float64: radians per position of each pair, base^(-2i/dim), slowed down for contexts longer than trained.

    ``scaling`` None: as they are.  "linear": every frequency divided by ``factor`` (positions interpolated).  "base": the base
    raised so that the slowest pair is slowed by ``factor`` and the fastest not at all.  "ramp": pairs that turn fewer than
    ``low`` times within ``trained_length`` positions divided by ``factor``, those that turn more than ``high`` times left
    alone, a linear blend between."""
    if dim <= 0 or dim % 2 != 0:
        raise ValueError("dim must be even and positive")
    if scaling not in (None, "linear", "base", "ramp"):
        raise ValueError("scaling must be None, 'linear', 'base' or 'ramp'")
    if not base > 0 or not factor > 0:
        raise ValueError("base and factor must be positive")
    if scaling == "base" and dim > 2:
        base = base * factor ** (dim / (dim - 2))
    f = base ** (-torch.arange(0, dim, 2, dtype=torch.float64) / dim)
    if scaling == "linear" or (scaling == "base" and dim == 2):
        f = f / factor
    elif scaling == "ramp":
        if trained_length is None or not high > low:
            raise ValueError("scaling 'ramp' needs trained_length, and low < high")
        keep = ((f * trained_length / (2 * math.pi) - low) / (high - low)).clamp(0.0, 1.0)
        f = f / factor * (1.0 - keep) + f * keep
    return f.to(device)


def _call(q, k, frequencies, positions, first, interleaved, amplitude, inverse):
    """positions: None or an integer tensor [B, T]."""
    B, T, Hq, D = q.shape
    dev = q.device
    q_out = new(dev, q.dtype, B, T, Hq, D)
    k_out = None if k is None else new(dev, k.dtype, *k.shape)
    if q_out.numel() == 0:
        return q_out, k_out
    if positions is None:
        where = 0, 0, 0, 0
    else:
        where = positions.data_ptr(), positions.element_size(), *positions.stride()
    p = _lib.ROTARY.pack(B, T, Hq, 0 if k is None else k.shape[2], D, 2 * frequencies.shape[0], DTYPES[q.dtype], int(interleaved),
                         int(inverse), amplitude, q.data_ptr(), *q.stride()[:3],
                         *((0, 0, 0, 0) if k is None else (k.data_ptr(), *k.stride()[:3])), frequencies.data_ptr(),
                         *where, first, q_out.data_ptr(), 0 if k is None else k_out.data_ptr())
    with on_device(dev):
        rc = _lib.lib().ringrnn_rotary(p, raw_stream(dev.index))
        if rc:
            _lib.check(rc)
    return q_out, k_out


class RotaryFunc(Function):
    """apply(q, k, frequencies, positions, first, interleaved, amplitude) -> (q', k')"""

    @staticmethod
    def forward(ctx, q, k, frequencies, positions, first, interleaved, amplitude):
        ctx.save_for_backward(frequencies, positions)
        ctx.args = first, interleaved, amplitude
        ctx.like = (q.shape, q.dtype, q.device), None if k is None else k.shape
        ctx.set_materialize_grads(False)
        return _call(q, k, frequencies, positions, first, interleaved, amplitude, False)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_q, d_k):
        refuse_tangents("the gradient of rotary", d_q, d_k)
        frequencies, positions = ctx.saved_tensors
        first, interleaved, amplitude = ctx.args
        got = [None, None]
        asked = [(i, last_contiguous(g)) for i, g in enumerate((d_q, d_k)) if g is not None and ctx.needs_input_grad[i]]
        if asked:
            (i, g), rest = asked[0], asked[1:]
            one, two = _call(g, rest[0][1] if rest else None, frequencies, positions, first, interleaved, amplitude, True)
            got[i] = one
            if rest:
                got[rest[0][0]] = two
        return got[0], got[1], None, None, None, None, None


def rotary(q, k, frequencies, positions=0, interleaved=False, amplitude=1.0):
    """(q', k'): the first ``2 * len(frequencies)`` elements of each head turned by position * frequency, the others copied.

    ``q`` [B,T,Hq,D] and ``k`` [B,T,Hk,D] (None: q alone, and k' is None): float32, bfloat16 or float16, any strides, numbers of
    heads of their own; one launch for both.  ``frequencies`` [R/2] float64 (``rotary_frequencies``), R <= D.  ``positions``: the
    position of the first token, or an int32 / int64 tensor [B,T] (an expanded one will do) with each token's.  Pairs are
    elements (2i, 2i+1) if ``interleaved``, else (i, i + R/2).  ``amplitude`` multiplies the turned elements.  Angles are formed
    in 64 bits, so that positions of millions are as exact as small ones.  Gradients: q and k; forward-mode derivatives are refused."""
    refuse_tangents("rotary", q, k, frequencies)
    if q.dtype not in DTYPES:
        raise RuntimeError("q must be float32, bfloat16 or float16")
    dev = q.device
    for name, t in (("q", q), ("k", k)):
        if t is None and name == "k":
            continue
        if not t.is_cuda:
            raise RuntimeError(f"{name} must be a CUDA tensor (the operator has no CPU path)")
        if t.dim() != 4 or t.dtype != q.dtype or t.device != dev or t.shape[:2] != q.shape[:2] or t.shape[3] != q.shape[3]:
            raise RuntimeError(f"{name} must be [batch, tokens, heads, width], of one type and device for q and k")
    if (frequencies.dtype != torch.float64 or frequencies.dim() != 1 or frequencies.device != dev
            or not 1 <= frequencies.shape[0] <= q.shape[3] // 2):
        raise RuntimeError("frequencies must be float64 [rotated / 2] on q's device, rotated <= width")
    if frequencies.requires_grad and torch.is_grad_enabled():
        raise RuntimeError("frequencies have no gradient: they are constants of the layer (pass frequencies.detach())")
    frequencies = frequencies.detach().contiguous()
    first = 0
    if torch.is_tensor(positions):
        if positions.dtype not in (torch.int32, torch.int64) or positions.shape != q.shape[:2] or positions.device != dev:
            raise RuntimeError("positions must be an integer, or int32 / int64 [batch, tokens] on q's device")
    else:
        try:
            first, positions = operator.index(positions), None
        except TypeError:
            raise RuntimeError("positions must be an integer, or int32 / int64 [batch, tokens] on q's device") from None
        if not -(1 << 63) <= first < 1 << 63:
            raise ValueError("positions must fit 64 bits")
    if k is not None and k.shape[2] == 0:
        raise RuntimeError("k must have a head (None: q alone)")
    if q.shape[2] == 0:
        raise RuntimeError("q must have a head")
    q = last_contiguous(q)
    k = None if k is None else last_contiguous(k)
    amplitude = float(amplitude)
    if torch.is_grad_enabled() and (q.requires_grad or (k is not None and k.requires_grad)):
        return RotaryFunc.apply(q, k, frequencies, positions, first, interleaved, amplitude)
    return _call(q, k, frequencies, positions, first, interleaved, amplitude, False)
