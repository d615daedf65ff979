"""Dropout whose mask is a function of numbers and never stored.

Element j of row r is kept or dropped by Philox4x32-10 on (seed, stream, first_row + r, j): as with ``inputs.generate_on_device``, a
row draws the same numbers in whatever batch it stands, so data-parallel ranks that pass their first row drop what one GPU with
the whole batch would, and the backward pass recomputes the mask instead of reading it.  The reference's comparison models use
torch's dropout (train/train_causal_transformer.py), which stores a mask.
"""
import operator

import torch
from torch.autograd import Function
from torch.autograd.function import once_differentiable

from . import _lib
from .linear_attention import DTYPES, raw_stream, refuse_tangents
from .ring_rnn_cuda import on_device


def _call(x, residual, p, seed, stream, first_row):
    y = torch.empty_like(x)  # (x is contiguous)
    if y.numel() == 0:
        return y
    rows = x.shape[0]
    dev = x.device
    numbers = seed if torch.is_tensor(seed) else None
    with on_device(dev):
        rc = _lib.lib().ringrnn_dropout(
            DTYPES[x.dtype], rows, x.numel() // rows, x.data_ptr(), None if residual is None else residual.data_ptr(),
            y.data_ptr(), p, 0 if numbers is not None else seed, stream, None if numbers is None else numbers.data_ptr(),
            first_row, raw_stream(dev.index))
        if rc:
            _lib.check(rc)
    return y


class DropoutFunc(Function):
    """apply(x, residual, p, seed, stream, first_row) -> y"""

    @staticmethod
    def forward(ctx, x, residual, p, seed, stream, first_row):
        # (a seed tensor is saved, so that autograd refuses a backward after it was overwritten)
        ctx.save_for_backward(seed if torch.is_tensor(seed) else None)
        ctx.args = p, seed if not torch.is_tensor(seed) else None, stream, first_row
        return _call(x, residual, p, seed, stream, first_row)

    @staticmethod
    @once_differentiable
    def backward(ctx, d_y):
        refuse_tangents("the gradient of dropout", d_y)
        p, seed, stream, first_row = ctx.args
        seed = ctx.saved_tensors[0] if seed is None else seed
        d_x = _call(d_y.contiguous(), None, p, seed, stream, first_row) if ctx.needs_input_grad[0] else None
        return d_x, d_y if ctx.needs_input_grad[1] else None, None, None, None, None


def dropout(x, p, seed, stream=0, first_row=0, residual=None):
    """residual + dropout(x): elements of ``x`` [rows, ...] are zeroed with probability ``p`` (to 2^-32), the others divided by
    1 - p; ``residual`` (same shape and type, or None) is added before the one rounding.

    ``seed``: an integer of 64 bits; ``stream`` (32 bits) tells apart what shares a seed, such as layers and steps.  Or ``seed`` is
    an int64 tensor [2] = (seed, stream) on the device, read when the kernel runs: a captured graph draws new numbers each time
    it is replayed if the tensor is advanced between.  ``first_row``: number of x's first row in the whole batch.  p = 1 drops
    everything.  What is dropped has no influence, infinities and NaN included.  float32, bfloat16 or float16, contiguous.
    Gradients: x and residual; forward-mode derivatives are refused."""
    refuse_tangents("dropout", x, residual)
    if x.dtype not in DTYPES:
        raise RuntimeError("x must be float32, bfloat16 or float16")
    if x.dim() < 1:
        raise RuntimeError("x must have a dimension of rows")
    for name, t in (("x", x), ("residual", residual)):
        if t is None:
            continue
        if not t.is_cuda:
            raise RuntimeError(f"{name} must be a CUDA tensor (the operator has no CPU path)")
        if t.shape != x.shape or t.dtype != x.dtype or t.device != x.device:
            raise RuntimeError("residual must have x's shape, type and device")
        if not t.is_contiguous():
            raise RuntimeError(f"{name} must be contiguous")
    p = float(p)
    if not 0.0 <= p <= 1.0:
        raise ValueError("p must be between 0 and 1")
    if torch.is_tensor(seed):
        if seed.dtype != torch.int64 or seed.shape != (2,) or seed.device != x.device or not seed.is_contiguous():
            raise RuntimeError("seed must be an integer, or a contiguous int64 tensor [2] (seed, stream) on x's device")
        if stream != 0:
            raise ValueError("stream is the second number of a seed tensor")
    else:
        seed = operator.index(seed)
        if not -(1 << 63) <= seed < 1 << 64:
            raise ValueError("seed must fit 64 bits")
        seed &= (1 << 64) - 1
    stream, first_row = operator.index(stream), operator.index(first_row)
    if not 0 <= stream < 1 << 32 or not 0 <= first_row < 1 << 63:
        raise ValueError("stream must fit 32 bits, first_row 63, and neither may be negative")
    if torch.is_grad_enabled() and (x.requires_grad or (residual is not None and residual.requires_grad)):
        return DropoutFunc.apply(x, residual, p, seed, stream, first_row)
    return _call(x, residual, p, seed, stream, first_row)
