"""Positions, seeds and rows are integers of at most 64 bits: nothing is cut off to make them so."""
import numpy as np
import pytest
import torch

from rnn_train_ring_attractor_b200.dropout import dropout
from rnn_train_ring_attractor_b200.rotary import rotary, rotary_frequencies

pytestmark = pytest.mark.gpu


def test_positions():
    q, f = torch.randn(1, 3, 2, 8, device="cuda"), rotary_frequencies(8)
    assert torch.equal(rotary(q, None, f, np.int64(7))[0], rotary(q, None, f, 7)[0])
    rotary(q, None, f, -(1 << 63))
    for bad in (2.5, 7.0, "7", None):
        with pytest.raises(RuntimeError, match="positions must be an integer"):
            rotary(q, None, f, bad)
    for bad in (1 << 63, -(1 << 63) - 1):
        with pytest.raises(ValueError, match="64 bits"):
            rotary(q, None, f, bad)


def test_seeds_streams_and_rows():
    x = torch.randn(4, 8, device="cuda")
    assert torch.equal(dropout(x, 0.5, np.int64(3), stream=np.uint32(2), first_row=np.int32(1)), dropout(x, 0.5, 3, stream=2, first_row=1))
    for bad in (dict(seed=1.5), dict(stream=0.5), dict(first_row=2.0)):
        with pytest.raises(TypeError):
            dropout(**{**dict(x=x, p=0.5, seed=1), **bad})
