"""Which long sequences are cut into segments: by the problem's own type, with operands that need no copy."""
import ctypes as C

import pytest

from rnn_train_ring_attractor_b200 import _lib
from rnn_train_ring_attractor_b200.build import build


@pytest.fixture(scope="module")
def L():
    build()
    return _lib.lib()


@pytest.mark.parametrize("dtype,B,T,H,dk,dv", [(0, 1, 2500, 1, 40, 24), (1, 1, 5003, 1, 128, 64), (1, 2, 4100, 1, 64, 128), (1, 1, 2600, 3, 20, 33),
                                               (2, 1, 3000, 1, 200, 64), (2, 1, 5003, 1, 64, 128), (1, 1, 30011, 8, 128, 128),
                                               (1, 1, 20003, 20, 64, 64)])
@pytest.mark.parametrize("backward", [False, True])
def test_long_sequences_of_few_heads_are_cut(L, dtype, B, T, H, dk, dv, backward):
    """The workspace is sums of segments then, two at least for each sequence and head; gradients have two sets."""
    def operand(width):
        row = (width + 7) // 8 * 8
        return _lib.Strided(1 << 20, T * H * row, H * row, row)
    p = _lib.LinearAttention(B, T, H, dk, dv, dtype, 1.0, operand(dk), operand(dk), operand(dv), 1 << 20, None, None)
    n = L.ringrnn_linear_attention_bytes(C.byref(p), C.byref(operand(dv)) if backward else None)
    sums = B * H * dk * dv * 4
    assert n != _lib.INVALID_BYTES and n >= (2 if backward else 1) * 2 * sums
    p.T = 32  # one chunk, of whichever kernel
    assert L.ringrnn_linear_attention_bytes(C.byref(p), None) == 0
