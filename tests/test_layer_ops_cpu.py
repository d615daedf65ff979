"""Host side of the layer operators: refusals, buffer sizes, frequencies, and the tests' own definitions against each other."""
import ctypes as C
import math

import pytest
import torch

import layer_reference as ref
from rnn_train_ring_attractor_b200 import _lib
from rnn_train_ring_attractor_b200.build import build
from rnn_train_ring_attractor_b200.dropout import dropout
from rnn_train_ring_attractor_b200.linear_attention import linear_attention, linear_attention_step
from rnn_train_ring_attractor_b200.rotary import rotary, rotary_frequencies


@pytest.fixture(scope="module")
def L():
    build()
    return _lib.lib()


def _linear(**kw):
    d = dict(B=2, T=40, H=3, dk=16, dv=24, dtype=1, scale=1.0)
    d.update({n: kw.pop(n) for n in list(kw) if n in d})
    s = [_lib.Strided(1 << 20, 4000, 100, 30) for _ in range(3)]
    p = _lib.LinearAttention(d["B"], d["T"], d["H"], d["dk"], d["dv"], d["dtype"], d["scale"], *s, 1 << 20, None, None)
    for n, x in kw.items():
        if n in "qkv":
            getattr(p, n).data = x
        else:
            setattr(p, n, x)
    return p


@pytest.mark.parametrize("bad,status", [(dict(B=0), 2), (dict(T=0), 2), (dict(H=-1), 2), (dict(dk=0), 2), (dict(dk=257), 2),
                                        (dict(dv=257), 2), (dict(dtype=3), 1), (dict(q=None), 1), (dict(k=None), 1),
                                        (dict(v=None), 1), (dict(log_decay=None), 1)])
def test_linear_attention_refuses_before_any_launch(L, bad, status):
    p = _linear(**bad)
    big = 1 << 40
    assert L.ringrnn_linear_attention_fwd(C.byref(p), 256, None, 256, big, None) == status
    g = _lib.Strided(1 << 20, 4000, 100, 30)
    assert L.ringrnn_linear_attention_bwd(C.byref(p), C.byref(g), None, 256, 256, 256, None, 256, big, None) == status
    if status == 2:
        assert L.ringrnn_linear_attention_bytes(C.byref(p), None) == _lib.INVALID_BYTES
    if bad not in (dict(T=0), dict(dk=257), dict(dv=257)):  # the step has no tokens and wider heads
        assert L.ringrnn_linear_attention_step(C.byref(p), 256, None, 256, None) == status


def test_linear_attention_refuses_missing_buffers(L):
    p = _linear()
    g = _lib.Strided(1 << 20, 4000, 100, 30)
    assert L.ringrnn_linear_attention_fwd(None, 256, None, None, 0, None) == 1
    assert L.ringrnn_linear_attention_fwd(C.byref(p), None, None, 256, 1 << 40, None) == 1
    assert L.ringrnn_linear_attention_bwd(C.byref(p), None, None, 256, 256, 256, None, 256, 1 << 40, None) == 1
    assert L.ringrnn_linear_attention_bwd(C.byref(p), C.byref(g), None, None, 256, 256, None, 256, 1 << 40, None) == 1
    assert L.ringrnn_linear_attention_step(C.byref(p), None, None, 256, None) == 1
    p = _linear(dk=1025)
    assert L.ringrnn_linear_attention_step(C.byref(p), 256, None, 256, None) == 2
    long = _linear(B=1, T=100000, H=1, dk=128, dv=128)  # one head: cut into segments, which needs room for their sums
    for backward in (None, C.byref(g)):
        n = L.ringrnn_linear_attention_bytes(C.byref(long), backward)
        assert 0 < n < 1 << 30
    n = L.ringrnn_linear_attention_bytes(C.byref(long), None)
    assert L.ringrnn_linear_attention_fwd(C.byref(long), 256, None, None, n, None) == 3
    assert L.ringrnn_linear_attention_fwd(C.byref(long), 256, None, 256, n - 1, None) == 3
    assert L.ringrnn_linear_attention_fwd(C.byref(long), 256, None, 257, n, None) == 3


def test_rotary_and_dropout_refuse_before_any_launch(L):
    def call(**kw):
        p = _lib.Rotary(2, 3, 4, 2, 16, 8, 1, 0, 0, 1.0, _lib.Strided(256, 1, 1, 1), _lib.Strided(256, 1, 1, 1), 256, None, 0, 0, 0, 0,
                        256, 256)
        for n, x in kw.items():
            if n in ("q", "k"):
                getattr(p, n).data = x
            else:
                setattr(p, n, x)
        return L.ringrnn_rotary(C.byref(p), None)
    assert L.ringrnn_rotary(None, None) == 1
    for bad in (dict(B=0), dict(T=0), dict(Hq=0), dict(Hk=0), dict(D=0), dict(rotated=0), dict(rotated=7), dict(rotated=18)):
        assert call(**bad) == 2, bad
    for bad in (dict(q=None), dict(q_out=None), dict(k_out=None), dict(frequency=None), dict(dtype=5), dict(position_bytes=2),
                dict(position_bytes=8)):
        assert call(**bad) == 1, bad

    def drop(dtype=1, rows=2, n=8, x=256, y=256, p=0.5, stream=0):
        return L.ringrnn_dropout(dtype, rows, n, x, None, y, p, 1, stream, None, 0, None)
    for bad in (dict(rows=0), dict(n=0), dict(n=(1 << 34) + 1), dict(rows=1 << 40, n=1 << 30)):
        assert drop(**bad) == 2, bad
    for bad in (dict(dtype=9), dict(x=None), dict(y=None), dict(p=-0.1), dict(p=1.1), dict(p=float("nan")), dict(stream=1 << 32)):
        assert drop(**bad) == 1, bad


def test_structures_as_bytes_are_the_structures():
    for packed, ctype in ((_lib.LINEAR_ATTENTION, _lib.LinearAttention), (_lib.STRIDED, _lib.Strided), (_lib.ROTARY, _lib.Rotary)):
        assert packed.size == C.sizeof(ctype)

    def fields(x):
        for name, _ in x._fields_:
            v = getattr(x, name)
            if isinstance(v, C.Structure):
                yield from fields(v)
            else:
                yield v
    for packed, ctype in ((_lib.LINEAR_ATTENTION, _lib.LinearAttention), (_lib.ROTARY, _lib.Rotary)):
        n = len(packed.unpack(bytes(packed.size)))
        values = list(range(1, n + 1))
        got = list(fields(ctype.from_buffer_copy(packed.pack(*values))))
        assert got == values


def test_python_surfaces_refuse_host_tensors():
    q = torch.zeros(1, 2, 1, 8)
    with pytest.raises(RuntimeError, match="CUDA"):
        linear_attention(q, q, q, torch.zeros(1))
    with pytest.raises(RuntimeError, match="CUDA"):
        linear_attention_step(q[0], q[0], q[0], torch.zeros(2, 1, 8, 8), torch.zeros(1))
    with pytest.raises(RuntimeError, match="CUDA"):
        rotary(q, None, torch.zeros(4, dtype=torch.float64))
    with pytest.raises(RuntimeError, match="CUDA"):
        dropout(torch.zeros(2, 4), 0.5, 1)
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        linear_attention(q.double(), q.double(), q.double(), torch.zeros(1))


def test_frequencies():
    kw = dict(device="cpu")
    f = rotary_frequencies(64, base=500.0, **kw)
    want = torch.tensor([500.0 ** (-2 * i / 64) for i in range(32)], dtype=torch.float64)
    assert f.dtype == torch.float64 and torch.allclose(f, want, rtol=1e-14, atol=0)
    assert torch.allclose(rotary_frequencies(64, 500.0, "linear", 4.0, **kw), want / 4, rtol=1e-14, atol=0)
    b = rotary_frequencies(64, 500.0, "base", 4.0, **kw)
    assert float(b[0]) == 1.0 and math.isclose(float(b[-1]), float(want[-1]) / 4, rel_tol=1e-12)
    r = rotary_frequencies(64, 500.0, "ramp", 4.0, trained_length=400, low=2.0, high=20.0, **kw)
    turns = want * 400 / (2 * math.pi)
    assert torch.equal(r[turns >= 20.0], f[turns >= 20.0]) and torch.allclose(r[turns <= 2.0], want[turns <= 2.0] / 4, rtol=1e-14)
    assert bool((r <= f).all()) and bool((r >= f / 4).all()) and bool((r.diff() < 0).all())
    for bad in (dict(dim=7), dict(dim=0), dict(dim=8, scaling="other"), dict(dim=8, base=-1.0), dict(dim=8, scaling="ramp"),
                dict(dim=8, scaling="ramp", trained_length=10, low=3.0, high=3.0), dict(dim=8, factor=0.0)):
        with pytest.raises(ValueError):
            rotary_frequencies(**bad, **kw)


def test_definitions_agree():
    g = torch.Generator().manual_seed(3)
    q, k = (torch.randn(2, 23, 3, 5, generator=g, dtype=torch.float64) for _ in range(2))
    v = torch.randn(2, 23, 3, 4, generator=g, dtype=torch.float64)
    s = torch.randn(2, 3, 5, 4, generator=g, dtype=torch.float64)
    l = torch.tensor([-0.01, -0.7, -40.0])
    for a, b in zip(ref.attend(q, k, v, l, 0.3, s), ref.attend_by_steps(q, k, v, l, 0.3, s)):
        assert torch.allclose(a, b, rtol=1e-12, atol=1e-12)
    # a sequence that ends after n tokens is the sequence of n tokens
    n = torch.tensor([9, 0])
    out, final = ref.attend(q, k, v, l, 0.3, s, n)
    a, b = ref.attend_by_steps(q[:1, :9], k[:1, :9], v[:1, :9], l, 0.3, s[:1])
    assert torch.allclose(out[:1, :9], a, rtol=1e-12, atol=1e-12) and torch.allclose(final[:1], b, rtol=1e-12, atol=1e-12)
    assert not out[0, 9:].any() and not out[1].any() and torch.equal(final[1], s[1])
    # known answers of the generator (Random123's test vectors for philox4x32 with ten rounds)
    assert ref.philox((0, 0, 0, 0), (0, 0)) == [0x6627E8D5, 0xE169C58D, 0xBC57AC4C, 0x9B00DBD8]
    f = 0xFFFFFFFF
    assert ref.philox((f, f, f, f), (f, f)) == [0x408F276D, 0x41C83B0E, 0xA20BC7C6, 0x6D5451FD]
