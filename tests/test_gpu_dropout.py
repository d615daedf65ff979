"""Counter-based dropout against its definition: which elements are kept is exact, their values are rounded once."""
import math

import pytest
import torch

import layer_reference as ref
from rnn_train_ring_attractor_b200.dropout import dropout

pytestmark = pytest.mark.gpu

FP32, BF16, FP16 = torch.float32, torch.bfloat16, torch.float16


def _randn(*shape, dtype, seed=0):
    return torch.randn(*shape, device="cuda", generator=torch.Generator(device="cuda").manual_seed(seed)).to(dtype)


def _want(x, kept, p, residual=None):
    y = torch.where(kept, x.double() / (1 - p) if p < 1 else 0.0, 0.0)
    return y if residual is None else y + residual.double()


def _room(x, kept, p, want):
    """1 / (1 - p), the product and the sum in fp32: three roundings of the kept value and one of the sum; then the type's."""
    top = torch.where(kept, x.double().abs() / max(1 - p, 1e-30), 0.0)
    f = 3 * 2.0 ** -24 * top + 2.0 ** -24 * want.abs()
    return f + ref.U[x.dtype] * (want.abs() + f) + ref.TINY[x.dtype]


CASES = [(FP32, 1, 1, 0.5), (BF16, 3, 8, 0.1), (FP16, 2, 37, 0.25), (BF16, 4, 100, 0.9), (FP32, 3, 130, 0.0), (BF16, 2, 64, 1.0), (BF16, 5, 7, 0.3),
         (FP32, 2, 4099, 0.37)]


@pytest.mark.parametrize("dtype,rows,n,p", CASES)
@pytest.mark.parametrize("numbers", [(0, 0, 0), (0xFEDCBA9876543210, 0xFFFFFFFF, (1 << 40) - 2)])
def test_mask_values_and_gradients(dtype, rows, n, p, numbers):
    seed, stream, first = numbers
    kept = ref.kept(rows, n, p, seed, stream, first).cuda()
    x, r, d = (_randn(rows, n, dtype=dtype, seed=i).requires_grad_() for i in range(3))
    kw = dict(stream=stream, first_row=first)
    y = dropout(x, p, seed, **kw)
    # a kept value is zero only if x is
    assert torch.equal(y != 0, kept & (x != 0))
    want = _want(x.detach(), kept, p)
    assert ref.worst(y.detach(), want, _room(x.detach(), kept, p, want)) <= 1.0
    z = dropout(x, p, seed, residual=r, **kw)
    want = _want(x.detach(), kept, p, r.detach())
    assert ref.worst(z.detach(), want, _room(x.detach(), kept, p, want)) <= 1.0
    gx, gr = torch.autograd.grad(z, (x, r), d.detach())
    want = _want(d.detach(), kept, p)
    assert ref.worst(gx, want, _room(d.detach(), kept, p, want)) <= 1.0 and torch.equal(gr, d)
    only, = torch.autograd.grad(dropout(x.detach(), p, seed, residual=r, **kw), r, d.detach())
    assert torch.equal(only, d)


@pytest.mark.parametrize("dtype", [FP32, BF16, FP16])
@pytest.mark.parametrize("rows,n", [(1, 1), (700, 1), (333, 3), (50, 7), (41, 9), (64, 31), (300, 250), (19, 1001), (7, 65537), (2, 3000006), (600, 12)])
def test_rows_of_any_length_and_offset_draw_like_whole_vectors(dtype, rows, n):
    """An element's number is its row's and its own: the same as where every row is padded to whole vectors."""
    wide = (n + 7) // 8 * 8
    x, r = _randn(rows, wide, dtype=dtype, seed=1), _randn(rows, wide, dtype=dtype, seed=2)
    numbers = torch.tensor([5, 9], device="cuda")
    want, more = dropout(x, 0.3, 5, stream=9, first_row=11)[:, :n], dropout(x, 0.3, 5, stream=9, first_row=11, residual=r)[:, :n]
    for at, at_r in ((0, 0), (1, 1), (3, 3), (1, 2), (0, 5)):
        flat, flat_r = torch.empty(rows * n + 8, device="cuda", dtype=dtype), torch.empty(rows * n + 8, device="cuda", dtype=dtype)
        y, z = flat[at:at + rows * n].view(rows, n), flat_r[at_r:at_r + rows * n].view(rows, n)
        y.copy_(x[:, :n]), z.copy_(r[:, :n])
        assert torch.equal(dropout(y, 0.3, 5, stream=9, first_row=11), want)
        assert torch.equal(dropout(y, 0.3, 5, stream=9, first_row=11, residual=z), more)
        assert torch.equal(dropout(y, 0.3, numbers, first_row=11, residual=z), more)


def test_rows_draw_the_same_in_every_batch():
    x = _randn(12, 3, 50, dtype=BF16)
    whole = dropout(x, 0.4, 77, stream=5, first_row=1000)
    for lo, hi in ((0, 5), (5, 6), (6, 12)):
        assert torch.equal(dropout(x[lo:hi].contiguous(), 0.4, 77, stream=5, first_row=1000 + lo), whole[lo:hi])
    for other in (dict(seed=78), dict(stream=6), dict(first_row=1012)):
        kw = dict(seed=77, stream=5, first_row=1000)
        kw.update(other)
        assert not torch.equal(dropout(x, 0.4, **kw) == 0, whole == 0)


def test_share_of_kept_elements():
    """2^22 draws at p: the count is within six standard deviations, a chance of 2e-9."""
    n = 1 << 22
    x = torch.ones(64, n // 64, device="cuda")
    for p in (0.03, 0.5, 0.8):
        kept = int((dropout(x, p, 123) != 0).sum())
        assert abs(kept - n * (1 - p)) <= 6 * math.sqrt(n * p * (1 - p))


def test_dropped_infinities_and_in_place_shapes():
    kept = ref.kept(4, 64, 0.5, 9, 0, 0).cuda()
    x = _randn(4, 64, dtype=BF16)
    bad = torch.where(kept, x, torch.tensor(float("nan"), device="cuda", dtype=BF16))
    assert torch.equal(dropout(bad, 0.5, 9), dropout(x, 0.5, 9))
    inf = torch.where(kept, x, torch.tensor(float("inf"), device="cuda", dtype=BF16))
    assert torch.equal(dropout(inf, 0.5, 9), dropout(x, 0.5, 9))
    # rows of any shape, at any address
    y = dropout(x, 0.5, 9)
    assert torch.equal(dropout(x.view(4, 2, 8, 4), 0.5, 9).view(4, 64), y)
    at = torch.cat((x.new_zeros(3), x.flatten()))[3:].view(4, 64)
    assert at.data_ptr() % 16 != 0 and torch.equal(dropout(at, 0.5, 9), y)
    assert torch.equal(dropout(x, 0.5, 9, residual=torch.zeros_like(x)), y)
    assert torch.equal(dropout(x, 0.5, -1), dropout(x, 0.5, (1 << 64) - 1))
    assert dropout(x[:0], 0.5, 9).shape == (0, 64)


def test_more_elements_than_32_bits_count():
    """Rows whose elements lie beyond 2^32: the last ones are as a short row's of the same number."""
    rows, n = 3, (1 << 31) + 8
    x = torch.ones(rows, n, device="cuda", dtype=BF16)
    y = dropout(x, 0.5, 4)
    for r in range(rows):
        assert torch.equal(y[r, :4096], dropout(x[r:r + 1, :4096].contiguous(), 0.5, 4, first_row=r)[0])
    last = []
    for r in range(rows):
        w = [ref.philox((g, 0, r, 0), (4, 0)) for g in ((n >> 2) - 2, (n >> 2) - 1)]
        last.append([x >= 1 << 31 for c in w for x in c])
    assert torch.equal(y[:, -8:] != 0, torch.tensor(last, device="cuda"))


def test_seed_tensor_in_a_captured_graph():
    x = _randn(8, 96, dtype=BF16).requires_grad_()
    d = _randn(8, 96, dtype=BF16, seed=1)
    numbers = torch.tensor([5, 0], device="cuda")

    def work():
        y = dropout(x, 0.3, numbers)
        return y, torch.autograd.grad(y, x, d)[0]

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        work()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = work()
        numbers[1] += 1
    for step in range(3):
        graph.replay()
        torch.cuda.synchronize()
        y = dropout(x, 0.3, 5, stream=step)
        for a, b in zip(held, (y, torch.autograd.grad(y, x, d)[0])):
            assert torch.equal(a, b)
    y = dropout(x, 0.3, numbers)
    numbers[1] += 1
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_refusals():
    x = _randn(4, 8, dtype=BF16)
    for bad in (dict(x=x.t()), dict(x=x.double()), dict(residual=x[:2]), dict(residual=x.float()), dict(seed=torch.zeros(2, device="cuda")),
                dict(seed=torch.zeros(2, dtype=torch.int64)), dict(residual=torch.zeros(8, 4, device="cuda", dtype=BF16).t())):
        with pytest.raises(RuntimeError):
            dropout(**{**dict(x=x, p=0.5, seed=1), **bad})
    for bad in (dict(p=-0.1), dict(p=1.5), dict(p=float("nan")), dict(stream=-1), dict(stream=1 << 32), dict(first_row=-1), dict(seed=1 << 64),
                dict(seed=torch.zeros(2, device="cuda", dtype=torch.int64), stream=1)):
        with pytest.raises(ValueError):
            dropout(**{**dict(x=x, p=0.5, seed=1), **bad})
