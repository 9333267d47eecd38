"""Dropout from the counter generator on the GPU against its definition in 64 bits."""
import pytest
import torch

import _rows as ref
from flextrain_amd import dropout

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
SEED = 0x9ABCDEF012345678


def _randn(cuda, shape, dtype, seed=0):
    return torch.randn(shape, device=cuda, generator=torch.Generator(device=cuda).manual_seed(seed)).to(dtype)


def _check(got, x, p, seed=SEED, residual=None, **kw):
    want, before = ref.dropout(x, p, seed, residual=residual, **kw)
    ref.assert_within(got, want, before)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("shape", [(1,), (7,), (8,), (9,), (1, 4096), (3, 1003), (2, 5, 64), (2049, 65), (513, 1024), ()])
@pytest.mark.parametrize("with_residual", [False, True])
def test_shapes(cuda, dtype, shape, with_residual):
    x = _randn(cuda, shape, dtype)
    residual = _randn(cuda, shape, dtype, 1) if with_residual else None
    got = dropout(x, 0.1, SEED, substream=3, residual=residual)
    assert got.shape == x.shape and got.dtype == dtype
    _check(got, x, 0.1, substream=3, residual=residual)


@pytest.mark.parametrize("x_dtype", TYPES)
@pytest.mark.parametrize("residual_dtype", TYPES)
def test_types(cuda, x_dtype, residual_dtype):
    x, residual = _randn(cuda, (33, 257), x_dtype), _randn(cuda, (33, 257), residual_dtype, 1)
    got = dropout(x, 0.3, SEED, residual=residual)
    assert got.dtype == residual_dtype
    _check(got, x, 0.3, residual=residual)


@pytest.mark.parametrize("p", [0.0, 2.0 ** -48, 1e-6, 2.0 ** -17, 0.1, 0.5, 0.999999, 1.0 - 2.0 ** -30, 1.0])
def test_probabilities(cuda, p):
    x = _randn(cuda, (1 << 20,), F32).abs() + 1.0
    got = dropout(x, p, 11)
    _check(got, x, p, seed=11)


def test_ties_are_decided_by_the_second_hash(cuda):
    """Probabilities whose limit is one element's own 48-bit number: that element stays, and with the
    next number it goes."""
    n = 1 << 12
    x = torch.ones(n, device=cuda)
    u = ref.numbers(torch.arange(n).numpy(), 5, 0)
    for i in (0, 1, 2, 3, 1001, n - 1):
        for limit in (int(u[i]), int(u[i]) + 1):
            got = dropout(x, limit * 2.0 ** -48, 5)
            assert (float(got[i]) != 0.0) == (limit == int(u[i]))
            assert torch.equal((got != 0).cpu(), torch.from_numpy(u >= limit))


@pytest.mark.parametrize("first", [0, 1, 2, 3, 4, 4095, (1 << 33) + 5, (1 << 62) - 1])
def test_index_offset(cuda, first):
    x = _randn(cuda, (31, 101), BF16)
    _check(dropout(x, 0.25, 3, substream=7, first_index=first), x, 0.25, seed=3, substream=7, first_index=first)


def test_a_split_tensor_has_the_mask_of_the_whole(cuda):
    x = _randn(cuda, (64, 1001), F16)
    whole = dropout(x, 0.4, 99)
    parts = [dropout(x[a:b], 0.4, 99, first_index=a * 1001) for a, b in ((0, 1), (1, 30), (30, 64))]
    assert torch.equal(torch.cat(parts), whole)


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("start,cols,wide", [(0, 1003, 1008), (1, 64, 67), (3, 1000, 1024), (0, 8, 9)])
def test_rows_that_lie_apart(cuda, dtype, start, cols, wide):
    """Slices of wider tensors; what lies between the rows stays."""
    x = _randn(cuda, (57, wide), dtype)[:, start:start + cols]
    residual = _randn(cuda, (57, wide + 2), dtype, 1)[:, 1:1 + cols]
    store = _randn(cuda, (57, wide + 5), dtype, 2)
    untouched = store.clone()
    got = dropout(x, 0.1, SEED, residual=residual, out=store[:, 2:2 + cols])
    _check(got, x, 0.1, residual=residual)
    untouched[:, 2:2 + cols] = got
    assert torch.equal(store, untouched)


def test_broadcast_rows(cuda):
    x = _randn(cuda, (1, 300), BF16).expand(40, 300)
    _check(dropout(x, 0.5, 1), x, 0.5, seed=1)


def test_in_place(cuda):
    x, residual = _randn(cuda, (100, 333), F16), _randn(cuda, (100, 333), F16, 1)
    want = dropout(x, 0.2, 4, residual=residual)
    a, b = x.clone(), residual.clone()
    assert torch.equal(dropout(a, 0.2, 4, residual=residual, out=a), want) and torch.equal(a, want)
    assert torch.equal(dropout(x, 0.2, 4, residual=b, out=b), want)


def test_infinities_and_nan(cuda):
    """Kept ones come through, dropped ones contribute nothing."""
    x = torch.full((4096,), float("nan"), device=cuda, dtype=BF16)
    x[::2] = float("inf")
    keep = ref.kept(x.shape, 0.5, 8) > 0
    got = dropout(x, 0.5, 8).cpu()
    assert torch.equal(got == 0, ~keep)
    assert bool(torch.isnan(got[1::2][keep[1::2]]).all()) and bool(torch.isinf(got[::2][keep[::2]]).all())
    residual = torch.ones(4096, device=cuda, dtype=BF16)
    assert bool((dropout(x, 0.5, 8, residual=residual).cpu()[~keep] == 1).all())


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("with_residual", [False, True])
def test_gradients(cuda, dtype, with_residual):
    x = _randn(cuda, (65, 130), dtype).requires_grad_()
    residual = _randn(cuda, (65, 130), F32, 1).requires_grad_() if with_residual else None
    y = dropout(x, 0.3, SEED, substream=2, residual=residual)
    dy = _randn(cuda, y.shape, y.dtype, 2)
    y.backward(dy)
    assert x.grad.dtype == dtype
    _check(x.grad, dy, 0.3, substream=2)
    if with_residual:
        assert torch.equal(residual.grad, dy)


def test_gradient_against_differences(cuda):
    """The operator is linear in x: the gradient of a weighted sum is its change per unit step."""
    x = _randn(cuda, (6, 11), F32)
    weights = _randn(cuda, (6, 11), F32, 1).double()
    leaf = x.clone().requires_grad_()
    (dropout(leaf, 0.4, 21).double() * weights).sum().backward()
    for i in range(x.numel()):
        up, down = x.clone(), x.clone()
        up.view(-1)[i] += 0.5
        down.view(-1)[i] -= 0.5
        step = float((up - down).view(-1)[i])
        slope = float((((dropout(up, 0.4, 21).double() - dropout(down, 0.4, 21).double()) * weights).sum() / step))
        # values below 8: four fp32 roundings of at most 8 / 0.6 * 2^-24 each, times a weight, over the step
        assert abs(slope - float(leaf.grad.view(-1)[i])) <= 6 * 8 / 0.6 * 2.0 ** -24 * float(weights.abs().view(-1)[i]) / step + 1e-12


def test_gradient_of_a_broadcast_result(cuda):
    """Gradients without memory of their own (sums hand out one number for all elements)."""
    x = _randn(cuda, (9, 77), F32).requires_grad_()
    dropout(x, 0.2, 6).sum().backward()
    _check(x.grad, torch.ones(9, 77), 0.2, seed=6)
    x.grad = None
    dropout(x, 0.2, 6).t().contiguous().t().mul(2.0).sum().backward()
    _check(x.grad, torch.full((9, 77), 2.0), 0.2, seed=6)


def test_seed_in_gpu_memory(cuda):
    x = _randn(cuda, (1000,), F32).requires_grad_()
    for value in (0, -1, 12345, -(1 << 63)):
        seed = torch.tensor([value], dtype=torch.int64, device=cuda)
        y = dropout(x, 0.5, seed, substream=1)
        _check(y, x, 0.5, seed=value & ref.MASK64, substream=1)
        (g,) = torch.autograd.grad(y, x, torch.ones_like(y))
        _check(g, torch.ones(1000), 0.5, seed=value & ref.MASK64, substream=1)
    y = dropout(x, 0.5, seed)
    seed.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_recorded_with_a_seed_that_changes(cuda):
    """A recorded forward and backward pass follows the seed's memory: other masks in every replay, and
    the backward pass's that of its forward pass."""
    x, dy = _randn(cuda, (300, 257), BF16), _randn(cuda, (300, 257), BF16, 1)
    seed = torch.tensor([50], dtype=torch.int64, device=cuda)

    def both():
        seed.add_(1)
        return dropout(x, 0.1, seed), dropout(dy, 0.1, seed)

    stream = torch.cuda.Stream()
    with torch.cuda.stream(stream):
        both()
    torch.cuda.current_stream().wait_stream(stream)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        y, dx = both()
    for _ in range(4):
        graph.replay()
        torch.cuda.synchronize()
        now = int(seed.item())
        assert torch.equal(y, dropout(x, 0.1, now)) and torch.equal(dx, dropout(dy, 0.1, now))
    assert now == 55


def test_streams(cuda):
    """Two calls in flight on two streams."""
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    x = _randn(cuda, (2048, 1024), F32)
    torch.cuda.synchronize()
    with torch.cuda.stream(a):
        ya = dropout(x, 0.1, 1)
    with torch.cuda.stream(b):
        yb = dropout(x, 0.1, 2)
    torch.cuda.synchronize()
    assert torch.equal(ya, dropout(x, 0.1, 1)) and torch.equal(yb, dropout(x, 0.1, 2))


def test_far_elements(cuda):
    """More than 2^32 elements: every row of a tall tensor has the mask of its own index."""
    rows, cols = (1 << 21) + 3, 2048
    x = torch.ones((1, cols), device=cuda, dtype=BF16).expand(rows, cols)
    y = dropout(x, 0.5, 77)
    for r in (0, 1, (1 << 20) - 1, 1 << 20, 1 << 21, rows - 1):
        assert torch.equal((y[r] != 0).cpu().double(), ref.kept((cols,), 0.5, 77, first_index=r * cols)), r
    z = dropout(y, 0.5, 78, out=y)  # flat: no row of its own
    for r in (0, (1 << 21) - 1, rows - 1):
        keep = ref.kept((cols,), 0.5, 77, first_index=r * cols) * ref.kept((cols,), 0.5, 78, first_index=r * cols)
        assert torch.equal((z[r] != 0).cpu().double(), keep), r


def test_share_of_kept_elements(cuda):
    """10^8 elements at p = 0.1: the share that stays lies within six standard deviations (3e-5 each), and
    neighbours, elements of one group and of the next agree as independent ones do."""
    n = 10 ** 8
    keep = (dropout(torch.ones(n, device=cuda), 0.1, 2024) != 0)
    assert abs(float(keep.double().mean()) - 0.9) < 6 * 3e-5
    for lag in (1, 2, 3, 4, 8, 4096):
        both = float((keep[lag:] & keep[:-lag]).double().mean())
        assert abs(both - 0.81) < 6 * 6e-5, lag
