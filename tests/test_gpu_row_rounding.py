"""Where the row operators round: the scaled product by itself, then the addition to what is there."""
import pytest
import torch

import _rows as ref
from flextrain_amd import dropout, embedding_grad_

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]


def _randn(cuda, shape, dtype, seed=0):
    return torch.randn(shape, device=cuda, generator=torch.Generator(device=cuda).manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("x_dtype", TYPES)
@pytest.mark.parametrize("residual_dtype", TYPES)
@pytest.mark.parametrize("p", [0.1, 0.3, 0.5])
def test_residual_is_added_to_the_dropped_out_rows(cuda, x_dtype, residual_dtype, p):
    """With a residual: the fp32 result without one, added in fp32, rounded once. One time in a thousand that sum of
    16-bit numbers lies on the border between two of the result's type."""
    x, residual = _randn(cuda, (513, 2056), x_dtype), _randn(cuda, (513, 2056), residual_dtype, 1)
    alone = dropout(x.float(), p, 5, substream=2)
    keep = ref.kept(x.shape, p, 5, 2).to(cuda) > 0
    assert torch.equal(alone, torch.where(keep, x.float() * (1.0 / (1.0 - p)), torch.zeros_like(alone)))
    assert torch.equal(dropout(x, p, 5, substream=2, residual=residual), (residual.float() + alone).to(residual_dtype))
    for wide in (x[:, 1:1001], x[:, :999]):  # rows that lie apart
        beside = residual[:, 3:3 + wide.shape[1]]
        want = (beside.float() + dropout(wide.float(), p, 6)).to(residual_dtype)
        assert torch.equal(dropout(wide, p, 6, residual=beside), want)


@pytest.mark.parametrize("dtype", TYPES)
def test_what_cancels_is_zero(cuda, dtype):
    """9 / (1 - 0.1) is 10: the factor's own rounding must not be seen in 10 - 10."""
    x, residual = torch.full((64, 1000), 9.0, device=cuda, dtype=dtype), torch.full((64, 1000), -10.0, device=cuda, dtype=dtype)
    keep = ref.kept(x.shape, 0.1, 3) > 0
    want = torch.where(keep, 0.0, -10.0).to(dtype)
    assert torch.equal(dropout(x, 0.1, 3, residual=residual).cpu(), want)


@pytest.mark.parametrize("n", [100, 700, 3000, 40000])
@pytest.mark.parametrize("g_dtype", TYPES)
def test_accumulated_gradient_is_the_written_one_added(cuda, n, g_dtype):
    rows, cols = 900, 264
    tokens = torch.randint(0, rows, (n,), device=cuda, generator=torch.Generator(device=cuda).manual_seed(1))
    acc, grads = _randn(cuda, (rows, cols), F32), _randn(cuda, (n, cols), g_dtype, 1)
    kw = dict(scale=0.7, dropout=0.1, seed=4)
    written = embedding_grad_(torch.empty_like(acc), tokens, grads, accumulate=False, **kw)
    assert torch.equal(embedding_grad_(acc.clone(), tokens, grads, **kw), acc + written)


@pytest.mark.parametrize("n", [100, 700, 3000, 40000])
@pytest.mark.parametrize("cols", [40, 41])
@pytest.mark.parametrize("g_dtype", TYPES)
@pytest.mark.parametrize("acc_dtype", TYPES)
def test_a_gradient_that_cancels_is_zero(cuda, n, cols, g_dtype, acc_dtype):
    """Rows with ten tokens, nine of them 1: the sum is 9, times 10 / 9 is 10."""
    tokens = torch.arange(n, device=cuda) % (n // 10)
    grads = torch.full((n, cols), 1.0, device=cuda, dtype=g_dtype)
    grads[:n // 10] = 0.0
    acc = torch.full((n // 10, cols), -10.0, device=cuda, dtype=acc_dtype)
    assert not bool(embedding_grad_(acc, tokens, grads, scale=10.0 / 9.0).any())
