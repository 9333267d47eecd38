"""What autograd is told by the row operators, and what it may be asked."""
import pytest
import torch

import _rows as ref
from flextrain_amd import FlexTrainAdam, dropout, embedding, embedding_grad_, embedding_lookup

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16


def _randn(cuda, shape, dtype, seed=0):
    return torch.randn(shape, device=cuda, generator=torch.Generator(device=cuda).manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("gradacc", [F32, BF16])
@pytest.mark.parametrize("used_before", [False, True])
def test_a_frozen_table_has_no_gradient(cuda, gradacc, used_before):
    table = torch.nn.Parameter(_randn(cuda, (50, 24), BF16))
    opt = FlexTrainAdam([{"params": [table]}], lr=1e-2, gradacc_dtype=gradacc)
    tokens, dy = torch.arange(30, device=cuda), torch.ones((30, 24), device=cuda, dtype=BF16)
    if used_before:
        opt.embedding(tokens, table).backward(dy)
    before = opt.gradient_of(table).clone()
    table.requires_grad_(False)
    x = opt.embedding(tokens, table, scale=2.0)
    assert not x.requires_grad and torch.equal(x, table[:30] * 2)
    weight = torch.ones((24,), device=cuda, dtype=BF16, requires_grad=True)
    (x * weight).sum().backward()
    assert torch.equal(opt.gradient_of(table), before)
    table.requires_grad_(True)
    opt.embedding(tokens, table).backward(dy)
    assert torch.equal(opt.gradient_of(table)[:30], before[:30] + 1) and torch.equal(opt.gradient_of(table)[30:], before[30:])
