"""Tokens that lie far apart: views of batches of long sequences."""
import pytest
import torch

from flextrain_amd import embedding, embedding_grad_, embedding_lookup

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
@pytest.mark.parametrize("view", ["cut", "transposed", "column", "every third", "broadcast"])
def test_views_of_long_batches(cuda, dtype, view):
    gen = torch.Generator(device=cuda).manual_seed(0)
    long = torch.randint(0, 700, (2, 65537), device=cuda, generator=gen).to(dtype)
    wide = torch.randint(0, 700, (64, 40000), device=cuda, generator=gen).to(dtype)
    tokens = {"cut": long[:, :-1], "transposed": wide.t()[:3000], "column": wide[:, 39999], "every third": wide[:5, 1::3],
              "broadcast": wide[::2, :1].expand(32, 900)}[view]
    table = torch.randn((700, 24), device=cuda, generator=gen)
    assert torch.equal(embedding_lookup(tokens, table), table[tokens.long()])
    grads = torch.randint(-8, 9, (*tokens.shape, 24), device=cuda, generator=gen).float()  # sums without rounding
    want = torch.zeros_like(table).index_add_(0, tokens.long().reshape(-1), grads.reshape(-1, 24))
    assert torch.equal(embedding_grad_(torch.zeros_like(table), tokens, grads), want)
    weight = table.clone().requires_grad_()
    embedding(tokens, weight).backward(grads)
    assert torch.equal(weight.grad, want)
