"""Rows that lie between each other, and results that share memory with what is read."""
import pytest
import torch

from flextrain_amd import dropout, embedding_grad_, embedding_lookup

pytestmark = pytest.mark.gpu


def _randn(cuda, shape, dtype, seed=0):
    return torch.randn(shape, device=cuda, generator=torch.Generator(device=cuda).manual_seed(seed)).to(dtype)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("swap", [False, True])
def test_slices_of_one_tensor(cuda, dtype, swap):
    """Columns side by side, rows behind each other, every second row: nothing is shared."""
    cut = [(slice(None), slice(0, 40)), (slice(None), slice(40, 80))], [(slice(0, 50), slice(None)), (slice(50, 100), slice(None))], \
        [(slice(0, 100, 2), slice(None)), (slice(1, 100, 2), slice(None))], [(slice(0, 30), slice(0, 40)), (slice(30, 90, 2), slice(0, 40))]
    for a, b in cut:
        if swap:
            a, b = b, a
        store = _randn(cuda, (100, 80), dtype)
        before = store.clone()
        want = dropout(before[a].clone(), 0.2, 3)
        assert torch.equal(dropout(store[a], 0.2, 3, out=store[b]), want) and torch.equal(store[a], before[a])
        store.copy_(before)
        want = dropout(before[a].clone(), 0.2, 3, residual=before[b].clone())
        assert torch.equal(dropout(store[a], 0.2, 3, residual=store[b], out=store[b]), want) and torch.equal(store[a], before[a])
        store.copy_(before)
        tokens = torch.arange(store[a].shape[0], device=cuda)
        assert torch.equal(embedding_lookup(tokens, store[a], out=store[b]), before[a])
        store.copy_(before)
        assert torch.equal(embedding_grad_(store[b], tokens, store[a]), (before[a].float() + before[b].float()).to(dtype))
        assert torch.equal(store[a], before[a])


def test_shared_memory_is_refused(cuda):
    store = _randn(cuda, (100, 80), torch.float32)
    before = store.clone()
    tokens = torch.arange(99, device=cuda)
    halves = store.view(-1)[:4000].view(100, 40)
    for call in (lambda: dropout(store[1:], 0.2, 3, out=store[:-1]), lambda: dropout(store[:, 1:], 0.2, 3, out=store[:, :-1]),
                 lambda: dropout(store[:1].expand(100, 80), 0.2, 3, out=store), lambda: dropout(store[:, :40], 0.2, 3, out=halves),
                 lambda: dropout(before[:98], 0.2, 3, residual=store[1:99], out=store[:98]),
                 lambda: dropout(store.view(torch.bfloat16)[:, :80], 0.2, 3, residual=before, out=store),
                 lambda: embedding_lookup(tokens, store[1:], out=store[:-1]), lambda: embedding_grad_(store[:-1], tokens, store[1:])):
        with pytest.raises(ValueError, match="overlaps"):
            call()
    assert torch.equal(store, before)
