"""Function transformations and the row operators: refused before anything else is looked at, so without a GPU too."""
import pytest
import torch

from flextrain_amd import dropout, embedding, embedding_grad_, embedding_lookup

X, IDS = torch.ones(3, 8), torch.arange(3)
CALLS = {
    "dropout": lambda x: dropout(x, 0.1, 1),
    "residual": lambda x: dropout(X, 0.1, 1, residual=x),
    "lookup": lambda x: embedding_lookup(IDS, x),
    "gradient": lambda x: embedding_grad_(torch.zeros(3, 8), IDS, x),
    "embedding": lambda x: embedding(IDS, x),
    "embedding into": lambda x: embedding(IDS, x, grad_into=torch.zeros(3, 8)),
}


@pytest.mark.parametrize("call", CALLS)
def test_forward_mode(call):
    with torch.autograd.forward_ad.dual_level():
        with pytest.raises(NotImplementedError, match="forward-mode"):
            CALLS[call](torch.autograd.forward_ad.make_dual(X.clone(), torch.ones(3, 8)))
        with pytest.raises(ValueError, match="GPU"):  # no tangent: looked at as ever
            CALLS[call](X)
