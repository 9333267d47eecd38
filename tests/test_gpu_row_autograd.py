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


WRITES = {
    "dropout": lambda t: dropout(torch.ones_like(t), 0.1, 1, out=t),
    "dropout in place": lambda t: dropout(t, 0.1, 1, out=t),
    "dropout onto the residual": lambda t: dropout(torch.ones_like(t), 0.1, 1, residual=t, out=t),
    "lookup": lambda t: embedding_lookup(torch.arange(t.shape[0], device=t.device), torch.ones_like(t), out=t),
    "gradient": lambda t: embedding_grad_(t, torch.arange(t.shape[0], device=t.device), torch.ones_like(t)),
}


@pytest.mark.parametrize("write", WRITES)
@pytest.mark.parametrize("through_a_view", [False, True])
def test_writes_into_given_tensors_are_found_out(cuda, write, through_a_view):
    """As with torch's own operators: a backward pass that needs the old values of a tensor that was written raises."""
    x, w = _randn(cuda, (20, 12), F32), _randn(cuda, (20, 12), F32, 1).requires_grad_()
    h = x * w  # w's gradient needs x
    before = x._version
    with torch.no_grad():
        WRITES[write](x[3:9] if through_a_view else x)
    assert x._version > before
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()


def test_a_gradient_added_by_a_backward_pass_is_found_out(cuda):
    weight, acc = _randn(cuda, (20, 12), F32), _randn(cuda, (20, 12), F32, 1)
    w = _randn(cuda, (20, 12), F32, 2).requires_grad_()
    h = acc * w
    embedding(torch.arange(9, device=cuda), weight, grad_into=acc).sum().backward()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        h.sum().backward()


@pytest.mark.parametrize("write", WRITES)
def test_writes_without_autograd(cuda, write):
    x = _randn(cuda, (20, 12), F32)
    want = WRITES[write](x.clone())
    with torch.inference_mode():
        inside = x.clone()
        assert inside.is_inference() and torch.equal(WRITES[write](inside), want)


def test_results_given_by_the_caller_must_not_require_gradients(cuda):
    leaf, ids = _randn(cuda, (5, 8), F32).requires_grad_(), torch.arange(5, device=cuda)
    kept = leaf.detach().clone()
    for call in (lambda: embedding_lookup(ids, kept, out=leaf), lambda: embedding_grad_(leaf, ids, kept),
                 lambda: embedding_lookup(ids, kept, out=leaf * 1.0)):
        with pytest.raises(ValueError, match="require gradients"):
            call()
    assert torch.equal(leaf, kept)
    with torch.no_grad():  # as an update of one's own
        embedding_grad_(leaf, ids, kept, scale=-1.0)
        assert not bool(leaf.any())
        assert torch.equal(embedding_lookup(ids, kept, out=leaf), kept)


@pytest.mark.parametrize("needs", [False, True])
def test_forward_mode_is_refused(cuda, needs):
    """A tangent must not vanish without a word."""
    x, ids = _randn(cuda, (6, 8), F32).requires_grad_(needs), torch.arange(6, device=cuda)
    plain = x.detach().clone()
    with torch.autograd.forward_ad.dual_level():
        dual = torch.autograd.forward_ad.make_dual(x, torch.ones_like(plain))
        for call in (lambda: dropout(dual, 0.1, 1), lambda: dropout(plain, 0.1, 1, residual=dual), lambda: embedding_lookup(ids, dual),
                     lambda: embedding(ids, dual), lambda: embedding(ids, dual, grad_into=plain.clone()),
                     lambda: embedding_grad_(plain.clone(), ids, dual)):
            with pytest.raises(NotImplementedError):
                call()
        assert torch.equal(embedding_lookup(ids, plain), plain)  # without a tangent, as ever
        assert torch.equal(dropout(plain, 0.0, 1), plain)
        assert torch.equal(embedding_grad_(torch.zeros_like(plain), ids, plain), plain)
    with torch.no_grad():
        assert torch.equal(embedding(ids, x), plain)


@pytest.mark.parametrize("dtype,residual_dtype", [(F32, None), (F32, F32), (BF16, F32), (F32, BF16), (F16, None)])
@pytest.mark.parametrize("seed_in_memory", [False, True])
def test_dropout_twice_differentiated(cuda, dtype, residual_dtype, seed_in_memory):
    """The operator is linear: its backward pass is the operator again, and so on."""
    p, shape = 0.25, (33, 40)
    seed = torch.tensor([9], dtype=torch.int64, device=cuda) if seed_in_memory else 9
    x = _randn(cuda, shape, dtype).requires_grad_()
    residual = None if residual_dtype is None else _randn(cuda, shape, residual_dtype, 1).requires_grad_()
    leaves = [x] if residual is None else [x, residual]
    factor = ref.kept(shape, p, 9, 3).to(cuda) / (1.0 - p)  # 4 / 3: each product is rounded to fp32, then to its type

    y = dropout(x, p, seed, substream=3, residual=residual)
    first = torch.autograd.grad((y * y).sum() / 2, leaves, create_graph=True)  # y * factor, and y
    assert all(g.requires_grad for g in first)
    u = [torch.ones_like(g) * 2.0 for g in first]
    second = torch.autograd.grad(first, leaves, u)
    # first = J' y, y = J leaves: second = J' J u with J = [diag(factor), 1]
    ju = 2.0 * factor + (0.0 if residual is None else 2.0)
    wants = [factor * ju] + ([] if residual is None else [ju])
    for got, want in zip(second, wants):
        # five values are rounded one behind the other, to fp32 and to the coarsest of the types
        coarse = max(ref.HALF_STEP[t] for t in (dtype, residual_dtype) if t is not None)
        assert bool(((got.double() - want).abs() <= 5 * 1.01 * (coarse + ref.F32) * want.abs()).all())


def test_gradient_of_a_gradient_penalty(cuda):
    """A gradient with respect to the gradient that came in, as a penalty on gradients needs it."""
    x, w = _randn(cuda, (20, 24), F32).requires_grad_(), _randn(cuda, (20, 24), F32, 1).requires_grad_()
    keep = ref.kept((20, 24), 0.5, 4).to(cuda).float() * 2.0  # exact in fp32
    g, = torch.autograd.grad((dropout(x, 0.5, 4) * w).sum(), x, create_graph=True)
    want, = torch.autograd.grad((x * keep * w).sum(), x, create_graph=True)
    assert torch.equal(g, want)
    got_w, = torch.autograd.grad(g.pow(2).sum(), w)
    want_w, = torch.autograd.grad(want.pow(2).sum(), w)
    assert torch.equal(got_w, want_w)
    # a transposed gradient of the gradient
    g, = torch.autograd.grad((dropout(x, 0.5, 4).t() * w.t()).sum(), x, create_graph=True)
    got_w, = torch.autograd.grad(g.t().pow(2).sum(), w)
    assert torch.equal(got_w, want_w)


def test_a_backward_pass_confined_to_some_leaves(cuda):
    """``inputs=`` and ``torch.autograd.grad`` leave the accumulator alone, as they do a leaf that is not named."""
    weight, acc = _randn(cuda, (20, 12), F32).requires_grad_(), torch.zeros((20, 12), device=cuda)
    w = _randn(cuda, (12,), F32, 1).requires_grad_()
    x = embedding(torch.arange(9, device=cuda), weight, grad_into=acc)
    torch.autograd.grad((x * w).sum(), w, retain_graph=True)
    (x * w).sum().backward(inputs=[w])
    assert not bool(acc.any())
    (x * w).sum().backward()
    assert torch.equal(acc[:9], w.detach().expand(9, 12)) and not bool(acc[9:].any()) and weight.grad is None
