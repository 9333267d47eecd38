"""The row operators together, as a training program uses them: embedding and dropout forward and
backward over micro-batches, the gradient in the optimizer's own accumulator, then the step."""
import pytest
import torch

import _rows as ref
from flextrain_amd import FlexTrainAdam, dropout, embedding_grad_, embedding_lookup
from flextrain_amd.loss_scaler import DynamicLossScaler

pytestmark = pytest.mark.gpu

ROWS, COLS = 1013, 72


def _optimizer(cuda, dtype, gradacc, **kw):
    gen = torch.Generator(device=cuda).manual_seed(0)
    table = torch.nn.Parameter((torch.randn((ROWS, COLS), device=cuda, generator=gen) * 0.02).to(dtype))
    head = torch.nn.Parameter((torch.randn((COLS, 5), device=cuda, generator=gen) * 0.1).to(dtype))
    return FlexTrainAdam([{"params": [head, table]}], lr=1e-2, gradacc_dtype=gradacc, **kw), table, head


def _ids(cuda, seed, shape=(3, 101)):
    return torch.randint(0, ROWS, shape, device=cuda, generator=torch.Generator(device=cuda).manual_seed(seed)) // 7 * 3


@pytest.mark.parametrize("dtype,gradacc", [(torch.bfloat16, torch.float32), (torch.float16, torch.float32), (torch.bfloat16, torch.bfloat16),
                                           (torch.float32, torch.float32)])
@pytest.mark.parametrize("offload", [False, True])
def test_micro_batches_into_the_step(cuda, dtype, gradacc, offload):
    opt, table, head = _optimizer(cuda, dtype, gradacc, offload=offload)
    twin, table2, head2 = _optimizer(cuda, dtype, gradacc, offload=offload)
    for step in range(2):
        want, slack = torch.zeros((ROWS, COLS), dtype=torch.float64), torch.zeros((ROWS, COLS), dtype=torch.float64)
        for k in range(3):
            tokens, seed = _ids(cuda, 10 * step + k), 1000 * step + k
            x = opt.embedding(tokens, table, scale=2.0, padding_token=3, dropout=0.1, seed=seed, substream=1)
            caught = []
            x.register_hook(caught.append)
            y = dropout(x, 0.2, seed, substream=2, residual=x)
            (y @ head).float().pow(2).mean().backward()
            # the gradient that reached the embedding, summed by the definition into what was there
            new, before = ref.gradient(want, tokens, caught[0], scale=2.0, padding_token=3, p=0.1, seed=seed, substream=1)
            slack = slack + before + torch.where(new != want, (new.abs() + slack) * ref.HALF_STEP[gradacc] + ref.TINY[gradacc], 0.0)
            want = new
        acc = opt.gradient_of(table)
        assert acc.dtype == gradacc and acc.shape == table.shape
        ref.assert_within(acc, want, slack)
        # a second optimizer, handed the same sums, takes the same step
        twin.gradient_of(table2).copy_(acc)
        twin.gradient_of(head2).copy_(opt.gradient_of(head))
        for o in (opt, twin):
            o.update_states()
            assert o.step()
        assert torch.equal(table, table2) and torch.equal(head, head2)
        assert not bool(opt.gradient_of(table).any())


def test_overflow_in_one_row_skips_the_step(cuda):
    opt, table, head = _optimizer(cuda, torch.float16, torch.float32, loss_scaler=DynamicLossScaler(init_scale=2.0 ** 12))
    before = table.detach().clone()
    for bad in (True, False):
        tokens = _ids(cuda, 1)
        x = opt.embedding(tokens, table, dropout=0.1, seed=5)
        dy = torch.full_like(x, 1e-3)
        if bad:
            keep = ref.kept(x.shape, 0.1, 5)
            at = int(torch.nonzero(keep.flatten())[7, 0])
            dy.view(-1)[at] = float("inf")
        x.backward(dy)
        opt.update_states()
        assert opt.step() != bad
        assert torch.equal(table, before) == bad


def test_recorded_step(cuda):
    """Lookup, dropout, gradient and update recorded once and replayed: the replays take the eager steps."""
    opt, table, _ = _optimizer(cuda, torch.bfloat16, torch.float32, loss_scaler=DynamicLossScaler(init_scale=256.0), capturable=True)
    twin, table2, _ = _optimizer(cuda, torch.bfloat16, torch.float32, loss_scaler=DynamicLossScaler(init_scale=256.0), capturable=True)
    tokens, seed = _ids(cuda, 0, (700,)), torch.tensor([9], dtype=torch.int64, device=cuda)
    dy = torch.randn((700, COLS), device=cuda, generator=torch.Generator(device=cuda).manual_seed(3)).bfloat16()

    def passes(o, t):
        x = embedding_lookup(tokens, t.detach(), dropout=0.1, seed=seed)
        y = dropout(x, 0.1, seed, substream=1, residual=x)
        dx = dropout(dy, 0.1, seed, substream=1, residual=dy)
        embedding_grad_(o.gradient_of(t), tokens, dx, dropout=0.1, seed=seed)
        o.enqueue_step()
        return y

    for o, t in ((opt, table), (twin, table2)):
        o.update_states()
        passes(o, t)
        assert o.complete_step()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        recorded = passes(opt, table)
    for k in range(4):
        tokens.copy_(_ids(cuda, k + 20, (700,)))
        seed.fill_(k + 77)
        for o in (opt, twin):
            o.update_states()
        graph.replay()
        eager = passes(twin, table2)
        assert opt.complete_step() and twin.complete_step()
        assert torch.equal(recorded, eager) and torch.equal(table, table2)


def test_refusals(cuda):
    opt, table, head = _optimizer(cuda, torch.bfloat16, torch.float32)
    tokens = _ids(cuda, 0)
    with pytest.raises(ValueError, match="steps itself"):
        opt.gradient_of(torch.nn.Parameter(torch.zeros(3, device=cuda)))
    with pytest.raises(ValueError, match="steps itself"):
        opt.embedding(tokens, torch.nn.Parameter(torch.zeros((4, 4), device=cuda)))
    with pytest.raises(ValueError, match="int64 or int32"):
        opt.embedding(tokens.float(), table)
    with pytest.raises(ValueError, match="grads have shape"):
        embedding_grad_(opt.gradient_of(table), tokens, torch.zeros((3, 100, COLS), device=cuda))
    with pytest.raises(ValueError, match="two dimensions"):
        embedding_lookup(tokens, table.view(-1))
    with pytest.raises(ValueError, match="grad_into has shape"):
        from flextrain_amd import embedding
        embedding(tokens, table, grad_into=opt.gradient_of(head))
    with pytest.raises(ValueError, match="out must have shape"):
        embedding_lookup(tokens, table, out=torch.zeros((3, 101, COLS + 1), device=cuda, dtype=torch.bfloat16))
    with pytest.raises(ValueError, match="unsupported dtype"):
        embedding_lookup(tokens, torch.zeros((5, 5), device=cuda, dtype=torch.float64))
    with pytest.raises(ValueError, match="overlap"):
        embedding_lookup(tokens, table, out=torch.zeros((1, COLS), device=cuda, dtype=torch.bfloat16).expand(3, 101, COLS))
    x = torch.zeros((4, 4), device=cuda)
    for p in (-0.1, 1.1, float("nan")):
        with pytest.raises(ValueError, match="probability"):
            dropout(x, p, 1)
        with pytest.raises(ValueError, match="probability"):
            embedding_lookup(tokens, table, dropout=p)
    for seed in (-1, 1 << 64, torch.zeros(2, dtype=torch.int64, device=cuda), torch.zeros(1, device=cuda), torch.zeros(1, dtype=torch.int64)):
        with pytest.raises(ValueError, match="seed"):
            dropout(x, 0.5, seed)
    for kw in (dict(substream=-1), dict(substream=1 << 32), dict(first_index=-1), dict(first_index=1 << 62)):
        with pytest.raises(ValueError):
            dropout(x, 0.5, 1, **kw)
    with pytest.raises(ValueError, match="residual has shape"):
        dropout(x, 0.5, 1, residual=x[:2])
    with pytest.raises(ValueError, match="rows"):
        dropout(x.t()[:, :3], 0.5, 1)
    with pytest.raises(ValueError, match="require gradients"):
        dropout(x.clone().requires_grad_(), 0.5, 1, out=x)
