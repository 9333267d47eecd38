"""The row operators on other streams than the default one. What a stream has to wait for is asked of the stream: while
another one is kept busy, an event behind the pass must not have been reached."""
import time

import pytest
import torch

from flextrain_amd import FlexTrainAdam, dropout, embedding, embedding_grad_, embedding_lookup

pytestmark = pytest.mark.gpu

ROWS, COLS = 900, 72


def _gen(cuda, seed):
    return torch.Generator(device=cuda).manual_seed(seed)


def _whole(cuda, shape, seed=0):
    """Whole numbers: sums without rounding."""
    return torch.randint(-8, 9, shape, device=cuda, generator=_gen(cuda, seed)).float()


def _ids(cuda, n, seed=0):
    return torch.randint(0, ROWS, (n,), device=cuda, generator=_gen(cuda, seed))


def _keep_busy(cuda, stream):
    """About a quarter of a second of work on the stream."""
    with torch.cuda.stream(stream):
        a = torch.ones((8192, 8192), device=cuda, dtype=torch.bfloat16)
        b = torch.empty_like(a)
        for _ in range(300):
            torch.mm(a, a, out=b)


def _waits_for(stream, busy):
    """Whether what is enqueued on ``stream`` now runs behind what ``busy`` still works on."""
    event = torch.cuda.Event()
    event.record(stream)
    time.sleep(0.02)  # an event on an idle stream is reached by then
    reached = event.query()
    assert not busy.query(), "the other stream should have been busy for longer"
    return not reached


@pytest.mark.parametrize("n", [100, 5000])
def test_backward_pass_is_joined_to_its_caller(cuda, n):
    """The lookup on a side stream, the backward pass called on the default one: what follows there (the step, which
    reads and clears the accumulator) waits for the gradient."""
    weight, acc, tokens, dy = _whole(cuda, (ROWS, COLS)), torch.zeros((ROWS, COLS), device=cuda), _ids(cuda, n), _whole(cuda, (n, COLS), 1)
    embedding(tokens, weight, grad_into=acc.clone()).backward(dy)  # loads the code
    side, caller = torch.cuda.Stream(), torch.cuda.current_stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        y = embedding(tokens, weight, grad_into=acc)
    caller.wait_stream(side)
    _keep_busy(cuda, side)
    y.backward(dy)
    assert _waits_for(caller, side)
    torch.cuda.synchronize()
    assert torch.equal(acc, torch.zeros_like(acc).index_add_(0, tokens, dy))


def test_step_behind_a_lookup_on_another_stream(cuda):
    """Forward on a side stream that is late in the backward pass, step on the default one: the same as on one stream."""
    side = torch.cuda.Stream()
    tables = []
    for use in (side, torch.cuda.current_stream()):
        table = torch.nn.Parameter(_whole(cuda, (ROWS, COLS)).bfloat16())
        opt = FlexTrainAdam([{"params": [table]}], lr=1e-2, gradacc_dtype=torch.float32)
        torch.cuda.synchronize()
        for k in range(2):
            use.wait_stream(torch.cuda.current_stream())
            with torch.cuda.stream(use):
                y = opt.embedding(_ids(cuda, 3000, k), table)
            torch.cuda.current_stream().wait_stream(use)
            if use is side:
                _keep_busy(cuda, side)
            y.backward(_whole(cuda, (3000, COLS), k + 5).bfloat16())
            opt.update_states()
            opt.step()
        torch.cuda.synchronize()
        tables.append(table.detach().clone())
    assert torch.equal(*tables) and not torch.equal(tables[0], _whole(cuda, (ROWS, COLS)).bfloat16())


@pytest.mark.parametrize("first", ["default", "side", "other side"])
@pytest.mark.parametrize("graphs", [1, 2])
def test_two_streams_add_into_one_accumulator(cuda, first, graphs):
    """Two lookups of one table, the one whose gradient comes first on a busy stream: the other stream's gradient waits,
    in one backward pass or two, and again with the streams changed."""
    weight, acc = _whole(cuda, (ROWS, COLS)), torch.zeros((ROWS, COLS), device=cuda)
    tokens = [_ids(cuda, n, n) for n in (300, 4000)]
    dy = [_whole(cuda, (n, COLS), n) for n in (300, 4000)]
    embedding(tokens[1], weight, grad_into=acc.clone()).backward(dy[1])
    caller = torch.cuda.current_stream()
    busy, free = {"default": (caller, torch.cuda.Stream()), "side": (torch.cuda.Stream(), caller), "other side": (torch.cuda.Stream(), torch.cuda.Stream())}[first]
    third = torch.cuda.Stream()  # the backward pass is called here: the default stream would wait for the side streams, or be busy itself
    torch.cuda.synchronize()
    for late, early in ((busy, free), (busy, free), (free, busy)):
        with torch.cuda.stream(early):
            y1 = embedding(tokens[1], weight, grad_into=acc[:, :])
        with torch.cuda.stream(late):  # made last: its gradient comes first
            y0 = embedding(tokens[0], weight, grad_into=acc)
        torch.cuda.synchronize()
        _keep_busy(cuda, late)
        with torch.cuda.stream(third):
            if graphs == 1:
                torch.autograd.backward([y0, y1], dy)
            else:
                y0.backward(dy[0])
                with torch.cuda.stream(torch.cuda.Stream()):  # a caller that waits for nothing
                    y1.backward(dy[1])
        assert _waits_for(early, late)
        torch.cuda.synchronize()
    want = torch.zeros_like(acc)
    for t, d in zip(tokens, dy):
        want.index_add_(0, t, d)
    assert torch.equal(acc, 3 * want)


def test_streams_of_a_recording(cuda):
    """Two lookups of one table on two streams of one recording, eager passes on other streams between the replays."""
    weight, acc = _whole(cuda, (ROWS, COLS)), torch.zeros((ROWS, COLS), device=cuda)
    tokens = [_ids(cuda, n, n) for n in (300, 4000)]
    dy = [_whole(cuda, (n, COLS), n) for n in (300, 4000)]
    side, other = torch.cuda.Stream(), torch.cuda.Stream()

    def both():
        main = torch.cuda.current_stream()
        side.wait_stream(main)
        with torch.cuda.stream(side):
            y1 = embedding(tokens[1], weight, grad_into=acc)
        y0 = embedding(tokens[0], weight, grad_into=acc)
        main.wait_stream(side)
        torch.autograd.backward([y0, y1], dy)

    want = torch.zeros_like(acc)
    for t, d in zip(tokens, dy):
        want.index_add_(0, t, d)
    graphs = []
    with torch.cuda.stream(other):
        both()  # eager, on streams that the recordings do not have
    torch.cuda.synchronize()
    assert torch.equal(acc, want)
    for _ in range(2):  # the second recording has nothing to do with the first one's
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            both()
    for k in range(3):
        for graph in graphs:
            acc.zero_()
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(acc, want)
        with torch.cuda.stream(other if k % 2 else torch.cuda.current_stream()):
            both()
        torch.cuda.synchronize()
        assert torch.equal(acc, 2 * want)


@pytest.mark.parametrize("gradacc", [torch.float32, torch.bfloat16])
@pytest.mark.parametrize("lookup_first", [True, False])
def test_a_table_with_another_gradient(cuda, gradacc, lookup_first):
    """A table that is looked up on one stream and used as a matrix on another: the gradient that comes second, in the hook
    or in autograd's own addition, waits for the first one's busy stream."""
    table = torch.nn.Parameter(_whole(cuda, (ROWS, COLS)).bfloat16())
    opt = FlexTrainAdam([{"params": [table]}], lr=1e-2, gradacc_dtype=gradacc)
    tokens, dy, dz = _ids(cuda, 300), _whole(cuda, (300, COLS), 1).bfloat16().sign(), _whole(cuda, (ROWS, COLS), 2).bfloat16()
    caller, side, third = torch.cuda.current_stream(), torch.cuda.Stream(), torch.cuda.Stream()

    def lookup():
        with torch.cuda.stream(side):
            return opt.embedding(tokens, table)

    opt.embedding(tokens, table).backward(dy)
    want = torch.zeros((ROWS, COLS), device=cuda).index_add_(0, tokens, dy.float())
    for k in range(2):
        torch.cuda.synchronize()
        if lookup_first:  # made last, its gradient comes first
            z, y = table * 2.0, lookup()
            first, second = side, caller
        else:
            y, z = lookup(), table * 2.0
            first, second = caller, side
        torch.cuda.synchronize()
        _keep_busy(cuda, first)
        with torch.cuda.stream(third):
            torch.autograd.backward([y, z], [dy, dz])
        assert _waits_for(second, first)
        torch.cuda.synchronize()
    want = 3 * want + 4.0 * dz.float()  # whole numbers; in 16 bits below 256: exact
    assert float(want.abs().max()) < 256 and torch.equal(opt.gradient_of(table).float(), want)
    assert len(torch.autograd.grad(table.sum(), table)) == 1 and opt.gradient_of(table).any()


def test_a_table_with_another_gradient_on_one_stream(cuda):
    """Lookup and output layer share the table, as models with tied weights do."""
    for gradacc in (torch.float32, torch.bfloat16):
        table = torch.nn.Parameter(_whole(cuda, (ROWS, COLS)).bfloat16())
        opt = FlexTrainAdam([{"params": [table]}], lr=1e-2, gradacc_dtype=gradacc)
        tokens, weights = _ids(cuda, 40), _whole(cuda, (40, ROWS), 3).bfloat16().sign()
        x = opt.embedding(tokens, table)
        (x @ table.t()).backward(weights)
        direct = weights.float().t() @ table.detach().float()[tokens]
        rows = weights.float() @ table.detach().float()
        want = direct.double().index_add_(0, tokens, rows.double())
        got = opt.gradient_of(table).double()
        # both gradients arrive rounded to bf16, their sum is rounded to the accumulator's type; tokens met twice add up rounded rows
        terms = direct.abs().double().index_add_(0, tokens, rows.abs().double())
        assert bool(((got - want).abs() <= 2.1 * 2.0 ** -8 * terms).all())


@pytest.mark.parametrize("call", ["dropout", "lookup", "gradient of few", "gradient of many", "gradient written", "embedding"])
def test_calls_run_on_the_current_stream(cuda, call):
    """Inputs that are ready late on a side stream, results that are read there: a kernel on another stream would take the
    old inputs, or come too late."""
    n = 100 if call == "gradient of few" else 20000
    new = dict(x=_whole(cuda, (n, COLS), 1), table=_whole(cuda, (ROWS, COLS), 2), tokens=_ids(cuda, n, 3), acc=_whole(cuda, (ROWS, COLS), 4))
    old = {k: torch.zeros_like(v) for k, v in new.items()}

    def run(x, table, tokens, acc):
        if call == "dropout":
            return dropout(x, 0.1, 3, residual=x)
        if call == "lookup":
            return embedding_lookup(tokens, table, dropout=0.1, seed=2)
        if call == "embedding":
            weight = table.detach().requires_grad_()
            y = embedding(tokens, weight, grad_into=acc)
            y.backward(x)
            return torch.cat([y.detach(), acc])
        return embedding_grad_(acc, tokens, x, accumulate=call != "gradient written")

    want = run(**{k: v.clone() for k, v in new.items()})
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    _keep_busy(cuda, side)
    with torch.cuda.stream(side):
        for k in new:
            old[k].copy_(new[k])
        got = run(**old).clone()
        assert not side.query(), "the stream should have been busy for longer"
        for v in old.values():
            v.zero_()
    torch.cuda.synchronize()
    assert torch.equal(got, want)
