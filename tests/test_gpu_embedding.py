"""Embedding lookup and its gradient by sorted tokens on the GPU against their definition in 64 bits."""
import pytest
import torch

import _rows as ref
from flextrain_amd import dropout, embedding, embedding_grad_, embedding_lookup

pytestmark = pytest.mark.gpu

F32, F16, BF16 = torch.float32, torch.float16, torch.bfloat16
TYPES = [F32, F16, BF16]
SEED = 0x123456789ABCDEF0


def _gen(cuda, seed):
    return torch.Generator(device=cuda).manual_seed(seed)


def _randn(cuda, shape, dtype, seed=0):
    return torch.randn(shape, device=cuda, generator=_gen(cuda, seed)).to(dtype)


def _ids(cuda, shape, rows, seed=0, dtype=torch.int64):
    """Frequent and rare tokens: the k-th about 1/k as often as the first."""
    u = torch.rand(shape, device=cuda, generator=_gen(cuda, seed), dtype=torch.float64)
    return ((rows + 1.0) ** u - 1).floor().clamp(0, rows - 1).to(dtype)


def _check_lookup(got, tokens, table, **kw):
    ref_kw = dict(kw)
    ref_kw["p"] = ref_kw.pop("dropout", 0.0)
    want, before = ref.lookup(tokens, table, **ref_kw)
    ref.assert_within(got, want, before)


def _check_grad(got, acc, tokens, grads, **kw):
    kw["p"] = kw.pop("dropout", 0.0)
    want, before = ref.gradient(acc, tokens, grads, **kw)
    ref.assert_within(got, want, before)
    if kw.get("accumulate", True):  # rows without a token keep their bits
        met = torch.zeros(acc.shape[0], dtype=torch.bool)
        at = tokens.cpu().long().reshape(-1) - kw.get("first_row", 0)
        met[at[(at >= 0) & (at < acc.shape[0])]] = True
        assert torch.equal(got.cpu()[~met], acc.cpu()[~met])


# ---- lookup ---------------------------------------------------------------------------------------


@pytest.mark.parametrize("table_dtype", TYPES)
@pytest.mark.parametrize("out_dtype", TYPES)
@pytest.mark.parametrize("p", [0.0, 0.2])
def test_lookup_types(cuda, table_dtype, out_dtype, p):
    table, tokens = _randn(cuda, (331, 200), table_dtype), _ids(cuda, (3, 50), 331)
    kw = dict(scale=7.3, dropout=p, seed=SEED, substream=1)
    got = embedding_lookup(tokens, table, dtype=out_dtype, **kw)
    assert got.shape == (3, 50, 200) and got.dtype == out_dtype
    _check_lookup(got, tokens, table, **kw)


@pytest.mark.parametrize("cols", [1, 7, 8, 9, 64, 127, 128, 129, 500, 512, 513, 1003, 2048, 4096, 5000, 8192])
@pytest.mark.parametrize("n", [1, 3, 4, 5, 700])
@pytest.mark.parametrize("p", [0.0, 0.1])
def test_lookup_sizes(cuda, cols, n, p):
    table, tokens = _randn(cuda, (97, cols), BF16), _ids(cuda, (n,), 97)
    _check_lookup(embedding_lookup(tokens, table, scale=0.5, dropout=p, seed=3), tokens, table, scale=0.5, dropout=p, seed=3)


@pytest.mark.parametrize("cols", [640, 1003, 2056, 4096])
def test_lookup_of_many_tokens(cuda, cols):
    """Enough wavefronts for the variant that takes several units per lane."""
    table, tokens = _randn(cuda, (1000, cols), F16), _ids(cuda, (17001,), 1000)
    assert torch.equal(embedding_lookup(tokens, table), table[tokens])
    got = embedding_lookup(tokens, table, dropout=0.1, seed=9)
    for lo in (0, 16900):
        _check_lookup(got[lo:lo + 100], tokens[lo:lo + 100], table, dropout=0.1, seed=9, first_index=lo * cols)


@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_lookup_token_layouts(cuda, dtype):
    table = _randn(cuda, (50, 96), F32)
    wide = _ids(cuda, (6, 40), 50, dtype=dtype)
    for tokens in (wide[:, :-1], wide[::2, 1::3], wide.t(), wide[2, ::5], wide[:, 0], wide[0, 0], wide[:1, 3:3], wide.view(2, 3, 40),
                   wide[:, :1].expand(6, 9)):
        got = embedding_lookup(tokens, table)
        assert got.shape == (*tokens.shape, 96) and torch.equal(got, table[tokens.long()])
        got = embedding_lookup(tokens, table, dropout=0.3, seed=5, first_index=9)
        _check_lookup(got, tokens, table, dropout=0.3, seed=5, first_index=9)
        if tokens.numel():
            grads, acc = _randn(cuda, got.shape, F32, 1), torch.zeros_like(table)
            _check_grad(embedding_grad_(acc.clone(), tokens, grads, dropout=0.3, seed=5), acc, tokens, grads, dropout=0.3, seed=5)


def test_lookup_outside_the_table(cuda):
    """Shards of a vocabulary: what lies elsewhere reads as zero, and the shards add up to the whole."""
    table = _randn(cuda, (300, 130), F32)
    tokens = _ids(cuda, (500,), 300)
    parts = [embedding_lookup(tokens, table[a:b], first_row=a, dtype=F32) for a, b in ((0, 100), (100, 101), (101, 300))]
    assert torch.equal(sum(parts), table[tokens])
    odd = torch.tensor([-1, -(1 << 63), (1 << 63) - 1, 300, 1 << 32, (1 << 32) + 5, 299, 0], device=cuda)
    got = embedding_lookup(odd, table, scale=float("inf"))
    assert not bool(got[:6].any()) and bool(torch.isinf(got[6:]).all())
    got = embedding_lookup(odd.int(), table)  # the low halves
    assert torch.equal(got[6:], table[[299, 0]])
    assert not bool(embedding_lookup(tokens, table[:0]).any())


def test_lookup_layouts(cuda):
    """Rows of table and result that lie apart; what lies between the result's rows stays."""
    table = _randn(cuda, (40, 150), BF16)[:, 3:104]
    tokens = _ids(cuda, (33,), 40)
    store = _randn(cuda, (33, 111), BF16, 1)
    untouched = store.clone()
    embedding_lookup(tokens, table, out=store[:, 5:106])
    untouched[:, 5:106] = table[tokens]
    assert torch.equal(store, untouched)


def test_lookup_far_rows(cuda):
    """A table of more than 2^32 elements, results beyond 2^31."""
    rows, cols = (1 << 20) + 9, 4104
    table = torch.zeros((rows, cols), device=cuda, dtype=BF16)
    tokens = torch.tensor([0, rows - 1, 1 << 20, 5], device=cuda)
    table[tokens] = _randn(cuda, (4, cols), BF16)
    assert torch.equal(embedding_lookup(tokens, table), table[tokens])
    acc_rows = table[tokens].clone()
    embedding_grad_(table, tokens, acc_rows)
    assert torch.equal(table[tokens], acc_rows * 2)
    many = tokens.repeat(200)
    embedding_grad_(table, many, acc_rows.repeat(200, 1), scale=1.0 / 256)
    want, before = ref.gradient(acc_rows * 2, torch.arange(4).repeat(200), acc_rows.repeat(200, 1), scale=1.0 / 256)
    ref.assert_within(table[tokens], want, before)
    assert not bool(table[1:5].any()) and not bool(table[rows - 5:rows - 1].any())


def test_lookup_far_results(cuda):
    """Results and gradients of more than 2^32 elements; masks of elements beyond 2^32."""
    n, cols = (1 << 20) + 77, 4104
    table, tokens = _randn(cuda, (50, cols), BF16), _ids(cuda, (n,), 50)
    out = embedding_lookup(tokens, table)
    for at in (0, 1 << 19, 1 << 20, n - 1):
        assert torch.equal(out[at], table[tokens[at]])
    out.zero_()
    rows = torch.tensor([0, 1 << 19, (1 << 20) - 1, 1 << 20, n - 1], device=cuda)
    out[rows] = torch.randint(-8, 9, (5, cols), device=cuda, generator=_gen(cuda, 4)).to(BF16)
    want = torch.zeros((50, cols)).index_add_(0, tokens[rows].cpu(), out[rows].float().cpu())
    assert torch.equal(embedding_grad_(torch.zeros((50, cols), device=cuda), tokens, out).cpu(), want)
    keep = torch.stack([ref.kept((cols,), 0.5, 3, first_index=int(r) * cols) for r in rows])
    want = torch.zeros((50, cols)).index_add_(0, tokens[rows].cpu(), out[rows].float().cpu() * keep.float()) * 2
    assert torch.equal(embedding_grad_(torch.zeros((50, cols), device=cuda), tokens, out, dropout=0.5, seed=3).cpu(), want)
    embedding_lookup(tokens, table, dropout=0.5, seed=3, out=out)
    for k, r in enumerate(rows.tolist()):
        assert torch.equal(out[r].cpu().float(), (table[tokens[r]].float().cpu() * 2 * keep[k].float()).to(BF16).float())


# ---- gradient -------------------------------------------------------------------------------------


@pytest.mark.parametrize("g_dtype", TYPES)
@pytest.mark.parametrize("acc_dtype", TYPES)
@pytest.mark.parametrize("n", [100, 2000])
@pytest.mark.parametrize("p", [0.0, 0.2])
def test_gradient_types(cuda, g_dtype, acc_dtype, n, p):
    acc, tokens, grads = _randn(cuda, (500, 200), acc_dtype), _ids(cuda, (n,), 500), _randn(cuda, (n, 200), g_dtype, 1)
    kw = dict(scale=0.7, dropout=p, seed=SEED, substream=4)
    got = embedding_grad_(acc.clone(), tokens, grads, **kw)
    _check_grad(got, acc, tokens, grads, **kw)
    kw["accumulate"] = False
    got = embedding_grad_(acc.clone().fill_(float("nan")), tokens, grads, **kw)
    _check_grad(got, acc, tokens, grads, **kw)


# around the limits of the variants: 1024 tokens of such rows without sorting, 16384 sorted in one launch
@pytest.mark.parametrize("n", [0, 1, 2, 63, 64, 65, 127, 128, 129, 1023, 1024, 1025, 8191, 8192, 8193, 16383, 16384, 16385, 20011])
@pytest.mark.parametrize("rows", [1, 2, 63, 64, 65, 511, 512, 513, 50257])
@pytest.mark.parametrize("accumulate", [True, False])
def test_gradient_counts(cuda, n, rows, accumulate):
    cols = 72
    acc, tokens, grads = _randn(cuda, (rows, cols), F32), _ids(cuda, (n,), rows, n), _randn(cuda, (n, cols), BF16, 1)
    got = embedding_grad_(acc.clone(), tokens, grads, accumulate=accumulate)
    _check_grad(got, acc, tokens, grads, accumulate=accumulate)


@pytest.mark.parametrize("cols", [1, 4, 7, 8, 9, 12, 100, 504, 511, 512, 513, 1003, 1024, 4096, 5001])
@pytest.mark.parametrize("n", [90, 1500])
@pytest.mark.parametrize("p", [0.0, 0.1])
def test_gradient_widths(cuda, cols, n, p):
    acc, tokens, grads = _randn(cuda, (120, cols), BF16), _ids(cuda, (n,), 120), _randn(cuda, (n, cols), F16, 1)
    kw = dict(scale=2.0, dropout=p, seed=6, first_index=cols * 3)
    _check_grad(embedding_grad_(acc.clone(), tokens, grads, **kw), acc, tokens, grads, **kw)


@pytest.mark.parametrize("n", [128, 129, 255, 4096, 8192, 30000, 140001])
@pytest.mark.parametrize("how", ["one", "two", "ends", "blocks", "all different", "sorted", "reversed", "two in a bucket"])
def test_gradient_runs(cuda, n, how):
    """Runs that begin and end everywhere: inside a wavefront, across wavefronts and workgroups, across all of them."""
    rows, cols = 150000, 64
    i = torch.arange(n, device=cuda)
    tokens = {"one": torch.full_like(i, 77), "two": torch.where(i % 3 == 0, 5, rows - 1), "ends": torch.where((i == 0) | (i == n - 1), i, 9),
              "blocks": i * 7 // 1000 * 3, "all different": (i * 7919) % rows, "sorted": i // 5, "reversed": (n - 1 - i) // 33,
              "two in a bucket": torch.where(i % 2 == 0, 512, torch.where(i % 5 == 0, 256 * (i % 400), 1024))}[how]
    acc, grads = torch.zeros((rows, cols), device=cuda), _randn(cuda, (n, cols), F32, 1)
    got = embedding_grad_(acc.clone(), tokens, grads)
    _check_grad(got, acc, tokens, grads)


@pytest.mark.parametrize("n,rows", [(131072, 70000), (131073, 300), (262144, 1 << 19), (262145, 200000), (1 << 20, 40), (1 << 21, 700),
                                    ((1 << 21) + 1, 50000), (5000, (1 << 26) + 5),
                                    (16384, 1 << 26), (16384, (1 << 17) + 1),
                                    (8192, 1 << 17), (300, 1 << 17), (16384, 100000), (8192, 100000)])
@pytest.mark.parametrize("how", ["frequent and rare", "one and others", "last rows", "one bucket"])
def test_gradient_sorting(cuda, n, rows, how):
    """Tiles that are counted directly and by a scan, digits of one, two and three passes, heavy buckets."""
    i = torch.arange(n, device=cuda)
    tokens = {"frequent and rare": _ids(cuda, (n,), rows), "one and others": torch.where(i % 4 == 0, i * 7919 % rows, rows // 3),
              "last rows": rows - 1 - i % 33, "one bucket": (i * 31 % 97 * 256 + 5) % rows}[how]
    grads = torch.randint(-8, 9, (n, 2), device=cuda, generator=_gen(cuda, 2)).to(BF16)  # sums without rounding
    want = torch.zeros((rows, 2)).index_add_(0, tokens.cpu(), grads.float().cpu())
    got = embedding_grad_(torch.empty((rows, 2), device=cuda), tokens, grads, accumulate=False)
    assert torch.equal(got.cpu(), want)


@pytest.mark.parametrize("n", [2, 7, 8, 9, 65, 511, 512, 513, 1023, 1024])
@pytest.mark.parametrize("cols", [5, 513, 2048, 2049, 4096, 4104, 9001])
@pytest.mark.parametrize("how", ["one", "eight and nine", "different", "few left"])
def test_gradient_without_sorting(cuda, n, cols, how):
    """Rows that one workgroup, some or all of its tokens' workgroups share, in one pass over the columns or several."""
    rows, i = 1500, torch.arange(n, device=cuda)
    tokens = {"one": torch.full_like(i, rows - 1), "eight and nine": torch.where(i % 17 < 8, i // 17 * 2, i // 17 * 2 + 1) % rows,
              "different": (i * 7) % rows, "few left": torch.where(i % 50 == 1, 3, 2000)}[how]
    for g_dtype, acc_dtype in ((BF16, F32), (F16, BF16)):
        grads = torch.randint(-8, 9, (n, cols), device=cuda, generator=_gen(cuda, 2)).to(g_dtype)
        acc = torch.randint(-8, 9, (rows, cols), device=cuda, generator=_gen(cuda, 3)).to(acc_dtype)
        inside = tokens < rows
        for accumulate in (True, False):
            # whole numbers below 2^24: the sum has no rounding, the result's type has one
            want = acc.double().cpu() if accumulate else torch.zeros((rows, cols), dtype=torch.float64)
            want.index_add_(0, tokens[inside].cpu(), grads[inside].double().cpu())
            got = embedding_grad_(acc.clone() if accumulate else torch.full_like(acc, float("nan")), tokens, grads, accumulate=accumulate)
            assert torch.equal(got.cpu(), want.to(acc_dtype)), (g_dtype, acc_dtype, accumulate)


@pytest.mark.parametrize("n,cols", [(512, 700), (1000, 4090), (300, 9000)])
@pytest.mark.parametrize("g_dtype,acc_dtype", [(BF16, F32), (F32, F32), (F16, F16)])
def test_masked_gradient_without_sorting(cuda, n, cols, g_dtype, acc_dtype):
    tokens = _ids(cuda, (n,), 40, 5)
    tokens[::3] = 39
    acc, grads = _randn(cuda, (40, cols), acc_dtype), _randn(cuda, (n, cols), g_dtype, 1)
    kw = dict(scale=0.5, dropout=0.3, seed=8, substream=2, first_index=7, padding_token=3)
    got = embedding_grad_(acc.clone(), tokens, grads, **kw)
    _check_grad(got, acc, tokens, grads, **kw)
    assert torch.equal(embedding_grad_(acc.clone(), tokens, grads, **kw), got)


def test_gradient_of_whole_numbers_is_exact(cuda):
    """Sums below 2^24 have no rounding: any order, any split gives the same number."""
    n, rows, cols = 100003, 3001, 136
    tokens = _ids(cuda, (n,), rows)
    grads = torch.randint(-8, 9, (n, cols), device=cuda, generator=_gen(cuda, 2)).to(BF16)
    want = torch.zeros((rows, cols), dtype=torch.float64).index_add_(0, tokens.cpu(), grads.cpu().double())
    got = embedding_grad_(torch.empty((rows, cols), device=cuda), tokens, grads, accumulate=False)
    assert torch.equal(got.cpu().double(), want)


@pytest.mark.parametrize("n", [100, 5000, 50000])
def test_gradient_skips_padding_and_other_shards(cuda, n):
    rows = 1000
    tokens = _ids(cuda, (n,), rows)
    tokens[::2] = 17
    tokens[5::7] = -100
    grads = _randn(cuda, (n, 80), F32, 1)
    grads[tokens == 17] = float("nan")  # nothing of it may come through
    acc = _randn(cuda, (rows, 80), F32, 2)
    kw = dict(padding_token=17)
    got = embedding_grad_(acc.clone(), tokens, grads, **kw)
    _check_grad(got, acc, tokens, grads, **kw)
    assert torch.equal(got[17], acc[17])
    a, b = 300, 777  # a shard, padding inside and outside of it
    for pad in (17, 400):
        kw = dict(padding_token=pad, first_row=a)
        part = torch.where(torch.isnan(grads), torch.zeros_like(grads), grads)
        got = embedding_grad_(acc[a:b].clone(), tokens, part, **kw)
        _check_grad(got, acc[a:b], tokens, part, **kw)
    for bad in (torch.full_like(tokens, 17), torch.full_like(tokens, -1), torch.full_like(tokens, rows)):  # nothing left
        assert torch.equal(embedding_grad_(acc.clone(), bad, grads, padding_token=17), acc)
        assert not bool(embedding_grad_(acc.clone(), bad, grads, padding_token=17, accumulate=False).any())


@pytest.mark.parametrize("n", [60, 3000])
@pytest.mark.parametrize("g_dtype,acc_dtype", [(BF16, F16), (F16, F32), (F32, BF16)])
@pytest.mark.parametrize("at", [1, 2, 3, 5])
def test_rows_at_any_element(cuda, n, g_dtype, acc_dtype, at):
    """Whole units of rows that begin at any element: all that an address is aligned to is one element."""
    tokens = _ids(cuda, (n,), 70)
    grads, store = _randn(cuda, (n, 133), g_dtype)[:, at:at + 128], _randn(cuda, (70, 133), acc_dtype, 1)
    acc = store[:, at - 1:at + 127]
    before = store.clone()
    embedding_grad_(acc, tokens, grads, scale=0.5, dropout=0.1, seed=2)
    _check_grad(acc, before[:, at - 1:at + 127], tokens, grads, scale=0.5, dropout=0.1, seed=2)
    assert torch.equal(store[:, :at - 1], before[:, :at - 1]) and torch.equal(store[:, at + 127:], before[:, at + 127:])
    out = torch.empty((n, 137), device=cuda, dtype=g_dtype)[:, at:at + 128]
    _check_lookup(embedding_lookup(tokens, acc, out=out, dropout=0.1, seed=2), tokens, acc, dropout=0.1, seed=2)


def test_one_token_without_a_dimension(cuda):
    acc, token, grad = _randn(cuda, (9, 40), F32), torch.tensor(7, device=cuda), _randn(cuda, (40,), F32, 1)
    _check_grad(embedding_grad_(acc.clone(), token, grad), acc, token, grad)


@pytest.mark.parametrize("n", [70, 900])
def test_everything_dropped(cuda, n):
    acc, tokens, grads = _randn(cuda, (50, 40), F32), _ids(cuda, (n,), 50), torch.full((n, 40), float("nan"), device=cuda)
    assert torch.equal(embedding_grad_(acc.clone(), tokens, grads, dropout=1.0, seed=3), acc)
    assert not bool(embedding_grad_(acc.clone(), tokens, grads, dropout=1.0, seed=3, accumulate=False).any())
    assert not bool(embedding_lookup(tokens, torch.full_like(acc, float("inf")), dropout=1.0, seed=3).any())


@pytest.mark.parametrize("n", [60, 3000])
def test_gradient_layouts(cuda, n):
    """Strided tokens, rows that lie apart; what lies between the accumulator's rows stays."""
    wide = _ids(cuda, (4, n // 4 + 1), 200, dtype=torch.int32)
    tokens = wide[:, :-1]
    grads = _randn(cuda, (*tokens.shape, 120), BF16)[..., 2:103]
    store = _randn(cuda, (200, 109), F16, 1)
    before = store.clone()
    embedding_grad_(store[:, 4:105], tokens, grads)
    _check_grad(store[:, 4:105], before[:, 4:105], tokens, grads)
    assert torch.equal(store[:, :4], before[:, :4]) and torch.equal(store[:, 105:], before[:, 105:])
    cleared = embedding_grad_(store[:, 4:105], tokens, grads, accumulate=False)
    _check_grad(cleared, before[:, 4:105], tokens, grads, accumulate=False)
    assert torch.equal(store[:, :4], before[:, :4]) and torch.equal(store[:, 105:], before[:, 105:])
    ones = torch.ones((1, 101), device=cuda).expand(*tokens.shape, 101)  # one row for all tokens
    acc = torch.zeros((200, 101), device=cuda)
    _check_grad(embedding_grad_(acc.clone(), tokens, ones), acc, tokens, ones)


def test_gradient_passes_infinities_and_nan_on(cuda):
    """An overflow must reach the optimizer's check: in the row that it belongs to and in no other."""
    for n in (100, 4000):
        tokens, grads = _ids(cuda, (n,), 50), _randn(cuda, (n, 64), F16)
        tokens[:4] = torch.tensor([3, 4, 5, 5], device=cuda)
        grads[0, 1], grads[1, 2], grads[2, 3], grads[3, 3] = float("inf"), float("nan"), float("inf"), float("-inf")
        got = embedding_grad_(torch.zeros((50, 64), device=cuda), tokens, grads).cpu()
        bad = torch.nonzero(~torch.isfinite(got)).tolist()
        assert bad == [[3, 1], [4, 2], [5, 3]] and bool(torch.isnan(got[5, 3]))


@pytest.mark.parametrize("n", [128, 6000, 40000])
def test_gradient_is_the_same_every_time(cuda, n):
    tokens, grads = _ids(cuda, (n,), 700), _randn(cuda, (n, 520), BF16)
    first = embedding_grad_(torch.zeros((700, 520), device=cuda), tokens, grads, dropout=0.1, seed=1)
    for _ in range(3):
        assert torch.equal(embedding_grad_(torch.zeros((700, 520), device=cuda), tokens, grads, dropout=0.1, seed=1), first)


def test_two_streams(cuda):
    a, b = torch.cuda.Stream(), torch.cuda.Stream()
    tokens, grads = _ids(cuda, (2, 20000), 5000), _randn(cuda, (2, 20000, 256), BF16)
    accs = torch.zeros((2, 5000, 256), device=cuda)
    torch.cuda.synchronize()
    for _ in range(3):
        with torch.cuda.stream(a):
            embedding_grad_(accs[0], tokens[0], grads[0], accumulate=False)
        with torch.cuda.stream(b):
            embedding_grad_(accs[1], tokens[1], grads[1], accumulate=False)
    torch.cuda.synchronize()
    for k in (0, 1):
        assert torch.equal(accs[k], embedding_grad_(torch.empty_like(accs[k]), tokens[k], grads[k], accumulate=False))


@pytest.mark.parametrize("n", [100, 3000, 20000])
def test_recorded(cuda, n):
    """Two recorded calls (each with its own workspace) replayed with new tokens between eager calls."""
    rows, cols = 900, 130
    tokens, grads, table = _ids(cuda, (n,), rows), _randn(cuda, (n, cols), BF16), _randn(cuda, (rows, cols), BF16, 1)
    acc, other = torch.zeros((rows, cols), device=cuda), torch.zeros((rows, cols), device=cuda, dtype=BF16)
    embedding_grad_(acc.clone(), tokens, grads)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rows_out = embedding_lookup(tokens, table)
        embedding_grad_(acc, tokens, grads, accumulate=False)
        embedding_grad_(other, tokens, grads, accumulate=False, scale=2.0)
    for k in range(4):
        tokens.copy_(_ids(cuda, (n,), rows, seed=k + 10))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(rows_out, table[tokens])
        assert torch.equal(acc, embedding_grad_(torch.empty_like(acc), tokens, grads, accumulate=False))
        assert torch.equal(other, embedding_grad_(torch.empty_like(other), tokens, grads, accumulate=False, scale=2.0))


# ---- autograd -------------------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("p", [0.0, 0.3])
def test_autograd_dense(cuda, dtype, p):
    weight = _randn(cuda, (300, 88), dtype).requires_grad_()
    tokens = _ids(cuda, (4, 300), 300)
    kw = dict(scale=1.5, dropout=p, seed=SEED, substream=9, first_index=4)
    y = embedding(tokens, weight, padding_token=2, **kw)
    _check_lookup(y, tokens, weight, **kw)
    dy = _randn(cuda, y.shape, dtype, 1)
    y.backward(dy)
    assert weight.grad.dtype == dtype
    _check_grad(weight.grad, weight.detach(), tokens, dy, padding_token=2, accumulate=False, **kw)


def test_autograd_against_differences(cuda):
    weight = _randn(cuda, (5, 9), F32)
    tokens = torch.tensor([[0, 3, 3], [4, 0, 3]], device=cuda)
    weights = _randn(cuda, (2, 3, 9), F32, 1).double()

    def loss(w):
        return (embedding(tokens, w, scale=2.0, dropout=0.3, seed=4).double() * weights).sum()

    leaf = weight.clone().requires_grad_()
    loss(leaf).backward()
    for i in range(weight.numel()):
        up, down = weight.clone(), weight.clone()
        up.view(-1)[i] += 0.5
        down.view(-1)[i] -= 0.5
        slope = float((loss(up) - loss(down)) / (up - down).view(-1)[i].double())
        # values below 8 * 2 / 0.7, two roundings of 2^-24 each at either end, at most three tokens, weights below 8
        assert abs(slope - float(leaf.grad.view(-1)[i])) <= 3 * 8 * 4 * 8 * 2 / 0.7 * 2.0 ** -24


@pytest.mark.parametrize("acc_dtype", TYPES)
def test_autograd_into_an_accumulator(cuda, acc_dtype):
    """Micro-batches one after the other; weight itself gets nothing, requires it or not."""
    for needs in (True, False):
        weight = _randn(cuda, (400, 72), BF16).requires_grad_(needs)
        acc = _randn(cuda, (400, 72), acc_dtype, 1)
        for k in range(3):
            before = acc.clone()
            tokens = _ids(cuda, (2, 250), 400, k)
            y = embedding(tokens, weight, scale=3.0, dropout=0.1, seed=k, grad_into=acc)
            dy = _randn(cuda, y.shape, BF16, k + 5)
            y.backward(dy)
            _check_grad(acc, before, tokens, dy, scale=3.0, dropout=0.1, seed=k)
        assert weight.grad is None
    with torch.no_grad():
        assert not embedding(tokens, weight, grad_into=acc).requires_grad


def test_autograd_layouts_of_the_gradient(cuda):
    weight = _randn(cuda, (60, 40), F32).requires_grad_()
    tokens = _ids(cuda, (3, 50), 60)
    for f in (lambda y: y.sum(), lambda y: (y.transpose(1, 2).contiguous() * 2.0).sum(), lambda y: y[:, ::2].sum() + y[:, :, 3].sum(),
              lambda y: y.mean(1).sum()):
        want, = torch.autograd.grad(f(weight[tokens]), weight)
        got, = torch.autograd.grad(f(embedding(tokens, weight)), weight)
        # sums of at most 150 equal or similar terms on either side
        assert float((got - want).abs().max()) <= 2 * 150 * 2.0 ** -24 * float(want.abs().max())


def test_changed_tokens_are_found_out(cuda):
    weight, tokens = _randn(cuda, (60, 40), F32).requires_grad_(), _ids(cuda, (30,), 60)
    y = embedding(tokens, weight)
    tokens.add_(1)
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        y.sum().backward()


def test_recorded_backward_pass(cuda):
    """Forward and backward recorded together, into an accumulator, while an eager graph of the same
    table is alive: the recording holds no leaf of it."""
    weight = _randn(cuda, (500, 64), BF16).requires_grad_()
    tokens, dy = _ids(cuda, (700,), 500), _randn(cuda, (700, 64), BF16, 1)
    acc, seed = torch.zeros((500, 64), device=cuda), torch.tensor([3], dtype=torch.int64, device=cuda)

    def step():
        y = embedding(tokens, weight, dropout=0.1, seed=seed, grad_into=acc)
        z = dropout(y, 0.1, seed, substream=1, residual=y)
        z.backward(dy)

    alive = embedding(tokens, weight, grad_into=acc.clone())
    stream = torch.cuda.Stream()
    stream.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(stream):
        step()
    torch.cuda.current_stream().wait_stream(stream)
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        step()
    for k in range(3):
        seed.fill_(100 + k)
        acc.zero_()
        graph.replay()
        torch.cuda.synchronize()
        got = acc.clone()
        acc.zero_()
        step()
        assert torch.equal(got, acc) and bool(acc.any())
    alive.sum().backward()
