"""What the row operators refuse, checked without a GPU: every check precedes any device work."""
import ctypes

import pytest
import torch

from flextrain_amd import _C, dropout, embedding, embedding_grad_, embedding_lookup
from flextrain_amd.rows import row_stride, token_record, with_even_rows

F32, F16, BF16 = _C.F32, _C.F16, _C.BF16
BUF = (ctypes.c_double * 64)()
ADDR = ctypes.addressof(BUF)
EINVAL, EALIGN = -1, -2


def _tokens(**kw):
    base = dict(ids=ADDR, outer=1, inner=4, outer_stride=0, inner_stride=1, first_row=0, padding=_C.NO_PADDING, id_bytes=8, reserved=0)
    base.update(kw)
    return _C.Tokens(**base)


def _drop(**kw):
    base = dict(p=0.5, seed=1, seed_dev=None, first_index=0, substream=0, reserved=0)
    base.update(kw)
    return _C.Dropout(**base)


def _lookup(tokens=None, table=ADDR, table_dtype=F32, rows=4, table_stride=8, out=ADDR, out_dtype=F32, out_stride=8, cols=8, scale=1.0, drop=None,
            null_tokens=False):
    t = None if null_tokens else ctypes.byref(tokens if tokens is not None else _tokens())
    return _C.lib().ft_embedding_lookup(t, table, table_dtype, rows, table_stride, out, out_dtype, out_stride, cols, scale,
                                        None if drop is None else ctypes.byref(drop), None)


def _grad(tokens=None, g=ADDR, g_dtype=F32, g_stride=8, acc=ADDR, acc_dtype=F32, rows=4, acc_stride=8, cols=8, accumulate=1, drop=None, ws=None,
          ws_bytes=0, null_tokens=False):
    t = None if null_tokens else ctypes.byref(tokens if tokens is not None else _tokens())
    return _C.lib().ft_embedding_grad(t, g, g_dtype, g_stride, acc, acc_dtype, rows, acc_stride, cols, 1.0, accumulate,
                                      None if drop is None else ctypes.byref(drop), ws, ws_bytes, None)


def _dropout(x=ADDR, x_dtype=F32, x_stride=8, residual=None, residual_stride=0, out=ADDR, out_dtype=F32, out_stride=8, rows=2, cols=8, drop=None,
             null_drop=False):
    return _C.lib().ft_dropout(x, x_dtype, x_stride, residual, residual_stride, out, out_dtype, out_stride, rows, cols,
                               None if null_drop else ctypes.byref(drop if drop is not None else _drop()), None)


BAD_TOKENS = [dict(id_bytes=2), dict(id_bytes=0), dict(first_row=-1), dict(ids=None), dict(inner=1 << 31), dict(outer=1 << 16, inner=1 << 16),
              dict(outer=1 << 40, inner=0), dict(inner_stride=1 << 40), dict(outer_stride=1 << 40)]


@pytest.mark.parametrize("bad", BAD_TOKENS, ids=str)
@pytest.mark.parametrize("call", [_lookup, _grad])
def test_bad_tokens(call, bad):
    assert call(tokens=_tokens(**bad)) == EINVAL


@pytest.mark.parametrize("call", [_lookup, _grad])
def test_tokens_missing_or_off_their_size(call):
    assert call(null_tokens=True) == EINVAL
    assert call(tokens=_tokens(ids=ADDR + 4)) == EALIGN
    assert call(tokens=_tokens(ids=ADDR + 2, id_bytes=4)) == EALIGN


@pytest.mark.parametrize("bad,code", [
    (dict(table=None), EINVAL), (dict(out=None), EINVAL), (dict(table_dtype=3), EINVAL), (dict(out_dtype=-1), EINVAL), (dict(table=ADDR + 2), EALIGN),
    (dict(out=ADDR + 1, out_dtype=BF16), EALIGN), (dict(out_stride=7), EINVAL), (dict(rows=1 << 31), EINVAL), (dict(cols=(1 << 24) + 1), EINVAL),
    (dict(table_stride=1 << 50), EINVAL), (dict(drop=_drop(p=1.5)), EINVAL), (dict(drop=_drop(p=-0.1)), EINVAL),
    (dict(drop=_drop(p=float("nan"))), EINVAL), (dict(drop=_drop(seed_dev=ADDR + 4)), EALIGN)], ids=str)
def test_lookup_refusals(bad, code):
    assert _lookup(**bad) == code and _C.lib().ft_last_error()


@pytest.mark.parametrize("bad,code", [
    (dict(g=None), EINVAL), (dict(acc=None), EINVAL), (dict(g_dtype=3), EINVAL), (dict(acc_dtype=7), EINVAL), (dict(g=ADDR + 2), EALIGN),
    (dict(acc=ADDR + 1, acc_dtype=F16), EALIGN), (dict(acc_stride=7), EINVAL), (dict(rows=1 << 31), EINVAL), (dict(cols=(1 << 24) + 1), EINVAL),
    (dict(acc_stride=1 << 50), EINVAL), (dict(g_stride=1 << 50), EINVAL), (dict(drop=_drop(p=2.0)), EINVAL),
    (dict(drop=_drop(seed_dev=ADDR + 2)), EALIGN)], ids=str)
def test_gradient_refusals(bad, code):
    assert _grad(**bad) == code and _C.lib().ft_last_error()


def test_gradient_workspace():
    need = _C.lib().ft_embedding_grad_workspace_bytes
    assert need(0, 1000, 64) == need(100, 1000, 64) == 0
    assert need(1 << 31, 10, 10) == need(1000, 1 << 31, 10) == need(1000, 10, (1 << 24) + 1) == 0  # calls that are refused anyway
    long = _tokens(inner=5000)
    assert need(5000, 4, 8) > 0
    assert _grad(tokens=long) == EINVAL and b"workspace" in _C.lib().ft_last_error()
    assert _grad(tokens=long, ws=ADDR, ws_bytes=need(5000, 4, 8) - 1) == EINVAL
    assert _grad(tokens=long, ws=ADDR + 8, ws_bytes=need(5000, 4, 8)) == EALIGN


@pytest.mark.parametrize("bad,code", [
    (dict(x=None), EINVAL), (dict(out=None), EINVAL), (dict(x_dtype=3), EINVAL), (dict(out_dtype=3), EINVAL), (dict(x=ADDR + 2), EALIGN),
    (dict(out=ADDR + 1, out_dtype=F16), EALIGN), (dict(residual=ADDR + 2), EALIGN), (dict(out_stride=7), EINVAL), (dict(null_drop=True), EINVAL),
    (dict(drop=_drop(p=1.0001)), EINVAL), (dict(rows=1 << 40, cols=1 << 20), EINVAL), (dict(cols=1 << 31, out_stride=1 << 32), EINVAL),
    (dict(x_stride=1 << 60), EINVAL), (dict(drop=_drop(seed_dev=ADDR + 1)), EALIGN)], ids=str)
def test_dropout_refusals(bad, code):
    assert _dropout(**bad) == code and _C.lib().ft_last_error()


def test_nothing_to_do_touches_no_device():
    assert _lookup(tokens=_tokens(inner=0, ids=None), out=None) == 0
    assert _lookup(cols=0) == 0
    assert _grad(tokens=_tokens(inner=0, ids=None), g=None) == 0
    assert _grad(rows=0, acc=None) == 0 and _grad(cols=0) == 0 and _grad(cols=0, accumulate=0) == 0
    assert _dropout(rows=0, x=None, out=None) == 0 and _dropout(cols=0) == 0


def test_host_tensors_are_refused():
    x, ids = torch.zeros(4, 8), torch.zeros(3, dtype=torch.int64)
    for call in (lambda: dropout(x, 0.1, 1), lambda: dropout(x.requires_grad_(), 0.1, 1), lambda: embedding_lookup(ids, x.detach()),
                 lambda: embedding(ids, x), lambda: embedding(ids, x, grad_into=torch.zeros(4, 8)),
                 lambda: embedding_grad_(torch.zeros(4, 8), ids, torch.zeros(3, 8))):
        with pytest.raises(ValueError, match="GPU"):
            call()


def test_row_strides():
    t = torch.zeros(4, 6, 10)
    assert row_stride("t", t, 10) == 10
    assert row_stride("t", t[..., 2:9], 7) == 10
    assert row_stride("t", t[:, :1, :3], 3) == 60 and row_stride("t", t[:1, ::2, :3], 3) == 20 and row_stride("t", t[:, ::2], 10) == 20
    assert row_stride("t", torch.zeros(1, 10).expand(5, 10), 10) == 0
    assert row_stride("t", t[..., :1], 1) == 10
    assert row_stride("t", torch.zeros(0, 3), 3) == 3
    for bad in (t.transpose(1, 2), t[:, ::4], t[:, 1:, :3], t[..., ::2], torch.zeros(()).expand(2, 3)):
        with pytest.raises(ValueError, match="rows"):
            row_stride("t", bad, bad.shape[-1])
        assert with_even_rows(bad).is_contiguous() and with_even_rows(t) is t


def test_token_records():
    t = torch.zeros(4, 10, dtype=torch.int64)
    for tokens, want in ((t, (1, 40, 0, 1)), (t[:, :-1], (4, 9, 10, 1)), (t.t(), (10, 4, 1, 10)), (t[0, ::3], (1, 4, 0, 3)), (t[:, :1].expand(4, 5), (4, 5, 10, 0))):
        record, n = token_record(tokens, 0, None)
        assert n == tokens.numel() and (record.outer, record.inner, record.outer_stride, record.inner_stride) == want
    for bad, kw in ((t.float(), {}), (t.to(torch.int16), {}), (torch.zeros(2, 3, 4, dtype=torch.int64)[..., 1:], {}), (t, dict(first_row=-1)),
                    (t, dict(padding=1 << 63))):
        with pytest.raises(ValueError):
            token_record(bad, kw.get("first_row", 0), kw.get("padding"))
