"""Results that share memory with what is read: refused before any device work, so without a GPU too."""
import ctypes

import pytest

from flextrain_amd import _C

F32, F16, BF16 = _C.F32, _C.F16, _C.BF16
BUF = (ctypes.c_double * 4096)()
ADDR = (ctypes.addressof(BUF) + 63) // 64 * 64
EINVAL = -1


def _refused(rc):
    assert rc == EINVAL and b"overlap" in _C.lib().ft_last_error()


def _dropout(x=0, out=0, x_dtype=F32, out_dtype=F32, x_stride=8, out_stride=8, rows=4, cols=8, residual=None, residual_stride=0):
    """x, out and residual: bytes from ADDR."""
    drop = ctypes.byref(_C.Dropout(0.5, 1, None, 0, 0, 0))
    return _C.lib().ft_dropout(ADDR + x, x_dtype, x_stride, None if residual is None else ADDR + residual, residual_stride, ADDR + out, out_dtype,
                               out_stride, rows, cols, drop, None)


@pytest.mark.parametrize("kw", [
    dict(out=4), dict(out=-4), dict(out=31 * 4), dict(out_stride=9), dict(x_stride=16, out_stride=16, out=7 * 4),
    dict(x_stride=16, out_stride=16, out=(16 - 7) * 4), dict(x_stride=24, out_stride=16, out=4 * 4), dict(x_stride=0), dict(x_stride=0, out=7 * 4),
    dict(rows=1, cols=32, out=31 * 4)], ids=str)
def test_dropout(kw):
    _refused(_dropout(**kw))
    kw = dict(kw)  # the same with the residual, x elsewhere
    _refused(_dropout(x=8192, residual=0, residual_stride=kw.pop("x_stride", 8), **kw))


@pytest.mark.parametrize("kw", [dict(x_dtype=BF16), dict(out_dtype=F16), dict(x_dtype=BF16, x_stride=32, out_stride=16, out=8)], ids=str)
def test_dropout_of_another_type(kw):
    _refused(_dropout(**kw))


def test_lookup():
    tokens = ctypes.byref(_C.Tokens(ADDR + 16384, 1, 4, 0, 1, 0, _C.NO_PADDING, 8, 0))
    for table, rows, stride in ((ADDR, 4, 8), (ADDR + 4, 4, 8), (ADDR + 31 * 4, 1, 8), (ADDR - 4, 1, 8), (ADDR + 60, 3, 16)):
        _refused(_C.lib().ft_embedding_lookup(tokens, table, F32, rows, stride, ADDR, F32, 8, 8, 1.0, None, None))


@pytest.mark.parametrize("inner", [4, 2000])
def test_gradient(inner):
    need = _C.lib().ft_embedding_grad_workspace_bytes(inner, 4, 8)
    tokens = ctypes.byref(_C.Tokens(ADDR + 8192, 1, inner, 0, 1, 0, _C.NO_PADDING, 8, 0))
    for g, stride in ((ADDR, 8), (ADDR + 4, 8), (ADDR + 31 * 4, 0), (ADDR - 4, 1)):
        _refused(_C.lib().ft_embedding_grad(tokens, g, F32, stride, ADDR, F32, 4, 8, 8, 1.0, 1, None, ADDR + 16384 if need else None, need, None))
