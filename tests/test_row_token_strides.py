"""How far the tokens of a call may lie apart, checked without a GPU: calls on rows of no elements check everything
and do nothing."""
import ctypes

import pytest
import torch

from flextrain_amd import _C
from flextrain_amd.rows import token_record

BUF = (ctypes.c_double * 8)()
ADDR = ctypes.addressof(BUF)
EINVAL = -1
MOST = 1 << 38  # ids; 1 TiB of 32-bit ones


def _lookup(record):
    return _C.lib().ft_embedding_lookup(ctypes.byref(record), ADDR, _C.F32, 4, 8, ADDR, _C.F32, 8, 0, 1.0, None, None)


def _grad(record):
    return _C.lib().ft_embedding_grad(ctypes.byref(record), ADDR, _C.F32, 8, ADDR, _C.F32, 4, 8, 0, 1.0, 1, None, None, 0, None)


@pytest.mark.parametrize("call", [_lookup, _grad])
@pytest.mark.parametrize("outer,inner,outer_stride,inner_stride,accepted", [
    (2, 65536, 65537, 1, True), (64, 40000, 40000, 1, True), (40000, 64, 1, 40000, True), (1, 64, 0, 40000, True), (8, 1 << 20, 1 << 21, 1, True),
    (3, 1000, 32769, 0, True), (2, 2, MOST // 2, 1, True), (2, 2, MOST // 2 + 1, 1, False), (1, 4, 0, MOST // 4, True),
    (1, 4, 0, MOST // 4 + 1, False), (1 << 15, 1 << 15, MOST >> 15, MOST >> 15, True), (1 << 15, 1 << 15, (MOST >> 15) + 1, 1, False),
    (2, 2, (1 << 64) - 1, 1, False), (2, 2, 1, 1 << 63, False)])
def test_distance_of_the_tokens(call, outer, inner, outer_stride, inner_stride, accepted):
    record = _C.Tokens(ADDR, outer, inner, outer_stride, inner_stride, 0, _C.NO_PADDING, 8, 0)
    assert call(record) == (0 if accepted else EINVAL)
    if not accepted:
        assert b"stride" in _C.lib().ft_last_error()


@pytest.mark.parametrize("call", [_lookup, _grad])
@pytest.mark.parametrize("dtype", [torch.int32, torch.int64])
def test_views_of_long_batches(call, dtype):
    """What a program cuts out of a batch of long sequences."""
    long, wide = torch.zeros((2, 65537), dtype=dtype), torch.zeros((64, 40000), dtype=dtype)
    for tokens in (long[:, :-1], wide.t(), wide[:, 0], wide[:, ::3], wide[::9, 5:], wide[:, :1].expand(64, 7)):
        record, n = token_record(tokens, 0, None)
        assert n == tokens.numel() and call(record) == 0
