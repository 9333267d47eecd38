"""How many elements a call of the row operators takes: past the stated limits it is refused before any device work.
No call here is one that would run."""
import ctypes

import pytest

from flextrain_amd import _C

F32, F16, BF16 = _C.F32, _C.F16, _C.BF16
BUF = (ctypes.c_double * 64)()
ADDR = (ctypes.addressof(BUF) + 15) // 16 * 16
FAR = 1 << 60  # nothing is read or written
EINVAL = -1


def _tokens(n):
    return ctypes.byref(_C.Tokens(ADDR, 1, n, 0, 1, 0, _C.NO_PADDING, 8, 0))


def _refused(rc):
    assert rc == EINVAL and b"too many" in _C.lib().ft_last_error()


@pytest.mark.parametrize("table_dtype,out_dtype,p,limit", [(BF16, BF16, 0.0, 1 << 35), (F16, F16, 0.0, 1 << 35), (F16, F32, 0.0, 1 << 35),
                                                           (F32, F32, 0.2, 1 << 35), (BF16, F16, 0.2, 1 << 36)])
@pytest.mark.parametrize("cols", [4096, 8192, 1 << 20])
def test_elements_of_a_lookup(table_dtype, out_dtype, p, limit, cols):
    """2^35 is 3.4e10."""
    drop = ctypes.byref(_C.Dropout(p, 1, None, 0, 0, 0))
    _refused(_C.lib().ft_embedding_lookup(_tokens(limit // cols), ADDR, table_dtype, 4, cols, FAR, out_dtype, cols, cols, 1.0, drop, None))


@pytest.mark.parametrize("g_dtype,acc_dtype,limit", [(BF16, F32, 2.41e11), (F32, F16, 2.41e11), (F16, BF16, 4.82e11)])
@pytest.mark.parametrize("cols", [4096, 8192, 1 << 20])
def test_elements_of_a_gradient(g_dtype, acc_dtype, limit, cols):
    _refused(_C.lib().ft_embedding_grad(_tokens(int(limit) // cols), ADDR, g_dtype, cols, ADDR, acc_dtype, 4, cols, cols, 1.0, 1, None, ADDR, 1 << 60, None))
