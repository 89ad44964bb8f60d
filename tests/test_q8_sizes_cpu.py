"""CPU: sizes of the 8-bit operators whose arithmetic in 32 bits would overflow are refused before anything is launched."""
import pytest

MOST = 2 ** 31 - 1024


@pytest.mark.parametrize("cols", [2 ** 31 - 1, 2 ** 31 - 8, 2 ** 31 - 31, 2 ** 31 - 512, MOST + 1])
@pytest.mark.parametrize("x", [4096, 4098])
def test_columns_that_would_overflow(ops, cols, x):
    for rows in (1, 3):
        assert ops.lib().b200attn_q8_quantize(x, ops.DTYPE_BF16, 2 ** 31, rows, cols, 4096, 2 ** 31, 4096, None) == ops.ERR_INVALID
        assert b"sizes" in ops.lib().b200attn_last_error()


def test_most_columns(ops):
    assert ops.lib().b200attn_q8_quantize(None, ops.DTYPE_BF16, MOST, 0, MOST, None, MOST, None, None) == 0
