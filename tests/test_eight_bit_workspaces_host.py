"""What the gradients of linear_8bit reserve beside their results, without a GPU."""
import pytest

from vtpack_amd import _lib

MIB = 1 << 20


def _up(n, to):
    return -(-n // to) * to


def _expanded(rows, out, width, lies):
    """bf16 copies: both second operands along the sums, and the gradient unless it is read where it lies."""
    return 2 * (width * _up(rows, 64) + width * _up(out, 64) + (0 if lies else rows * _up(out, 64)))


@pytest.mark.parametrize("rows,out,width", [(32768, 4096, 1024), (65536, 1024, 4096), (131072, 1024, 4096)])
def test_a_sum_that_is_not_cut_reserves_no_parts(rows, out, width):
    """dx of many rows goes straight to its place.  (dW is cut into 32 parts at most.)"""
    bytes_ = _lib.load().vtdge_linear_8bit_backward_workspace(rows, out, width, 1, _lib.BF16)
    rest = bytes_ - _expanded(rows, out, width, True)
    assert 0 <= rest < 4 * rows * width
    assert rest % (4 * out * (width + 1)) <= 4096 and rest <= 32 * 4 * out * (width + 1) + 4096
    # all of it read where it lies and nothing cut: the expanded operands alone
    assert _lib.load().vtdge_linear_8bit_backward_workspace(8192, 8192, 8192, 1, _lib.BF16) == _expanded(8192, 8192, 8192, True) == 256 * MIB


def test_a_sum_that_is_cut_reserves_its_parts():
    """Few tiles and long sums: 64 x 64 results of 65536 rows."""
    rows, out, width = 65536, 64, 64
    rest = _lib.load().vtdge_linear_8bit_backward_workspace(rows, out, width, 1, _lib.BF16) - _expanded(rows, out, width, True)
    assert rest >= 2 * 4 * out * (width + 1) and rest < 4 * rows * width
