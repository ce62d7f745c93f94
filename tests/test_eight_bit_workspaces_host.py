"""What the gradients of linear_8bit reserve beside their results, without a GPU."""
import pytest

from vtpack_amd import _lib

MIB = 1 << 20
LIES, NO_DX, NO_DWEIGHT, NO_DBIAS = 1, 2, 4, 8


def _up(n, to):
    return -(-n // to) * to


def _expanded(rows, out, width, lies):
    """bf16 copies: both second operands along the sums, and the gradient unless it is read where it lies."""
    return 2 * (width * _up(rows, 64) + width * _up(out, 64) + (0 if lies else rows * _up(out, 64)))


@pytest.mark.parametrize("rows,out,width", [(32768, 4096, 1024), (65536, 1024, 4096), (131072, 1024, 4096)])
def test_a_sum_that_is_not_cut_reserves_no_parts(rows, out, width):
    """dx of many rows goes straight to its place.  (dW is cut into 32 parts at most.)"""
    bytes_ = _lib.load().vtdge_linear_8bit_backward_workspace(rows, out, width, LIES, _lib.BF16)
    rest = bytes_ - _expanded(rows, out, width, True)
    assert 0 <= rest < 4 * rows * width
    assert rest % (4 * out * (width + 1)) <= 4096 and rest <= 32 * 4 * out * (width + 1) + 4096
    # all of it read where it lies and nothing cut: the expanded operands alone
    assert _lib.load().vtdge_linear_8bit_backward_workspace(8192, 8192, 8192, LIES, _lib.BF16) == _expanded(8192, 8192, 8192, True) == 256 * MIB


def test_a_sum_that_is_cut_reserves_its_parts():
    """Few tiles and long sums: 64 x 64 results of 65536 rows."""
    rows, out, width = 65536, 64, 64
    rest = _lib.load().vtdge_linear_8bit_backward_workspace(rows, out, width, LIES, _lib.BF16) - _expanded(rows, out, width, True)
    assert rest >= 2 * 4 * out * (width + 1) and rest < 4 * rows * width


@pytest.mark.parametrize("lies,dtype", [(LIES, _lib.BF16), (0, _lib.BF16), (0, _lib.F32)])
def test_gradients_that_are_not_wanted_reserve_nothing(lies, dtype):
    """dx alone (a frozen weight) has no use for x, dweight alone (a first layer) none for the weight."""
    size = _lib.load().vtdge_linear_8bit_backward_workspace
    rows, out, width = 65536, 1024, 4096
    g = 0 if lies else 2 * rows * out
    assert size(rows, out, width, lies | NO_DWEIGHT | NO_DBIAS, dtype) == g + 2 * width * out
    only = size(rows, out, width, lies | NO_DX | NO_DBIAS, dtype) - g - 2 * width * rows
    assert only % (4 * out * width) == 0                    # (parts of dweight)
    assert size(rows, out, width, lies | NO_DX | NO_DWEIGHT, dtype) <= g + 32 * 4 * out
    for rows, out, width in ((100, 70, 50), (65536, 64, 64), (4112, 384, 384)):
        whole = size(rows, out, width, lies, dtype)
        assert all(0 <= size(rows, out, width, lies | no, dtype) <= whole for no in range(0, 16, 2))


def test_less_than_what_is_wanted_takes_is_refused():
    lib, p = _lib.load(), 4096                              # never read: the arguments are refused first
    rows, out, width = 65536, 1024, 4096
    for dx, dw, db, no in ((p, None, None, NO_DWEIGHT | NO_DBIAS), (None, p, None, NO_DX | NO_DBIAS), (p, p, None, NO_DBIAS), (p, p, p, 0)):
        bytes_ = lib.vtdge_linear_8bit_backward_workspace(rows, out, width, LIES | no, _lib.BF16)
        args = [p, out, p, p, rows, out, width, p, bytes_ - 1, dx, dw, db, _lib.BF16, None]
        assert lib.vtdge_linear_8bit_backward(*args) == _lib.ERR_ARG and str(bytes_).encode() in lib.vtdge_last_error()
        args[7], args[8] = None, bytes_
        assert lib.vtdge_linear_8bit_backward(*args) == _lib.ERR_ARG
