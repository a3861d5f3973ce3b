"""Where ``residual_out`` of the 8-bit norm may lie: it may be x or residual, row for row, or between their rows; any
other overlap is refused before a launch, since one workgroup's store would meet another's load."""
import pytest

from specdec_nanovllm_amd import _lib
from test_w8a8_cpu import A, no_gpu

BF16 = _lib.SD_BF16
K = 1024  # a row of x is 2048 bytes


def norm(x=A[0], xs=K, res=A[1], rs=K, out=A[5], os=K, rows=4):
    lib = _lib.load()
    rc = lib.sd_rmsnorm_int8(x, xs, res, rs, A[2], A[3], K, A[4], out, os, rows, K, 1e-6, BF16, None)
    return rc, lib.sd_last_error().decode()


@no_gpu
@pytest.mark.parametrize("change", [
    dict(out=A[0] + 2048), dict(out=A[0] - 2048), dict(out=A[1] + 2048),  # a row further
    dict(out=A[0] + 16), dict(out=A[1] - 16),                             # inside the same row
    dict(out=A[0], os=2 * K), dict(out=A[0], xs=2 * K),                   # other row strides
    dict(out=A[0], xs=0), dict(out=A[1], rs=0), dict(x=A[0] + 6144, out=A[0], xs=-K),  # (the last: rows in the other order)
    dict(out=A[0], res=A[0] + 2048), dict(out=A[1], x=A[1] + 2048),       # one of the two only
    dict(out=A[0] + 2032, xs=2 * K, os=2 * K),                            # between the rows, 16 bytes too early
    dict(out=A[0] + 2064, xs=2 * K, os=2 * K), dict(out=A[0] - 2032, xs=2 * K, os=2 * K),
    dict(out=A[0] + 16, rows=1), dict(out=A[1] - 2032, rows=1, rs=0, os=0),
    dict(out=A[0], x=A[0] + 3 * 2048, rows=4),                            # the last row alone
])
def test_residual_out_that_is_partly_an_input_is_refused(change):
    rc, says = norm(**change)
    assert rc == 1 and "share memory" in says, (rc, says)


@no_gpu
@pytest.mark.parametrize("change", [
    dict(out=A[0]), dict(out=A[1]), dict(out=A[0], res=A[0]),
    dict(out=A[0], rows=1, xs=0), dict(out=A[0], rows=1, os=8 * K),
    dict(out=A[0] + 2048, xs=2 * K, os=2 * K), dict(out=A[0] - 2048, xs=2 * K, os=2 * K),  # columns of one buffer
    dict(out=A[1] + 2048, rs=3 * K, os=3 * K), dict(out=A[0] + 4 * 2048), dict(out=A[0] - 4 * 2048),
    dict(out=A[0] + 6144, xs=-K), dict(x=A[0] + 24 * 2048, xs=-8 * K, out=A[0] + 2048),  # below it; in a gap
])
def test_other_places_are_taken(change):
    """(a launch without a GPU is an error of the runtime, none of the arguments')"""
    rc, says = norm(**change)
    assert rc == _lib.SD_ERR_HIP, (rc, says)
