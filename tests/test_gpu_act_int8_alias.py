"""The 8-bit norm with ``residual_out`` in its place: x, the residual, or other columns of their buffer, through the C entry
(``ops.rmsnorm_int8`` allocates it)."""
import pytest
import torch

import test_gpu_act_int8 as ta
from specdec_nanovllm_amd import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def norm(x, w, residual, residual_out):
    rows, k = x.shape
    codes = torch.empty((rows, k), dtype=torch.int8, device=DEV)
    scale = torch.empty(rows, dtype=torch.float32, device=DEV)
    _lib.check(_lib.load().sd_rmsnorm_int8(
        x.data_ptr(), x.stride(0), residual.data_ptr(), residual.stride(0), w.data_ptr(), codes.data_ptr(), k,
        scale.data_ptr(), residual_out.data_ptr(), residual_out.stride(0), rows, k, 1e-6, _lib.dtype_code(x.dtype),
        _lib.stream_ptr(codes.device)))
    return codes, scale, residual_out


@pytest.mark.parametrize("rows,k", [(1, 1024), (700, 528), (300, 2560), (40, 9728)])
@pytest.mark.parametrize("place", ["x", "residual", "columns", "both"])
def test_in_place(place, rows, k):
    x, r, w = ta.make(rows, k, "bf16"), ta.make(rows, k, "bf16", seed=7), ta.weight(k, "bf16")
    if place == "both":
        r = x
    want = ops.rmsnorm_int8(x, w, 1e-6, r)
    ta.check_norm(x, w, want, r)
    if place == "columns":
        room = torch.full((rows, 3 * k), 7.0, dtype=torch.bfloat16, device=DEV)
        room[:, :k], room[:, 2 * k:] = x, r
        got = norm(room[:, :k], w, room[:, 2 * k:], room[:, k:2 * k])
        assert torch.equal(room[:, :k], x) and torch.equal(room[:, 2 * k:], r)
    else:
        got = norm(x, w, r, r if place == "residual" else x)
    assert all(torch.equal(a, b) for a, b in zip(got, want))


def test_a_row_further_is_refused():
    room = torch.zeros((9, 1024), dtype=torch.bfloat16, device=DEV)
    w, r = ta.weight(1024, "bf16"), ta.make(8, 1024, "bf16")
    with pytest.raises(ValueError, match="share memory"):
        norm(room[:8], w, r, room[1:])
