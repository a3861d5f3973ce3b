"""Rows of the 8-bit norm whose product with the weight leaves fp32 though s and the weight are finite (bf16 only: fp16
values cannot): the norm of such a row is finite, and its codes and scale are those of the formula. Where the squares'
sum leaves fp32 too the row is zeros, as ``ops.rmsnorm``'s.

The products are compared after a division by 2^128, which is exact for every product that is not 2^8 below the row's
largest, whose code is 0 either way; the scale's tolerance is that of tests/test_gpu_act_int8.py.
"""
import numpy as np
import pytest
import torch

import test_gpu_act_int8 as ta
from conftest import to_np
from oracle import w8a8 as o8
from specdec_nanovllm_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
EPS = 1e-6
# every launch: rows and columns by the number of threads and chunks
LAUNCHES = [(9, 512), (9, 208), (600, 1024), (9, 1024), (9, 2048), (9, 4096), (600, 4096), (9, 8192), (9, 9728), (9, 32768)]


def reference(x, w, residual=None):
    s, v = o8.norm_products(to_np(x.float()), to_np(w.float()), None if residual is None else to_np(residual.float()))
    past = np.isinf(v).any(-1) & np.isfinite(s).all(-1) & np.isfinite(to_np(w.float())).all()
    with np.errstate(over="ignore", invalid="ignore"):
        v = np.where(past[:, None], (s.astype(np.float64) * to_np(w.float()).astype(np.float64) * 2.0**-128).astype(np.float32), v)
    codes, most = o8.codes(v)
    scale = o8.norm_scale(np.where(past, most * 2.0**128, most), s, EPS)
    zeros = np.square(s.astype(np.float64)).sum(-1) > float(np.finfo(np.float32).max)
    return codes, np.where(zeros & ~np.isnan(scale), 0.0, scale), past


def check(x, w, residual=None):
    codes, scale, past = reference(x, w, residual)
    got = ops.rmsnorm_int8(x, w, EPS, residual)
    assert np.array_equal(to_np(got[0]), codes)
    have = to_np(got[1]).astype(np.float64)
    assert np.array_equal(np.isnan(have), np.isnan(scale))
    ok = ~np.isnan(scale)
    assert (np.abs(have - scale)[ok] <= 36 * 2.0**-24 * scale[ok]).all()
    if residual is not None:
        want = (x.float() + residual.float()).to(x.dtype)
        assert bool(((got[2] == want) | (got[2].isnan() & want.isnan())).all())
    return past, got


@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("rows,k", LAUNCHES)
def test_large_weights(rows, k, with_residual):
    """Weights of 1e30: rows of 1e10 leave fp32, rows of 1 do not."""
    x, w = ta.make(rows, k, "bf16"), (ta.weight(k, "bf16").float() * 1e30).to(torch.bfloat16)
    x[1::2] *= 1e10
    r = ta.make(rows, k, "bf16", seed=4) if with_residual else None
    past, got = check(x, w, r)
    assert past[1::2].all() and not past[::2].any()
    assert bool((got[1] > 0).all()) and bool(got[1].isfinite().all())


@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("rows,k", LAUNCHES)
def test_squares_and_products_past_fp32_give_zeros_as_rmsnorm(rows, k, with_residual):
    x, w = ta.make(rows, k, "bf16"), ta.weight(k, "bf16")
    w[k // 2] = 1.5
    x[1::2, k // 2] = 3e38  # times 1.5
    x[2] = 3e38
    r = ta.make(rows, k, "bf16", seed=4) if with_residual else None
    past, got = check(x, w, r)
    assert past[1::2].all() and past[2] and bool((got[1][1::2] == 0).all()) and float(got[1][2]) == 0
    assert bool((ops.rmsnorm(x[1:3], w, EPS) == 0).all()) if k <= 8192 else True
    assert bool((ops.dequantize_rows_int8(*got[:2])[1:3] == 0).all())


@pytest.mark.parametrize("with_residual", [False, True])
@pytest.mark.parametrize("rows,k", LAUNCHES)
def test_an_infinity_or_nan_next_to_it_still_has_no_scale(rows, k, with_residual):
    x, w = ta.make(rows, k, "bf16"), ta.weight(k, "bf16")
    w[k // 2] = 1.5
    x[1:, k // 2] = 3e38
    x[2, 0], x[3, k - 1], x[4, k // 3] = float("inf"), float("-inf"), float("nan")
    r = ta.make(rows, k, "bf16", seed=4) if with_residual else None
    if with_residual:
        x[5, 1] = r[5, 1] = 3e38  # finite values, an infinite sum
    _, got = check(x, w, r)
    assert bool(got[1][2:5].isnan().all()) and bool((got[0][2:5] == 0).all())
    assert bool(got[1][5].isnan()) == with_residual
    for bad in (float("inf"), float("nan")):
        w[k - 1] = bad
        assert bool(ops.rmsnorm_int8(x, w, EPS, r)[1].isnan().all())


def test_in_place():
    """The row is formed again from what was loaded: residual_out may have taken its place."""
    from test_gpu_act_int8_alias import norm

    for rows, k in LAUNCHES:
        w = (ta.weight(k, "bf16").float() * 1e30).to(torch.bfloat16)
        for place in (0, 1):
            x, r = ta.make(rows, k, "bf16", std=1e10), ta.make(rows, k, "bf16", seed=4, std=1e10)
            want = ops.rmsnorm_int8(x, w, EPS, r)
            assert bool((want[1] > 0).all())
            assert all(torch.equal(a, b) for a, b in zip(norm(x, w, r, (x, r)[place]), want))
