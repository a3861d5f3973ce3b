"""The linear with 4-bit weights (csrc/w4a16.hip through ``ops``) against the 64-bit oracle.

Tolerance: the output's rounding, eps / 2 |y|, and the fp32 sums: terms of size |x| (31 + 24) s, at most
32 + 4 roundings inside a group's chain of MFMAs and one for each group, wave and the bias after it.
"""
import numpy as np
import pytest
import torch

from oracle import int4 as o4
from specdec_nanovllm_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def f64(t):
    return t.detach().double().cpu().numpy()


def make(m, n, k, group, kind, scale_kind=None, seed=0):
    g = torch.Generator().manual_seed(seed)
    w = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8)
    s = ((torch.rand((n, k // group), generator=g) + 0.2) * 0.02).to(DTYPES[scale_kind or kind])
    x = torch.randn((m, k), generator=g).to(DTYPES[kind])
    b = torch.randn((n,), generator=g).to(DTYPES[kind])
    return x.to(DEV), w.to(DEV), s.to(DEV), b.to(DEV)


def check(got, x, w, s, b, kind):
    eps = float(torch.finfo(DTYPES[kind]).eps)
    wx, sx = o4.weights(w.cpu().numpy(), f64(s)), np.repeat(f64(s), 2 * w.shape[1] // s.shape[1], -1)
    want = f64(x) @ wx.T + (0 if b is None else f64(b))
    groups = s.shape[1]
    size = 55 * np.abs(f64(x)) @ np.abs(sx).T + (0 if b is None else np.abs(f64(b)))
    tol = eps / 2 * np.abs(want) + (36 + 4 * groups + 16) * 2**-24 * size + 1e-7
    off = np.abs(f64(got) - want)
    assert (off <= tol).all(), f"off by {off.max():.3g} where {tol[off > tol].max():.3g} is allowed"


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("group", [32, 64, 96, 128, 256])
@pytest.mark.parametrize("m", [1, 5, 16, 17, 40, 130, 300])
def test_rows_and_groups(kind, group, m):
    n, k = 200, 768
    x, w, s, b = make(m, n, k, group, kind)
    check(ops.w4a16_linear(x, w, s, b), x, w, s, b, kind)


@pytest.mark.parametrize("m", [1, 3, 33, 257])
@pytest.mark.parametrize("n,k,group", [(1, 32, 32), (15, 96, 96), (16, 160, 32), (17, 128, 128),
                                       (513, 1056, 32), (64, 1600, 64), (1000, 9728, 128)])
def test_odd_sizes(m, n, k, group):
    x, w, s, b = make(m, n, k, group, "bf16", seed=m + n)
    check(ops.w4a16_linear(x, w, s), x, w, s, None, "bf16")


@pytest.mark.parametrize("scale_kind", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("m", [2, 50])
def test_scale_types(scale_kind, m):
    x, w, s, b = make(m, 100, 512, 64, "bf16", scale_kind)
    check(ops.w4a16_linear(x, w, s, b), x, w, s, b, "bf16")


@pytest.mark.parametrize("m", [1, 20])
def test_strided_rows_batches_and_out(m):
    x, w, s, b = make(m, 96, 256, 64, "bf16", seed=3)
    wide = torch.full((m, 320), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[:, :256] = x
    out = torch.full((m, 200), 5.0, dtype=torch.bfloat16, device=DEV)
    ops.w4a16_linear(wide[:, :256], w, s, b, out=out[:, 3:99])
    check(out[:, 3:99], x, w, s, b, "bf16")
    assert bool((out[:, :3] == 5).all()) and bool((out[:, 99:] == 5).all())
    y = ops.w4a16_linear(x.view(m, 1, 256), w, s, b)
    assert y.shape == (m, 1, 96) and torch.equal(y[:, 0], out[:, 3:99])
    assert ops.w4a16_linear(x[:0], w, s).shape == (0, 96)


@pytest.mark.parametrize("m", [1, 20])
def test_zero_weights_and_one_row_of_nan(m):
    x, w, s, _ = make(m, 64, 256, 64, "bf16", seed=4)
    w[:32] = 0x88  # every code 8: weight 0
    y = ops.w4a16_linear(x * 100, w, s)
    # 24 sum x taken off in fp32: nothing but its rounding is left
    size = 55 * (100 * x.double().abs()) @ s.double().repeat_interleave(64, 1).T
    assert bool((y[:, :32].double().abs() <= 52 * 2**-24 * size[:, :32]).all())
    if m > 1:
        x[3] = float("nan")
        y = ops.w4a16_linear(x, w, s)
        assert bool(y[3].isnan().all()) and bool(y[:3].isfinite().all()) and bool(y[4:].isfinite().all())


def test_repeats_bit_for_bit_in_a_graph():
    x, w, s, b = make(7, 300, 1024, 128, "bf16", seed=5)
    first = ops.w4a16_linear(x, w, s, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.w4a16_linear(x, w, s, b)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, first)
        x.mul_(1.5)
        first = ops.w4a16_linear(x, w, s, b)
