"""The linears in 8-bit integers (csrc/w8a8.hip through ``ops``) against the oracle.

The sums are exact and the fp32 steps single operations in a fixed order, so the linear equals the oracle's fp32
arithmetic bit for bit. With SiLU, gate and up are those same fp32 values; what is left is exp2(-gate log2(e)): the
product's rounding, |gate| log2(e) 2^-24, and the constant's, 2^-26 of the same, in the exponent, (1 + 1/4) |gate| 2^-24
of the exponential, and one unit, 2^-23, of v_exp_f32; the sum's rounding, one unit of v_rcp_f32, two products:
2^-24 (1.25 |gate| + 2 + 1 + 2 + 2), and the output's own half step or least value. Where the reciprocal is less than
2^-126 it may be 0: |gate up| 2^-126.
"""
import numpy as np
import pytest
import torch

from conftest import to_np
from oracle import w8a8 as o8
from specdec_nanovllm_amd import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "fp32": torch.float32}


def make(m, n, k, kind="bf16", scale_kind="bf16", seed=0):
    g = torch.Generator().manual_seed(seed + 31 * m + n + k)
    x = torch.randint(-127, 128, (m, k), generator=g, dtype=torch.int8)
    w = torch.randint(-127, 128, (n, k), generator=g, dtype=torch.int8)
    xs = torch.rand((m,), generator=g) * 0.05 + 1e-3
    ws = ((torch.rand((n,), generator=g) + 0.1) * 1e-3).to(DTYPES[scale_kind])
    b = torch.randn((n,), generator=g).to(DTYPES[kind])
    return x.to(DEV), xs.to(DEV), w.to(DEV), ws.to(DEV), b.to(DEV)


def equal(got, x, xs, w, ws, b, kind):
    want = o8.linear32(to_np(x), to_np(xs), to_np(w), to_np(ws.float()), None if b is None else to_np(b.float()))
    want = torch.from_numpy(want).to(DTYPES[kind])
    assert got.dtype == DTYPES[kind] and got.shape == want.shape
    bad = (got.cpu() != want).nonzero()
    assert not len(bad), f"{len(bad)} outputs differ, the first at {bad[0].tolist()}"


def near(got, x, xs, w, ws, b, kind):
    y = o8.linear32(to_np(x), to_np(xs), to_np(w), to_np(ws.float()), None if b is None else to_np(b.float()))
    gate, up = (np.abs(t) for t in np.split(y.astype(np.float64), 2, axis=-1))
    want = o8.silu_up(y.astype(np.float64))
    tiny = float(torch.finfo(DTYPES[kind]).tiny) * float(torch.finfo(DTYPES[kind]).eps)
    tol = np.abs(want) * (float(torch.finfo(DTYPES[kind]).eps) / 2 + 2.0**-24 * (1.25 * gate + 7)) + tiny + gate * up * 2.0**-126
    off = np.abs(to_np(got).astype(np.float64) - want)
    assert got.dtype == DTYPES[kind] and got.shape == want.shape
    assert (off <= tol).all(), f"off by {off.max():.3g} where {tol[off > tol].max():.3g} is allowed"


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 32, 33, 64, 65, 129, 300])
def test_rows(kind, m):
    x, xs, w, ws, b = make(m, 272, 768, kind)
    equal(ops.w8a8_linear(x, xs, w, ws, b, DTYPES[kind]), x, xs, w, ws, b, kind)
    near(ops.w8a8_gate_up_silu(x, xs, w, ws, b, DTYPES[kind]), x, xs, w, ws, b, kind)


@pytest.mark.parametrize("m", [1, 5, 40, 131])
@pytest.mark.parametrize("n,k", [(2, 16), (30, 48), (34, 112), (66, 128), (130, 144), (514, 1040), (1000, 4112), (254, 9728)])
def test_odd_sizes(m, n, k):
    x, xs, w, ws, b = make(m, n, k)
    equal(ops.w8a8_linear(x, xs, w, ws), x, xs, w, ws, None, "bf16")
    equal(ops.w8a8_linear(x, xs, w[:n - 1], ws[:n - 1], b[:n - 1]), x, xs, w[:n - 1], ws[:n - 1], b[:n - 1], "bf16")
    near(ops.w8a8_gate_up_silu(x, xs, w, ws), x, xs, w, ws, None, "bf16")


@pytest.mark.parametrize("m,n,k", [(200, 6144, 2560), (777, 2560, 1040), (1100, 5000, 272), (64, 256, 9728), (2100, 2200, 528)])
def test_tiles_and_slices(m, n, k):
    x, xs, w, ws, b = make(m, n, k)
    equal(ops.w8a8_linear(x, xs, w, ws, b), x, xs, w, ws, b, "bf16")
    near(ops.w8a8_gate_up_silu(x, xs, w, ws, b), x, xs, w, ws, b, "bf16")


# (gated, rows, outputs, K, (tile rows, weight rows, workgroups a compute unit), in slices)
ROUTES = [
    (0, 40, 34, 144, (32, 64, 4), False), (0, 40, 34, 1040, (32, 64, 4), False), (0, 20, 34, 9744, (32, 64, 4), True),
    (0, 40, 8200, 528, (64, 64, 2), False), (0, 40, 8200, 1040, (64, 64, 2), False),
    (0, 1500, 34, 9744, (64, 64, 2), True), (0, 40, 8200, 144, (64, 128, 2), False),
    (0, 100, 8200, 1040, (64, 128, 2), False), (0, 2000, 1030, 1040, (96, 96, 1), False),
    (0, 70, 8200, 9744, (96, 96, 1), True), (0, 200, 8200, 1040, (128, 128, 1), False),
    (0, 100, 8200, 9744, (128, 128, 1), True), (0, 400, 12000, 144, (128, 256, 1), False),
    (0, 400, 12000, 1040, (128, 256, 1), False), (0, 500, 8200, 144, (192, 128, 1), False),
    (0, 500, 8200, 1040, (192, 128, 1), False), (0, 900, 8200, 144, (192, 256, 1), False),
    (0, 900, 8200, 1040, (192, 256, 1), False), (0, 1000, 12000, 144, (256, 256, 1), False),
    (0, 1000, 12000, 1040, (256, 256, 1), False), (1, 40, 34, 144, (32, 64, 4), False),
    (1, 40, 34, 1040, (32, 64, 4), False), (1, 20, 34, 9744, (32, 64, 4), True),
    (1, 40, 4100, 528, (64, 64, 2), False), (1, 40, 4100, 1040, (64, 64, 2), False),
    (1, 700, 34, 9744, (64, 64, 2), True), (1, 16, 8200, 144, (64, 128, 2), False),
    (1, 40, 8200, 1040, (64, 128, 2), False), (1, 70, 12000, 528, (96, 96, 1), False),
    (1, 70, 8200, 1040, (96, 96, 1), False), (1, 70, 4100, 9744, (96, 96, 1), True),
    (1, 100, 8200, 1040, (128, 128, 1), False), (1, 100, 4100, 9744, (128, 128, 1), True),
    (1, 200, 8200, 144, (128, 256, 1), False), (1, 200, 8200, 1040, (128, 256, 1), False),
    (1, 130, 12000, 144, (192, 128, 1), False), (1, 130, 12000, 1040, (192, 128, 1), False),
    (1, 900, 4100, 144, (192, 256, 1), False), (1, 400, 8200, 1040, (192, 256, 1), False),
    (1, 400, 12000, 144, (256, 256, 1), False), (1, 400, 12000, 1040, (256, 256, 1), False),
]


@pytest.mark.parametrize("gated,m,n,k,tile,sliced", ROUTES)
def test_every_tile(gated, m, n, k, tile, sliced):
    """Every tile, in slices too, at shapes that end inside it; K ends inside a step. Odd N: rows that start anywhere."""
    plan = _lib.load().sd_w8a8_plan(m, n, k, gated)
    if torch.cuda.get_device_properties(0).multi_processor_count == 256:
        assert ((plan >> 20) & 4095, (plan >> 8) & 4095, plan >> 32) == tile and (plan & 255 > 1) == sliced
    for cols in (n, n - 1):
        x, xs, w, ws, b = make(m, cols * (1 + gated), k)
        if gated:
            near(ops.w8a8_gate_up_silu(x, xs, w, ws, b), x, xs, w, ws, b, "bf16")
        else:
            equal(ops.w8a8_linear(x, xs, w, ws, b), x, xs, w, ws, b, "bf16")


@pytest.mark.parametrize("scale_kind", ["bf16", "fp16", "fp32"])
@pytest.mark.parametrize("m", [2, 50])
def test_scale_types(scale_kind, m):
    x, xs, w, ws, b = make(m, 100, 512, "fp16", scale_kind)
    equal(ops.w8a8_linear(x, xs, w, ws, b, torch.float16), x, xs, w, ws, b, "fp16")


@pytest.mark.parametrize("m", [3, 200])
def test_largest_sums(m):
    """All codes -128: 2^14 K, the longest K there is."""
    k = (1 << 17) - 16
    x = torch.full((m, k), -128, dtype=torch.int8, device=DEV)
    w = torch.full((40, k), -128, dtype=torch.int8, device=DEV)
    w[1::2] = 127
    xs = torch.full((m,), 2.0**-20, device=DEV)
    ws = torch.ones(40, device=DEV)
    y = ops.w8a8_linear(x, xs, w, ws)
    want = torch.tensor([128.0 * 128 * k, -128.0 * 127 * k], dtype=torch.float64).float() * 2.0**-20
    assert torch.equal(y.cpu(), want.to(torch.bfloat16).repeat(20).expand(m, 40))


def test_rows_do_not_depend_on_the_call():
    """A row's outputs are the same bits in every route."""
    x, xs, w, ws, b = make(700, 1040, 2064)
    all_rows = ops.w8a8_linear(x, xs, w, ws, b)
    gated = ops.w8a8_gate_up_silu(x, xs, w, ws, b)
    routes = set()
    for m in (1, 8, 17, 33, 70, 140, 300, 699):
        routes.add(_lib.load().sd_w8a8_plan(m, 1040, 2064, 0))
        assert torch.equal(ops.w8a8_linear(x[:m], xs[:m], w, ws, b), all_rows[:m])
        assert torch.equal(ops.w8a8_gate_up_silu(x[:m], xs[:m], w, ws, b), gated[:m])
    assert len(routes) > 1


@pytest.mark.parametrize("m", [1, 20, 70])
def test_strided_rows_batches_and_out(m):
    x, xs, w, ws, b = make(m, 96, 256, seed=3)
    wide = torch.full((m, 320), 99, dtype=torch.int8, device=DEV)
    wide[:, 16:272] = x
    wwide = torch.full((96, 272), 99, dtype=torch.int8, device=DEV)
    wwide[:, :256] = w
    out = torch.full((m + 1, 200), 5.0, dtype=torch.bfloat16, device=DEV)
    ops.w8a8_linear(wide[:, 16:272], xs, wwide[:, :256], ws, b, out=out[:m, 3:99])
    equal(out[:m, 3:99], x, xs, w, ws, b, "bf16")
    assert bool((out[:, :3] == 5).all()) and bool((out[:, 99:] == 5).all()) and bool((out[m:] == 5).all())
    ops.w8a8_gate_up_silu(wide[:, 16:272], xs, wwide[:, :256], ws, b, out=out[:m, 3:51])
    near(out[:m, 3:51], x, xs, w, ws, b, "bf16")
    y = ops.w8a8_linear(x.view(m, 1, 256), xs.view(m, 1), w, ws, b)
    assert y.shape == (m, 1, 96) and torch.equal(y[:, 0], ops.w8a8_linear(x, xs, w, ws, b))
    for odd in (wide[:, 1:257], wide[:, 16:272].t().contiguous().t()):  # copied: any address, any order
        equal(ops.w8a8_linear(odd, xs, w, ws), odd, xs, w, ws, None, "bf16")
    assert ops.w8a8_linear(x[:0], xs[:0], w, ws).shape == (0, 96)
    assert ops.w8a8_gate_up_silu(x[:0], xs[:0], w, ws).shape == (0, 48)


@pytest.mark.parametrize("m", [4, 100])
def test_rows_without_a_scale(m):
    """NaN scales (rows that held a NaN) and zero scales stay in their rows."""
    x, xs, w, ws, b = make(m, 64, 256, seed=4)
    xs[1], xs[3] = float("nan"), 0.0
    x[1] = 0
    for y in (ops.w8a8_linear(x, xs, w, ws, b), ops.w8a8_gate_up_silu(x, xs, w, ws)):
        assert bool(y[1].isnan().all()) and not bool(y[[0, 2]].isnan().any()) and not bool(y[3:].isnan().any())
    assert torch.equal(ops.w8a8_linear(x, xs, w, ws, b)[3], b)


def test_without_its_workspace_one_slice():
    x, xs, w, ws, _ = make(40, 64, 9728, seed=6)
    lib = _lib.load()
    assert lib.sd_w8a8_workspace_size(40, 64, 9728, 0) > 0
    y = torch.empty((40, 64), dtype=torch.bfloat16, device=DEV)
    rc = lib.sd_w8a8_linear(x.data_ptr(), 9728, xs.data_ptr(), w.data_ptr(), 9728, ws.data_ptr(), _lib.SD_BF16, None,
                            y.data_ptr(), 64, 40, 64, 9728, _lib.SD_BF16, None, 0, _lib.stream_ptr(y.device))
    _lib.check(rc)
    assert torch.equal(y, ops.w8a8_linear(x, xs, w, ws))


@pytest.mark.parametrize("m", [7, 40, 150])
def test_graph_replays_and_streams(m):
    x, xs, w, ws, b = make(m, 192, 4096, seed=5)
    ops.w8a8_linear(x, xs, w, ws, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.w8a8_linear(x, xs, w, ws, b)
        gated = ops.w8a8_gate_up_silu(x, xs, w, ws, b)
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.w8a8_linear(x, xs, w, ws, b))
        assert torch.equal(gated, ops.w8a8_gate_up_silu(x, xs, w, ws, b))
        x.copy_(x.flip(0))
    torch.cuda.synchronize()
    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        y = ops.w8a8_linear(x, xs, w, ws, b)
    side.synchronize()
    assert torch.equal(y, ops.w8a8_linear(x, xs, w, ws, b))
