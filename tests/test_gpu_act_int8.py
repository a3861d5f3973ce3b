"""Activations in 8 bits (csrc/act_int8.hip through ``ops``) against the oracle.

Codes are equal. A scale without a norm is one correctly rounded division: 2^-24. With the norm, the sum of K squares
has at most 56 roundings in a row (8 or 32 of a thread's, 6 in the wave, 1 to 16 of the waves' sums), half of which pass
the root, then the mean, eps, root, inverse and two products: (28 + 8) 2^-24.
"""
import numpy as np
import pytest
import torch

from conftest import to_np
from oracle import w8a8 as o8
from specdec_nanovllm_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
EPS = 1e-6


def make(rows, k, kind, seed=0, std=1.0):
    g = torch.Generator().manual_seed(seed + rows * 7919 + k)
    x = torch.randn((rows, k), generator=g) * torch.exp(0.5 * torch.randn((k,), generator=g)) * std
    return x.to(DTYPES[kind]).to(DEV)


def weight(k, kind, seed=1):
    g = torch.Generator().manual_seed(seed)
    return (1 + 0.1 * torch.randn((k,), generator=g)).to(DTYPES[kind]).to(DEV)


def check_quantized(x, codes, scale):
    c, most = o8.codes(to_np(x.float()).reshape(-1, x.shape[-1]))
    assert codes.dtype == torch.int8 and scale.dtype == torch.float32
    assert np.array_equal(to_np(codes).reshape(c.shape), c)
    s = to_np(scale).astype(np.float64).reshape(-1)
    assert np.array_equal(np.isnan(s), np.isnan(most))
    ok = ~np.isnan(s)
    assert (np.abs(s - most / 127)[ok] <= 2.0**-24 * most[ok] / 127 + 2.0**-150).all()


def check_norm(x, w, got, residual=None, eps=EPS):
    k = x.shape[-1]
    codes, scale = got[:2]
    s, v = o8.norm_products(to_np(x.float()).reshape(-1, k), to_np(w.float()),
                            None if residual is None else to_np(residual.float()).reshape(-1, k))
    c, most = o8.codes(v)
    assert np.array_equal(to_np(codes).reshape(c.shape), c)
    want = o8.norm_scale(most, s, eps)
    have = to_np(scale).astype(np.float64).reshape(-1)
    assert np.array_equal(np.isnan(have), np.isnan(want))
    ok = ~np.isnan(want)
    assert (np.abs(have - want)[ok] <= 36 * 2.0**-24 * want[ok]).all()
    if residual is not None:
        assert torch.equal(got[2], (x.float() + residual.float()).to(x.dtype))


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("rows,k", [(1, 16), (3, 32), (5, 496), (4, 512), (7, 528), (1, 1024), (9, 1040), (2, 2048),
                                    (3, 2064), (5, 2560), (2, 4096), (3, 4112), (7, 9728), (2, 8192), (3, 8208),
                                    (2, 16384), (2, 16400), (3, 32768), (1000, 1024), (777, 2560)])
def test_rows_and_columns(kind, rows, k):
    x = make(rows, k, kind)
    check_quantized(x, *ops.quantize_rows_int8(x))
    w, r = weight(k, kind), make(rows, k, kind, seed=5)
    check_norm(x, w, ops.rmsnorm_int8(x, w, EPS))
    check_norm(x, w, ops.rmsnorm_int8(x, w, EPS, r), r)


@pytest.mark.parametrize("k", [496, 528, 1024, 1040, 2048, 2064, 4096, 4112, 9728])
def test_rows_do_not_depend_on_the_call(k):
    """Few rows take more threads each, sums of squares the same steps."""
    x, r, w = make(1030, k, "bf16"), make(1030, k, "bf16", seed=5), weight(k, "bf16")
    want, plain = ops.rmsnorm_int8(x, w, EPS, r), ops.quantize_rows_int8(x)
    for part in (slice(0, 1), slice(3, 10), slice(17, 529), slice(0, 513), slice(5, 1029)):
        assert all(torch.equal(a, b[part]) for a, b in zip(ops.rmsnorm_int8(x[part], w, EPS, r[part]), want))
        assert all(torch.equal(a, b[part]) for a, b in zip(ops.quantize_rows_int8(x[part]), plain))


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_ties_go_to_the_even_code(kind):
    """max |x| = 127 * 2^j: the quotients are x / 2^j, every half among them."""
    half = torch.arange(-254, 255, dtype=torch.float32) / 2
    x = torch.zeros((4, 512))
    x[:, :509] = half
    x = (x * torch.tensor([1.0, 2.0**-10, 2.0**6, 0.25])[:, None]).to(DTYPES[kind]).to(DEV)
    codes, scale = ops.quantize_rows_int8(x)
    check_quantized(x, codes, scale)
    assert torch.equal(codes[0, :509].cpu().long(), torch.round(half.double()).long())


def test_quotients_next_to_a_tie():
    """Rows whose products with the weight have 24 bits, quotients within 2^-16 of n + 1/2 among them."""
    g = torch.Generator().manual_seed(3)
    x = torch.randn((64, 4096), generator=g).half().to(DEV)
    w = (torch.rand((4096,), generator=g) + 0.5).half().to(DEV)
    _, v = o8.norm_products(to_np(x.float()), to_np(w.float()))
    q = 127 * v.astype(np.float64) / np.abs(v).max(-1, keepdims=True)
    assert (np.abs(np.abs(q - np.rint(q)) - 0.5) < 2.0**-16).any()
    check_norm(x, w, ops.rmsnorm_int8(x, w, EPS))


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_zeros_nan_and_infinities(kind):
    x = make(8, 1040, kind)
    x[1] = 0
    x[2, 1039] = float("nan")
    x[3, 0] = float("inf")
    x[4, 500] = -float("inf")
    x[5] = -0.0
    codes, scale = ops.quantize_rows_int8(x)
    check_quantized(x, codes, scale)
    assert float(scale[1]) == 0 and bool(scale[2:5].isnan().all()) and float(scale[5]) == 0
    w = weight(1040, kind)
    for eps in (EPS, 0.0):
        codes, scale = ops.rmsnorm_int8(x, w, eps)
        assert float(scale[1]) == 0 and float(scale[5]) == 0  # also 0 / 0
        assert bool(scale[2:5].isnan().all()) and bool((codes[1:6] == 0).all())
        check_norm(x[[0, 6, 7]], w, (codes[[0, 6, 7]], scale[[0, 6, 7]]), eps=eps)


@pytest.mark.parametrize("kind,std", [("bf16", 1e-38), ("bf16", 1e-20), ("bf16", 1e36), ("fp16", 1e-6), ("fp16", 2e4)])
def test_small_and_large_values(kind, std):
    x = make(5, 768, kind, std=std).clamp(torch.finfo(DTYPES[kind]).min, torch.finfo(DTYPES[kind]).max)
    check_quantized(x, *ops.quantize_rows_int8(x))


def test_squares_past_fp32_give_zeros_as_rmsnorm():
    x = make(2, 512, "bf16", std=1e30)
    w = weight(512, "bf16")
    codes, scale = ops.rmsnorm_int8(x, w, EPS)
    assert bool((ops.rmsnorm(x, w, EPS) == 0).all()) and bool((scale == 0).all())


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("rows,k", [(1, 16), (3, 2048), (5, 2064), (130, 1040), (3, 9728)])
def test_read_back(kind, rows, k):
    codes, scale = ops.quantize_rows_int8(make(rows, k, kind))
    want = to_np(codes).astype(np.float64) * to_np(scale).astype(np.float64)[:, None]
    for dt in (torch.bfloat16, torch.float16, torch.float32):
        got = ops.dequantize_rows_int8(codes, scale, dt)
        assert got.dtype == dt and got.shape == codes.shape
        half = float(torch.finfo(dt).eps) / 2 + (2.0**-24 if dt != torch.float32 else 0)
        assert (np.abs(to_np(got).astype(np.float64) - want) <= half * np.abs(want) + 2.0**-25).all()
    # a row is off by half a level and the value's roundings at most
    x = make(rows, k, kind)
    back = to_np(ops.dequantize_rows_int8(codes, scale, torch.float32)).astype(np.float64)
    s = to_np(scale).astype(np.float64)[:, None]
    assert (np.abs(back - to_np(x.float()).astype(np.float64)) <= 0.5 * s + 3 * 2.0**-24 * 127 * s).all()


def test_strides_batches_and_empty():
    x = make(6, 1024, "bf16")
    wide = torch.full((6, 1200), float("nan"), dtype=torch.bfloat16, device=DEV)
    wide[:, 8:1032] = x
    want = ops.quantize_rows_int8(x)
    for view in (wide[:, 8:1032], wide[:, 8:1032].clone().t().contiguous().t(), x.view(2, 3, 1024)):
        got = ops.quantize_rows_int8(view)
        assert got[0].shape == view.shape and got[1].shape == view.shape[:-1]
        assert torch.equal(got[0].view(6, -1), want[0]) and torch.equal(got[1].view(6), want[1])
    odd = torch.zeros(6 * 1024 + 3, dtype=torch.bfloat16, device=DEV)[3:].view(6, 1024)  # starts anywhere
    odd.copy_(x)
    assert torch.equal(ops.quantize_rows_int8(odd)[0], want[0])
    w, r = weight(1024, "bf16"), make(6, 1024, "bf16", seed=9)
    want = ops.rmsnorm_int8(x, w, EPS, r)
    wide[:, 8:1032] = r
    got = ops.rmsnorm_int8(x.view(3, 2, 1024), w.float(), EPS, wide[:, 8:1032].view(3, 2, 1024))
    assert all(torch.equal(a.reshape(-1), b.reshape(-1)) for a, b in zip(got, want))
    assert got[0].shape == (3, 2, 1024) and got[1].shape == (3, 2) and got[2].shape == (3, 2, 1024)
    back = ops.dequantize_rows_int8(want[0].view(3, 2, 1024), want[1].view(3, 2))
    assert torch.equal(back.view(6, 1024), ops.dequantize_rows_int8(want[0], want[1]))
    for t in (ops.quantize_rows_int8(x[:0]), ops.rmsnorm_int8(x[:0], w, EPS, r[:0])):
        assert t[0].shape == (0, 1024) and t[1].shape == (0,)
    assert ops.dequantize_rows_int8(want[0][:0], want[1][:0]).shape == (0, 1024)
    one = ops.quantize_rows_int8(x[0])  # a vector
    assert one[0].shape == (1024,) and one[1].shape == ()


def test_graph_replays():
    x, w, r = make(5, 2560, "bf16"), weight(2560, "bf16"), make(5, 2560, "bf16", seed=3)
    ops.rmsnorm_int8(x, w, EPS, r)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = ops.rmsnorm_int8(x, w, EPS, r)
        back = ops.dequantize_rows_int8(got[0], got[1])
    for _ in range(3):
        graph.replay()
        torch.cuda.synchronize()
        want = ops.rmsnorm_int8(x, w, EPS, r)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        assert torch.equal(back, ops.dequantize_rows_int8(want[0], want[1]))
        x.mul_(1.5)
        r.copy_(x.flip(0))
