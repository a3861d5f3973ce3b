"""The 4-bit KV cache (csrc/int4_cache.hip through ``ops``) against the 64-bit oracle.

Tolerances: a rounding to the 16-bit type moves a value by at most half a step, eps / 2 of it; fp32
intermediates add 2^-24 each. A code is the nearest level of the row's own (stored) scale and zero:
its quotient, taken in fp32 from an exact input, is off by at most 2^-22 * 15 < 2^-18 levels. A
rotated key is one fp32 chain of 15 roundings or less (squares over 16 lanes of 8: 12 of them halve
in the square root; rsqrt 2; products and the sum 7), below 2^-20 (|a| + |b|) for the two dims of its
pair.
"""
import numpy as np
import pytest
import torch

from oracle import int4 as o4
from specdec_nanovllm_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


def f64(t):
    return t.detach().double().cpu().numpy()


def rand(shape, kind, seed, std=1.0):
    g = torch.Generator().manual_seed(seed)
    return (torch.randn(shape, generator=g) * std).to(DTYPES[kind]).to(DEV)


def make_cache(blocks, page, heads, group, kind, interleaved=False):
    codes, scales = ops.int4_kvcache(blocks, page, heads, group, DTYPES[kind])
    if interleaved:
        codes, scales = codes.contiguous(), scales.contiguous()
    return codes, scales


def rows_at(codes, scales, slots):
    page = codes.shape[1]
    s = slots.long().cpu()
    return codes.cpu()[s // page, s % page].numpy(), f64(scales)[s // page, s % page]


def check_rows(codes, scales, x, err, kind, part):
    """Stored codes and scales (rows) against the exact values x, each known to ``err``."""
    eps = float(torch.finfo(DTYPES[kind]).eps)
    tiny = float(torch.finfo(DTYPES[kind]).smallest_normal) * eps
    ng = scales.shape[-1] // 4
    sz = scales[..., 2 * ng * part:2 * ng * (part + 1)]
    dims = o4.key_dim if part == 0 else o4.value_dim
    c = o4.unpack(codes[..., 64 * part:64 * part + 64], dims).reshape(*x.shape[:-1], ng, -1)
    xg, eg = x.reshape(c.shape), err.reshape(c.shape)
    s, z = sz[..., 0::2], sz[..., 1::2]
    lo, hi, e = xg.min(-1), xg.max(-1), eg.max(-1)
    assert (np.abs(z - lo) <= eps / 2 * np.abs(lo) + 1.01 * e + tiny).all(), "zero"
    want = np.maximum(hi - z, 0) / 15
    assert (np.abs(s - want) <= eps / 2 * (1 + 2**-10) * want + e / 7 + tiny).all(), "scale"
    safe = np.where(s > 0, s, 1)[..., None]
    level = np.clip((xg - z[..., None]) / safe, 0, 15) * (s > 0)[..., None]
    assert (np.abs(c - level) <= 0.5 + 2**-18 + eg / safe).all(), "code"


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("tokens,heads,page,interleaved", [(1, 1, 16, False), (37, 8, 16, True),
                                                           (300, 3, 48, False)])
def test_store_and_load(kind, group, tokens, heads, page, interleaved):
    k, v = rand((tokens, heads, 128), kind, 1, 3.0), rand((tokens, heads, 128), kind, 2)
    k[0, 0, 5] = 40.0
    v[-1, -1] = 0.75  # a constant row: scale 0
    v[0, 0, :32] = 0
    blocks = -(-tokens // page) + 2
    codes, scales = make_cache(blocks, page, heads, group, kind, interleaved)
    slots = torch.randperm(blocks * page, generator=torch.Generator().manual_seed(3))[:tokens]
    slots = slots.to(torch.int32).to(DEV)
    ops.store_kvcache_int4(k, v, codes, scales, slots)
    c, s = rows_at(codes, scales, slots)
    zero = np.zeros((tokens, heads, 128))
    check_rows(c, s, f64(k), zero, kind, 0)
    check_rows(c, s, f64(v), zero, kind, 1)
    untouched = torch.ones(blocks * page, dtype=torch.bool)
    untouched[slots.long().cpu()] = False
    assert int(codes.cpu().reshape(blocks * page, -1)[untouched].abs().max()) == 0
    eps = float(torch.finfo(DTYPES[kind]).eps)
    got = ops.load_kvcache_int4(codes, scales, slots)
    for g, want in zip(got, o4.values(c, s)):
        tol = np.abs(want) * (eps / 2 + 2**-23) + float(torch.finfo(DTYPES[kind]).smallest_normal) * eps
        assert (np.abs(f64(g) - want) <= tol).all()


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("tokens,hq,hkv,norm,key_out", [(1, 16, 8, True, True), (7, 32, 8, False, False),
                                                        (611, 32, 8, True, True), (33, 5, 5, True, True)])
def test_append(kind, group, tokens, hq, hkv, norm, key_out):
    eps_t, page = float(torch.finfo(DTYPES[kind]).eps), 64
    qkv = rand((tokens, (hq + 2 * hkv) * 128), kind, 4)
    q, k, v = (x.unflatten(-1, (-1, 128)) for x in qkv.split([hq * 128, hkv * 128, hkv * 128], -1))
    before = qkv.clone()
    qw, kw = (1 + rand((128,), kind, 5, 0.2), 1 + rand((128,), kind, 6, 0.2)) if norm else (None, None)
    angles = torch.arange(2000, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(64).double() / 64)
    cs = torch.cat((angles.cos(), angles.sin()), -1).float().to(DEV)
    pos = torch.randint(0, 2000, (tokens,), generator=torch.Generator().manual_seed(7))
    if tokens > 4:
        pos[2], pos[3] = 2000, -1  # no row in the table: not rotated
    blocks = -(-tokens // page) + 1
    codes, scales = make_cache(blocks, page, hkv, group, kind)
    slots = torch.randperm(blocks * page, generator=torch.Generator().manual_seed(8))[:tokens].to(torch.int32)
    if tokens > 4:
        slots[1] = -1
    qo, ko = ops.qk_norm_rope_store_int4(q, k, v, pos.to(DEV), cs, codes, scales, slots.to(DEV), qw, kw,
                                         1e-6, key_out=key_out)
    assert torch.equal(qkv, before), "the projection's output is left as it was"
    assert (ko is None) == (not key_out)
    inside = (pos >= 0) & (pos < 2000)
    row = f64(cs)[np.where(inside, pos, 0)]
    cos = np.where(inside[:, None], row[:, :64], 1.0)
    sin = np.where(inside[:, None], row[:, 64:], 0.0)
    exact = {}
    for name, x, w in (("q", q, qw), ("k", k, kw)):
        wn = None if w is None else f64(w)
        y = o4.norm_rotate(f64(x), wn, 1e-6, cos, sin)
        flat = o4.norm_rotate(f64(x), wn, 1e-6, np.ones_like(cos), np.zeros_like(sin))
        size = np.tile(np.abs(flat[..., :64]) + np.abs(flat[..., 64:]), 2)
        exact[name] = y, 2**-20 * size
    for name, got in (("q", qo), ("k", ko)):
        if got is None:
            continue
        y, err = exact[name]
        assert (np.abs(f64(got) - y) <= eps_t / 2 * np.abs(y) + 1.01 * err + 1e-7).all(), name
    kept = slots >= 0
    c, s = rows_at(codes, scales, slots[kept])
    y, err = exact["k"]
    check_rows(c, s, y[kept.numpy()], err[kept.numpy()], kind, 0)
    check_rows(c, s, f64(v)[kept.numpy()], np.zeros_like(y[kept.numpy()]), kind, 1)


def test_load_of_absent_rows_is_zero():
    codes, scales = make_cache(2, 16, 4, 64, "bf16")
    codes.fill_(255)
    scales.fill_(1.0)
    k, v = ops.load_kvcache_int4(codes, scales, torch.tensor([-1, 5, 32, 31], dtype=torch.int32, device=DEV))
    for t in (k, v):
        assert f64(t)[[0, 2]].any() == False and (f64(t)[[1, 3]] == 16).all()  # noqa: E712


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_group_that_is_not_finite_comes_back_as_nan(bad):
    k, v = rand((2, 2, 128), "bf16", 9), rand((2, 2, 128), "bf16", 10)
    k[1, 0, 40] = bad
    v[0, 1, 127] = bad
    codes, scales = make_cache(1, 16, 2, 32, "bf16")
    slots = torch.tensor([3, 4], dtype=torch.int32, device=DEV)
    ops.store_kvcache_int4(k, v, codes, scales, slots)
    kk, vv = ops.load_kvcache_int4(codes, scales, slots)
    nan_k, nan_v = torch.zeros(2, 2, 128, dtype=torch.bool), torch.zeros(2, 2, 128, dtype=torch.bool)
    nan_k[1, 0, 32:64] = True
    nan_v[0, 1, 96:] = True
    assert torch.equal(kk.isnan().cpu(), nan_k) and torch.equal(vv.isnan().cpu(), nan_v)


def test_values_halfway_between_two_codes_go_to_the_even_one():
    x = torch.zeros((1, 1, 128))
    x[0, 0, :31] = torch.arange(31) * 0.5  # scale 1: every other value lies between two codes
    k = x.to(torch.bfloat16).to(DEV)
    codes, scales = make_cache(1, 16, 1, 32, "bf16")
    slots = torch.zeros(1, dtype=torch.int32, device=DEV)
    ops.store_kvcache_int4(k, k, codes, scales, slots)
    for t in ops.load_kvcache_int4(codes, scales, slots):
        assert torch.equal(t.float().cpu()[0, 0, :31], torch.round(x[0, 0, :31]))


def test_a_captured_append_follows_its_inputs():
    kind, tokens = "bf16", 5
    q, k, v = (rand((tokens, h, 128), kind, i) for i, h in ((11, 4), (12, 2), (13, 2)))
    angles = torch.arange(64.0)[:, None] * torch.rand(64, generator=torch.Generator().manual_seed(1))
    cs = torch.cat((angles.cos(), angles.sin()), -1).to(DEV)
    pos, slots = torch.arange(tokens, device=DEV), torch.arange(tokens, dtype=torch.int32, device=DEV)
    codes, scales = make_cache(1, 16, 2, 64, kind)

    def step():
        qk = ops.qk_norm_rope_store_int4(q, k, v, pos, cs, codes, scales, slots)
        return (*qk, *ops.load_kvcache_int4(codes, scales, slots))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    for i in range(3):
        for t, s in ((q, 20), (k, 30), (v, 40)):
            t.copy_(rand(t.shape, kind, s + i))
        graph.replay()
        torch.cuda.synchronize()
        got = [t.clone() for t in out]
        for a, b in zip(got, step()):
            assert torch.equal(a, b)
