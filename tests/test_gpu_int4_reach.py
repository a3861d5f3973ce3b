"""The 4-bit operators where sizes, streams and graphs reach further than one small call: caches and
weights past 4 GB, the tile widths that only many rows and columns take, tensors made on another stream,
graphs that share a workspace, padded batches.

Large caches are written and read back, which compares stored values with their own quantization:
half a level of the group's range, and the 16-bit rounding of scale and zero (eps / 2 of each, the scale's
15 times) and of the value. Everything else is compared bit for bit with the same call on small
tensors, or as in the operators' own tests.
"""
import numpy as np
import pytest
import torch

from oracle import int4 as o4
from specdec_nanovllm_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
SCALE = 128 ** -0.5


def f64(t):
    return t.detach().double().cpu().numpy()


def rand(shape, seed, dtype=torch.bfloat16):
    g = torch.Generator().manual_seed(seed)
    return torch.randn(shape, generator=g).to(dtype).to(DEV)


def check_linear(got, x, w, s, eps=2.0**-7):
    """As tests/test_gpu_w4a16.py: the output's rounding and the fp32 sums."""
    wx, sx = o4.weights(w.cpu().numpy(), f64(s)), np.repeat(f64(s), 2 * w.shape[1] // s.shape[1], -1)
    want, size = f64(x) @ wx.T, 55 * np.abs(f64(x)) @ np.abs(sx).T
    tol = eps / 2 * np.abs(want) + (36 + 4 * s.shape[1] + 16) * 2**-24 * size + 1e-7
    assert (np.abs(f64(got) - want) <= tol).all()


@pytest.mark.parametrize("n,cols", [(16300, 128), (24500, 192), (32760, 256), (33000, 256)])
@pytest.mark.parametrize("k,group", [(128, 128), (192, 64), (96, 32)])
def test_wide_tiles(n, cols, k, group):
    """Two row tiles whose second has 2 rows; columns past the last whole tile and, at 33000, past one
    round of ``cols`` columns; half a block of columns with group 64."""
    g = torch.Generator().manual_seed(n)
    w = torch.randint(0, 256, (n, k // 2), generator=g, dtype=torch.uint8).to(DEV)
    s = ((torch.rand((n, k // group), generator=g) + 0.2) * 0.02).to(torch.bfloat16).to(DEV)
    x = rand((130, k), 1)
    check_linear(ops.w4a16_linear(x, w, s), x, w, s)
    out = torch.full((130, n + 3), 7.0, dtype=torch.bfloat16, device=DEV)  # odd stride and start
    ops.w4a16_linear(x, w, s, out=out[:, 1:n + 1])
    check_linear(out[:, 1:n + 1], x, w, s)
    assert bool((out[:, 0] == 7).all()) and bool((out[:, n + 1:] == 7).all())


@pytest.mark.parametrize("m", [1, 7, 20])
@pytest.mark.parametrize("k", [1 << 15, 1 << 17])
def test_scales_that_fill_the_lds(m, k):
    """A row of 1024 groups of 32 leaves room for few waves; of 4096, for none."""
    g = torch.Generator().manual_seed(k)
    w = torch.randint(0, 256, (37, k // 2), generator=g, dtype=torch.uint8).to(DEV)
    s = ((torch.rand((37, k // 32), generator=g) + 0.2) * 0.02).to(torch.bfloat16).to(DEV)
    x = rand((m, k), 8)
    check_linear(ops.w4a16_linear(x, w, s), x, w, s)


@pytest.mark.parametrize("m", [1, 20, 100])
def test_weights_past_4_gb(m):
    n, k, group = 1 << 21, 4608, 512
    w = torch.randint(0, 256, (n, k // 2), dtype=torch.uint8, device=DEV)  # 4.8 GB
    s = (torch.rand((n, k // group), device=DEV) * 0.02 + 0.004).to(torch.bfloat16)
    x = rand((m, k), 2)
    y = ops.w4a16_linear(x, w, s)
    for at in (0, (1 << 32) // (k // 2) - 20, n - 40):
        rows = slice(at, at + 40)
        check_linear(y[:, rows], x, w[rows], s[rows])


def test_a_cache_past_4_gb():
    page, heads, group = 256, 8, 32
    blocks = (1 << 32) // (page * heads * 128) + 40  # 4.3 GB of codes, 1.1 GB of scales
    codes, scales = ops.int4_kvcache(blocks, page, heads, group)
    small, small_s = ops.int4_kvcache(4, page, heads, group)
    far = torch.tensor([blocks - 1, blocks - 17, 3, blocks - 30], dtype=torch.int32, device=DEV)
    near = torch.arange(4, dtype=torch.int32, device=DEV)
    place = torch.arange(4 * page, device=DEV)

    def slots(table):
        return (table[place // page].long() * page + place % page).to(torch.int32)

    k, v, q = rand((4 * page, heads, 128), 3), rand((4 * page, heads, 128), 4), rand((4 * page, 16, 128), 5)
    angles = torch.arange(64.0)[:, None] * torch.rand(64, generator=torch.Generator().manual_seed(1))
    cs = torch.cat((angles.cos(), angles.sin()), -1).to(DEV)
    pos = place % 64
    ops.store_kvcache_int4(k, v, codes, scales, slots(far))
    kk, vv = ops.load_kvcache_int4(codes, scales, slots(far))
    for got, x in ((kk, k), (vv, v)):
        xs, off = f64(x).reshape(-1, 4, 32), np.abs(f64(got) - f64(x)).reshape(-1, 4, 32)
        span, high = xs.max(-1) - xs.min(-1), np.abs(xs).max(-1)
        eps = 2.0**-7
        allowed = (span / 30) * (1 + eps) + eps / 2 * (span + 2 * high)
        assert (off.max(-1) <= allowed).all()
    for table, (c, s) in ((far, (codes, scales)), (near, (small, small_s))):
        ops.qk_norm_rope_store_int4(q, k, v, pos, cs, c, s, slots(table), key_out=False)
    for a, b in zip(ops.load_kvcache_int4(codes, scales, slots(far)),
                    ops.load_kvcache_int4(small, small_s, slots(near))):
        assert torch.equal(a, b)
    lens = torch.tensor([4 * page - 3], dtype=torch.int32, device=DEV)
    for rows in (1, 3):
        cuq = torch.tensor([0, rows], dtype=torch.int32, device=DEV)
        out = [ops.paged_attention_int4(q[:rows], c, s, t[None], SCALE, context_lens=lens, cu_seqlens_q=cuq,
                                        max_seqlen_q=rows)
               for t, (c, s) in ((far, (codes, scales)), (near, (small, small_s)))]
        assert torch.equal(*out) and bool(out[0].isfinite().all())


def _decode(lens, seed):
    """A small cache filled by its own store, a table and a query for ``lens``."""
    page, heads = 64, 4
    width = -(-max(lens) // page)
    codes, scales = ops.int4_kvcache(len(lens) * width, page, heads, 64)
    n = len(lens) * width * page
    ops.store_kvcache_int4(rand((n, heads, 128), seed), rand((n, heads, 128), seed + 1), codes, scales,
                           torch.arange(n, dtype=torch.int32, device=DEV))
    table = torch.arange(len(lens) * width, dtype=torch.int32, device=DEV).view(len(lens), width)
    return rand((len(lens), 16, 128), seed + 2), codes, scales, table, torch.tensor(lens, dtype=torch.int32, device=DEV)


def test_tensors_of_another_stream():
    q, codes, scales, table, lens = _decode([3000, 100], 6)
    w = torch.randint(0, 256, (2560, 1024), dtype=torch.uint8, device=DEV)
    s = (torch.rand((2560, 16), device=DEV) * 0.02).to(torch.bfloat16)
    x = rand((200, 2048), 7)
    want = (ops.paged_attention_int4(q, codes, scales, table, SCALE, context_lens=lens), ops.w4a16_linear(x, w, s))
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    for _ in range(4):  # both at once: neither stream's workspace is the other's
        with torch.cuda.stream(side):
            a = (ops.paged_attention_int4(q, codes, scales, table, SCALE, context_lens=lens),
                 ops.w4a16_linear(x, w, s))
        b = (ops.paged_attention_int4(q, codes, scales, table, SCALE, context_lens=lens), ops.w4a16_linear(x, w, s))
        torch.cuda.synchronize()
        for got in (a, b):
            assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])


def test_two_graphs_and_eager_calls_between():
    sets = [_decode([2000, 900, 17], 20), _decode([4000], 30)]
    w = torch.randint(0, 256, (1024, 512), dtype=torch.uint8, device=DEV)
    s = (torch.rand((1024, 8), device=DEV) * 0.02).to(torch.bfloat16)
    xs = [rand((40, 1024), 40), rand((150, 1024), 41)]

    def step(i):
        q, codes, scales, table, lens = sets[i]
        return (ops.paged_attention_int4(q, codes, scales, table, SCALE, context_lens=lens),
                ops.w4a16_linear(xs[i], w, s))

    side = torch.cuda.Stream()
    with torch.cuda.stream(side):
        step(0), step(1)
    torch.cuda.synchronize()
    graphs, outs = [], []
    for i in (0, 1):
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[i]):
            outs.append(step(i))
    for r in range(3):
        for i in (0, 1):
            sets[i][0].mul_(1.25)
            xs[i].add_(0.125)
        graphs[0].replay()
        graphs[1].replay()
        got = [[t.clone() for t in o] for o in outs]
        for i in (0, 1):
            assert all(torch.equal(a, b) for a, b in zip(got[i], step(i))), (r, i)
        graphs[1].replay()
        graphs[0].replay()
        torch.cuda.synchronize()
        for i in (0, 1):
            assert all(torch.equal(a, b) for a, b in zip(got[i], outs[i])), (r, i)


def test_a_padded_batch():
    """Rows that only fill a captured batch: no context, an unused table, slot -1."""
    q, codes, scales, table, lens = _decode([700, 65], 50)
    want = ops.paged_attention_int4(q, codes, scales, table, SCALE, context_lens=lens)
    kept = (codes.clone(), scales.clone())
    q4 = torch.cat((q, torch.full_like(q, float("nan"))))
    t4 = torch.cat((table, torch.full_like(table, -1)))
    l4 = torch.cat((lens, torch.zeros_like(lens)))
    got = ops.paged_attention_int4(q4, codes, scales, t4, SCALE, context_lens=l4)
    assert torch.equal(got[:2], want) and bool((got[2:] == 0).all())
    k = torch.full((4, 4, 128), float("nan"), dtype=torch.bfloat16, device=DEV)
    ops.store_kvcache_int4(k, k, codes, scales, torch.full((4,), -1, dtype=torch.int32, device=DEV))
    assert torch.equal(codes, kept[0]) and torch.equal(scales, kept[1])
