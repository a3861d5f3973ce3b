"""The 8-bit operators at the ends of what they take: the most rows and outputs, matrices past 4 GiB, calls at once on two
streams, graphs that are replayed in turn, activations that are one row for all.

The linear equals the oracle's fp32 steps bit for bit (tests/test_gpu_w8a8.py), also where they are written in torch: sums
of 16 products stay below 2^24, exact in fp32 in any order, and without a bias the last step is one product.
"""
import pytest
import torch

import test_gpu_act_int8 as ta
import test_gpu_w8a8 as tw
from specdec_nanovllm_amd import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"


def codes(rows, k, seed):
    g = torch.Generator(device=DEV).manual_seed(seed)
    return torch.randint(-127, 128, (rows, k), generator=g, dtype=torch.int8, device=DEV)


def short(x, xs, w, ws):
    assert x.shape[1] <= 64
    return ((x.float() @ w.float().T * ws) * xs[:, None]).to(torch.bfloat16)


def test_most_rows():
    m = 1 << 24
    x, w = codes(m, 16, 1), codes(48, 16, 2)
    xs, ws = torch.rand(m, device=DEV) + 0.5, torch.rand(48, device=DEV) * 1e-3 + 1e-4
    got = ops.w8a8_linear(x, xs, w, ws)
    for r in range(0, m, 1 << 22):
        assert torch.equal(got[r:r + (1 << 22)], short(x[r:r + (1 << 22)], xs[r:r + (1 << 22)], w, ws))
    with pytest.raises(RuntimeError, match="too large"):
        ops.w8a8_linear(torch.cat((x, x[:1])), torch.cat((xs, xs[:1])), w, ws)


@pytest.mark.parametrize("m", [1, 4, 12, 40, 260])
def test_most_outputs(m):
    n = 1 << 21
    x, w = codes(m, 16, 3), codes(n, 16, 4)
    xs, ws = torch.rand(m, device=DEV) + 0.5, torch.rand(n, device=DEV) * 1e-3 + 1e-4
    assert torch.equal(ops.w8a8_linear(x, xs, w, ws), short(x, xs, w, ws))
    half = ops.w8a8_gate_up_silu(x, xs, w, ws)
    tw.near(half[:, -100:], x, xs, torch.cat((w[n // 2 - 100:n // 2], w[-100:])),
            torch.cat((ws[n // 2 - 100:n // 2], ws[-100:])), None, "bf16")


@pytest.mark.parametrize("m", [1, 20, 100])
def test_weights_past_4_gib(m):
    n, k = 600_000, 8192
    w = torch.empty((n, k), dtype=torch.int8, device=DEV)
    for r in range(0, n, 100_000):
        w[r:r + 100_000] = codes(100_000, k, 10 + r)
    x, xs, ws = codes(m, k, 5), torch.rand(m, device=DEV) + 0.5, torch.rand(n, device=DEV) * 1e-4 + 1e-5
    for f, rows in ((ops.w8a8_linear, n), (ops.w8a8_gate_up_silu, n // 2)):
        y = f(x, xs, w, ws)
        for at in (0, 262_100, rows - 50):  # 262 144 rows are 2 GiB
            if f is ops.w8a8_linear:
                tw.equal(y[:, at:at + 50], x, xs, w[at:at + 50], ws[at:at + 50], None, "bf16")
            else:
                tw.near(y[:, at:at + 50], x, xs, torch.cat((w[at:at + 50], w[rows + at:rows + at + 50])),
                        torch.cat((ws[at:at + 50], ws[rows + at:rows + at + 50])), None, "bf16")


def test_rows_and_outputs_past_4_gib():
    m, k = 600_000, 8192
    x = torch.empty((m, k), dtype=torch.int8, device=DEV)
    for r in range(0, m, 100_000):
        x[r:r + 100_000] = codes(100_000, k, 20 + r)
    xs, w, ws = torch.rand(m, device=DEV) + 0.5, codes(80, k, 6), torch.rand(80, device=DEV) * 1e-4 + 1e-5
    out = torch.full((m, 4096), 7.0, dtype=torch.bfloat16, device=DEV)  # 4.6 GiB, a part of each row written
    ops.w8a8_linear(x, xs, w, ws, out=out[:, 4000:4080])
    for at in (0, 262_100, 524_250, m - 50):
        tw.equal(out[at:at + 50, 4000:4080], x[at:at + 50], xs[at:at + 50], w, ws, None, "bf16")
        assert bool((out[at:at + 50, :4000] == 7).all()) and bool((out[at:at + 50, 4080:] == 7).all())
    back = ops.dequantize_rows_int8(x, xs)
    for at in (0, 262_100, m - 50):
        assert torch.equal(back[at:at + 50], (x[at:at + 50].float() * xs[at:at + 50, None]).to(torch.bfloat16))


def test_quantized_rows_past_4_gib():
    rows, k = 600_000, 4096
    x = torch.empty((rows, k), dtype=torch.bfloat16, device=DEV)
    for r in range(0, rows, 100_000):
        x[r:r + 100_000].normal_(generator=torch.Generator(device=DEV).manual_seed(r))
    w = ta.weight(k, "bf16")
    q, n = ops.quantize_rows_int8(x), ops.rmsnorm_int8(x, w, 1e-6, x)
    for at in (0, 262_100, 524_250, rows - 50):
        part = slice(at, at + 50)
        ta.check_quantized(x[part], q[0][part], q[1][part])
        ta.check_norm(x[part], w, tuple(t[part] for t in n), x[part])


def test_most_rows_of_activations():
    rows = (1 << 24) - 1
    x = torch.empty((rows, 16), dtype=torch.bfloat16, device=DEV).normal_()
    c, s = ops.quantize_rows_int8(x)
    ta.check_quantized(x[-5000:], c[-5000:], s[-5000:])
    want = x.float().abs().amax(-1).double() / 127  # (in fp32 torch multiplies by the rounded 1 / 127)
    assert bool(((s.double() - want).abs() <= 2.0**-24 * want).all())
    assert torch.equal(ops.dequantize_rows_int8(c, s), (c.float() * s[:, None]).to(torch.bfloat16))
    with pytest.raises(RuntimeError, match="rows below"):
        ops.quantize_rows_int8(torch.cat((x, x[:1])))


@pytest.mark.parametrize("m", [3, 30, 200])
def test_one_row_for_all(m):
    x, xs, w, ws, b = tw.make(1, 96, 512, seed=8)
    y = ops.w8a8_linear(x.expand(m, 512), xs.expand(m), w, ws, b)
    assert torch.equal(y, ops.w8a8_linear(x, xs, w, ws, b).expand(m, 96))
    c, s = ops.quantize_rows_int8(ta.make(1, 512, "bf16").expand(m, 512))
    assert torch.equal(c, c[:1].expand(m, 512)) and torch.equal(s, s[:1].expand(m))


def test_two_streams_at_once():
    """Calls in slices, whose sums pass through memory, side by side."""
    args = [tw.make(40, 64, 9728, seed=s) for s in (1, 2)]
    assert _lib.load().sd_w8a8_workspace_size(40, 64, 9728, 0) > 0
    want = [ops.w8a8_linear(*a) for a in args]
    streams = [torch.cuda.Stream() for _ in args]
    torch.cuda.synchronize()
    got = [[], []]
    for _ in range(20):
        for i, (a, s) in enumerate(zip(args, streams)):
            with torch.cuda.stream(s):
                got[i].append(ops.w8a8_linear(*a))
    torch.cuda.synchronize()
    assert all(torch.equal(y, w) for w, ys in zip(want, got) for y in ys)


def test_graphs_replayed_in_turn():
    args = [tw.make(40, 64, 9728, seed=s) for s in (3, 4)]
    graphs, out = [], []
    for a in args:
        ops.w8a8_linear(*a)
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g):
            out.append((ops.w8a8_linear(*a), ops.quantize_rows_int8(ops.w8a8_gate_up_silu(*a))))
        graphs.append(g)
    for _ in range(3):
        for a in args:
            a[0].copy_(a[0].flip(0))
        for g in graphs:
            g.replay()
        torch.cuda.synchronize()
        for a, (y, (c, s)) in zip(args, out):
            assert torch.equal(y, ops.w8a8_linear(*a))
            wc, ws = ops.quantize_rows_int8(ops.w8a8_gate_up_silu(*a))
            assert torch.equal(c, wc) and torch.equal(s, ws)


def test_out_may_not_be_an_input():
    x, xs, w, ws, b = tw.make(8, 64, 512)
    room = torch.zeros(8 * 64 + 64, dtype=torch.bfloat16, device=DEV)
    with pytest.raises(ValueError, match="shares memory"):
        ops.w8a8_linear(x, xs, w, ws, room[512 - 64:512], out=room[:512].view(8, 64))
    tw.equal(ops.w8a8_linear(x, xs, w, ws, room[512:], out=room[:512].view(8, 64)), x, xs, w, ws, room[512:], "bf16")
