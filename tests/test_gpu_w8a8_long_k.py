"""Few rows with sums so long that they are sliced over the device (w8a8_linear, w8a8_gate_up_silu), with the workspace and
without: the oracle's fp32 steps bit for bit, as in tests/test_gpu_w8a8.py, which derives SiLU's tolerance too."""
import pytest
import torch

import test_gpu_w8a8 as tw
from specdec_nanovllm_amd import _lib, ops

pytestmark = pytest.mark.gpu
SHAPES = [(1, 512, 65536), (1, 30, 131056), (2, 1024, 28672), (4, 512, 20496), (5, 254, 16400), (8, 1024, 28672),
          (16, 2560, 14352), (16, 5120, 9728), (16, 514, 65536), (12, 100, 131056), (3, 96, 16384), (3, 96, 16400)]


@pytest.mark.parametrize("m,n,k", SHAPES)
def test_long_sums(m, n, k):
    x, xs, w, ws, b = tw.make(m, n, k)
    tw.equal(ops.w8a8_linear(x, xs, w, ws, b), x, xs, w, ws, b, "bf16")
    tw.near(ops.w8a8_gate_up_silu(x, xs, w, ws, b), x, xs, w, ws, b, "bf16")
    tw.equal(ops.w8a8_linear(x, xs, w[:n - 1], ws[:n - 1]), x, xs, w[:n - 1], ws[:n - 1], None, "bf16")


@pytest.mark.parametrize("m", [1, 16])
def test_without_a_workspace(m):
    """The same bits, from the kernel for few rows."""
    x, xs, w, ws, _ = tw.make(m, 512, 65536)
    lib, y = _lib.load(), torch.empty((m, 512), dtype=torch.bfloat16, device=x.device)
    assert lib.sd_w8a8_workspace_size(m, 512, 65536, 0) > 0
    _lib.check(lib.sd_w8a8_linear(x.data_ptr(), 65536, xs.data_ptr(), w.data_ptr(), 65536, ws.data_ptr(), _lib.SD_BF16,
                                  None, y.data_ptr(), 512, m, 512, 65536, _lib.SD_BF16, None, 0, _lib.stream_ptr(y.device)))
    assert torch.equal(y, ops.w8a8_linear(x, xs, w, ws))


def test_one_row_of_a_strided_tensor():
    """A single row's stride counts nothing."""
    x, xs, w, ws, b = tw.make(1, 256, 28672)
    wide = torch.zeros((2, 1 << 24), dtype=torch.int8, device=x.device)[::2]
    wide[:, :28672] = x
    got = ops.w8a8_linear(wide[:, :28672], xs, w, ws, b)
    tw.equal(got, x, xs, w, ws, b, "bf16")


def test_graph_replays():
    x, xs, w, ws, b = tw.make(4, 512, 65536)
    ops.w8a8_linear(x, xs, w, ws, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = ops.w8a8_linear(x, xs, w, ws, b)
    for _ in range(3):
        x.copy_(x.flip(0))
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(out, ops.w8a8_linear(x, xs, w, ws, b))
