"""The route of few rows by the number of weight rows and columns: sums so long that a few workgroups would walk them
while the others idle are sliced over the device, all others stay with the kernel for few rows."""
import pytest
import torch

from specdec_nanovllm_amd import _lib


@pytest.fixture(autouse=True)
def of_256_compute_units():
    if torch.cuda.device_count() and torch.cuda.get_device_properties(0).multi_processor_count != 256:
        pytest.skip("the routes of 256 compute units")


def route(m, n, k, gated=0):
    """(tile rows, 0 for the kernel for few rows, K slices)"""
    lib = _lib.load()
    plan, ws = lib.sd_w8a8_plan(m, n, k, gated), lib.sd_w8a8_workspace_size(m, n, k, gated)
    rows = (plan >> 20) & 4095
    slices = plan & 255 if rows else 0
    assert ws == (slices * m * n * 4 * (1 + gated) if slices > 1 else 0)
    return rows, slices


@pytest.mark.parametrize("m,n,k", [(16, 512, 65536), (16, 2560, 28672), (16, 5120, 9728), (8, 1024, 28672), (5, 512, 65536),
                                   (4, 512, 65536), (1, 1024, 65536), (1, 512, 131056)])
def test_long_sums_are_sliced(m, n, k):
    assert route(m, n, k)[1] > 1
    assert route(m, n // 2, k, 1)[1] > 1


@pytest.mark.parametrize("m,n,k", [(1, 512, 16384), (1, 2560, 9728), (4, 4096, 28672), (16, 2560, 9728), (16, 512, 9728),
                                   (8, 9000, 4096), (16, 4096, 10240), (1, 151936, 1024), (4, 19456, 20480)])
def test_others_are_not(m, n, k):
    assert route(m, n, k) == (0, 0)
