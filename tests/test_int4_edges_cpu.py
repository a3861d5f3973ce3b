"""What the 4-bit entries accept at the edges of their ranges, as far as the host decides it."""
import pytest

from specdec_nanovllm_amd import _lib


@pytest.mark.parametrize("m", [1, 2, 3, 8])
@pytest.mark.parametrize("n", [1, 37, 4096, 16384, 151936, 1 << 21])
def test_few_rows_need_a_workspace_only_past_512_groups(m, n):
    """``ops.w4a16_linear`` does not ask up to there."""
    f = _lib.load().sd_w4a16_workspace_size
    for group in (32, 64, 96, 128, 1024):
        for groups in (1, 2, 15, 100, 511, 512):
            if group * groups <= 1 << 20:
                assert f(m, n, group * groups, group) == 0
    assert f(m, 37, 1 << 17, 32) > 0
