"""What the 4-bit entries accept at the edges of their ranges, as far as the host decides it."""
import pytest
import torch

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


@pytest.mark.skipif(torch.cuda.device_count() > 0, reason="fake device addresses: only where no GPU can be reached")
@pytest.mark.parametrize("m,n,x_stride,w_stride,says", [
    (1, 64, 1 << 40, 512, "shares memory"),   # as far as the call gets: the stride is that of no second row
    (1, 1, 1 << 25, 1 << 40, "shares memory"),
    (2, 64, (1 << 24) + 8, 512, "too large"),
    (1, 2, 1024, (1 << 24) + 16, "too large"),
    (2, 64, 1 << 24, 1 << 24, "shares memory")])
def test_row_strides_count_where_there_are_rows(m, n, x_stride, w_stride, says):
    lib, at = _lib.load(), 0x10000000
    rc = lib.sd_w4a16_linear(at, x_stride, at << 4, w_stride, at << 3, _lib.SD_BF16, 128, None, at + 16, 4096, m, n,
                             1024, _lib.SD_BF16, None, 0, None)
    assert rc != 0 and says in lib.sd_last_error().decode()


def test_the_attention_layer_aligns_rows_that_start_anywhere():
    from specdec_nanovllm_amd.layers.attention import _aligned

    for t in (torch.empty(3 * 4 * 128 + 1, dtype=torch.bfloat16)[1:].view(3, 4, 128),
              torch.empty((3, 4, 129), dtype=torch.bfloat16)[..., :128],
              torch.empty((3, 128, 4), dtype=torch.bfloat16).transpose(1, 2)):
        t.copy_(torch.arange(t.numel()).view(t.shape) % 251)
        a = _aligned(t)
        assert a.data_ptr() % 16 == 0 and a.is_contiguous() and torch.equal(a, t)
    t = torch.empty((3, 4, 256), dtype=torch.bfloat16)[..., 128:]
    assert _aligned(t) is t  # a view of aligned rows stays one
