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


def test_a_cached_prefix_is_read_back_as_far_as_there_are_keys(monkeypatch):
    """A table as wide as the longest sequence that may come is not read to its end."""
    from specdec_nanovllm_amd import ops
    from specdec_nanovllm_amd.layers.attention import Attention
    from specdec_nanovllm_amd.utils.context import reset_context, set_context

    page, heads, asked = 16, 2, {}

    def load(codes, scales, slots):
        asked["slots"] = slots
        return torch.zeros((slots.numel(), heads, 128)), torch.zeros((slots.numel(), heads, 128))

    def prefill(q, k, v, cu_q, cu_k, n, scale, block_table):
        asked["k"], asked["table"] = k, block_table
        return q

    monkeypatch.setattr(ops, "load_kvcache_int4", load)
    monkeypatch.setattr(ops, "prefill_attention", prefill)
    monkeypatch.setattr(ops, "store_kvcache_int4", lambda *a: None)
    layer = Attention(4, 128, 0.1, heads)
    layer.k_cache, layer.v_cache = ops.int4_kvcache(9, page, heads, device="cpu")
    table = torch.full((2, 1000), -1, dtype=torch.int32)
    table[0, :3], table[1, :2] = torch.tensor([7, 1, 4], dtype=torch.int32), torch.tensor([0, 8], dtype=torch.int32)
    cu_q, cu_k = torch.tensor([0, 20, 40]), torch.tensor([0, 41, 41 + 24])
    q, k = torch.zeros((40, 4, 128)), torch.zeros((40, heads, 128))
    try:
        set_context(True, cu_q, cu_k, 20, 41, torch.zeros(40, dtype=torch.int32), None, table)
        layer(q, k, k)
    finally:
        reset_context()
    rows = torch.arange(page)
    want = torch.stack([torch.cat([b * page + rows if b >= 0 else torch.full((page,), -1) for b in seq])
                        for seq in ([7, 1, 4], [0, 8, -1])])
    assert torch.equal(asked["slots"].reshape(2, -1).long(), want)
    assert asked["k"].shape == (6, page, heads, 128)
    assert torch.equal(asked["table"], torch.arange(6, dtype=torch.int32).view(2, 3))


@pytest.mark.parametrize("group", [0, -32])
def test_apply_int4_quant_refuses_groups_of_no_columns(group):
    from specdec_nanovllm_amd.layers.linear import ReplicatedLinear
    from specdec_nanovllm_amd.layers.quant import apply_int4_quant

    m = torch.nn.ModuleDict(dict(a=ReplicatedLinear(64, 8)))
    m["a"].weight.data = torch.zeros((8, 64), dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="multiple of 32"):
        apply_int4_quant(m, ["a"], group)
    assert m["a"].weight.dtype == torch.bfloat16


def test_w4a16_plans_agree_with_their_workspaces():
    lib = _lib.load()
    for m in (1, 3, 9, 17, 40, 66, 130, 777, 5000):
        for n, k, group in ((1, 32, 32), (2570, 9728, 64), (4100, 1312, 32), (19456, 2560, 128), (1 << 21, 128, 128)):
            plan, need = lib.sd_w4a16_plan(m, n, k, group), lib.sd_w4a16_workspace_size(m, n, k, group)
            rows, columns, parts = plan >> 20, plan >> 8 & 0xfff, plan & 0xff
            if rows:
                assert (rows, columns) in ((32, 64), (32, 128), (64, 64), (64, 128), (128, 128), (128, 192), (128, 256))
                assert 1 <= parts <= 16 and need == (parts * m * n * 4 if parts > 1 else 0)
            else:
                assert m <= 32 and columns in (16, 32) and 1 <= parts <= 16 and need == 0
    for bad in ((0, 64, 64, 32), (4, 64, 64, 48), (4, 64, 96, 64), (4, 1 << 30, 64, 64), (4, 64, 1 << 21, 64)):
        assert lib.sd_w4a16_plan(*bad) == 0
