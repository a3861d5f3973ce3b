"""The 4-bit operators at the edges of what their entries accept: each call is held to the 64-bit
oracle with the tolerance of the operator's own tests, or bit for bit to the same call on compact
tensors."""
import pytest
import torch

import test_gpu_int4_attention as ta
import test_gpu_w4a16 as tw
from specdec_nanovllm_amd import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
SCALE = 128 ** -0.5


def position_major(t, stride):
    """A copy of the cache tensor ``t`` whose positions lie ``stride`` elements apart, all pages of a
    position side by side."""
    blocks, page, heads, width = t.shape
    assert blocks * heads * width <= stride
    room = torch.empty((page - 1) * stride + blocks * heads * width, dtype=t.dtype, device=t.device)
    return room.as_strided(t.shape, (heads * width, stride, width, 1)).copy_(t)


# (keys left in the sequence) x (bytes between positions) passes 2^32 in each
@pytest.mark.parametrize("page,keys,stride", [
    (64, 200, 1 << 25),            # the largest stride there is; one page a step
    (16, 200, 1 << 25),            # a page for each half of a step
    (64, 1100, 1 << 22),
    (64, 1100, 36864 * 128),       # a stride that is no power of two wraps between rows
    (48, 2100, 1 << 21),
    (40, 1100, 1 << 22)])          # pages anywhere in a step
@pytest.mark.parametrize("rows,hq,group", [(1, 8, 64), (2, 16, 128), (7, 8, 32)])
def test_far_apart_positions(page, keys, stride, rows, hq, group):
    """One, one and two row tiles of two kv heads (4 rows, 16 and 28 of each)."""
    c = ta.make([keys, 70], page, hq, 2, group, "bf16", nq=[rows, rows], seed=page)
    lens = torch.tensor(c["lens"], dtype=torch.int32, device=DEV)

    def attend(codes, scales):
        return ops.paged_attention_int4(c["q"], codes, scales, c["table"], SCALE, context_lens=lens,
                                        cu_seqlens_q=ta.cu(c["nq"]), max_seqlen_q=rows)

    compact = attend(c["codes"], c["scales"])
    ta.check(c, compact, "bf16")
    far = attend(position_major(c["codes"], stride), position_major(c["scales"], stride >> 4))
    assert torch.equal(far, compact)


@pytest.mark.parametrize("m", [1, 7])
def test_few_rows_with_very_many_scales_take_their_slices(monkeypatch, m):
    """Rows whose scales leave LDS no room run in K slices, whose workspace the call gives."""
    given = []
    make = ops._workspace
    monkeypatch.setattr(ops, "_workspace", lambda n, dev: given.append(n) or make(n, dev))
    k = 1 << 17
    x, w, s, b = tw.make(m, 37, k, 32, "bf16", seed=m)
    y = ops.w4a16_linear(x, w, s, b)
    tw.check(y, x, w, s, b, "bf16")
    assert given == [_lib.load().sd_w4a16_workspace_size(m, 37, k, 32)] and given[0] > 0


@pytest.mark.parametrize("m", [1, 3, 20, 70])
def test_activations_that_start_anywhere(m):
    x, w, s, b = tw.make(m, 96, 256, 64, "bf16", seed=m)
    room = torch.empty(x.numel() + 1, dtype=x.dtype, device=DEV)
    moved = room[1:].view(x.shape).copy_(x)
    assert moved.is_contiguous() and moved.data_ptr() % 16
    want = ops.w4a16_linear(x, w, s, b)
    tw.check(want, x, w, s, b, "bf16")
    assert torch.equal(ops.w4a16_linear(moved, w, s, b), want)
    assert torch.equal(ops.w4a16_linear(moved.view(m, 1, 256), w, s, b).view(m, 96), want)


@pytest.mark.parametrize("m", [1, 2])
def test_the_last_token_of_a_long_prompt(m):
    """Rows further apart than the kernels' strides reach."""
    hidden = torch.empty((m, 8200, 2560), dtype=torch.bfloat16, device=DEV)
    x, w, s, b = tw.make(m, 100, 2560, 128, "bf16", seed=9)
    hidden[:, -1] = x
    last = hidden[:, -1]
    assert last.stride(0) > 1 << 24
    y = ops.w4a16_linear(last, w, s, b)
    tw.check(y, x, w, s, b, "bf16")


def test_a_cached_prefix_under_a_table_of_the_longest_sequence():
    from specdec_nanovllm_amd.layers.attention import Attention
    from specdec_nanovllm_amd.utils.context import reset_context, set_context

    heads, page, new, keys = 8, 64, [40, 90], [168, 154]
    c = ta.make(keys, page, 16, heads, 64, "bf16", seed=11)
    layer = Attention(16, 128, SCALE, heads)
    layer.k_cache, layer.v_cache = c["codes"], c["scales"]
    wide = torch.full((2, 140_000), -1, dtype=torch.int32, device=DEV)  # 9 M positions a sequence
    wide[:, :c["table"].shape[1]] = c["table"]
    g = torch.Generator().manual_seed(12)
    q, k, v = (torch.randn((sum(new), h, 128), generator=g).to(torch.bfloat16).to(DEV) for h in (16, heads, heads))
    out = []
    for table in (c["table"], wide):
        slots = torch.cat([table[b, p // page] * page + p % page for b in (0, 1)
                           for p in [torch.arange(keys[b] - new[b], keys[b], device=DEV)]]).to(torch.int32)
        try:
            set_context(True, ta.cu(new), ta.cu(keys), max(new), max(keys), slots, None, table)
            out.append(layer(q, k, v))
        finally:
            reset_context()
    assert torch.equal(*out) and bool(out[0].isfinite().all())
