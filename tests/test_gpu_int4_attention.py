"""Attention over the 4-bit cache (csrc/int4_attention.hip through ``ops``) against the 64-bit oracle
on the very codes and scales.

Tolerance of an output o = sum_j p_j v_j: its rounding, eps / 2 |o|; the scores: a product of 128 terms
of size |q| (16 + 15) s + |q| |z| rounds at most 32 + 4 times in fp32 (four chained MFMAs of 32), so a
score is off by at most E = 40 * 2^-24 * sum_d |q_d| (31 s + |z|) * scale, and p, o and the sum l
by a factor of 1 + 2 E; the weights' two bf16 parts keep 2^-16 of each p_j (31 s' + |z'|), and their fp32 sums
as much again.
"""
import numpy as np
import pytest
import torch

from oracle import int4 as o4
from specdec_nanovllm_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda"
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}
SCALE = 128 ** -0.5


def f64(t):
    return t.detach().double().cpu().numpy()


def make(lens, page, hq, hkv, group, kind, nq=None, width=None, interleaved=False, seed=0):
    """A cache with ``lens`` keys per sequence on shuffled pages; everything else in it is garbage
    (NaN scales), the table's unused entries -1."""
    g = torch.Generator().manual_seed(seed)
    need = [-(-n // page) for n in lens]
    width = width or max(1, max(need))
    blocks = sum(need) + 1
    codes = torch.randint(0, 256, (blocks, hkv, page, 128), generator=g, dtype=torch.uint8)
    ng = 128 // group
    scales = torch.empty((blocks, hkv, page, 4 * ng))
    scales[..., 0::2] = torch.rand((blocks, hkv, page, 2 * ng), generator=g) * 0.4 + 0.1
    scales[..., 1::2] = -3 * torch.rand((blocks, hkv, page, 2 * ng), generator=g)
    table = torch.full((len(lens), width), -1, dtype=torch.int32)
    perm, at = torch.randperm(blocks, generator=g), 0
    live = torch.zeros((blocks, page), dtype=torch.bool)
    for b, n in enumerate(need):
        table[b, :n] = perm[at:at + n].to(torch.int32)
        at += n
        for i in range(n):
            live[table[b, i], :min(page, lens[b] - i * page)] = True
    scales.transpose(1, 2)[~live] = float("nan")
    nq = nq or [1] * len(lens)
    q = torch.randn((sum(nq), hq, 128), generator=g).to(DTYPES[kind]).to(DEV)
    codes, scales = codes.transpose(1, 2), scales.transpose(1, 2).to(DTYPES[kind])
    if interleaved:
        codes, scales = codes.contiguous(), scales.contiguous()
        codes, scales = codes.to(DEV), scales.to(DEV)
    else:
        codes = codes.transpose(1, 2).to(DEV).transpose(1, 2)
        scales = scales.transpose(1, 2).contiguous().to(DEV).transpose(1, 2)
    return dict(q=q, codes=codes, scales=scales, table=table.to(DEV), lens=lens, nq=nq)


def check(c, out, kind):
    eps = float(torch.finfo(DTYPES[kind]).eps)
    codes, scales, table = c["codes"].cpu().numpy(), f64(c["scales"]), c["table"].cpu().numpy()
    page, hkv = codes.shape[1], codes.shape[2]
    q, got = f64(c["q"]), f64(out)
    share, at = q.shape[1] // hkv, 0
    ng = scales.shape[-1] // 4
    for b, (n, rows) in enumerate(zip(c["lens"], c["nq"])):
        pages = table[b, :-(-n // page)]
        cc = codes[pages].reshape(-1, hkv, 128)[:n]
        ss = scales[pages].reshape(-1, hkv, 4 * ng)[:n]
        key, value = o4.values(cc, ss)
        reach = [31 * np.abs(ss[..., 2 * ng * i:2 * ng * (i + 1)][..., 0::2]).repeat(128 // ng, -1)
                 + np.abs(ss[..., 2 * ng * i:2 * ng * (i + 1)][..., 1::2]).repeat(128 // ng, -1) for i in (0, 1)]
        for h in range(q.shape[1]):
            kv = h // share
            qq = q[at:at + rows, h]
            want, p = o4.attention(qq, key[:, kv], value[:, kv], SCALE, n - rows)
            tol = eps / 2 * np.abs(want) + 1e-7
            if n:
                E = 40 * 2**-24 * (np.abs(qq) @ reach[0][:, kv].T).max(-1, keepdims=True) * SCALE
                tol = tol + (2**-16 + 2 * E) * (p @ reach[1][:, kv])
            bad = np.abs(got[at:at + rows, h] - want) > tol
            assert not bad.any(), (f"sequence {b} ({n} keys, {rows} rows) head {h}: off by "
                                   f"{np.abs(got[at:at + rows, h] - want).max():.3g}")
        at += rows


def cu(n):
    return torch.tensor([0, *np.cumsum(n)], dtype=torch.int32, device=DEV)


ODD = [1, 0, 31, 32, 33, 127, 128, 129, 300, 1000]


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("page,interleaved", [(16, False), (48, True), (64, True), (256, False)])
@pytest.mark.parametrize("keys", [1024, 4000])  # a workgroup a pair, and split
def test_decode(kind, group, page, interleaved, keys):
    c = make(ODD, page, 16, 4, group, kind, interleaved=interleaved, width=keys // page)
    out = ops.paged_attention_int4(c["q"], c["codes"], c["scales"], c["table"], SCALE,
                                   context_lens=torch.tensor(ODD, dtype=torch.int32, device=DEV))
    check(c, out, kind)


@pytest.mark.parametrize("hq,hkv", [(1, 1), (8, 8), (5, 5), (32, 2), (32, 1), (12, 4)])
def test_head_layouts(hq, hkv):
    lens = [700, 5, 64]
    c = make(lens, 64, hq, hkv, 64, "bf16", seed=1)
    out = ops.paged_attention_int4(c["q"], c["codes"], c["scales"], c["table"], SCALE,
                                   cu_seqlens_k=cu(lens))
    check(c, out, "bf16")


@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("width", [1, 2, 3, 4, 8, 300])
def test_short_and_wide_tables(width, group):
    # few keys a table: one workgroup a pair; a wide table with short sequences: split
    lens = [min(256 * width, n) for n in (200, 0, 256, 511, 77)]
    c = make(lens, 256, 8, 4, group, "bf16", width=width, seed=2)
    out = ops.paged_attention_int4(c["q"], c["codes"], c["scales"], c["table"], SCALE,
                                   context_lens=torch.tensor(lens, dtype=torch.int32, device=DEV))
    check(c, out, "bf16")


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("group", [32, 64, 128])
@pytest.mark.parametrize("keys", [960, 3000])
@pytest.mark.parametrize("page", [64, 16, 40])
def test_verify_rows(kind, group, keys, page):
    lens, nq = [900, 3, 40, 0, 129, 8], [7, 7, 1, 2, 0, 8]  # rows 0 .. 3 of the second see no key
    c = make(lens, page, 16, 4, group, kind, nq=nq, seed=3, width=keys // page)
    out = ops.paged_attention_int4(c["q"], c["codes"], c["scales"], c["table"], SCALE,
                                   context_lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                                   cu_seqlens_q=cu(nq), max_seqlen_q=8)
    check(c, out, kind)
    assert float(out[7:11].abs().max()) == 0 and float(out[15:17].abs().max()) == 0


@pytest.mark.parametrize("splits", [1, 3, 40])
def test_splits(splits):
    lens = [3000, 100, 1500]
    c = make(lens, 16, 8, 2, 64, "bf16", seed=4)
    out = ops.paged_attention_int4(c["q"], c["codes"], c["scales"], c["table"], SCALE,
                                   context_lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                                   num_splits=splits)
    check(c, out, "bf16")


def test_more_sequences_than_a_wave():
    g = torch.Generator().manual_seed(5)
    lens = torch.randint(0, 400, (150,), generator=g).tolist()
    c = make(lens, 32, 4, 2, 64, "bf16", seed=5)
    for width in (13, 40):
        table = torch.full((150, width), -1, dtype=torch.int32, device=DEV)
        table[:, :c["table"].shape[1]] = c["table"]
        out = ops.paged_attention_int4(c["q"], c["codes"], c["scales"], table, SCALE,
                                       context_lens=torch.tensor(lens, dtype=torch.int32, device=DEV))
        check(c, out, "bf16")


def test_strided_rows_and_rows_past_the_last_are_left():
    lens, nq = [500, 60], [3, 2]
    c = make(lens, 64, 8, 4, 64, "bf16", nq=nq, seed=6)
    wide = torch.zeros((7, 8, 256), dtype=torch.bfloat16, device=DEV)
    wide[:5, :, :128] = c["q"]
    out = torch.full((7, 8, 160), 7.0, dtype=torch.bfloat16, device=DEV)
    ops.paged_attention_int4(wide[..., :128], c["codes"], c["scales"], c["table"], SCALE,
                             context_lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                             cu_seqlens_q=cu(nq), max_seqlen_q=4, out=out[..., :128])
    check(c, out[:5, :, :128], "bf16")
    assert bool((out[5:] == 7).all()) and bool((out[..., 128:] == 7).all())


def test_keys_that_no_row_sees_may_hold_nan():
    # rows of a verify step: the earlier rows do not see the last key, whose scales are NaN
    lens, nq = [65], [2]
    c = make(lens, 64, 4, 4, 64, "bf16", nq=nq, seed=7)
    last = int(c["table"][0, 1])
    c["scales"][last, 0] = float("nan")
    out = ops.paged_attention_int4(c["q"], c["codes"], c["scales"], c["table"], SCALE,
                                   context_lens=torch.tensor(lens, dtype=torch.int32, device=DEV),
                                   cu_seqlens_q=cu(nq), max_seqlen_q=2)
    assert bool(out[0].isfinite().all()) and bool(out[1].isnan().all())
    c["lens"], c["nq"] = [64], [1]
    c["q"] = c["q"][:1]
    check(c, out[:1], "bf16")


def test_a_query_of_nan_gives_nan():
    c = make([40, 700], 64, 4, 4, 64, "bf16", seed=8)
    c["q"][:, 1] = float("nan")
    out = ops.paged_attention_int4(c["q"], c["codes"], c["scales"], c["table"], SCALE,
                                   context_lens=torch.tensor([40, 700], dtype=torch.int32, device=DEV))
    assert bool(out[:, 1].isnan().all()) and bool(out[:, [0, 2, 3]].isfinite().all())


def test_large_scores_and_rising_maxima():
    c = make([2000, 130], 64, 8, 4, 64, "bf16", seed=9)
    c["q"].mul_(30)  # scores of hundreds: the running maximum moves many times
    lens = torch.tensor([2000, 130], dtype=torch.int32, device=DEV)
    out = ops.paged_attention_int4(c["q"], c["codes"], c["scales"], c["table"], SCALE, context_lens=lens)
    check(c, out, "bf16")


def test_repeats_bit_for_bit_and_follows_its_inputs_in_a_graph():
    lens = [1200, 300, 64]
    c = make(lens, 64, 8, 4, 64, "bf16", seed=10)
    ctx = torch.tensor(lens, dtype=torch.int32, device=DEV)

    def step():
        return ops.paged_attention_int4(c["q"], c["codes"], c["scales"], c["table"], SCALE, context_lens=ctx)

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        first = step()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step()
    graph.replay()
    assert torch.equal(out, first) and torch.equal(step(), first)
    for i, now in enumerate(([1, 300, 0], [1199, 7, 64], lens)):
        ctx.copy_(torch.tensor(now, dtype=torch.int32))
        c["q"].add_(0.25)
        graph.replay()
        got = out.clone()
        torch.cuda.synchronize()
        assert torch.equal(got, step()), i
        c["lens"] = now
        check(c, got, "bf16")
