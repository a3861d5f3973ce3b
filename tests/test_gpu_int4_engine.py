"""The 4-bit operators as they are used together: one decoder layer's decode step, the attention layer
with a 4-bit cache, and the draft chain. Every stage is held to the 64-bit oracle on the very inputs
that it got (the tolerances of the operators' own tests)."""
import numpy as np
import pytest
import torch

import test_gpu_int4_attention as ta
import test_gpu_int4_cache as tc
import test_gpu_w4a16 as tw
from conftest import assert_close_attn
from oracle import int4 as o4
from specdec_nanovllm_amd import ops
from specdec_nanovllm_amd.draft_chain import DraftChain
from specdec_nanovllm_amd.layers.attention import Attention
from specdec_nanovllm_amd.layers.linear import ReplicatedLinear
from specdec_nanovllm_amd.layers.quant import apply_int4_quant
from specdec_nanovllm_amd.utils.context import reset_context, set_context

pytestmark = pytest.mark.gpu
DEV = "cuda"
HQ, HKV, D, PAGE = 16, 8, 128, 64


def f64(t):
    return t.detach().double().cpu().numpy()


def filled(lens, kind, seed):
    """A 4-bit cache of ``lens`` keys per sequence (as a prefill would leave it) and room for 8 more each."""
    c = ta.make([n + 8 for n in lens], PAGE, HQ, HKV, 64, kind, seed=seed)
    return c["codes"], c["scales"], c["table"]


def slots_of(table, first, count):
    out = []
    for b, (p0, n) in enumerate(zip(first, count)):
        p = torch.arange(p0, p0 + n)
        out.append(table[b].cpu()[p // PAGE].long() * PAGE + p % PAGE)
    return torch.cat(out).to(torch.int32).to(DEV)


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
def test_a_decode_step_stage_by_stage(kind):
    lens, hidden = [1, 130, 700, 64], 512
    codes, scales, table = filled(lens, kind, 1)
    g = torch.Generator().manual_seed(2)
    lin = torch.nn.ModuleDict(dict(qkv=ReplicatedLinear(hidden, (HQ + 2 * HKV) * D), o=ReplicatedLinear(HQ * D, hidden)))
    for p in lin.parameters():
        p.data = (torch.randn(p.shape, generator=g) * 0.05).to(torch.bfloat16)
    lin.to(DEV)
    apply_int4_quant(lin, ["qkv", "o"], 128)
    x = torch.randn((4, hidden), generator=g).to(ta.DTYPES[kind]).to(DEV)
    qkv = lin["qkv"](x)
    tw.check(qkv, x, lin["qkv"].weight, lin["qkv"].weight_scale, None, kind)
    q, k, v = (t.unflatten(-1, (-1, D)) for t in qkv.split([HQ * D, HKV * D, HKV * D], -1))
    angles = torch.arange(800, dtype=torch.float64)[:, None] * 1e4 ** (-torch.arange(64).double() / 64)
    cs = torch.cat((angles.cos(), angles.sin()), -1).float().to(DEV)
    w = (1 + 0.1 * torch.randn((D,), generator=g)).to(ta.DTYPES[kind]).to(DEV)
    slots = slots_of(table, lens, [1] * 4)
    qr, _ = ops.qk_norm_rope_store_int4(q, k, v, torch.tensor(lens, device=DEV), cs, codes, scales, slots, w, w, 1e-6,
                                        key_out=False)
    row = f64(cs)[lens]
    want = o4.norm_rotate(f64(k), f64(w), 1e-6, row[:, :64], row[:, 64:])
    flat = o4.norm_rotate(f64(k), f64(w), 1e-6, np.ones((4, 64)), np.zeros((4, 64)))
    err = 2**-20 * np.tile(np.abs(flat[..., :64]) + np.abs(flat[..., 64:]), 2)
    c, s = tc.rows_at(codes, scales, slots)
    tc.check_rows(c, s, want, err, kind, 0)
    tc.check_rows(c, s, f64(v), np.zeros_like(want), kind, 1)
    keys = [n + 1 for n in lens]
    o = ops.paged_attention_int4(qr, codes, scales, table, D ** -0.5,
                                 context_lens=torch.tensor(keys, dtype=torch.int32, device=DEV))
    ta.check(dict(q=qr, codes=codes, scales=scales, table=table, lens=keys, nq=[1] * 4), o, kind)
    y = lin["o"](o.view(4, -1))
    tw.check(y, o.view(4, -1), lin["o"].weight, lin["o"].weight_scale, None, kind)


def layer(codes, scales):
    a = Attention(HQ, D, D ** -0.5, HKV)
    a.k_cache, a.v_cache = codes, scales
    return a


def rows(n, heads, seed):
    return torch.randn((n, heads, D), generator=torch.Generator().manual_seed(seed)).to(torch.bfloat16).to(DEV)


def test_the_attention_layer_decodes_and_verifies_over_a_4_bit_cache():
    lens = [1, 130, 700]
    codes, scales, table = filled(lens, "bf16", 3)
    a = layer(codes, scales)
    for n in (1, 4):
        total, keys = 3 * n, [x + n for x in lens]
        q, k, v = rows(total, HQ, 4), rows(total, HKV, 5), rows(total, HKV, 6)
        slots = slots_of(table, lens, [n] * 3)
        try:
            if n == 1:
                set_context(False, slot_mapping=slots, block_tables=table,
                            context_lens=torch.tensor(keys, dtype=torch.int32, device=DEV))
                o = a(q, k, v)
                assert o.shape == (3, 1, HQ, D)
                o = o.squeeze(1)
            else:
                set_context(True, ta.cu([n] * 3), ta.cu(keys), n, max(keys), slots, None, table)
                o = a(q, k, v)
        finally:
            reset_context()
        c, s = tc.rows_at(codes, scales, slots)
        tc.check_rows(c, s, f64(k), np.zeros((total, HKV, D)), "bf16", 0)
        ta.check(dict(q=q, codes=codes, scales=scales, table=table, lens=keys, nq=[n] * 3), o, "bf16")


def test_the_attention_layer_prefills_with_and_without_a_cached_prefix():
    cached, new = [128, 64], [40, 90]
    keys = [a + b for a, b in zip(cached, new)]
    c = ta.make(keys, PAGE, HQ, HKV, 64, "bf16", seed=7)
    codes, scales, table = c["codes"], c["scales"], c["table"]
    a = layer(codes, scales)
    total = sum(new)
    q, k, v = rows(total, HQ, 8), rows(total, HKV, 9), rows(total, HKV, 10)
    slots = slots_of(table, cached, new)
    try:
        set_context(True, ta.cu(new), ta.cu(keys), max(new), max(keys), slots, None, table)
        o = a(q, k, v)
        set_context(True, ta.cu(new), ta.cu(new), max(new), max(new), slots, None, None)
        plain = a(q, k, v)
    finally:
        reset_context()
    at = 0
    for b, n in enumerate(new):
        pages = table[b, :-(-keys[b] // PAGE)].long()
        kk, vv = o4.values(codes[pages].cpu().numpy().reshape(-1, HKV, D)[:keys[b]],
                           f64(scales)[pages.cpu()].reshape(-1, HKV, 8)[:keys[b]])
        kk, vv = o4.round16(kk, "bf16"), o4.round16(vv, "bf16")  # read back in 16 bits
        for h in range(HQ):
            part = slice(at, at + n)
            want, _ = o4.attention(f64(q)[part, h], kk[:, h // 2], vv[:, h // 2], D ** -0.5, cached[b])
            assert_close_attn(f64(o)[part, h], want, what=f"cached prefix, sequence {b} head {h}")
            want, _ = o4.attention(f64(q)[part, h], f64(k)[part, h // 2], f64(v)[part, h // 2], D ** -0.5, 0)
            assert_close_attn(f64(plain)[part, h], want, what=f"sequence {b} head {h}")
        at += n


@pytest.mark.parametrize("weight_bits,kv_bits", [(4, 4), (8, 4), (4, 16)])
@pytest.mark.parametrize("context", ["prefill", "randn"])
def test_the_draft_chain_in_4_bits_replays_from_a_graph(weight_bits, kv_bits, context):
    c = DraftChain(2, ctx_len=70, k=3, layers=2, hidden=256, heads=4, kv_heads=2, inter=512, vocab=1000, block_size=16,
                   weight_bits=weight_bits, kv_bits=kv_bits, context=context)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        c.chain()
    torch.cuda.synchronize()
    first = c.tokens.clone()
    logits = c.step(0)
    assert bool(logits.isfinite().all()) and torch.equal(logits.argmax(-1), first[1])
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        c.chain()
    for _ in range(3):
        c.tokens[1:].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(c.tokens, first)
    assert c.step_bytes() > 0
    c.gemv_chain()
    c.attention_chain()
