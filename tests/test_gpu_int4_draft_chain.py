"""The numbers of the draft step in 4 bits: logits against the float32 restatement of
tests/test_gpu_draft_chain.py on the dequantized weights, with its tolerance (2e-2 of the largest logit,
for the bf16 roundings between operators). With a 4-bit cache the restatement attends over the rows
that the cache holds after the step, read back; the rows that the step itself appended are held to
the restatement's own keys and values: half a level of their group's range, 2^-7 of the value and of the range
for scale and zero in bf16, and the logits' 2e-2 of the largest for the roundings before them.
"""
import copy

import pytest
import torch

import test_gpu_draft_chain as td
from specdec_nanovllm_amd import ops
from specdec_nanovllm_amd.draft_chain import DraftChain
from specdec_nanovllm_amd.layers.quant import dequantize_weight, dequantize_weight_int4

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("weight_bits,kv_bits", [(4, 4), (8, 4), (4, 16)])
@pytest.mark.parametrize("batch,context", [(1, "prefill"), (3, "prefill"), (3, "randn")])
def test_logits_match_the_float32_reference(monkeypatch, weight_bits, kv_bits, batch, context):
    monkeypatch.setattr(td, "dequantize_weight", dequantize_weight_int4 if weight_bits == 4 else dequantize_weight)
    ch = DraftChain(batch, weight_bits=weight_bits, kv_bits=kv_bits, context=context, **td.SMALL)
    blocks, rows = batch * ch.pages_per_seq, torch.arange(batch, device=ch.dev, dtype=torch.int32)
    every = torch.arange(blocks * ch.bs, dtype=torch.int32, device=ch.dev)
    ref = copy.copy(ch)
    ref.slots = (blocks * ch.bs + rows).expand(ch.k, batch)  # the restatement's rows: a page of their own
    for s in range(ch.k):
        logits = ch.step(s).float()
        kv = torch.zeros((2, ch.L, blocks + 1, ch.bs, ch.Hkv, ch.D), dtype=ch.dtype, device=ch.dev)
        for li in range(ch.L):
            held = ops.load_kvcache_int4(*ch.kv4[li], every) if kv_bits == 4 else ch.kv[:, li].flatten(1, 2)
            for part in (0, 1):
                kv[part, li, :blocks] = held[part].view(blocks, ch.bs, ch.Hkv, ch.D)
        want = td.ref_step(ref, kv, ch.tokens[s], s)
        off = (logits - want).abs().max().item()
        assert off <= 2e-2 * want.abs().max().item(), f"step {s}: off by {off:.4g}"
        flat = kv.flatten(2, 3).float()
        got, own = flat[:, :, ch.slots[s].long()], flat[:, :, ref.slots[s].long()]
        group = own.unflatten(-1, (-1, 64))
        span = (group.amax(-1, keepdim=True) - group.amin(-1, keepdim=True)).expand_as(group).flatten(-2)
        most = own.abs().amax((1, 2, 3, 4), keepdim=True)
        allowed = (span / 30 + 2**-7 * (span + own.abs()) if kv_bits == 4 else 0) + 2e-2 * most
        assert bool(((got - own).abs() <= allowed).all()), f"step {s}: off by {(got - own).abs().max().item():.4g}"
        assert torch.equal(ch.tokens[s + 1], logits.argmax(-1))


@pytest.mark.parametrize("weight_bits,kv_bits", [(4, 4), (8, 4), (4, 16)])
def test_fused_changes_nothing_in_4_bits(weight_bits, kv_bits):
    a, b = (DraftChain(2, weight_bits=weight_bits, kv_bits=kv_bits, context="randn", fused=fused, **td.SMALL)
            for fused in (False, True))
    assert torch.equal(a.step(0), b.step(0)) and torch.equal(a.tokens, b.tokens)
