"""The 8-bit operators as they are used together: a decoder layer stage by stage, the layers' modules, the draft chain
with activations in 8 bits, and what a caller may do that the operators' own tests do not.

The draft chain's operators are each held to the oracle on the inputs that the step gives them, and its logits with a
16-bit cache to a restatement of the step with the operators' own rounding points (``ref_step``): what is left between
the two are last bits of attention, of sums of squares and of exponentials, which move a bf16 value or an 8-bit code by
a level now and then. The tolerance is that of tests/test_gpu_draft_chain.py, whose restatement differs from its chain in
more places: 2e-2 of the largest logit.
"""
import pytest
import torch

import test_gpu_act_int8 as ta
import test_gpu_draft_chain as td
import test_gpu_w8a8 as tw
from conftest import to_np
from oracle import w8a8 as o8
from specdec_nanovllm_amd import ops
from specdec_nanovllm_amd.draft_chain import DraftChain
from specdec_nanovllm_amd.layers.layernorm import RMSNorm
from specdec_nanovllm_amd.layers.linear import ReplicatedLinear
from specdec_nanovllm_amd.layers.quant import (apply_int8_activations, apply_int8_quant, dequantize_weight,
                                               int8_linear_a8, quantize_weight)

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("rows", [1, 7, 70, 300])
def test_an_mlp_stage_by_stage(kind, rows):
    """norm -> gate_up -> quantize -> down, each stage held to the oracle on the very inputs that it got."""
    hidden, inter = 528, 1040
    g = torch.Generator().manual_seed(rows)
    w = [quantize_weight((torch.randn(s, generator=g) * 0.05).to(torch.bfloat16).to(DEV))
         for s in ((2 * inter, hidden), (hidden, inter))]
    x, r, nw = ta.make(rows, hidden, kind), ta.make(rows, hidden, kind, seed=1), ta.weight(hidden, kind)
    codes, scale, new = ops.rmsnorm_int8(x, nw, 1e-6, r)
    ta.check_norm(x, nw, (codes, scale, new), r)
    act = ops.w8a8_gate_up_silu(codes, scale, *w[0], dtype=ta.DTYPES[kind])
    tw.near(act, codes, scale, *w[0], None, kind)
    c2, s2 = ops.quantize_rows_int8(act)
    ta.check_quantized(act, c2, s2)
    tw.equal(ops.w8a8_linear(c2, s2, *w[1], dtype=ta.DTYPES[kind]), c2, s2, *w[1], None, kind)


@pytest.mark.parametrize("rows", [1, 5, 90])
def test_modules(rows):
    g = torch.Generator().manual_seed(3)
    m = torch.nn.ModuleDict(dict(norm=RMSNorm(256), up=ReplicatedLinear(256, 272, bias=True), down=ReplicatedLinear(272, 64)))
    for p in m.parameters():
        p.data = (torch.randn(p.shape, generator=g) * 0.1 + (1 if p.dim() == 1 and p.numel() == 256 else 0)).to(torch.bfloat16)
    m.to(DEV)
    apply_int8_quant(m, ["up"], act_bits=8)
    apply_int8_quant(m, ["down"])
    apply_int8_activations(m, ["down"])
    x, r = ta.make(rows, 256, "bf16"), ta.make(rows, 256, "bf16", seed=2)
    up, down = m["up"], m["down"]
    h, new = m["norm"].forward_int8(x, r)
    assert torch.equal(new, (x.float() + r.float()).to(torch.bfloat16))
    y = up(h)
    tw.equal(y, *h, up.weight, up.weight_scale, up.bias, "bf16")
    z = down(y)
    q = ops.quantize_rows_int8(y)
    tw.equal(z, *q, down.weight, down.weight_scale, None, "bf16")
    assert torch.equal(down(q), z) and torch.equal(int8_linear_a8(y, down.weight, down.weight_scale), z)
    assert torch.equal(m["norm"].forward_int8(x)[0], ops.rmsnorm_int8(x, m["norm"].weight, 1e-6)[0])
    # near the product of the unquantized rows: a value is off by half a level at most, 1/254 of its row's largest
    ref = y.double() @ dequantize_weight(down.weight, down.weight_scale).double().T.contiguous()
    bound = (y.double().abs().amax(-1, keepdim=True) / 254) * (down.weight.double().abs() @ torch.ones(272, 1, device=DEV).double()).T \
        * down.weight_scale.double()
    assert bool(((z.double() - ref).abs() <= bound * 1.001 + 2.0**-7 * ref.abs() + 1e-6).all())
    apply_int8_activations(m, ["down"], 16)
    with pytest.raises(TypeError, match="quant_act_bits"):
        down(q)


def ref_linear(codes, scale, qw):
    """A product of codes with its scales, in 64 bits."""
    return codes.double() @ qw[0].double().T.contiguous() * qw[1].double() * scale[:, None]


def ref_quantize(v):
    """(codes, scale) of rows in 64 bits."""
    c, most = o8.codes(to_np(v.float()))
    return torch.from_numpy(c).double().to(v.device), torch.from_numpy(most / 127).to(v.device)


def ref_norm(x, w, eps, residual):
    s = x.float() + residual.float() if residual is not None else x.float()
    codes, scale = ref_quantize(s * w.float())
    return codes, scale / (s.double().square().mean(-1) + eps).sqrt(), s.to(x.dtype)


def ref_step(ch, tokens, s, attend):
    """Logits of draft step s: ``attend(layer, q, k, v)`` is attention over the cached rows and the new ones."""
    B, Hq, Hkv, D, bf = ch.B, ch.Hq, ch.Hkv, ch.D, torch.bfloat16
    pos, h, res = ch.positions[s], ch.embed[tokens], None

    def rope(x, w):
        x = x.float()
        x = x * torch.rsqrt(x.pow(2).mean(-1, keepdim=True) + ch.eps)
        # the 16-bit append keeps the module's roundings, the 4-bit one has none on the way
        x = (x.to(bf).float() * w.float()).to(bf).float() if ch.kv_bits == 16 else x * w.float()
        c, sn = ch.cos[pos][:, None, :], ch.sin[pos][:, None, :]
        x1, x2 = x.chunk(2, dim=-1)
        return torch.cat((x1 * c - x2 * sn, x2 * c + x1 * sn), dim=-1).to(bf)

    for li, lw in enumerate(ch.layers):
        codes, scale, res = ref_norm(h, lw["in_norm"], ch.eps, res)
        q, k, v = ref_linear(codes, scale, lw["qkv"]).to(bf).split([Hq * D, Hkv * D, Hkv * D], dim=-1)
        q, k = rope(q.reshape(B, Hq, D), lw["q_norm"]), rope(k.reshape(B, Hkv, D), lw["k_norm"])
        o = attend(li, q, k, v.reshape(B, Hkv, D))
        h = ref_linear(*ref_quantize(o.reshape(B, -1)), lw["o"]).to(bf)
        codes, scale, res = ref_norm(h, lw["post_norm"], ch.eps, res)
        gate, up = ref_linear(codes, scale, lw["gate_up"]).chunk(2, dim=-1)
        h = ref_linear(*ref_quantize((gate * torch.sigmoid(gate) * up).to(bf)), lw["down"]).to(bf)
    codes, scale, _ = ref_norm(h, ch.final_norm, ch.eps, res)
    return ref_linear(codes, scale, ch.lm_head)


@pytest.mark.parametrize("batch,context", [(1, "prefill"), (3, "prefill"), (3, "randn")])
def test_draft_chain_logits(batch, context):
    ch = DraftChain(batch, act_bits=8, context=context, **td.SMALL)
    pages = ch.block_table.long()
    for s in range(ch.k):
        logits = ch.step(s).float()
        n = ch.ctx_len + s + 1

        def attend(li, q, k, v):
            held = ch.kv[:, li].flatten(1, 2)
            for got, own in zip(held, (k, v)):  # the rows that the step itself appended
                off = (got[ch.slots[s].long()].double() - own.double()).norm() / own.double().norm()
                assert float(off) < 2e-2
            rows = (pages[:, :, None] * ch.bs + torch.arange(ch.bs, device=ch.dev)).flatten(1)[:, :n]
            kk, vv = (held[i][rows].double().repeat_interleave(ch.Hq // ch.Hkv, 2) for i in (0, 1))
            p = torch.softmax((q.double()[:, None] * kk).sum(-1) * ch.scale, 1)
            return (p[..., None] * vv).sum(1).to(torch.bfloat16)

        want = ref_step(ch, ch.tokens[s], s, attend)
        off = (logits - want).abs().max().item()
        assert off <= 2e-2 * want.abs().max().item(), f"step {s}: off by {off:.4g} of {want.abs().max().item():.4g}"
        assert torch.equal(ch.tokens[s + 1], logits.argmax(-1))


@pytest.mark.parametrize("kv_bits", [16, 4])
@pytest.mark.parametrize("batch", [1, 3, 20])
def test_draft_chain_stage_by_stage(monkeypatch, batch, kv_bits):
    """Every 8-bit operator of a step against the oracle on its own inputs, and what each of them is given."""
    ch = DraftChain(batch, act_bits=8, kv_bits=kv_bits, context="randn", **td.SMALL)
    calls = []

    def recorded(name):
        real = getattr(ops, name)

        def call(*args, **kw):
            held = [a.clone() if isinstance(a, torch.Tensor) else a for a in args]
            out = real(*args, **kw)
            # (a copy of what came out too: q and k are rotated in place)
            calls.append((name, args, held, out, out.clone() if isinstance(out, torch.Tensor) else out))
            return out

        monkeypatch.setattr(ops, name, call)

    for name in ("rmsnorm_int8", "quantize_rows_int8", "w8a8_linear", "w8a8_gate_up_silu"):
        recorded(name)
    logits = ch.step(0)
    layer = ["rmsnorm_int8", "w8a8_linear", "quantize_rows_int8", "w8a8_linear", "rmsnorm_int8", "w8a8_gate_up_silu",
             "quantize_rows_int8", "w8a8_linear"]
    assert [c[0] for c in calls] == layer * ch.L + ["rmsnorm_int8", "w8a8_linear"]
    weights = [lw[n][0] for lw in ch.layers for n in ("qkv", "o", "gate_up", "down")] + [ch.lm_head[0]]
    norms = [lw[n] for lw in ch.layers for n in ("in_norm", "post_norm")] + [ch.final_norm]
    assert [c[1][2] is w for c, w in zip((c for c in calls if c[0].startswith("w8a8")), weights)] == [True] * len(weights)
    assert [c[1][1] is w for c, w in zip((c for c in calls if c[0] == "rmsnorm_int8"), norms)] == [True] * len(norms)
    residual = None
    for i, (name, args, held, _, out) in enumerate(calls):
        if name == "rmsnorm_int8":
            r = held[3] if len(held) > 3 else None
            assert (residual is None) == (r is None) or i == 4
            assert residual is None or args[3] is residual
            ta.check_norm(held[0], held[1], out, r, ch.eps)
            residual = out[2] if r is not None else args[0]
            if i:
                assert args[0] is calls[i - 1][3]
        elif name == "quantize_rows_int8":
            ta.check_quantized(held[0], *out)
            assert calls[i - 1][0] != "w8a8_gate_up_silu" or args[0] is calls[i - 1][3]
        else:
            assert args[0] is calls[i - 1][3][0] and args[1] is calls[i - 1][3][1]
            (tw.near if name == "w8a8_gate_up_silu" else tw.equal)(out, *held[:4], None, "bf16")
    assert logits is calls[-1][3]


@pytest.mark.parametrize("kv_bits", [16, 4])
def test_draft_chain_prefill_is_the_step_over_all_rows(kv_bits):
    """The rows that the prefill leaves are near those of the prefill with 16-bit activations."""
    a = DraftChain(2, act_bits=8, kv_bits=kv_bits, **td.SMALL)
    b = DraftChain(2, kv_bits=kv_bits, **td.SMALL)
    every = torch.arange(2 * a.pages_per_seq * a.bs, dtype=torch.int32, device=a.dev)
    for li in range(a.L):
        ka, kb = ([ops.load_kvcache_int4(*c.kv4[li], every) if kv_bits == 4 else c.kv[:, li].flatten(1, 2)][0]
                  for c in (a, b))
        for x, y in zip(ka, kb):
            x, y = x.double(), y.double()
            assert float((x - y).norm() / y.norm()) < (0.02 if kv_bits == 16 else 0.06) * (li + 1)


def test_draft_chain_graph_replays():
    ch = DraftChain(3, act_bits=8, context="randn", **td.SMALL)
    ch.chain()
    want = ch.tokens.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ch.chain()
    for _ in range(3):
        ch.tokens[1:].zero_()
        graph.replay()
        torch.cuda.synchronize()
        assert torch.equal(ch.tokens, want)
    ch.gemv_chain()
    fused = DraftChain(3, act_bits=8, context="randn", fused=True, **td.SMALL)
    fused.chain()
    assert torch.equal(fused.tokens, want)
