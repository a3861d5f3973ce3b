"""Modules with activations in 8 bits give the type of the rows that they were given, quantized before or not."""
import pytest
import torch

import test_gpu_act_int8 as ta
import test_gpu_w8a8 as tw
from specdec_nanovllm_amd import ops
from specdec_nanovllm_amd.layers.layernorm import RMSNorm
from specdec_nanovllm_amd.layers.linear import ReplicatedLinear
from specdec_nanovllm_amd.layers.quant import apply_int8_quant

pytestmark = pytest.mark.gpu
DEV = "cuda"


@pytest.mark.parametrize("kind", ["bf16", "fp16"])
@pytest.mark.parametrize("rows", [1, 90])
def test_the_type_of_the_rows(kind, rows):
    dtype = ta.DTYPES[kind]
    m = torch.nn.ModuleDict(dict(up=ReplicatedLinear(256, 272, bias=True))).to(DEV, torch.bfloat16)
    g = torch.Generator().manual_seed(4)
    for p in m.parameters():
        p.data = (torch.randn(p.shape, generator=g) * 0.1).to(torch.bfloat16).to(DEV)
    apply_int8_quant(m, ["up"], act_bits=8)
    up, norm = m["up"], RMSNorm(256).to(DEV, dtype)
    x, r = ta.make(rows, 256, kind), ta.make(rows, 256, kind, seed=2)
    for h in (norm.forward_int8(x), norm.forward_int8(x, r)[0], ops.quantize_rows_int8(x)):
        y = up(h)
        tw.equal(y, *h, up.weight, up.weight_scale, up.bias.to(dtype), kind)
    assert torch.equal(up(x), y) and torch.equal(up(ops.quantize_rows_int8(x.view(rows, 1, 256)))[:, 0], y)
