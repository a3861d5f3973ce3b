"""Modules with activations in 8 bits: what ``apply_int8_quant`` and ``apply_int8_activations`` accept can run."""
import pytest
import torch

from specdec_nanovllm_amd.layers.linear import ReplicatedLinear
from specdec_nanovllm_amd.layers.quant import apply_int8_activations, apply_int8_quant


def model(dtype=torch.int8, **shapes):
    """{name: (outputs, columns)} as modules with zero weights; int8 ones with a scale a row."""
    m = torch.nn.ModuleDict({name: ReplicatedLinear(1, 1) for name in shapes})
    for name, shape in shapes.items():
        m[name].weight = torch.nn.Parameter(torch.zeros(shape, dtype=dtype), requires_grad=False)
        if dtype == torch.int8:
            m[name].weight_scale = torch.nn.Parameter(torch.ones(shape[0], dtype=torch.bfloat16), requires_grad=False)
    return m


# quantize_rows_int8 takes up to 32768 columns, w8a8_linear up to 2^21 outputs
@pytest.mark.parametrize("shape,says", [((8, 32784), "32768"), ((8, 40960), "32768"), (((1 << 21) + 1, 16), "2097152")])
def test_sizes_that_cannot_run_are_refused_before_a_change(shape, says):
    for dtype, call in ((torch.int8, apply_int8_activations), (torch.bfloat16, lambda *a: apply_int8_quant(*a, act_bits=8))):
        m = model(dtype, a=(8, 64), b=shape)
        with pytest.raises(ValueError, match=says):
            call(m, ["a", "b"])
        assert m["a"].quant_act_bits == m["b"].quant_act_bits == 16
        assert m["a"].weight.dtype == m["b"].weight.dtype == dtype


def test_the_largest_sizes_are_taken():
    m = model(a=(8, 32768), b=(1 << 21, 16))
    apply_int8_activations(m, ["a", "b"])
    assert m["a"].quant_act_bits == m["b"].quant_act_bits == 8


def test_any_int8_module_goes_back_to_16_bits():
    """Also one whose weights were replaced since, by group scales or a K that 8 bits do not take."""
    m = model(a=(8, 64), b=(8, 64))
    apply_int8_activations(m, ["a", "b"])
    m["a"].quant_granularity, m["a"].quant_group_size = "per_group", 32
    m["a"].weight_scale = torch.nn.Parameter(torch.ones((8, 2), dtype=torch.bfloat16), requires_grad=False)
    m["b"].weight = torch.nn.Parameter(torch.zeros((8, 72), dtype=torch.int8), requires_grad=False)
    for names in (["a"], ["b"]):
        with pytest.raises(ValueError):
            apply_int8_activations(m, names)
    apply_int8_activations(m, ["a", "b"], act_bits=16)
    assert m["a"].quant_act_bits == m["b"].quant_act_bits == 16


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_quantized_rows_keep_their_type(monkeypatch, dtype):
    """(codes, scale) from a norm or of a tensor: the linear's outputs have the type that the rows came from."""
    import copy
    import pickle

    from specdec_nanovllm_amd import _lib, ops
    from specdec_nanovllm_amd.layers.layernorm import RMSNorm
    from specdec_nanovllm_amd.layers.quant import int8_linear_a8

    class NoLaunch:
        def __getattr__(self, name):
            return lambda *args: 0

    monkeypatch.setattr(_lib, "load", NoLaunch)
    monkeypatch.setattr(_lib, "require_device", lambda *t: torch.device("cpu"))
    monkeypatch.setattr(_lib, "on_device", lambda dev: torch.no_grad())
    monkeypatch.setattr(_lib, "stream_ptr", lambda dev: 0)
    m = model(a=(8, 64))
    apply_int8_activations(m, ["a"])
    norm, x = RMSNorm(64).to(dtype), torch.zeros((2, 64), dtype=dtype)
    rows = [ops.quantize_rows_int8(x), norm.forward_int8(x), norm.forward_int8(x, x)[0],
            norm.forward_int8(x.view(1, 2, 64))]
    rows += [copy.deepcopy(rows[0]), pickle.loads(pickle.dumps(rows[1]))]
    for r in rows:
        assert isinstance(r, tuple) and len(r) == 2
        assert m["a"](r).dtype == int8_linear_a8(r, m["a"].weight, m["a"].weight_scale).dtype == dtype
        assert int8_linear_a8(r, m["a"].weight, m["a"].weight_scale, dtype=torch.bfloat16).dtype == torch.bfloat16
    assert m["a"](x).dtype == dtype
    assert m["a"](tuple(rows[0])).dtype == torch.bfloat16  # where nothing says
