"""The 8-bit activations' and integer linears' entry points without a GPU: refusals of the C ABI and of ``ops`` (before
any launch), the oracle on hand-made rows, the plans and a sweep of hostile arguments."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import w8a8 as o8
from specdec_nanovllm_amd import _lib, ops

A = [0x10000000 + i * 0x4000000 for i in range(16)]  # 16-byte aligned, never dereferenced
BF16, F32 = _lib.SD_BF16, _lib.SD_F32

_LINEAR = [A[0], 1024, A[1], A[2], 1024, A[3], BF16, None, A[4], 4096, 4, 4096, 1024, 7, None, 0, None]
CALLS = {  # valid calls but for their dtype (7), so that nothing is launched
    "sd_quantize_rows_int8": [A[0], 1024, A[1], 1024, A[2], 4, 1024, 7, None],
    "sd_rmsnorm_int8": [A[0], 1024, A[1], 1024, A[2], A[3], 1024, A[4], A[5], 1024, 4, 1024, 1e-6, 7, None],
    "sd_dequantize_rows_int8": [A[0], 1024, A[1], A[2], 1024, 4, 1024, 7, None],
    "sd_w8a8_linear": _LINEAR,
    "sd_w8a8_gate_up_silu": _LINEAR,
}
DTYPE_AT = {"sd_quantize_rows_int8": -2, "sd_rmsnorm_int8": -2, "sd_dequantize_rows_int8": -2,
            "sd_w8a8_linear": -4, "sd_w8a8_gate_up_silu": -4}
no_gpu = pytest.mark.skipif(torch.cuda.device_count() > 0,
                            reason="fake device addresses: only where no GPU can be reached")


def call(name, **change):
    """The call with arguments replaced by position (``a3=...``)."""
    args = list(CALLS[name])
    for k, v in change.items():
        args[int(k[1:])] = v
    lib = _lib.load()
    return getattr(lib, name)(*args), lib.sd_last_error().decode()


_BF = {"a13": BF16}
_REFUSED = [
    ("sd_quantize_rows_int8", {}, 2, "dtype"),
    ("sd_quantize_rows_int8", {"a7": F32}, 2, "dtype"),
    ("sd_quantize_rows_int8", {"a6": 1000}, 2, "multiple of 16"),
    ("sd_quantize_rows_int8", {"a6": 32784}, 2, "up to 32768"),
    ("sd_quantize_rows_int8", {"a5": 1 << 24}, 2, "rows below"),
    ("sd_quantize_rows_int8", {"a5": 1 << 22, "a6": 8208}, 2, "rows below"),
    ("sd_quantize_rows_int8", {"a5": 1 << 22, "a6": 4112}, 2, "rows below"),
    ("sd_quantize_rows_int8", {"a5": -1}, 1, "invalid sizes"),
    ("sd_quantize_rows_int8", {"a6": 0}, 1, "invalid sizes"),
    ("sd_quantize_rows_int8", {"a7": BF16, "a0": None}, 1, "null"),
    ("sd_quantize_rows_int8", {"a7": BF16, "a0": A[0] + 2}, 2, "aligned"),
    ("sd_quantize_rows_int8", {"a7": BF16, "a1": 1028}, 2, "aligned"),
    ("sd_quantize_rows_int8", {"a7": BF16, "a3": 1032}, 2, "aligned"),
    ("sd_quantize_rows_int8", {"a7": BF16, "a3": 1008}, 1, "overlap"),
    ("sd_quantize_rows_int8", {"a7": BF16, "a1": 1 << 41}, 1, "strides"),
    ("sd_rmsnorm_int8", {"a13": BF16, "a4": None}, 1, "null"),
    ("sd_rmsnorm_int8", {"a13": BF16, "a8": None}, 1, "null"),
    ("sd_rmsnorm_int8", {"a13": BF16, "a4": A[2] + 8}, 2, "aligned"),
    ("sd_rmsnorm_int8", {"a13": BF16, "a9": 1020}, 1, "overlap"),
    ("sd_rmsnorm_int8", {"a13": BF16, "a9": 1028}, 2, "aligned"),
    ("sd_quantize_rows_int8", {"a7": BF16, "a2": A[0] + 2048}, 1, "share memory"),
    ("sd_quantize_rows_int8", {"a7": BF16, "a4": A[2] + 4, "a2": A[2]}, 1, "share memory"),
    ("sd_quantize_rows_int8", {"a7": BF16, "a1": -1024, "a2": A[0] - 6144}, 1, "share memory"),
    ("sd_rmsnorm_int8", {"a13": BF16, "a5": A[1]}, 1, "share memory"),
    ("sd_rmsnorm_int8", {"a13": BF16, "a7": A[2] + 2044}, 1, "share memory"),
    ("sd_rmsnorm_int8", {"a13": BF16, "a8": A[4] - 1024}, 1, "share memory"),
    ("sd_dequantize_rows_int8", {"a7": F32, "a3": A[0] + 4080}, 1, "shares memory"),
    ("sd_dequantize_rows_int8", {"a7": F32, "a3": A[1] - 16368}, 1, "shares memory"),
    ("sd_dequantize_rows_int8", {}, 2, "dtype"),
    ("sd_dequantize_rows_int8", {"a5": 1 << 26}, 2, "2\\^26"),
    ("sd_dequantize_rows_int8", {"a7": BF16, "a2": None}, 1, "null"),
    ("sd_dequantize_rows_int8", {"a7": F32, "a4": 1026}, 2, "aligned"),
    ("sd_dequantize_rows_int8", {"a7": BF16, "a4": 1000}, 1, "overlap"),
]
for _name in ("sd_w8a8_linear", "sd_w8a8_gate_up_silu"):
    _REFUSED += [
        (_name, {}, 2, "dtype"),
        (_name, {**_BF, "a6": 5}, 2, "scales"),
        (_name, {**_BF, "a12": 1000}, 2, "multiple of 16"),
        (_name, {**_BF, "a12": 1 << 17}, 2, "too large"),
        (_name, {**_BF, "a12": 1 << 40}, 2, "too large"),
        (_name, {**_BF, "a12": -16}, 1, "invalid sizes"),
        (_name, {**_BF, "a11": 0}, 1, "invalid sizes"),
        (_name, {**_BF, "a11": (1 << 21) + 1}, 2, "too large"),
        (_name, {**_BF, "a10": 1 << 24, "a11": 1 << 14, "a9": 1 << 14}, 2, "too large"),
        (_name, {**_BF, "a1": (1 << 23) + 16}, 2, "too large"),
        (_name, {**_BF, "a2": None}, 1, "null"),
        (_name, {**_BF, "a1": 1032}, 2, "aligned"),
        (_name, {**_BF, "a4": 1032}, 2, "aligned"),
        (_name, {**_BF, "a0": A[0] + 8}, 2, "aligned"),
        (_name, {**_BF, "a4": -1024}, 1, "strides"),
        (_name, {**_BF, "a9": 4095}, 1, "overlap"),
        (_name, {**_BF, "a8": A[0] + 1024}, 1, "shares memory"),
        (_name, {**_BF, "a8": A[1] + 8}, 1, "shares memory"),
        (_name, {**_BF, "a8": A[2] + (1 << 20)}, 1, "shares memory"),
        (_name, {**_BF, "a8": A[3] + 4096}, 1, "shares memory"),
        (_name, {**_BF, "a7": A[5], "a8": A[5] - 32766}, 1, "shares memory"),
    ]


@no_gpu
@pytest.mark.parametrize("name,change,rc,says", _REFUSED)
def test_refusals_say_what_is_wrong(name, change, rc, says):
    got, message = call(name, **change)
    assert got == rc and says.replace("\\", "") in message, (got, message)


@no_gpu
def test_hostile_arguments_return_status_codes():
    hostile = {ctypes.c_void_p: [None, 0x1001, 0xFFFFFFFFFFFFF000], ctypes.c_int64: [0, -1, 2**31, 2**62, -(2**63)],
               ctypes.c_int32: [0, -1, 2**31 - 1, -(2**31)], ctypes.c_float: [float("nan"), float("inf")],
               ctypes.c_size_t: [0, 2**63]}
    lib = _lib.load()
    for name, base in CALLS.items():
        types = _lib.SIGNATURES[name][1]
        for i, t in enumerate(types[:-1]):
            if i - len(types) == DTYPE_AT[name]:
                continue
            for v in hostile[t]:
                args = list(base)
                args[i] = v
                assert 0 <= getattr(lib, name)(*args) < _lib.SD_ERR_HIP, (name, i, v)


def test_no_rows_are_no_work():
    lib = _lib.load()
    assert lib.sd_quantize_rows_int8(None, 0, None, 0, None, 0, 64, BF16, None) == 0
    assert lib.sd_rmsnorm_int8(None, 0, None, 0, None, None, 0, None, None, 0, 0, 64, 1e-6, BF16, None) == 0
    assert lib.sd_dequantize_rows_int8(None, 0, None, None, 0, 0, 64, F32, None) == 0
    assert lib.sd_w8a8_linear(None, 0, None, None, 0, None, BF16, None, None, 0, 0, 64, 64, BF16, None, 0, None) == 0


def test_workspace_and_plan():
    ws, plan = _lib.load().sd_w8a8_workspace_size, _lib.load().sd_w8a8_plan
    assert ws(1, 4096, 1024, 0) == ws(0, 64, 64, 0) == ws(4096, 19456, 2560, 1) == ws(64, 64, 1 << 17, 0) == 0
    # few tiles, a long K: a whole number of slices
    for gated in (0, 1):
        assert ws(40, 64, 9728, gated) % (40 * 64 * 4 * (1 + gated)) == 0 and ws(40, 64, 9728, gated) > 0
    assert plan(1, 4096, 1000, 0) == plan(0, 1, 16, 0) == plan(1 << 25, 64, 64, 0) == 0
    assert plan(1, 4096, 1024, 0) >> 20 == 0 and plan(4096, 19456, 2560, 0) >> 20 >= 128


def test_ops_refuse_wrong_tensors():
    x = torch.zeros((2, 64), dtype=torch.bfloat16)
    c, s = torch.zeros((2, 64), dtype=torch.int8), torch.ones(2)
    w, ws = torch.zeros((8, 64), dtype=torch.int8), torch.ones(8)
    for f in (lambda: ops.quantize_rows_int8(x), lambda: ops.rmsnorm_int8(x, x[0], 1e-6),
              lambda: ops.dequantize_rows_int8(c, s), lambda: ops.w8a8_linear(c, s, w, ws),
              lambda: ops.w8a8_gate_up_silu(c, s, w, ws)):
        with pytest.raises(RuntimeError, match="ROCm GPU"):
            f()
    with pytest.raises(AssertionError, match="hidden"):
        ops.rmsnorm_int8(x, torch.ones(32, dtype=torch.bfloat16), 1e-6)
    with pytest.raises(AssertionError):
        ops.rmsnorm_int8(x, x[0], 1e-6, x[:1])
    with pytest.raises(AssertionError, match="one scale a row"):
        ops.dequantize_rows_int8(c, s[:1])
    with pytest.raises(AssertionError):
        ops.dequantize_rows_int8(c, s.half())
    for f in (ops.w8a8_linear, ops.w8a8_gate_up_silu):
        with pytest.raises(AssertionError, match="int8"):
            f(x, s, w, ws)
        with pytest.raises(AssertionError, match="K mismatch"):
            f(c[:, :32], s, w, ws)
        with pytest.raises(AssertionError, match="one scale a row"):
            f(c, ws, w, ws)
        with pytest.raises(AssertionError, match="one entry"):
            f(c, s, w, ws[:7])
        with pytest.raises(AssertionError, match="bias"):
            f(c, s, w, ws, torch.zeros(7))
    with pytest.raises(AssertionError, match="gate; up"):
        ops.w8a8_gate_up_silu(c, s, w[:7], ws[:7])


def test_out_has_the_result_s_shape(monkeypatch):
    monkeypatch.setattr(_lib, "require_device", lambda *t: torch.device("cpu"))
    c, s = torch.zeros((2, 64), dtype=torch.int8), torch.ones(2)
    w, ws = torch.zeros((8, 64), dtype=torch.int8), torch.ones(8)
    for out in (torch.empty((8, 2), dtype=torch.bfloat16), torch.empty((2, 8)), torch.empty((8, 2), dtype=torch.bfloat16).t()):
        with pytest.raises(AssertionError):
            ops.w8a8_linear(c, s, w, ws, out=out)
    with pytest.raises(AssertionError, match="out must be"):
        ops.w8a8_gate_up_silu(c, s, w, ws, out=torch.empty((2, 8), dtype=torch.bfloat16))


def test_oracle():
    v = np.array([[0.5, -127, 1.5, 2.5, 126.5], [0, 0, 0, 0, 0], [1, np.nan, 2, 3, 4], [1, np.inf, 2, 3, 4],
                  [1e-40, 1e-41, 0, 0, 0]], dtype=np.float32)
    c, most = o8.codes(v)
    assert c.tolist()[:4] == [[0, -127, 2, 2, 126], [0] * 5, [0] * 5, [0] * 5] and c[4].tolist() == [127, 13, 0, 0, 0]
    assert most[0] == 127 and most[1] == 0 and np.isnan(most[2:4]).all()
    s, p = o8.norm_products(np.ones((1, 2)), np.array([2.0, 3.0]), np.ones((1, 2)))
    assert s.tolist() == [[2, 2]] and p.tolist() == [[4, 6]]
    assert np.allclose(o8.norm_scale(np.array([127.0]), np.full((1, 4), 2.0), 0.0), [0.5])
    x, w = np.array([[1, 2], [3, 4]], dtype=np.int8), np.array([[5, 6], [7, -128]], dtype=np.int8)
    one = np.ones(2, dtype=np.float32)
    assert o8.linear32(x, one, w, one).tolist() == [[17, -249], [39, -491]] == o8.linear64(x, one, w, one).tolist()
    assert o8.linear32(x, one * 2, w, one, one).tolist() == [[35, -497], [79, -981]]
    assert np.allclose(o8.silu_up(np.array([[0.0, 1.0, 5.0, 2.0]])), [[0, 2 / (1 + np.exp(-1))]])


def test_layers_check_before_they_change():
    from specdec_nanovllm_amd.draft_chain import DraftChain
    from specdec_nanovllm_amd.layers.linear import ReplicatedLinear
    from specdec_nanovllm_amd.layers.quant import apply_int8_activations, apply_int8_quant

    m = torch.nn.ModuleDict(dict(a=ReplicatedLinear(64, 8), b=ReplicatedLinear(72, 8), c=torch.nn.Linear(64, 8)))
    for p in m.parameters():
        p.data = torch.zeros(p.shape, dtype=torch.bfloat16)
    for names, kw, error in ((["a", "x"], {}, KeyError), (["a", "c"], {}, TypeError), (["a", "b"], {}, ValueError),
                             (["a"], dict(granularity="per_group", group_size=64), ValueError)):
        with pytest.raises(error):
            apply_int8_quant(m, names, act_bits=8, **kw)
    with pytest.raises(ValueError, match="8 or 16"):
        apply_int8_quant(m, ["a"], act_bits=4)
    assert m["a"].weight.dtype == torch.bfloat16 and m["a"].quant_act_bits == 16
    with pytest.raises(AssertionError, match="int8"):
        apply_int8_activations(m, ["a"])
    for name, k in (("a", 64), ("b", 72)):
        m[name].weight = torch.nn.Parameter(torch.zeros((8, k), dtype=torch.int8), requires_grad=False)
        m[name].weight_scale = torch.nn.Parameter(torch.ones(8, dtype=torch.bfloat16), requires_grad=False)
    with pytest.raises(ValueError, match="multiple of 16"):
        apply_int8_activations(m, ["a", "b"])
    assert m["a"].quant_act_bits == 16
    with pytest.raises(ValueError, match="8 or 16"):
        apply_int8_activations(m, ["a"], 4)
    scale = m["a"].weight_scale
    for other in (None, torch.nn.Parameter(torch.ones((8, 2)), requires_grad=False)):  # of groups, whatever the name says
        m["a"].weight_scale = other
        with pytest.raises(ValueError, match="one weight scale a row"):
            apply_int8_activations(m, ["a"])
    m["a"].weight_scale = scale
    assert m["a"].quant_act_bits == 16
    apply_int8_activations(m, ["a"])
    assert m["a"].quant_act_bits == 8
    x = torch.zeros((2, 64), dtype=torch.bfloat16)
    with pytest.raises(RuntimeError, match="ROCm GPU"):  # dispatched to the integer linear, which has no CPU form
        m["a"](x)
    apply_int8_activations(m, ["a"], 16)
    with pytest.raises(TypeError, match="quant_act_bits"):
        m["a"]((x.to(torch.int8), torch.ones(2)))
    for bits in (dict(act_bits=4), dict(act_bits=8, weight_bits=4)):
        with pytest.raises(ValueError, match="8"):
            DraftChain(1, device="cpu", **bits)
