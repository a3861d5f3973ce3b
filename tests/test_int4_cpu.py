"""The 4-bit entry points without a GPU: refusals of the C ABI and of ``ops`` (before any launch),
the 64-bit oracle on hand-made rows, and a sweep of hostile arguments."""
import ctypes

import numpy as np
import pytest
import torch

from oracle import int4 as o4
from specdec_nanovllm_amd import _lib, ops

A = [0x10000000 + i * 0x1000000 for i in range(16)]  # 16-byte aligned, never dereferenced
CACHE = (A[0], 256 * 1024, 128, 256 * 128, A[1], 256 * 64, 8, 256 * 8, 64)
BF16, F32 = _lib.SD_BF16, _lib.SD_F32

CALLS = {  # valid calls with one plausible thing left out (dtype 7), so that nothing is launched
    "sd_store_kvcache_int4": [A[2], 1024, 128, A[3], 1024, 128, *CACHE, A[4], 16, 8, 128, 256, 64, 7, None],
    "sd_qk_norm_rope_store_int4": [A[2], 4096, 128, A[3], 1024, 128, A[4], 1024, 128, 16, 32, 8, 128, A[5], A[6],
                                   1e-6, A[7], A[8], 128, 4096, A[9], A[10], *CACHE, 64, 256, A[11], 7, None],
    "sd_load_kvcache_int4": [*CACHE, A[2], 16, 8, 128, 256, 64, 7, A[3], A[4], None],
    "sd_paged_attention_int4": [A[2], 4096, 128, *CACHE, 64, 256, A[3], 16, 16, A[4], None, None, 1, 16, 16, 32, 8,
                                128, 0.1, BF16, A[5], 4096, 128, None, 0, 0, None],
    "sd_w4a16_linear": [A[2], 1024, A[3], 512, A[4], BF16, 128, None, A[5], 4096, 4, 4096, 1024, 7, None, 0, None],
}
DTYPE_AT = {"sd_store_kvcache_int4": -2, "sd_qk_norm_rope_store_int4": -2, "sd_load_kvcache_int4": -4,
            "sd_w4a16_linear": -4}
no_gpu = pytest.mark.skipif(torch.cuda.device_count() > 0,
                            reason="fake device addresses: only where no GPU can be reached")


def call(name, **change):
    """The call with arguments replaced by position (``a3=...``)."""
    args = list(CALLS[name])
    for k, v in change.items():
        args[int(k[1:])] = v
    lib = _lib.load()
    return getattr(lib, name)(*args), lib.sd_last_error().decode()


@no_gpu
@pytest.mark.parametrize("name,change,rc,says", [
    ("sd_store_kvcache_int4", {}, 2, "dtype"),
    ("sd_store_kvcache_int4", {"a14": 48}, 2, "groups of 32, 64 or 128"),
    ("sd_store_kvcache_int4", {"a18": 64}, 2, "head_dim 128"),
    ("sd_store_kvcache_int4", {"a16": -1}, 1, "invalid sizes"),
    ("sd_load_kvcache_int4", {"a15": BF16, "a14": 1 << 31}, 2, "too large"),
    ("sd_load_kvcache_int4", {"a8": 96}, 2, "groups of 32"),
    ("sd_qk_norm_rope_store_int4", {"a19": 0}, 1, "positions"),
    ("sd_paged_attention_int4", {}, 3, "workspace"),
    ("sd_paged_attention_int4", {"a23": 30}, 1, "GQA"),
    ("sd_paged_attention_int4", {"a20": 9, "a19": A[6]}, 2, "exceeds 32"),
    ("sd_paged_attention_int4", {"a20": 2}, 1, "max_qlen must be 1"),
    ("sd_paged_attention_int4", {"a25": 64}, 2, "head_dim 128"),
    ("sd_paged_attention_int4", {"a16": 1 << 24}, 2, "too much work"),
    ("sd_paged_attention_int4", {"a7": A[1] + 8}, 2, "aligned"),
    ("sd_paged_attention_int4", {"a4": 120}, 2, "aligned"),
    ("sd_paged_attention_int4", {"a5": -128}, 2, "position strides"),
    ("sd_paged_attention_int4", {"a27": F32}, 2, "dtype"),
    ("sd_paged_attention_int4", {"a17": None}, 1, "null"),
    ("sd_w4a16_linear", {}, 2, "dtype"),
    ("sd_w4a16_linear", {"a6": 48}, 2, "multiple of 32"),
    ("sd_w4a16_linear", {"a6": 384}, 2, "divide K"),
    ("sd_w4a16_linear", {"a10": -1}, 1, "invalid sizes"),
    ("sd_w4a16_linear", {"a13": BF16, "a8": A[2] + 512}, 1, "shares memory"),
    ("sd_w4a16_linear", {"a13": BF16, "a1": 1020}, 2, "aligned"),
    ("sd_w4a16_linear", {"a13": BF16, "a3": -512}, 1, "strides"),
    ("sd_w4a16_linear", {"a13": BF16, "a9": 4095}, 1, "overlap"),
    ("sd_w4a16_linear", {"a13": BF16, "a11": 1 << 30}, 2, "too large"),
    ("sd_w4a16_linear", {"a13": BF16, "a10": 1 << 24, "a11": 8128, "a9": 8128}, 2, "too large"),
])
def test_refusals_say_what_is_wrong(name, change, rc, says):
    got, message = call(name, **change)
    assert got == rc and says in message, (got, message)


@no_gpu
def test_hostile_arguments_return_status_codes():
    hostile = {ctypes.c_void_p: [None, 0x1001, 0xFFFFFFFFFFFFF000], ctypes.c_int64: [0, -1, 2**31, 2**62, -(2**63)],
               ctypes.c_int32: [0, -1, 2**31 - 1, -(2**31)], ctypes.c_float: [float("nan"), float("inf")],
               ctypes.c_size_t: [0, 2**63]}
    lib = _lib.load()
    for name, base in CALLS.items():
        types = _lib.SIGNATURES[name][1]
        for i, t in enumerate(types[:-1]):
            if i - len(types) == DTYPE_AT.get(name):
                continue
            for v in hostile[t]:
                args = list(base)
                args[i] = v
                assert 0 <= getattr(lib, name)(*args) < _lib.SD_ERR_HIP, (name, i, v)


def test_workspace_queries():
    f = _lib.load().sd_paged_attention_int4_workspace_size
    assert f(0, 1, 32, 8, 4096, 0) == 0
    assert f(4, 1, 32, 8, 512, 0) == 0  # few keys a pair: one launch, no workspace
    assert f(4, 1, 32, 8, 4096, 5) == 2 * 4 * 8 * 5 * 4 * 132 * 4
    assert f(4, 9, 32, 8, 4096, 0) == f(1 << 30, 1, 32, 8, 4096, 0) == f(1, 1, 32, 8, 1 << 31, 0) == 2**64 - 1


def test_w4a16_workspace():
    f = _lib.load().sd_w4a16_workspace_size
    assert f(16, 4096, 4096, 64) == f(0, 64, 64, 64) == f(640, 1 << 30, 64, 64) == f(1000, 19456, 2560, 128) == 0
    # few tiles, a long K: a whole number of slices
    assert f(65, 256, 8192, 128) % (65 * 256 * 4) == 0 and f(65, 256, 8192, 128) > 65 * 256 * 4


def test_ops_refuse_wrong_tensors():
    codes, scales = ops.int4_kvcache(2, 16, 4, 64, device="cpu")
    assert codes.shape == (2, 16, 4, 128) and scales.shape == (2, 16, 4, 8)
    k = torch.zeros((1, 4, 128), dtype=torch.bfloat16)
    slot = torch.zeros(1, dtype=torch.int32)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        ops.store_kvcache_int4(k, k, codes, scales, slot)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        ops.load_kvcache_int4(codes, scales, slot)
    with pytest.raises(AssertionError, match="as the activations"):
        ops.store_kvcache_int4(k.half(), k.half(), codes, scales, slot)
    with pytest.raises(AssertionError):
        ops.store_kvcache_int4(k[:, :2], k[:, :2], codes, scales, slot)
    with pytest.raises(AssertionError, match="group_size"):
        ops.int4_kvcache(2, 16, 4, 48, device="cpu")
    table, ctx = torch.zeros((1, 1), dtype=torch.int32), torch.ones(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="exactly one"):
        ops.paged_attention_int4(k, codes, scales, table, 0.1)
    with pytest.raises(ValueError, match="one query row"):
        ops.paged_attention_int4(k.expand(2, 4, 128), codes, scales, table, 0.1, context_lens=ctx)
    with pytest.raises(AssertionError, match="uint8"):
        ops.paged_attention_int4(k, codes.float(), scales, table, 0.1, context_lens=ctx)
    with pytest.raises(AssertionError, match="GQA"):
        ops.paged_attention_int4(k[:, :3], codes, scales, table, 0.1, context_lens=ctx)
    x, w = torch.zeros((1, 64), dtype=torch.bfloat16), torch.zeros((8, 32), dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="ROCm GPU"):
        ops.w4a16_linear(x, w, torch.ones((8, 2)))
    with pytest.raises(AssertionError, match="scale"):
        ops.w4a16_linear(x, w, torch.ones((8, 3)))
    with pytest.raises(AssertionError, match="K mismatch"):
        ops.w4a16_linear(x[:, :32], w, torch.ones((8, 2)))
    with pytest.raises(AssertionError, match="uint8"):
        ops.w4a16_linear(x, w.to(torch.int8), torch.ones((8, 2)))


def test_w4a16_out_has_the_result_s_shape(monkeypatch):
    monkeypatch.setattr(_lib, "require_device", lambda *t: torch.device("cpu"))
    x, w, s = torch.zeros((4, 64), dtype=torch.bfloat16), torch.zeros((8, 32), dtype=torch.uint8), torch.ones((8, 2))
    with pytest.raises(AssertionError, match="out must be"):
        ops.w4a16_linear(x, w, s, out=torch.empty((8, 4), dtype=torch.bfloat16))


@pytest.mark.parametrize("n,k,group", [(3, 64, 32), (70, 256, 128), (1, 96, 96)])
def test_quantize_weight_int4(n, k, group):
    from specdec_nanovllm_amd.layers.quant import dequantize_weight_int4, quantize_weight_int4

    w = torch.randn((n, k), generator=torch.Generator().manual_seed(n)).to(torch.bfloat16)
    w[0, :group] = 0
    q, s = quantize_weight_int4(w, group)
    assert q.shape == (n, k // 2) and s.shape == (n, k // group) and s.dtype == torch.bfloat16
    x = w.double().numpy().reshape(n, -1, group)
    exact = np.maximum(np.abs(x).max(-1) / 7, 1e-8)
    assert (np.abs(s.double().numpy() - exact) <= 2**-8 * exact * 1.001).all()  # rounded to bf16 once
    code = np.empty((n, k), dtype=np.int64)
    code[:, 0::2], code[:, 1::2] = q.numpy() & 15, q.numpy() >> 4
    assert code.min() >= 1 and code.max() <= 15
    # the nearest level of the unrounded scale; 2^-20: its fp32 quotient
    assert (np.abs(code.reshape(x.shape) - 8 - x / exact[..., None]) <= 0.5 + 2**-20).all()
    assert np.array_equal(dequantize_weight_int4(q, s).double().numpy(), o4.weights(q.numpy(), s.double().numpy()))
    for bad in (48, 0, 2 * k):
        with pytest.raises(AssertionError, match="groups"):
            quantize_weight_int4(w, bad)


def test_apply_int4_quant_checks_before_it_changes():
    from specdec_nanovllm_amd.layers.linear import ReplicatedLinear
    from specdec_nanovllm_amd.layers.quant import apply_int4_quant

    m = torch.nn.ModuleDict(dict(a=ReplicatedLinear(64, 8), b=ReplicatedLinear(96, 8), c=torch.nn.Linear(64, 8)))
    for p in m.parameters():
        p.data = torch.randn(p.shape, generator=torch.Generator().manual_seed(0)).to(torch.bfloat16)
    for names, group, error in ((["a", "x"], 32, KeyError), (["a", "c"], 32, TypeError), (["a", "b"], 64, ValueError)):
        with pytest.raises(error):
            apply_int4_quant(m, names, group)
        assert m["a"].weight.dtype == torch.bfloat16
    report = apply_int4_quant(m, ["a", "b"], 32)
    assert [r["name"] for r in report] == ["a", "b"] and all(0 < r["rel_err"] < 0.15 for r in report)
    assert m["a"].weight.dtype == torch.uint8 and m["b"].weight_scale.shape == (8, 3)
    with pytest.raises(RuntimeError, match="ROCm GPU"):  # dispatched to the 4-bit linear, which has no CPU form
        m["a"](torch.zeros((1, 64), dtype=torch.bfloat16))


def test_oracle_orders_are_permutations_and_rounding_is_to_even():
    for f in (o4.key_dim, o4.value_dim):
        assert sorted(f(i) for i in range(128)) == list(range(128))
    row = np.zeros(64, dtype=np.uint8)
    row[4 * 7 + 2] = 0x50  # dword 7 (g 1, i 3), nibble 5: dim 96 + 8 + 2 + 1; as a value: 16 * 5 + 7
    assert np.flatnonzero(o4.unpack(row, o4.key_dim)).tolist() == [107]
    assert np.flatnonzero(o4.unpack(row, o4.value_dim)).tolist() == [87]
    x = torch.randn(1000, generator=torch.Generator().manual_seed(0)) * 1e-3
    assert np.array_equal(o4.round16(x.double().numpy(), "fp16"), x.half().double().numpy())
    assert np.array_equal(o4.round16(x.double().numpy(), "bf16"), x.bfloat16().double().numpy())
