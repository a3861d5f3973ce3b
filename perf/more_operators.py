"""Linears in 8-bit integers and what makes their activations, as measurable cases.

Four kinds: RMSNorm with the residual's addition and its output in 8 bits (read back in 16), rows quantized to 8 bits
(read back), the linear of 8-bit activations and 8-bit weights with a scale per token and per channel, and the gated
projections of an MLP with SiLU and the product on the same integers. Geometries are the library's own: layers of hidden
1024 and 2560 (intermediate 9728, q/k/v of 4096 and 6144 columns), and generic ones around them.

Format: a row's codes are -127 .. 127 with one fp32 scale, value = code * scale, scale = max |v| / 127 and
code = round(127 v / max |v|), half to even. The norm quantizes its unrounded result.
"""
from __future__ import annotations

import math

import torch

own = False

EPS = 1e-6
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16}


# ------------------------------------------------------------------------------------- cases
def listed():
    return [
        # one token of a draft step: the norm before its q/k/v projection
        dict(name="norm_1", kind="norm", rows=1, k=1024, residual=True, dtype="bf16"),
        # a prompt of odd length, before the first layer's projection
        dict(name="norm_777", kind="norm", rows=777, k=2560, residual=False, dtype="fp16"),
        # a prefill batch
        dict(name="norm_8192", kind="norm", rows=8192, k=2560, residual=True, dtype="bf16"),
        # a verify step's rows before the down projection
        dict(name="quantize_7", kind="quantize", rows=7, k=9728, dtype="bf16"),
        # a long prompt's attention output before the o projection
        dict(name="quantize_4001", kind="quantize", rows=4001, k=4096, dtype="bf16"),
        # one token through a small decoder layer's q/k/v projection: the latency of a step
        dict(name="linear_1", kind="linear", rows=1, n=4096, k=1024, bias=False, dtype="bf16"),
        # a batch of users through the down projection: few tiles, a long sum
        dict(name="linear_16_down", kind="linear", rows=16, n=2560, k=9728, bias=False, dtype="bf16"),
        # a batch of verify steps through the q/k/v projection
        dict(name="linear_200_qkv", kind="linear", rows=200, n=6144, k=2560, bias=True, dtype="fp16"),
        # a prompt of odd length through the down projection
        dict(name="linear_777_down", kind="linear", rows=777, n=2560, k=9728, bias=False, dtype="bf16"),
        # one token through the gated projections of a larger layer
        dict(name="gate_up_1", kind="gate_up", rows=1, n=9728, k=2560, dtype="bf16"),
        # a short prompt
        dict(name="gate_up_130", kind="gate_up", rows=130, n=9728, k=2560, dtype="bf16"),
        # a prefill batch
        dict(name="gate_up_4096", kind="gate_up", rows=4096, n=9728, k=2560, dtype="bf16"),
    ]


def _log_int(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["norm", "quantize", "linear", "linear", "linear", "gate_up", "gate_up"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    k = 16 * _log_int(rng, 16, 608)
    if kind in ("norm", "quantize"):
        rows = _log_int(rng, 1, min(8192, 8192 * 2560 // k))
        case = dict(kind=kind, rows=rows, k=k, dtype=dtype)
        return dict(case, residual=rng.random() < 0.6) if kind == "norm" else case
    n = _log_int(rng, 200, 19456 if kind == "linear" else 9728)  # of gate_up: its outputs, twice as many weight rows
    most = 4096 * 9728 * 2560 * 2 // (n * k * (1 if kind == "linear" else 2))
    case = dict(kind=kind, rows=_log_int(rng, 1, min(4096, most)), n=n, k=k, dtype=dtype)
    return dict(case, bias=rng.random() < 0.5) if kind == "linear" else case


# ------------------------------------------------------------------------------------- inputs
def _randn(g, shape, std=1.0):
    return torch.randn(shape, generator=g, device="cuda") * std


def _rows(g, rows, k):
    """Activations: some channels are larger than others."""
    return _randn(g, (rows, k)) * torch.exp(0.5 * _randn(g, (k,)))


def _codes(g, rows, k, activations):
    """Codes and scales of rows that are quantized already."""
    x = _rows(g, rows, k) if activations else _randn(g, (rows, k), 0.02)
    most = x.abs().amax(-1, keepdim=True)
    return torch.round(x * (127 / most)).to(torch.int8), most[:, 0] / 127


def prepare(case, seed):
    g = torch.Generator(device="cuda")
    g.manual_seed(seed)
    dtype, rows, k = DTYPES[case["dtype"]], case["rows"], case["k"]
    st = dict(case=case)
    if case["kind"] in ("norm", "quantize"):
        st["x"] = _rows(g, rows, k).to(dtype)
        if case["kind"] == "norm":
            st["weight"] = (1 + _randn(g, (k,), 0.1)).to(dtype)
            st["residual"] = _rows(g, rows, k).to(dtype) if case["residual"] else None
        return st
    st["codes"], st["x_scale"] = _codes(g, rows, k, True)
    n = case["n"] * (2 if case["kind"] == "gate_up" else 1)
    st["w"], scale = _codes(g, n, k, False)
    st["scale"] = scale.to(torch.bfloat16)
    st["bias"] = _randn(g, (n,), 0.1).to(dtype) if case.get("bias") else None
    return st


# ----------------------------------------------------------------------------------- plain forms
def _plain_quantize(v):
    """Codes and max |v| of rows; 64 bits, so that a value next to a border takes the code that its formula says."""
    most = v.abs().amax(-1, keepdim=True)
    return torch.where(most > 0, torch.round(127 * v / torch.where(most > 0, most, 1)), 0), most


def _plain_norm(st):
    dtype = st["x"].dtype
    s = st["x"].float()
    if st["residual"] is not None:
        s = s + st["residual"].float()
    code, most = _plain_quantize(s.double() * st["weight"].double())
    scale = most.float() * torch.rsqrt((s * s).mean(-1, keepdim=True) + EPS) / 127
    value = (code.float() * scale).to(dtype)
    return (value, s.to(dtype)) if st["residual"] is not None else value


def _plain_rows(st):
    code, most = _plain_quantize(st["x"].double())
    return (code.float() * (most.float() / 127)).to(st["x"].dtype)


def _plain_product(st):
    y = st["codes"].float() @ st["w"].float().T
    y = y * st["scale"].float() * st["x_scale"][:, None]
    return y if st["bias"] is None else y + st["bias"].float()


def _plain_gate_up(st):
    gate, up = _plain_product(st).chunk(2, -1)
    return gate / (1 + torch.exp(-gate)) * up


# ---------------------------------------------------------------------------------------- a pass
_OPS = []  # the package, once it is asked for


def _ops():
    if not _OPS:
        import __graft_entry__

        _OPS.append(__graft_entry__.load_package().ops)
    return _OPS[0]


def _own_run(st):
    ops, kind, dtype = _ops(), st["case"]["kind"], DTYPES[st["case"]["dtype"]]
    if kind == "norm":
        codes, scale, *residual = ops.rmsnorm_int8(st["x"], st["weight"], EPS, st["residual"])
        value = ops.dequantize_rows_int8(codes, scale, dtype)
        return (value, *residual) if residual else value
    if kind == "quantize":
        return ops.dequantize_rows_int8(*ops.quantize_rows_int8(st["x"]), dtype)
    if kind == "linear":
        return ops.w8a8_linear(st["codes"], st["x_scale"], st["w"], st["scale"], st["bias"], dtype)
    return ops.w8a8_gate_up_silu(st["codes"], st["x_scale"], st["w"], st["scale"], dtype=dtype)


def run(state):
    if own:
        return _own_run(state)
    kind, dtype = state["case"]["kind"], DTYPES[state["case"]["dtype"]]
    if kind == "norm":
        return _plain_norm(state)
    if kind == "quantize":
        return _plain_rows(state)
    return (_plain_product(state) if kind == "linear" else _plain_gate_up(state)).to(dtype)


# ------------------------------------------------------------------------------------------ work
def work(case):
    m, k = case["rows"], case["k"]
    if case["kind"] in ("norm", "quantize"):
        moved = m * k * 3 + 4 * m + m * k * 3 + 4 * m  # rows in, codes and scales out; read back
        if case["kind"] == "norm":
            moved += 2 * k + (4 * m * k if case["residual"] else 0)
        return dict(bytes=moved, flops=m * k * (12 if case["kind"] == "norm" else 5))
    n = case["n"]
    rows = n * (2 if case["kind"] == "gate_up" else 1)
    moved = rows * k + m * k + 2 * m * n + 2 * rows + 4 * m + (2 * n if case.get("bias") else 0)
    return dict(bytes=moved, flops=2 * m * rows * k)


# ----------------------------------------------------------------------------------------- exact
def _x_levels(v):
    """Each value moved to the nearest of its row's 255 levels, ties to the even one."""
    step = v.abs().max(1, keepdim=True).values / 127
    return torch.nan_to_num(v / step, nan=0.0).round() * step


def exact(case, seed):
    st = prepare(case, seed)
    if case["kind"] == "quantize":
        return _x_levels(st["x"].double())
    if case["kind"] == "norm":
        h = st["x"].double()
        if case["residual"]:
            h = h + st["residual"].double()
        # the levels of a row are those of its unnormed products, each over the row's root mean square
        value = _x_levels(h * st["weight"].double()) / (h.square().sum(1, keepdim=True) / case["k"] + EPS).sqrt()
        return [value, h] if case["residual"] else value
    m, n = case["rows"], st["w"].shape[0]
    y = torch.matmul(st["codes"].double(), st["w"].double().t().contiguous())  # whole numbers below 2^53
    y = y * torch.outer(st["x_scale"].double(), st["scale"].double())
    if case.get("bias"):
        y = y + st["bias"].double().expand(m, n)
    if case["kind"] == "linear":
        return y
    return y[:, :n // 2] * torch.sigmoid(y[:, :n // 2]) * y[:, n // 2:]
