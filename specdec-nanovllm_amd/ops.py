"""Torch-facing wrappers of the three hot-path kernels.

Each function validates shapes the way the reference does (``assert`` where the
reference asserts), allocates the output and the split workspace with torch's
caching allocator on the current stream (so the call is graph-capturable and
reentrant across streams), and enqueues the HIP kernels through the C ABI on
``torch.cuda.current_stream()``. Nothing here computes on the CPU.
"""
from __future__ import annotations

import torch

from . import _lib


def _workspace(nbytes: int, dev: torch.device) -> torch.Tensor | None:
    if nbytes <= 0:
        return None
    return torch.empty(nbytes, dtype=torch.uint8, device=dev)


def _ptr(t: torch.Tensor | None) -> int | None:
    return None if t is None else t.data_ptr()


def _i32(t: torch.Tensor | None) -> torch.Tensor | None:
    if t is None:
        return None
    if t.dtype != torch.int32:
        t = t.to(torch.int32)
    return t.contiguous()


# --------------------------------------------------------------------------- store
def store_kvcache(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor,
                  v_cache: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """Write token rows of key/value into the paged cache at ``slot_mapping``.

    Contract of ``store_kvcache`` (nanovllm/layers/attention.py:33-40): key and
    value are (N, num_kv_heads, head_dim) with contiguous heads, the caches are
    (num_blocks, block_size, num_kv_heads, head_dim) with stride(1) equal to
    num_kv_heads * head_dim, and slot -1 skips the row.
    """
    N, num_heads, head_dim = key.shape
    D = num_heads * head_dim
    assert key.stride(-1) == 1 and value.stride(-1) == 1
    assert key.stride(1) == head_dim and value.stride(1) == head_dim
    assert k_cache.stride(1) == D and v_cache.stride(1) == D
    assert slot_mapping.numel() == N
    assert k_cache.stride() == v_cache.stride() and k_cache.shape == v_cache.shape
    assert key.dtype == value.dtype == k_cache.dtype == v_cache.dtype
    assert k_cache.dim() == 4 and k_cache.shape[2] == num_heads and k_cache.shape[3] == head_dim
    dev = _lib.require_device(key, value, k_cache, v_cache, slot_mapping)
    if N == 0:
        return
    slots = _i32(slot_mapping.reshape(-1))
    lib = _lib.load()
    with _lib.on_device(dev):
        rc = lib.sd_store_kvcache(
            key.data_ptr(), key.stride(0), key.stride(1),
            value.data_ptr(), value.stride(0), value.stride(1),
            k_cache.data_ptr(), v_cache.data_ptr(),
            k_cache.stride(0), k_cache.stride(1), k_cache.stride(2),
            slots.data_ptr(), N, num_heads, head_dim, k_cache.shape[1], k_cache.shape[0],
            key.element_size(), _lib.stream_ptr(dev))
    _lib.check(rc)


# ----------------------------------------------------------------------- attention
def _cache_geometry(k_cache: torch.Tensor, layout: str):
    if layout == "head_major":
        # (num_blocks, num_kv_heads, block_size, head_dim)
        num_blocks, num_kv_heads, block_size, head_dim = k_cache.shape
        sb, sh, sp = k_cache.stride(0), k_cache.stride(1), k_cache.stride(2)
    elif layout == "interleaved":
        # (num_blocks, block_size, num_kv_heads, head_dim): nano-vllm / flash-attn layout
        num_blocks, block_size, num_kv_heads, head_dim = k_cache.shape
        sb, sp, sh = k_cache.stride(0), k_cache.stride(1), k_cache.stride(2)
    else:
        raise ValueError(f"unknown layout: {layout}")
    return num_blocks, block_size, num_kv_heads, head_dim, sb, sp, sh


def paged_attention_workspace_bytes(num_seqs: int, max_seqlen_q: int, num_q_heads: int,
                                    num_kv_heads: int, max_ctx: int, num_splits: int = 0,
                                    device: torch.device | str | None = None) -> int:
    """Bytes of the split-KV workspace ``paged_attention`` uses for these sizes on
    ``device`` (the plan follows the device's compute units)."""
    lib = _lib.load()
    with torch.cuda.device(torch.device(device) if device is not None else
                           torch.cuda.current_device()):
        return int(lib.sd_paged_attention_workspace_size(
            int(num_seqs), int(max_seqlen_q), int(num_q_heads), int(num_kv_heads), 128,
            int(max_ctx), int(num_splits)))


def paged_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                    block_table: torch.Tensor, scale: float, *,
                    context_lens: torch.Tensor | None = None,
                    cu_seqlens_k: torch.Tensor | None = None,
                    cu_seqlens_q: torch.Tensor | None = None, max_seqlen_q: int = 1,
                    layout: str = "interleaved", num_splits: int = 0,
                    out: torch.Tensor | None = None, main_only: bool = False,
                    key: torch.Tensor | None = None, value: torch.Tensor | None = None,
                    slot_mapping: torch.Tensor | None = None,
                    no_alloc: bool = False, twin: str | None = None,
                    workspace: torch.Tensor | None = None) -> torch.Tensor:
    """Paged decode (``cu_seqlens_q is None``: one query row per sequence) or
    speculative-verify attention (rows ``cu_seqlens_q[b]:cu_seqlens_q[b+1]``,
    bottom-right causal), GQA, split-KV.

    q: (total_q, num_q_heads, head_dim); keys per sequence from ``context_lens``
    (B,) or ``cu_seqlens_k`` (B+1,). Returns ``out`` (same shape/dtype as q).
    ``main_only`` runs only the split-KV main kernel (measurement twin; the
    same as ``twin="main"``). The other measurement twins: ``twin="combine"``
    runs only the merge over ``workspace`` as a ``twin="main"`` call with the
    same arguments left it; ``twin="floor"`` issues only the main kernel's loads
    (no math, ``out`` untouched). ``workspace`` (uint8, at least the size the
    library asks for) replaces the workspace otherwise allocated per call.

    ``key``/``value`` (total_q, num_kv_heads, head_dim) with ``slot_mapping``
    (total_q,): store_kvcache of these rows fused into the same launch — the
    ``Attention.forward`` sequence (nanovllm/layers/attention.py:59-82). The
    same cache as ``store_kvcache`` and the output of attention afterwards up to
    rounding (the new keys are scored in fp32 in the merge launch), for the
    engine's slot layout: sequence b's rows are its last n_b keys (slot -1: not
    written).

    ``no_alloc`` runs the same kernels on the library's static device scratch
    (``sd_paged_attention_noalloc``) instead of a workspace from torch's
    allocator; pass ``out`` as well to allocate nothing at all. Calls that
    overlap in time on one device share that scratch and race.
    """
    if q.dim() != 3:
        raise ValueError(f"q must be (tokens, heads, head_dim), got {tuple(q.shape)}")
    total_q, num_q_heads, head_dim = q.shape
    num_blocks, block_size, num_kv_heads, hd_c, sb, sp, sh = _cache_geometry(k_cache, layout)
    assert num_q_heads % num_kv_heads == 0, \
        f"GQA needs num_q_heads divisible by num_kv_heads: {num_q_heads} vs {num_kv_heads}"
    assert hd_c == head_dim, f"head_dim mismatch: q {head_dim} vs cache {hd_c}"
    assert k_cache.shape == v_cache.shape and k_cache.stride() == v_cache.stride()
    assert k_cache.dtype == v_cache.dtype == q.dtype, "q and caches must share one dtype"
    assert k_cache.stride(-1) == 1 and q.stride(-1) == 1
    assert block_table.dim() == 2, "block_table must be (num_seqs, max_blocks)"
    if (context_lens is None) == (cu_seqlens_k is None):
        raise ValueError("give exactly one of context_lens / cu_seqlens_k")
    dev = _lib.require_device(q, k_cache, v_cache, block_table, context_lens, cu_seqlens_k,
                              cu_seqlens_q, out)
    num_seqs = block_table.shape[0]
    bt = _i32(block_table)
    ctx = _i32(context_lens)
    cuk = _i32(cu_seqlens_k)
    cuq = _i32(cu_seqlens_q)
    if cuq is None:
        max_seqlen_q = 1
        if total_q != num_seqs:
            raise ValueError(f"decode expects one query row per sequence: q has {total_q} rows, "
                             f"block_table {num_seqs}")
    if out is None:
        out = torch.empty_like(q)
    else:
        assert out.shape == q.shape and out.dtype == q.dtype and out.stride(-1) == 1
    if main_only:
        twin = "main"
    if twin not in (None, "main", "combine", "floor"):
        raise ValueError(f"unknown twin: {twin}")
    fused = key is not None
    assert not (no_alloc and (fused or twin)), "no_alloc is the plain attention call"
    assert not (fused and twin), "the measurement twins are plain attention calls"
    if fused:
        assert value is not None and slot_mapping is not None
        assert key.shape == (total_q, num_kv_heads, head_dim) and value.shape == key.shape
        assert key.dtype == value.dtype == q.dtype
        assert key.stride(-1) == 1 and value.stride(-1) == 1
        assert slot_mapping.numel() == total_q
        _lib.require_device(key, value, slot_mapping)
    if total_q == 0 or (num_seqs == 0 and not fused):
        return out  # (num_seqs == 0 with new rows: the library only stores them)
    lib = _lib.load()
    max_blocks = bt.shape[1]
    fn = {None: lib.sd_paged_attention, "main": lib.sd_paged_attention_partial,
          "combine": lib.sd_paged_attention_combine,
          "floor": lib.sd_paged_attention_floor}[twin]
    new_rows = ()
    if fused:
        slots = _i32(slot_mapping.reshape(-1))
        fn = lib.sd_paged_attention_store
        new_rows = (key.data_ptr(), key.stride(0), key.stride(1),
                    value.data_ptr(), value.stride(0), value.stride(1), slots.data_ptr())
    if no_alloc:
        with _lib.on_device(dev):
            rc = lib.sd_paged_attention_noalloc(
                q.data_ptr(), q.stride(0), q.stride(1),
                k_cache.data_ptr(), v_cache.data_ptr(), sb, sp, sh, num_blocks,
                block_size, bt.data_ptr(), bt.stride(0), max_blocks,
                _ptr(ctx), _ptr(cuk), _ptr(cuq),
                int(max_seqlen_q), total_q, num_seqs, num_q_heads, num_kv_heads, head_dim,
                float(scale), _lib.dtype_code(q.dtype),
                out.data_ptr(), out.stride(0), out.stride(1), int(num_splits),
                _lib.stream_ptr(dev))
        _lib.check(rc)
        return out
    with _lib.on_device(dev):
        # the plan (and so the workspace) depends on the device's compute units
        ws_bytes = lib.sd_paged_attention_workspace_size(
            num_seqs, int(max_seqlen_q), num_q_heads, num_kv_heads, head_dim,
            max_blocks * block_size, int(num_splits))
        if workspace is not None:
            assert workspace.dtype == torch.uint8 and workspace.is_contiguous()
            if workspace.numel() < ws_bytes:
                raise RuntimeError(f"workspace of {workspace.numel()} bytes, {ws_bytes} needed")
            _lib.require_device(workspace)
            ws, ws_bytes = workspace, workspace.numel()
        else:
            ws = _workspace(ws_bytes, dev)
        rc = fn(*new_rows, q.data_ptr(), q.stride(0), q.stride(1),
                k_cache.data_ptr(), v_cache.data_ptr(), sb, sp, sh, num_blocks,
                block_size, bt.data_ptr(), bt.stride(0), max_blocks,
                _ptr(ctx), _ptr(cuk), _ptr(cuq),
                int(max_seqlen_q), total_q, num_seqs, num_q_heads, num_kv_heads, head_dim,
                float(scale), _lib.dtype_code(q.dtype),
                out.data_ptr(), out.stride(0), out.stride(1),
                _ptr(ws), ws_bytes, int(num_splits), _lib.stream_ptr(dev))
    _lib.check(rc)
    return out


def prefill_attention(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                      cu_seqlens_q: torch.Tensor, cu_seqlens_k: torch.Tensor,
                      max_seqlen_q: int, scale: float, block_table: torch.Tensor | None = None,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """Variable-length causal attention (the prefill call of the attention layer,
    nanovllm/layers/attention.py:64-70): q (total_q, Hq, 128); ``k``/``v`` are
    contiguous (total_k, Hkv, 128) rows when ``block_table`` is None, else the
    paged caches (num_blocks, block_size, Hkv, 128). Row t of sequence b sees
    keys [0, nk_b - nq_b + t]. Returns (total_q, Hq, 128)."""
    total_q, num_q_heads, head_dim = q.shape
    assert k.shape == v.shape and k.stride() == v.stride()
    assert q.stride(-1) == 1 and k.stride(-1) == 1
    num_seqs = cu_seqlens_q.numel() - 1
    cuq, cuk = _i32(cu_seqlens_q), _i32(cu_seqlens_k)
    assert cuk.numel() == num_seqs + 1
    if block_table is None:
        assert k.dim() == 3, "contiguous k/v must be (total_k, Hkv, D)"
        num_kv_heads = k.shape[1]
        s_tok, s_head, s_blk, num_blocks, block_size = k.stride(0), k.stride(1), 0, 0, 0
        bt, bt_stride, max_blocks = None, 0, 0
    else:
        assert k.dim() == 4, "paged k/v cache must be (num_blocks, block_size, Hkv, D)"
        num_blocks, block_size, num_kv_heads, _ = k.shape
        s_blk, s_tok, s_head = k.stride(0), k.stride(1), k.stride(2)
        bt = _i32(block_table)
        bt_stride, max_blocks = bt.stride(0), bt.shape[1]
    assert num_q_heads % num_kv_heads == 0, "GQA needs num_q_heads % num_kv_heads == 0"
    dev = _lib.require_device(q, k, v, cuq, cuk, bt, out)
    if out is None:
        out = torch.empty_like(q)
    if num_seqs <= 0 or total_q == 0:
        return out
    lib = _lib.load()
    with _lib.on_device(dev):
        rc = lib.sd_prefill_attention(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(),
                                      v.data_ptr(), s_tok, s_head, s_blk, num_blocks, block_size,
                                      _ptr(bt), bt_stride, max_blocks, cuq.data_ptr(),
                                      cuk.data_ptr(), int(max_seqlen_q), total_q, num_seqs,
                                      num_q_heads, num_kv_heads, head_dim, float(scale),
                                      _lib.dtype_code(q.dtype), out.data_ptr(), out.stride(0),
                                      out.stride(1), _lib.stream_ptr(dev))
    _lib.check(rc)
    return out


# -------------------------------------------------------------------------- w8a16
def w8a16_linear(x: torch.Tensor, qweight: torch.Tensor, scale: torch.Tensor,
                 bias: torch.Tensor | None = None, group_size: int = 0,
                 out: torch.Tensor | None = None, twin: str | None = None) -> torch.Tensor:
    """y = x @ (qweight * scale)^T + bias with the dequantization fused.

    x: (..., K) fp16/bf16; qweight: (N, K) int8; scale: (N,) when
    ``group_size == 0`` else (N, K // group_size); returns (..., N) in x.dtype.
    ``twin="floor"``: the measurement twin instead (sd_w8a16_floor: the same
    plan, grid and loads with no math; per-channel scales only); the output
    is left unwritten.
    """
    if twin not in (None, "floor"):
        raise ValueError(f"unknown twin {twin!r}")
    assert qweight.dtype == torch.int8, f"qweight must be int8, got {qweight.dtype}"
    assert qweight.dim() == 2
    N, K = qweight.shape
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    M = x2.shape[0]
    assert x2.shape[1] == K, f"K mismatch: x {tuple(x2.shape)} vs w {tuple(qweight.shape)}"
    if x2.stride(-1) != 1 or (M > 1 and x2.stride(0) % 8 != 0):
        x2 = x2.contiguous()
    qw = qweight if qweight.is_contiguous() else qweight.contiguous()
    sc = scale.contiguous()
    if group_size:
        assert sc.numel() == N * (K // group_size), "per-group scale must be (N, K // group_size)"
    else:
        assert sc.numel() == N, "per-channel scale must have N entries"
    b = None if bias is None else bias.to(x.dtype).contiguous()
    dev = _lib.require_device(x2, qw, sc, b, out)
    if out is None:
        y = torch.empty((M, N), device=dev, dtype=x.dtype)
    else:
        y = out.reshape(M, N)
        assert y.dtype == x.dtype and y.stride(-1) == 1
    if M == 0:
        return y.view(*x.shape[:-1], N)
    lib = _lib.load()
    if twin == "floor":
        if group_size:
            raise RuntimeError("w8a16 floor twin: per-channel scales only")
        with _lib.on_device(dev):
            rc = lib.sd_w8a16_floor(
                x2.data_ptr(), x2.stride(0), qw.data_ptr(), qw.stride(0),
                sc.data_ptr(), _lib.dtype_code(sc.dtype), _ptr(b),
                y.data_ptr(), y.stride(0), M, N, K, _lib.dtype_code(x.dtype),
                _lib.stream_ptr(dev))
        _lib.check(rc)
        return y.view(*x.shape[:-1], N)
    with _lib.on_device(dev):
        # the plan (and so the workspace) depends on the device's compute units
        ws_bytes = lib.sd_w8a16_workspace_size(M, N, K, int(group_size))
        ws = _workspace(ws_bytes, dev)
        rc = lib.sd_w8a16_linear(
            x2.data_ptr(), x2.stride(0), qw.data_ptr(), qw.stride(0),
            sc.data_ptr(), _lib.dtype_code(sc.dtype), int(group_size), _ptr(b),
            y.data_ptr(), y.stride(0), M, N, K, _lib.dtype_code(x.dtype),
            _ptr(ws), ws_bytes, _lib.stream_ptr(dev))
    _lib.check(rc)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], N)



def _many_rows(M: int, N: int, K: int, group_size: int, dev: torch.device) -> bool:
    """Whether the plain linear leaves the 16-row kernels that the fused forms share
    (never up to 16 rows; past them a matter of sizes and compute units)."""
    if M <= 16 or dev.type != "cuda":
        return False
    with _lib.on_device(dev):
        return _lib.load().sd_w8a16_plan(M, N, K, int(group_size)) != 0


def w8a16_silu_linear(gate_up: torch.Tensor, qweight: torch.Tensor, scale: torch.Tensor,
                      bias: torch.Tensor | None = None, group_size: int = 0,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """w8a16_linear(silu_mul(gate_up), ...): the MLP's act_fn and down_proj
    (layers/activation.py:6-11 then the W8A16 linear). gate_up: (..., 2K); the
    activation is SiluAndMul's, bit for bit. One launch while the fused form
    stages its activation rows in LDS (min(M, 16) (2K + 16) <= 33,024 bytes)
    and the plain linear stays on the 16-row kernels it shares (sd_w8a16_plan),
    up to 128 rows (every workgroup repeats the SiLU of its rows: 1024 x 1024 at
    192 rows 17.4 us, 9.3 in two launches); the two separate launches otherwise."""
    assert qweight.dtype == torch.int8 and qweight.dim() == 2
    N, K = qweight.shape
    g2 = gate_up.reshape(-1, gate_up.shape[-1])
    M = g2.shape[0]
    assert g2.shape[1] == 2 * K, f"gate_up {tuple(g2.shape)} needs 2K = {2 * K} columns"
    if g2.stride(-1) != 1 or (M > 1 and g2.stride(0) % 8 != 0) or g2.data_ptr() % 16:
        g2 = g2.contiguous()
    qw = qweight if qweight.is_contiguous() else qweight.contiguous()
    sc = scale.contiguous()
    if group_size:
        assert sc.numel() == N * (K // group_size), "per-group scale must be (N, K // group_size)"
    else:
        assert sc.numel() == N, "per-channel scale must have N entries"
    if min(M, 16) * (2 * K + 16) > 33024 or M > 128 or \
            _many_rows(M, N, K, group_size, g2.device):
        y = w8a16_linear(silu_mul(g2), qw, sc, bias, group_size, out)
        return y.view(*gate_up.shape[:-1], N)
    b = None if bias is None else bias.to(gate_up.dtype).contiguous()
    dev = _lib.require_device(g2, qw, sc, b, out)
    if out is None:
        y = torch.empty((M, N), device=dev, dtype=gate_up.dtype)
    else:
        y = out.reshape(M, N)
        assert y.dtype == gate_up.dtype and y.stride(-1) == 1
    if M == 0:
        return y.view(*gate_up.shape[:-1], N)
    lib = _lib.load()
    with _lib.on_device(dev):
        rc = lib.sd_w8a16_silu_linear(
            g2.data_ptr(), g2.stride(0), qw.data_ptr(), qw.stride(0),
            sc.data_ptr(), _lib.dtype_code(sc.dtype), int(group_size), _ptr(b),
            y.data_ptr(), y.stride(0), M, N, K, _lib.dtype_code(gate_up.dtype),
            _lib.stream_ptr(dev))
    _lib.check(rc)
    return y.view(*gate_up.shape[:-1], N)


# Rows up to which the add + RMSNorm runs inside the projection's launch (the
# fused entry points accept more; past this the two launches measured faster):
# up to 16 rows of at most 1024 columns, where each wave of a workgroup
# normalises up to 4 rows in one round trip, and up to 4 rows of wider ones,
# where the waves take their rows one at a time.
NORM_FUSED_MAX_ROWS = 16
NORM_FUSED_MAX_ROWS_WIDE = 4


def _norm_fused(M: int, K: int) -> bool:
    limit = NORM_FUSED_MAX_ROWS if K <= 1024 else NORM_FUSED_MAX_ROWS_WIDE
    return M <= limit and K % 8 == 0 and K <= 8192


def w8a16_rmsnorm_linear(x: torch.Tensor, norm_weight: torch.Tensor, eps: float,
                         qweight: torch.Tensor, scale: torch.Tensor,
                         bias: torch.Tensor | None = None, group_size: int = 0,
                         residual: torch.Tensor | None = None,
                         residual_out: torch.Tensor | None = None,
                         out: torch.Tensor | None = None) -> torch.Tensor:
    """w8a16_linear(rmsnorm(x, norm_weight, eps, residual)[0], ...): a decoder
    layer's RMSNorm (layers/layernorm.py:16-47) feeding the next projection.
    The normalised rows equal ``rmsnorm``'s bit for bit. With ``residual``,
    ``residual_out`` (sharing no byte with x, residual or the output; None:
    not written)
    receives bf16(x + residual), ``rmsnorm``'s second output. One launch for
    up to 16 rows at K <= 1024 and up to 4 rows above: at one or two rows
    every wave of the row-streaming GEMV forms the norm of its columns; from
    three rows the tiled kernel's workgroups normalise their rows while
    staging them. More rows, or rows that do not fit the staging LDS, take the
    two separate launches (same results)."""
    assert qweight.dtype == torch.int8 and qweight.dim() == 2
    N, K = qweight.shape
    assert x.shape[-1] == K and norm_weight.shape == (K,)
    assert residual_out is None or residual is not None, "residual_out needs a residual"
    x2 = _rows16(x, "x")
    M = x2.shape[0]
    nw = norm_weight.to(x.dtype).contiguous()
    qw = qweight if qweight.is_contiguous() else qweight.contiguous()
    sc = scale.contiguous()
    if group_size:
        assert sc.numel() == N * (K // group_size), "per-group scale must be (N, K // group_size)"
    else:
        assert sc.numel() == N, "per-channel scale must have N entries"
    r2 = ro = None
    if residual is not None:
        assert residual.shape == x.shape and residual.dtype == x.dtype
        r2 = _rows16(residual, "residual")
    if residual_out is not None:
        assert residual_out.shape == x.shape and residual_out.dtype == x.dtype
        ro = residual_out.reshape(M, K)
        assert ro.stride(-1) == 1 and ro.data_ptr() % 16 == 0 and (M <= 1 or ro.stride(0) % 8 == 0)
    b = None if bias is None else bias.to(x.dtype).contiguous()
    dev = _lib.require_device(x2, nw, qw, sc, b, r2, ro, out)
    if out is None:
        y = torch.empty((M, N), device=dev, dtype=x.dtype)
    else:
        y = out.reshape(M, N)
        assert y.dtype == x.dtype and y.stride(-1) == 1
    shape = (*x.shape[:-1], N)
    if M == 0:
        return y.view(shape)
    rc = _lib.SD_ERR_UNSUPPORTED
    if _norm_fused(M, K):
        lib = _lib.load()
        with _lib.on_device(dev):
            rc = lib.sd_w8a16_rmsnorm_linear(
                x2.data_ptr(), x2.stride(0), _ptr(r2), 0 if r2 is None else r2.stride(0),
                _ptr(ro), 0 if ro is None else ro.stride(0), nw.data_ptr(), float(eps),
                qw.data_ptr(), qw.stride(0), sc.data_ptr(), _lib.dtype_code(sc.dtype),
                int(group_size), _ptr(b), y.data_ptr(), y.stride(0), M, N, K,
                _lib.dtype_code(x.dtype), _lib.stream_ptr(dev))
    if rc == _lib.SD_ERR_UNSUPPORTED:
        # more rows, or rows that do not fit the staging LDS: the RMSNorm launch
        # (writing residual_out itself), then the plain linear
        h = torch.empty_like(x2)
        rsum = ro if ro is not None or r2 is None else torch.empty_like(r2)
        lib = _lib.load()
        with _lib.on_device(dev):
            rc = lib.sd_rmsnorm(x2.data_ptr(), x2.stride(0), _ptr(r2),
                                0 if r2 is None else r2.stride(0), nw.data_ptr(), h.data_ptr(),
                                h.stride(0), _ptr(rsum), 0 if rsum is None else rsum.stride(0), M,
                                K, float(eps), _lib.dtype_code(x.dtype), _lib.stream_ptr(dev))
        _lib.check(rc)
        w8a16_linear(h, qw, sc, b, group_size, y)
        return y.view(shape)
    _lib.check(rc)
    return y.view(shape)


def w8a16_gate_up_silu(x: torch.Tensor, qweight: torch.Tensor, scale: torch.Tensor,
                       norm_weight: torch.Tensor | None = None, eps: float = 1e-6,
                       residual: torch.Tensor | None = None,
                       residual_out: torch.Tensor | None = None,
                       bias: torch.Tensor | None = None,
                       out: torch.Tensor | None = None) -> torch.Tensor:
    """silu_mul(w8a16_linear(a, qweight, scale)) of the MLP (models/qwen3.py
    Qwen3MLP.forward: gate_up_proj then act_fn), with a = x, or a =
    rmsnorm(x, norm_weight, eps, residual) when ``norm_weight`` is given
    (``residual_out`` as in ``w8a16_rmsnorm_linear``). qweight (2I, K) =
    [gate; up], per-channel scale (2I,); returns (..., I), bit for bit the
    separate calls. One launch on the row-streaming path (one or two rows,
    weights up to 32 MiB: a wave streams gate row i with up row I + i and
    forms the pair's SiLU once) and on the K-split path of narrow layers (a
    workgroup takes gate tile g and up tile g with the plain projection's K
    split; with the norm, above 16 rows at K <= 1024 or 4 rows above, the
    RMSNorm launch comes first);
    other shapes take the separate launches."""
    assert qweight.dtype == torch.int8 and qweight.dim() == 2
    N, K = qweight.shape
    assert N % 2 == 0 and x.shape[-1] == K
    assert residual_out is None or residual is not None, "residual_out needs a residual"
    assert residual is None or norm_weight is not None, "a residual needs the norm weight"
    x2 = _rows16(x, "x")
    M = x2.shape[0]
    nw = None if norm_weight is None else norm_weight.to(x.dtype).contiguous()
    qw = qweight if qweight.is_contiguous() else qweight.contiguous()
    sc = scale.contiguous()
    assert sc.numel() == N, "per-channel scale must have N entries"
    r2 = ro = None
    if residual is not None:
        assert residual.shape == x.shape and residual.dtype == x.dtype
        r2 = _rows16(residual, "residual")
    if residual_out is not None:
        assert residual_out.shape == x.shape and residual_out.dtype == x.dtype
        ro = residual_out.reshape(M, K)
        assert ro.stride(-1) == 1 and ro.data_ptr() % 16 == 0 and (M <= 1 or ro.stride(0) % 8 == 0)
    b = None if bias is None else bias.to(x.dtype).contiguous()
    dev = _lib.require_device(x2, nw, qw, sc, b, r2, ro, out)
    shape = (*x.shape[:-1], N // 2)
    if out is None:
        y = torch.empty((M, N // 2), device=dev, dtype=x.dtype)
    else:
        y = out.reshape(M, N // 2)
        assert y.dtype == x.dtype and y.stride(-1) == 1
    if M == 0:
        return y.view(shape)
    lib = _lib.load()
    xa, ra, roa, nwa = x2, r2, ro, nw
    if nw is not None and not _norm_fused(M, K) and K % 8 == 0 and K <= 8192:
        # past the rows where the staged norm pays (every workgroup normalises
        # all of them): the RMSNorm launch (writing residual_out itself), then
        # the paired projection on the normalised rows
        xa = torch.empty_like(x2)
        rsum = ro if ro is not None or r2 is None else torch.empty_like(r2)
        with _lib.on_device(dev):
            rc = lib.sd_rmsnorm(x2.data_ptr(), x2.stride(0), _ptr(r2),
                                0 if r2 is None else r2.stride(0), nw.data_ptr(), xa.data_ptr(),
                                xa.stride(0), _ptr(rsum), 0 if rsum is None else rsum.stride(0), M,
                                K, float(eps), _lib.dtype_code(x.dtype), _lib.stream_ptr(dev))
        _lib.check(rc)
        ra = roa = nwa = None
    rc = _lib.SD_ERR_UNSUPPORTED  # past the 16-row kernels: the tiled projection first
    if not _many_rows(M, N, K, 0, dev):
        with _lib.on_device(dev):
            rc = lib.sd_w8a16_gate_up_silu(
                xa.data_ptr(), xa.stride(0), _ptr(ra), 0 if ra is None else ra.stride(0),
                _ptr(roa), 0 if roa is None else roa.stride(0), _ptr(nwa), float(eps),
                qw.data_ptr(), qw.stride(0), sc.data_ptr(), _lib.dtype_code(sc.dtype), _ptr(b),
                y.data_ptr(), y.stride(0), M, N, K, _lib.dtype_code(x.dtype), _lib.stream_ptr(dev))
    if rc == _lib.SD_ERR_UNSUPPORTED and (nwa is None or (K % 8 == 0 and K <= 8192)):
        # neither the row-streaming nor the K-split path (or a faster tiled
        # projection): the projection, then the SiLU launch
        if nwa is None:
            gu = w8a16_linear(xa, qw, sc, b)
        else:
            gu = w8a16_rmsnorm_linear(x2, nw, eps, qw, sc, b, residual=r2, residual_out=ro)
        silu_mul(gu, out=y)
        return y.view(shape)
    _lib.check(rc)
    return y.view(shape)


# ------------------------------------------------------------------- 4-bit KV cache
def int4_kvcache(num_blocks: int, block_size: int, num_kv_heads: int, group_size: int = 64,
                 dtype: torch.dtype = torch.bfloat16,
                 device: torch.device | str = "cuda") -> tuple[torch.Tensor, torch.Tensor]:
    """An empty 4-bit KV cache for heads of 128 dims: (kv_codes (num_blocks, block_size,
    num_kv_heads, 128) uint8, kv_scales (..., 512 // group_size) of ``dtype``, the activations').

    A row of codes is one token's key (64 bytes) and value of one head; a scale and a zero per
    group of 32, 64 or 128 dims: value = zero + scale * code (include/specdec_amd.h has the
    order of the half bytes). The tensors are views of head-major memory (a head's rows of a
    page side by side), which attention reads in the longest runs; any strides with aligned rows
    work. 144 bytes a token and head at group 64, against 512 in 16 bits."""
    assert group_size in (32, 64, 128), f"group_size must be 32, 64 or 128, got {group_size}"
    codes = torch.zeros((num_blocks, num_kv_heads, block_size, 128), dtype=torch.uint8, device=device)
    scales = torch.zeros((num_blocks, num_kv_heads, block_size, 512 // group_size), dtype=dtype,
                         device=device)
    return codes.transpose(1, 2), scales.transpose(1, 2)


# (The checks below are written for their cost: a small call is bound by the host, where a tensor's
# ``reshape`` or ``to`` takes 1 us even if it changes nothing, a launch 4.)
def _cache4(kv_codes: torch.Tensor, kv_scales: torch.Tensor, dtype: torch.dtype) -> tuple:
    """(num_blocks, block_size, num_kv_heads) of a 4-bit cache and the C ABI's arguments of it
    (codes, strides, scales, strides, group size)."""
    assert kv_codes.dim() == 4 and kv_codes.dtype == torch.uint8 and kv_codes.shape[3] == 128, \
        "kv_codes must be (num_blocks, block_size, num_kv_heads, 128) uint8"
    assert kv_scales.dim() == 4 and kv_scales.dtype == dtype, \
        f"kv_scales must be 4-D and {dtype}, as the activations"
    nb, bs, heads, _ = kv_codes.shape
    nb2, bs2, heads2, n = kv_scales.shape
    assert nb == nb2 and bs == bs2 and heads == heads2 and n in (4, 8, 16), \
        "kv_scales must be kv_codes' blocks, 512 / group_size each"
    c0, c1, c2, c3 = kv_codes.stride()
    s0, s1, s2, s3 = kv_scales.stride()
    assert c3 == 1 and s3 == 1
    return nb, bs, heads, (kv_codes.data_ptr(), c0, c1, c2, kv_scales.data_ptr(), s0, s1, s2, 512 // n)


def _flat(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """1-D contiguous ``t`` of ``dtype``."""
    if t.dim() != 1:
        t = t.reshape(-1)
    if t.dtype != dtype:
        t = t.to(dtype)
    return t if t.is_contiguous() else t.contiguous()


def store_kvcache_int4(key: torch.Tensor, value: torch.Tensor, kv_codes: torch.Tensor,
                       kv_scales: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """``store_kvcache`` into a 4-bit cache (``int4_kvcache``): key / value (N, num_kv_heads,
    128) quantized to ``slot_mapping`` (slots of one call differ; -1 skips the row)."""
    dt = key.dtype
    assert key.dim() == 3 and key.shape == value.shape and dt == value.dtype
    N, Hkv, D = key.shape
    nb, bs, heads, cache = _cache4(kv_codes, kv_scales, dt)
    slots = _flat(slot_mapping, torch.int32)
    assert heads == Hkv and slots.numel() == N
    k0, k1, k2 = key.stride()
    v0, v1, v2 = value.stride()
    assert k2 == 1 and v2 == 1
    dev = _lib.require_device(key, value, kv_codes, kv_scales, slots)
    if N == 0:
        return
    with _lib.on_device(dev):
        rc = _lib.load().sd_store_kvcache_int4(
            key.data_ptr(), k0, k1, value.data_ptr(), v0, v1, *cache, slots.data_ptr(), N, Hkv, D,
            bs, nb, _lib.dtype_code(dt), _lib.stream_ptr(dev))
    _lib.check(rc)


def qk_norm_rope_store_int4(q: torch.Tensor, k: torch.Tensor, v: torch.Tensor,
                            positions: torch.Tensor, cos_sin_cache: torch.Tensor,
                            kv_codes: torch.Tensor, kv_scales: torch.Tensor,
                            slot_mapping: torch.Tensor, q_weight: torch.Tensor | None = None,
                            k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                            key_out: bool = True):
    """A step's append to a 4-bit cache in one launch: per-head RMSNorm of q (T, Hq, 128) and
    k (T, Hkv, 128) (skipped without weights), rotate-half RoPE at ``positions`` from
    ``cos_sin_cache`` (max_pos, [1,] 128) fp32 = [cos | sin], then the rotated key and v
    (T, Hkv, 128) quantized to ``slot_mapping``. Strided views of a qkv projection work and are
    left as they are; returns (q, k) as new contiguous tensors (k None with ``key_out=False``,
    for decode, where attention reads the cache). fp32 throughout, each output rounded once
    (``qk_norm_rope`` keeps the module's own roundings); the key is quantized unrounded."""
    dt = q.dtype
    assert q.dim() == 3 and k.dim() == 3 and v.shape == k.shape and dt == k.dtype == v.dtype
    T, Hq, D = q.shape
    T2, Hkv, D2 = k.shape
    assert T == T2 and D == D2
    assert (q_weight is None) == (k_weight is None)
    q0, q1, q2 = q.stride()
    k0, k1, k2 = k.stride()
    v0, v1, v2 = v.stride()
    assert q2 == 1 and k2 == 1 and v2 == 1
    nb, bs, heads, cache = _cache4(kv_codes, kv_scales, dt)
    assert heads == Hkv
    cs = cos_sin_cache if cos_sin_cache.dim() == 2 else \
        cos_sin_cache.reshape(cos_sin_cache.shape[0], -1)
    positions_max, width = cs.shape
    cs0, cs1 = cs.stride()
    assert cs.dtype == torch.float32 and width >= 128 and cs1 == 1
    pos, slots = _flat(positions, torch.int64), _flat(slot_mapping, torch.int32)
    assert pos.numel() == T and slots.numel() == T
    qw = kw = None
    if q_weight is not None:
        qw, kw = _flat(q_weight, dt), _flat(k_weight, dt)
        assert qw.numel() == D and kw.numel() == D
    dev = _lib.require_device(q, k, v, pos, cs, kv_codes, kv_scales, slots, qw, kw)
    q_out = torch.empty((T, Hq, D), dtype=dt, device=dev)
    k_out = torch.empty((T, Hkv, D), dtype=dt, device=dev) if key_out else None
    if T == 0:
        return q_out, k_out
    with _lib.on_device(dev):
        rc = _lib.load().sd_qk_norm_rope_store_int4(
            q.data_ptr(), q0, q1, k.data_ptr(), k0, k1, v.data_ptr(), v0, v1, T, Hq, Hkv, D,
            _ptr(qw), _ptr(kw), eps, pos.data_ptr(), cs.data_ptr(), cs0, positions_max,
            q_out.data_ptr(), _ptr(k_out), *cache, nb, bs, slots.data_ptr(), _lib.dtype_code(dt),
            _lib.stream_ptr(dev))
    _lib.check(rc)
    return q_out, k_out


def load_kvcache_int4(kv_codes: torch.Tensor, kv_scales: torch.Tensor,
                      slot_mapping: torch.Tensor) -> tuple[torch.Tensor, torch.Tensor]:
    """The rows of a 4-bit cache at ``slot_mapping`` (N,) in the activations' type: (key, value),
    each (N, num_kv_heads, 128); rows of slot -1 are zero. Prefill over a cached prefix reads its
    pages this way."""
    dt = kv_scales.dtype
    nb, bs, Hkv, cache = _cache4(kv_codes, kv_scales, dt)
    slots = _flat(slot_mapping, torch.int32)
    dev = _lib.require_device(kv_codes, kv_scales, slots)
    N = slots.numel()
    k = torch.empty((N, Hkv, 128), dtype=dt, device=dev)
    v = torch.empty((N, Hkv, 128), dtype=dt, device=dev)
    if N == 0:
        return k, v
    with _lib.on_device(dev):
        rc = _lib.load().sd_load_kvcache_int4(
            *cache, slots.data_ptr(), N, Hkv, 128, bs, nb, _lib.dtype_code(dt), k.data_ptr(),
            v.data_ptr(), _lib.stream_ptr(dev))
    _lib.check(rc)
    return k, v


def paged_attention_int4(q: torch.Tensor, kv_codes: torch.Tensor, kv_scales: torch.Tensor,
                         block_table: torch.Tensor, scale: float, *,
                         context_lens: torch.Tensor | None = None,
                         cu_seqlens_k: torch.Tensor | None = None,
                         cu_seqlens_q: torch.Tensor | None = None, max_seqlen_q: int = 1,
                         num_splits: int = 0, out: torch.Tensor | None = None) -> torch.Tensor:
    """``paged_attention`` over a 4-bit cache (``int4_kvcache``): decode (one query row per
    sequence) or speculative verify (``cu_seqlens_q``, bottom-right causal), GQA, split over the
    keys; (num_q_heads // num_kv_heads) * max_seqlen_q <= 32. q (total_q, num_q_heads, 128)."""
    if q.dim() != 3:
        raise ValueError(f"q must be (tokens, heads, head_dim), got {tuple(q.shape)}")
    total_q, Hq, D = q.shape
    num_blocks, block_size, Hkv, cache = _cache4(kv_codes, kv_scales, q.dtype)
    assert Hq % Hkv == 0, f"GQA needs num_q_heads divisible by num_kv_heads: {Hq} vs {Hkv}"
    assert block_table.dim() == 2, "block_table must be (num_seqs, max_blocks)"
    if (context_lens is None) == (cu_seqlens_k is None):
        raise ValueError("give exactly one of context_lens / cu_seqlens_k")
    bt, ctx, cuk, cuq = _i32(block_table), _i32(context_lens), _i32(cu_seqlens_k), _i32(cu_seqlens_q)
    num_seqs, max_blocks = bt.shape
    assert ctx is None or ctx.numel() == num_seqs
    assert cuk is None or cuk.numel() == num_seqs + 1
    if cuq is None:
        max_seqlen_q = 1
        if total_q != num_seqs:
            raise ValueError(f"decode expects one query row per sequence: q has {total_q} rows, "
                             f"block_table {num_seqs}")
    else:
        assert cuq.numel() == num_seqs + 1
    dev = _lib.require_device(q, kv_codes, kv_scales, bt, ctx, cuk, cuq, out)
    if out is None:
        out = torch.empty_like(q)
    else:
        assert out.shape == q.shape and out.dtype == q.dtype
    if total_q == 0 or num_seqs == 0:
        return out
    lib = _lib.load()
    qs, os = q.stride(), out.stride()
    assert qs[2] == 1 and os[2] == 1
    max_seqlen_q = int(max_seqlen_q)
    with _lib.on_device(dev):
        # the plan (and so the workspace) depends on the device's compute units
        ws_bytes = lib.sd_paged_attention_int4_workspace_size(
            num_seqs, max_seqlen_q, Hq, Hkv, max_blocks * block_size, int(num_splits))
        # (past the library's limits the size is the largest there is: the call says what is wrong)
        ws = _workspace(ws_bytes, dev) if ws_bytes < 1 << 60 else None
        rc = lib.sd_paged_attention_int4(
            q.data_ptr(), qs[0], qs[1], *cache, num_blocks, block_size, bt.data_ptr(), bt.stride(0),
            max_blocks, _ptr(ctx), _ptr(cuk), _ptr(cuq), max_seqlen_q, total_q, num_seqs, Hq, Hkv,
            D, float(scale), _lib.dtype_code(q.dtype), out.data_ptr(), os[0], os[1], _ptr(ws),
            ws_bytes if ws is not None else 0, int(num_splits), _lib.stream_ptr(dev))
    _lib.check(rc)
    return out


# ---------------------------------------------------------------------------- w4a16
def w4a16_linear(x: torch.Tensor, qweight: torch.Tensor, scale: torch.Tensor,
                 bias: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """y = x @ w^T + bias with 4-bit weights, w[n, k] = (code - 8) * scale[n, k // group].

    x: (..., K) fp16/bf16; qweight: (N, K // 2) uint8, byte j the codes of columns 2j (low half)
    and 2j + 1; scale: (N, K // group) bf16/fp16/fp32, the group a multiple of 32. Returns
    (..., N) in x.dtype; fp32 sums, rounded once (``layers.quant.quantize_weight_int4`` makes
    the weights)."""
    assert qweight.dtype == torch.uint8, f"qweight must be uint8, got {qweight.dtype}"
    assert qweight.dim() == 2 and scale.dim() == 2
    N, K = qweight.shape[0], 2 * qweight.shape[1]
    x2 = x if x.dim() == 2 else x.reshape(-1, x.shape[-1])
    M = x2.shape[0]
    assert x2.shape[1] == K, f"K mismatch: x {tuple(x2.shape)} vs w {tuple(qweight.shape)}"
    groups = scale.shape[1]
    assert scale.shape[0] == N and groups and K % groups == 0, "scale must be (N, K // group)"
    x0, x1 = x2.stride()
    if x1 != 1 or x2.data_ptr() % 16 or (M > 1 and (x0 % 8 or x0 > 1 << 24)):
        # (not contiguous(): a contiguous view may start anywhere, and stays where it is)
        x2, x0 = x2.clone(memory_format=torch.contiguous_format), K
    qw = qweight if qweight.is_contiguous() else qweight.contiguous()
    sc = scale if scale.is_contiguous() else scale.contiguous()
    b = None
    if bias is not None:
        assert bias.shape == (N,), "bias must be (N,)"
        b = _flat(bias, x.dtype)
    dev = _lib.require_device(x2, qw, sc, b, out)
    if out is None:
        y = torch.empty((M, N), device=dev, dtype=x.dtype)
    else:
        assert out.shape == (*x.shape[:-1], N), f"out must be {(*x.shape[:-1], N)}, got {tuple(out.shape)}"
        y = out.view(M, N)
        assert y.dtype == x.dtype and (N == 1 or y.stride(1) == 1)
    if M:
        lib = _lib.load()
        with _lib.on_device(dev):
            # the plan (and so the workspace) depends on the device's compute units; up to 8 rows there is
            # none unless a row's scales leave LDS no room, which 512 of them never do (the question takes 1 us)
            ws_bytes = lib.sd_w4a16_workspace_size(M, N, K, K // groups) if M > 8 or groups > 512 else 0
            ws = _workspace(ws_bytes, dev)
            rc = lib.sd_w4a16_linear(
                x2.data_ptr(), x0, qw.data_ptr(), K // 2, sc.data_ptr(), _lib.dtype_code(sc.dtype),
                K // groups, _ptr(b), y.data_ptr(), y.stride(0), M, N, K, _lib.dtype_code(x.dtype),
                _ptr(ws), ws_bytes, _lib.stream_ptr(dev))
        _lib.check(rc)
    return y if x.dim() == 2 else y.view(*x.shape[:-1], N)


# ------------------------------------------------------------------- 8-bit activations
def _rows8(t: torch.Tensor) -> tuple[torch.Tensor, int, int]:
    """2-D (rows, width) view with a unit last stride and rows at 16-byte addresses, a copy where they are not;
    with its row stride and address."""
    if t.dim() != 2:
        t = t.reshape(-1, t.shape[-1])
    s0, s1 = t.stride()
    p = t.data_ptr()
    if s1 != 1 or p % 16 or (s0 < 0 or s0 * t.itemsize % 16) and t.shape[0] > 1:
        # (not contiguous(): a contiguous view may start anywhere, and stays where it is)
        t = t.clone(memory_format=torch.contiguous_format)
        s0, p = t.shape[1], t.data_ptr()
    return t, s0, p


def _like(t: torch.Tensor, dtype: torch.dtype) -> torch.Tensor:
    """An empty row-major tensor of ``t``'s shape (``empty_like`` takes 1 us less than ``empty``)."""
    return torch.empty_like(t, dtype=dtype) if t.is_contiguous() else torch.empty(t.shape, dtype=dtype, device=t.device)


_BF16 = torch.bfloat16


class Int8Rows(tuple):
    """(codes, scale) of rows in 8 bits that know the type they came from, ``dtype``, which a layer's
    linear gives its outputs."""
    dtype = _BF16


def int8_rows(codes: torch.Tensor, scale: torch.Tensor, dtype: torch.dtype) -> Int8Rows:
    rows = Int8Rows((codes, scale))
    if dtype is not _BF16:  # (an attribute of its own takes 0.1 us)
        rows.dtype = dtype
    return rows


def quantize_rows_int8(x: torch.Tensor) -> Int8Rows:
    """Rows of activations in 8 bits: x (..., K) bf16/fp16 -> (codes int8 (..., K), scale fp32
    (...,)), value = code * scale, scale = max|x| / 127 and code = round_half_even(127 x / max|x|).
    A row with a NaN or an infinity has scale NaN, a row of zeros scale 0. K a multiple of 16 up
    to 32768. (``quantize_int8`` makes weights: a bf16 scale, rounded after the codes.)"""
    x2, x0, xp = _rows8(x)
    rows, K = x2.shape
    dt = x2.dtype
    dev = _lib.require_device(x2)
    codes = _like(x2, torch.int8)
    scale = torch.empty(rows, dtype=torch.float32, device=dev)
    with _lib.on_device(dev):
        rc = _lib.load().sd_quantize_rows_int8(
            xp, x0, codes.data_ptr(), K, scale.data_ptr(), rows, K, _lib.dtype_code(dt),
            _lib.stream_ptr(dev))
    if rc:
        _lib.check(rc)
    if x2 is not x and x.dim() != 2:
        codes, scale = codes.view(x.shape), scale.view(x.shape[:-1])
    return Int8Rows((codes, scale)) if dt is _BF16 else int8_rows(codes, scale, dt)


def rmsnorm_int8(x: torch.Tensor, weight: torch.Tensor, eps: float,
                 residual: torch.Tensor | None = None):
    """``rmsnorm`` whose result goes to 8 bits as ``quantize_rows_int8``'s, without a rounding to 16
    bits on the way: returns (codes, scale), with ``residual`` (codes, scale, residual_out), where s =
    x + residual in fp32, residual_out = s rounded to the dtype and the codes are of the norm of s."""
    x2, x0, xp = _rows8(x)
    rows, H = x2.shape
    dt = x2.dtype
    assert weight.shape == (H,), "weight must be (hidden,)"
    w = weight if weight.dtype == dt else weight.to(dt)
    wp = w.data_ptr()
    if wp % 16 or not w.is_contiguous():
        w = w.clone(memory_format=torch.contiguous_format)
        wp = w.data_ptr()
    r2 = ro = rp = rop = None
    r0 = 0
    if residual is not None:
        assert residual.shape == x.shape and residual.dtype == dt
        r2, r0, rp = _rows8(residual)
    dev = _lib.require_device(x2, w, r2)
    codes = _like(x2, torch.int8)
    scale = torch.empty(rows, dtype=torch.float32, device=dev)
    if r2 is not None:
        ro = _like(x2, dt)
        rop = ro.data_ptr()
    with _lib.on_device(dev):
        rc = _lib.load().sd_rmsnorm_int8(
            xp, x0, rp, r0, wp, codes.data_ptr(), H, scale.data_ptr(), rop, H, rows, H, eps,
            _lib.dtype_code(dt), _lib.stream_ptr(dev))
    if rc:
        _lib.check(rc)
    if x2 is not x and x.dim() != 2:
        codes, scale = codes.view(x.shape), scale.view(x.shape[:-1])
        ro = None if ro is None else ro.view(x.shape)
    if ro is not None:
        return codes, scale, ro
    return Int8Rows((codes, scale)) if dt is _BF16 else int8_rows(codes, scale, dt)


def dequantize_rows_int8(codes: torch.Tensor, scale: torch.Tensor,
                         dtype: torch.dtype = torch.bfloat16) -> torch.Tensor:
    """The values of 8-bit rows: codes (..., K) int8 times scale (...,) fp32, rounded to ``dtype``
    (bf16, fp16 or fp32). Per-channel int8 weights with their scale in fp32 too."""
    assert codes.dtype == torch.int8 and scale.dtype == torch.float32
    shape = codes.shape
    assert scale.shape == shape[:-1], f"one scale a row: {tuple(scale.shape)} for {tuple(shape)}"
    c2, c0, cp = _rows8(codes)
    s = scale if scale.is_contiguous() else scale.contiguous()
    rows, K = c2.shape
    dev = _lib.require_device(c2, s)
    out = _like(c2, dtype)
    with _lib.on_device(dev):
        rc = _lib.load().sd_dequantize_rows_int8(
            cp, c0, s.data_ptr(), out.data_ptr(), K, rows, K, _lib.dtype_code(dtype),
            _lib.stream_ptr(dev))
    if rc:
        _lib.check(rc)
    return out if len(shape) == 2 else out.view(shape)


# ----------------------------------------------------------------------------- w8a8
def _w8a8(gated: bool, x, x_scale, qweight, scale, bias, dtype, out):
    assert x.dtype == qweight.dtype == torch.int8, f"x and qweight must be int8, got {x.dtype} and {qweight.dtype}"
    assert qweight.dim() == 2 and x_scale.dtype == torch.float32
    wrows, K = qweight.shape
    N = wrows
    if gated:
        assert wrows % 2 == 0, "qweight must be [gate; up]"
        N = wrows // 2
    xshape = x.shape
    assert xshape[-1] == K, f"K mismatch: x {tuple(xshape)} vs w {tuple(qweight.shape)}"
    assert x_scale.shape == xshape[:-1], f"one scale a row: {tuple(x_scale.shape)} for {tuple(xshape)}"
    assert scale.numel() == wrows, "scale must have one entry per weight row"
    x2, x0, xp = _rows8(x)
    qw, w0, wp = _rows8(qweight)
    M = x2.shape[0]
    if M > 1 and x0 > 1 << 23:
        x2, x0 = x2.clone(memory_format=torch.contiguous_format), K
        xp = x2.data_ptr()
    xs = x_scale if x_scale.is_contiguous() else x_scale.contiguous()
    sc = scale if scale.is_contiguous() else scale.contiguous()
    b = None
    if bias is not None:
        assert bias.shape == (wrows,), "bias must have one entry per weight row"
        b = _flat(bias, dtype)
    dev = _lib.require_device(x2, xs, qw, sc, b, out)
    if out is None:
        y = torch.empty((M, N), device=dev, dtype=dtype)
        y0 = N
    else:
        shape = (*xshape[:-1], N)
        assert out.shape == shape, f"out must be {shape}, got {tuple(out.shape)}"
        y = out.view(M, N)
        y0, y1 = y.stride()
        assert y.dtype == dtype and (N == 1 or y1 == 1)
    if M:
        lib = _lib.load()
        with _lib.on_device(dev):
            # the plan (and so the workspace) depends on the device's compute units; up to 4 rows of up to 16384
            # columns there is none (the question takes 1 us, 2 to 3 where tiles are compared)
            ws_bytes = lib.sd_w8a8_workspace_size(M, N, K, gated) if M > 4 or K > 16384 else 0
            ws = torch.empty(ws_bytes, dtype=torch.uint8, device=dev) if ws_bytes else None
            rc = (lib.sd_w8a8_gate_up_silu if gated else lib.sd_w8a8_linear)(
                xp, x0, xs.data_ptr(), wp, w0, sc.data_ptr(), _lib.dtype_code(sc.dtype), _ptr(b), y.data_ptr(),
                y0, M, N, K, _lib.dtype_code(dtype), _ptr(ws), ws_bytes, _lib.stream_ptr(dev))
        if rc:
            _lib.check(rc)
    return y if len(xshape) == 2 else y.view(*xshape[:-1], N)


def w8a8_linear(x: torch.Tensor, x_scale: torch.Tensor, qweight: torch.Tensor, scale: torch.Tensor,
                bias: torch.Tensor | None = None, dtype: torch.dtype = torch.bfloat16,
                out: torch.Tensor | None = None) -> torch.Tensor:
    """y = (x @ qweight^T) * scale * x_scale + bias in 8-bit integers.

    x (..., K) int8 and x_scale (...,) fp32: activations of ``quantize_rows_int8`` or
    ``rmsnorm_int8``; qweight (N, K) int8 and scale (N,): the weights of ``w8a16_linear``, per
    channel. K a multiple of 16 below 2^17. Exact integer sums, fp32 scales, one rounding to
    ``dtype`` (bf16 or fp16); returns (..., N). Rows that do not start at 16-byte addresses are
    copied first, in every call, weights too: keep those aligned."""
    return _w8a8(False, x, x_scale, qweight, scale, bias, dtype, out)


def w8a8_gate_up_silu(x: torch.Tensor, x_scale: torch.Tensor, qweight: torch.Tensor,
                      scale: torch.Tensor, bias: torch.Tensor | None = None,
                      dtype: torch.dtype = torch.bfloat16,
                      out: torch.Tensor | None = None) -> torch.Tensor:
    """silu(gate) * up of the MLP's gate_up projection as ``w8a8_linear``: qweight (2I, K) =
    [gate; up], scale (2I,); returns (..., I). gate and up are not rounded on the way
    (``w8a16_gate_up_silu`` keeps the module's own roundings)."""
    return _w8a8(True, x, x_scale, qweight, scale, bias, dtype, out)


def quantize_int8(w: torch.Tensor, group_size: int = 0):
    """Symmetric int8 quantization of a 2-D weight on the GPU (the W8A16
    format's producer, nanovllm/layers/quant.py:123-148): per row (group_size
    0) or per group of columns, scale = max(max|w| / 127, 1e-8) in fp32,
    q = clamp(round_half_even(w / scale), -127, 127). Returns (q int8 (N, K),
    scale bf16 (N, K // group) — the fp32 scale rounded after q)."""
    assert w.dim() == 2, f"expects a 2-D weight, got {tuple(w.shape)}"
    N, K = w.shape
    G = group_size if group_size > 0 else K
    assert K % G == 0, "group_size must divide K"
    if w.stride(-1) != 1 or w.data_ptr() % 16 or (N > 1 and w.stride(0) % 8):
        w = w.contiguous()
    dev = _lib.require_device(w)
    q = torch.empty((N, K), dtype=torch.int8, device=dev)
    scale = torch.empty((N, K // G), dtype=torch.bfloat16, device=dev)
    if N:
        lib = _lib.load()
        with _lib.on_device(dev):
            rc = lib.sd_quantize_int8(w.data_ptr(), w.stride(0), _lib.dtype_code(w.dtype),
                                      q.data_ptr(), q.stride(0), scale.data_ptr(), N, K,
                                      int(group_size), _lib.stream_ptr(dev))
        _lib.check(rc)
    return q, scale


# --------------------------------------------------------------- draft-step neighbours
def _rows16(t: torch.Tensor, what: str) -> torch.Tensor:
    """2-D (rows, width) view with a unit last stride and 16-byte aligned rows."""
    t2 = t if t.dim() == 2 else t.reshape(-1, t.shape[-1])
    if t2.stride(-1) != 1 or t2.data_ptr() % 16 or (t2.shape[0] > 1 and t2.stride(0) % 8):
        t2 = t2.contiguous()
    return t2


def rmsnorm(x: torch.Tensor, weight: torch.Tensor, eps: float,
            residual: torch.Tensor | None = None, out: torch.Tensor | None = None):
    """RMSNorm.forward (nanovllm/layers/layernorm.py:16-47) over the last dim.

    ``residual is None``: returns ``bf16(bf16(x * rsqrt(mean(x^2) + eps)) * weight)``.
    Otherwise returns ``(out, residual_out)`` with ``s = x + residual`` in fp32,
    ``residual_out = s`` rounded to the dtype and ``out`` the norm of ``s``.
    """
    H = x.shape[-1]
    x2 = _rows16(x, "x")
    assert weight.shape == (H,), "weight must be (hidden,)"
    w = weight.to(x.dtype).contiguous()
    r2 = None if residual is None else _rows16(residual, "residual")
    if r2 is not None:
        assert residual.shape == x.shape and residual.dtype == x.dtype
    dev = _lib.require_device(x2, w, r2, out)
    o = torch.empty_like(x2) if out is None else out.reshape(-1, H)
    ro = None if r2 is None else torch.empty_like(r2)
    rows = x2.shape[0]
    if rows:
        lib = _lib.load()
        with _lib.on_device(dev):
            rc = lib.sd_rmsnorm(x2.data_ptr(), x2.stride(0), _ptr(r2), 0 if r2 is None else r2.stride(0),
                                w.data_ptr(), o.data_ptr(), o.stride(0), _ptr(ro),
                                0 if ro is None else ro.stride(0), rows, H, float(eps),
                                _lib.dtype_code(x.dtype), _lib.stream_ptr(dev))
        _lib.check(rc)
    if x.dim() != 2 or out is not None:
        o = o.view(x.shape)
    if residual is None:
        return o
    return o, ro if x.dim() == 2 else ro.view(x.shape)


def qk_norm_rope(q: torch.Tensor, k: torch.Tensor, positions: torch.Tensor,
                 cos_sin_cache: torch.Tensor, q_weight: torch.Tensor | None = None,
                 k_weight: torch.Tensor | None = None, eps: float = 1e-6,
                 v: torch.Tensor | None = None, k_cache: torch.Tensor | None = None,
                 v_cache: torch.Tensor | None = None,
                 slot_mapping: torch.Tensor | None = None) -> None:
    """In place on q (T, Hq, 128) and k (T, Hkv, 128) (strided views allowed):
    per-head RMSNorm with q_weight / k_weight (skipped when None), then
    rotate-half RoPE at ``positions`` from ``cos_sin_cache`` (max_pos, [1,] 128)
    fp32 = [cos | sin] (nanovllm/models/qwen3.py:80-88,
    layers/rotary_embedding.py:6-48).

    With ``v``, ``k_cache``, ``v_cache`` and ``slot_mapping``: also
    store_kvcache of the finished k rows and of v (layers/attention.py:33-40)
    in the same launch; caches (num_blocks, block_size, Hkv, 128)."""
    assert q.dim() == 3 and k.dim() == 3 and q.shape[0] == k.shape[0]
    assert q.shape[-1] == 128 and k.shape[-1] == 128 and q.stride(-1) == 1 and k.stride(-1) == 1
    assert q.dtype == k.dtype
    assert (q_weight is None) == (k_weight is None)
    T = q.shape[0]
    cs = cos_sin_cache.reshape(cos_sin_cache.shape[0], -1)
    assert cs.dtype == torch.float32 and cs.shape[1] >= 128 and cs.stride(-1) == 1
    pos = positions.reshape(-1)
    if pos.dtype != torch.int64:
        pos = pos.to(torch.int64)
    pos = pos.contiguous()
    assert pos.numel() == T
    qw = None if q_weight is None else q_weight.to(q.dtype).contiguous()
    kw = None if k_weight is None else k_weight.to(q.dtype).contiguous()
    dev = _lib.require_device(q, k, pos, cs, qw, kw)
    if T == 0:
        return
    lib = _lib.load()
    if k_cache is not None:
        assert v is not None and v_cache is not None and slot_mapping is not None
        assert v.shape == k.shape and v.stride(-1) == 1 and v.dtype == k.dtype
        assert k_cache.shape == v_cache.shape and k_cache.stride() == v_cache.stride()
        assert k_cache.dtype == k.dtype and k_cache.shape[2:] == k.shape[1:]
        slots = _i32(slot_mapping.reshape(-1)).contiguous()
        assert slots.numel() == T
        _lib.require_device(v, k_cache, v_cache, slots)
        with _lib.on_device(dev):
            rc = lib.sd_qk_norm_rope_store(
                q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0), k.stride(1),
                v.data_ptr(), v.stride(0), v.stride(1), T, q.shape[1], k.shape[1], 128,
                _ptr(qw), _ptr(kw), float(eps), pos.data_ptr(), cs.data_ptr(), cs.stride(0),
                cs.shape[0], k_cache.data_ptr(), v_cache.data_ptr(), k_cache.stride(0),
                k_cache.stride(1), k_cache.stride(2), k_cache.shape[0], k_cache.shape[1],
                slots.data_ptr(), _lib.dtype_code(q.dtype), _lib.stream_ptr(dev))
        _lib.check(rc)
        return
    with _lib.on_device(dev):
        rc = lib.sd_qk_norm_rope(q.data_ptr(), q.stride(0), q.stride(1), k.data_ptr(), k.stride(0),
                                 k.stride(1), T, q.shape[1], k.shape[1], 128, _ptr(qw), _ptr(kw),
                                 float(eps), pos.data_ptr(), cs.data_ptr(), cs.stride(0),
                                 cs.shape[0], _lib.dtype_code(q.dtype), _lib.stream_ptr(dev))
    _lib.check(rc)


def silu_mul(x: torch.Tensor, out: torch.Tensor | None = None) -> torch.Tensor:
    """SiluAndMul (nanovllm/layers/activation.py:6-11): x (..., 2I) -> (..., I)."""
    W = x.shape[-1]
    assert W % 2 == 0
    x2 = _rows16(x, "x")
    dev = _lib.require_device(x2, out)
    o = torch.empty((x2.shape[0], W // 2), dtype=x.dtype, device=dev) if out is None \
        else out.reshape(-1, W // 2)
    if x2.shape[0]:
        lib = _lib.load()
        with _lib.on_device(dev):
            rc = lib.sd_silu_mul(x2.data_ptr(), x2.stride(0), o.data_ptr(), o.stride(0),
                                 x2.shape[0], W // 2, _lib.dtype_code(x.dtype),
                                 _lib.stream_ptr(dev))
        _lib.check(rc)
    return o if x.dim() == 2 and out is None else o.view(*x.shape[:-1], W // 2)


# Philox (seed, offset) per device for calls that bring no rng_state: seeded
# from torch's initial seed, its offset advanced on the stream after each draw
# (so graph replays draw fresh noise too).
_RNG_STATES: dict = {}


def default_rng_state(dev: torch.device) -> torch.Tensor:
    st = _RNG_STATES.get(dev.index)
    if st is None:
        st = torch.tensor([torch.initial_seed() & 0x7FFFFFFFFFFFFFFF, 0], dtype=torch.int64,
                          device=dev)
        _RNG_STATES[dev.index] = st
    return st


def sample(logits: torch.Tensor, temperatures: torch.Tensor | None = None,
           rng_state: torch.Tensor | None = None, out: torch.Tensor | None = None) -> torch.Tensor:
    """One token per row of logits (rows, vocab): greedy argmax when
    ``temperatures`` is None (or a row's temperature is <= 0), otherwise the
    exponential-race draw of ``Sampler.forward`` (nanovllm/layers/sampler.py:6-12)
    with Philox noise keyed by ``rng_state`` = (seed, offset) int64 on the device.
    A given ``rng_state`` is the caller's to advance; without one the device's
    default state is used and advanced."""
    assert logits.dim() == 2 and logits.stride(-1) == 1
    rows, V = logits.shape
    t = None
    advance = False
    if temperatures is not None:
        t = temperatures.reshape(-1).to(torch.float32).contiguous()
        assert t.numel() == rows
        if rng_state is None:
            rng_state, advance = default_rng_state(logits.device), True
        assert rng_state.numel() == 2 and rng_state.dtype == torch.int64
    dev = _lib.require_device(logits, t, rng_state, out)
    o = torch.empty(rows, dtype=torch.int64, device=dev) if out is None else out
    assert o.dtype == torch.int64 and o.numel() == rows and o.is_contiguous()
    if rows:
        lib = _lib.load()
        with _lib.on_device(dev):
            ws_bytes = lib.sd_sample_workspace_size(rows, V)
            ws = _workspace(ws_bytes, dev)
            rc = lib.sd_sample(logits.data_ptr(), logits.stride(0), _lib.dtype_code(logits.dtype),
                               rows, V, _ptr(t), _ptr(rng_state), o.data_ptr(), _ptr(ws),
                               ws_bytes, _lib.stream_ptr(dev))
        _lib.check(rc)
        if advance:
            rng_state[1:].add_(1)
    return o


def verify_batch(draft: torch.Tensor, target_logits: torch.Tensor, draft_tokens: torch.Tensor,
                 temperatures: torch.Tensor | None = None, draft_is_point_mass: bool = False,
                 rng_state: torch.Tensor | None = None):
    """Rejection-sampling verification (nanovllm/spec_decode/verify.py:39-183):
    returns (accepted (B,) int64, bonus (B,) int64, accept_mask (B, k) bool).

    ``draft`` (B, k, V): the draft's raw logits, or its probabilities with
    ``draft_is_point_mass``; ``target_logits`` (B, k + 1, V); the row dims may
    be strided, the vocabulary contiguous. Noise is Philox keyed by
    ``rng_state`` (seed, offset) on the device; without one the device's
    default state is used and advanced."""
    assert draft.dim() == 3 and target_logits.dim() == 3 and draft_tokens.dim() == 2
    B, k, V = draft.shape
    assert target_logits.shape[0] == B and target_logits.shape[2] == V
    assert target_logits.shape[1] == k + 1, "target_logits must hold k + 1 rows"
    assert draft_tokens.shape == (B, k)
    assert draft.stride(-1) == 1 and target_logits.stride(-1) == 1
    tok = draft_tokens if draft_tokens.dtype == torch.int64 else draft_tokens.to(torch.int64)
    if tok.stride(-1) != 1:
        tok = tok.contiguous()
    t = None if temperatures is None else temperatures.reshape(-1).to(torch.float32).contiguous()
    if t is not None and t.numel() == 1 and B > 1:
        t = t.expand(B).contiguous()
    advance = rng_state is None
    if advance:
        rng_state = default_rng_state(draft.device)
    dev = _lib.require_device(draft, target_logits, tok, t, rng_state)
    accepted = torch.empty(B, dtype=torch.int64, device=dev)
    bonus = torch.empty(B, dtype=torch.int64, device=dev)
    mask = torch.empty((B, k), dtype=torch.bool, device=dev)
    if B:
        lib = _lib.load()
        with _lib.on_device(dev):
            ws_bytes = lib.sd_verify_batch_workspace_size(B, k, V)
            ws = _workspace(ws_bytes, dev)
            rc = lib.sd_verify_batch(draft.data_ptr(), draft.stride(0), draft.stride(1),
                                     _lib.dtype_code(draft.dtype), target_logits.data_ptr(),
                                     target_logits.stride(0), target_logits.stride(1),
                                     _lib.dtype_code(target_logits.dtype), tok.data_ptr(),
                                     tok.stride(0), _ptr(t), int(bool(draft_is_point_mass)),
                                     rng_state.data_ptr(), B, k, V, accepted.data_ptr(),
                                     bonus.data_ptr(), mask.data_ptr(), _ptr(ws), ws_bytes,
                                     _lib.stream_ptr(dev))
        _lib.check(rc)
        if advance:
            rng_state[1:].add_(1)
    return accepted, bonus, mask


# ---------------------------------------------------------------------- measurement
def stream_read(buf: torch.Tensor, sink: torch.Tensor, workgroups: int = 0) -> None:
    """One streaming read of ``buf`` (sd_stream_read): the box's read ceiling,
    the bench's second denominator beside the 8 TB/s data-sheet peak.
    ``sink``: at least one int32 of device memory, practically never written.
    ``workgroups`` <= 0 takes the library's default (six per CU)."""
    assert buf.is_contiguous() and sink.dtype == torch.int32 and sink.numel() >= 1
    dev = _lib.require_device(buf, sink)
    nbytes = buf.numel() * buf.element_size() // 16 * 16
    with _lib.on_device(dev):
        rc = _lib.load().sd_stream_read(buf.data_ptr(), nbytes, sink.data_ptr(),
                                         int(workgroups), _lib.stream_ptr(dev))
    _lib.check(rc)
