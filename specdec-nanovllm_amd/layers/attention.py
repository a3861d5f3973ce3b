"""Attention call site — drop-in for ``nanovllm/layers/attention.py``.

``store_kvcache`` keeps the reference signature and asserts
(attention.py:33-40) and runs the gfx950 slot-write kernel. ``Attention`` keeps
the constructor and ``forward(q, k, v)`` contract (attention.py:43-82): write
the new K/V rows through the slot mapping, then (both in one fused launch)

* decode (``not context.is_prefill``): paged attention of one query row per
  sequence over ``context_lens`` keys; the output has flash-attn's
  (B, 1, Hq, D) shape, as at attention.py:77-81;
* verify / prefix-cache prefill (``block_tables`` set): paged varlen attention
  with bottom-right causal masking, (total_q, Hq, D);
* plain prefill (contiguous k / v, no block table): the store, then the
  varlen causal prefill kernel over the contiguous rows.

A 4-bit cache (``k_cache, v_cache = ops.int4_kvcache(...)``: the codes of both and
their scales) takes the same calls: the store quantizes, decode and verify attend
over the codes, and a prefix-cached prefill reads the table's pages back in 16 bits.
"""
from __future__ import annotations

import torch
from torch import nn

from .. import ops
from ..utils.context import get_context


def store_kvcache(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor,
                  v_cache: torch.Tensor, slot_mapping: torch.Tensor):
    ops.store_kvcache(key, value, k_cache, v_cache, slot_mapping)


def _aligned(t: torch.Tensor) -> torch.Tensor:
    """``t`` with 16-byte aligned rows (views of a projection's output are)."""
    s = t.stride()
    if s[2] == 1 and not (s[0] % 8 or s[1] % 8 or t.data_ptr() % 16):
        return t
    return t.clone(memory_format=torch.contiguous_format)  # a contiguous tensor may start anywhere


def _pages_in_16_bits(kv_codes: torch.Tensor, kv_scales: torch.Tensor, block_tables: torch.Tensor,
                      max_keys: int = 0):
    """The pages of a block table read back from a 4-bit cache: paged K and V of their own, and
    the table over them (entry (b, i) is page b * width + i; unused entries are zero pages).
    max_keys: the longest sequence's keys, past which a table (as wide as the longest sequence
    there may be, say) is not read; 0: all of it."""
    page, heads = kv_codes.shape[1], kv_codes.shape[2]
    if max_keys > 0:
        block_tables = block_tables[:, :-(-max_keys // page)]
    B, width = block_tables.shape
    rows = torch.arange(page, dtype=torch.int32, device=block_tables.device)
    slots = torch.where(block_tables[..., None] >= 0, block_tables[..., None] * page + rows, -1)
    k, v = ops.load_kvcache_int4(kv_codes, kv_scales, slots)
    table = torch.arange(B * width, dtype=torch.int32, device=block_tables.device).view(B, width)
    return k.view(-1, page, heads, 128), v.view(-1, page, heads, 128), table


class Attention(nn.Module):

    def __init__(self, num_heads, head_dim, scale, num_kv_heads):
        super().__init__()
        self.num_heads = num_heads
        self.head_dim = head_dim
        self.scale = scale
        self.num_kv_heads = num_kv_heads
        self.k_cache = self.v_cache = torch.tensor([])

    def forward(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor):
        context = get_context()
        k_cache, v_cache = self.k_cache, self.v_cache
        has_cache = bool(k_cache.numel() and v_cache.numel())
        if k_cache.dtype == torch.uint8 and has_cache:
            return self._forward_int4(q, k, v, context)
        if context.is_prefill:  # attention.py:62-70
            G = self.num_heads // self.num_kv_heads
            if (has_cache and context.block_tables is not None
                    and G * int(context.max_seqlen_q) <= 32):
                # speculative verify / short prefix-cache rows: store_kvcache of k / v
                # and the paged attention in one call
                return ops.paged_attention(q, k_cache, v_cache, context.block_tables,
                                           self.scale, cu_seqlens_k=context.cu_seqlens_k,
                                           cu_seqlens_q=context.cu_seqlens_q,
                                           max_seqlen_q=int(context.max_seqlen_q),
                                           key=k, value=v, slot_mapping=context.slot_mapping)
            if has_cache:
                store_kvcache(k, v, k_cache, v_cache, context.slot_mapping)
            if context.block_tables is not None:  # prefix cache: keys come from the pages
                if not has_cache:
                    raise RuntimeError("prefix-cached prefill needs the paged k_cache / v_cache")
                k, v = k_cache, v_cache
            return ops.prefill_attention(q, k, v, context.cu_seqlens_q, context.cu_seqlens_k,
                                         int(context.max_seqlen_q), self.scale,
                                         block_table=context.block_tables)
        if not has_cache:
            raise RuntimeError("Attention needs its paged k_cache / v_cache")
        # decode (attention.py:71-81): q is (B, Hq, D), or (Hq, D) for one sequence;
        # the result has flash_attn_with_kvcache's (B, 1, Hq, D) shape
        if q.dim() == 2:
            q, k, v = q.unsqueeze(0), k.reshape(1, *k.shape[-2:]), v.reshape(1, *v.shape[-2:])
        if not (q.stride(-1) == 1 and q.stride(0) % 8 == 0 and q.stride(1) % 8 == 0):
            q = q.contiguous()
        o = ops.paged_attention(q, k_cache, v_cache, context.block_tables, self.scale,
                                context_lens=context.context_lens,
                                key=k, value=v, slot_mapping=context.slot_mapping)
        return o.unsqueeze(1)

    def _forward_int4(self, q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, context):
        """``forward`` over a 4-bit cache (k_cache: codes, v_cache: scales)."""
        codes, scales = self.k_cache, self.v_cache
        if not context.is_prefill and q.dim() == 2:
            q, k, v = q.unsqueeze(0), k.reshape(1, *k.shape[-2:]), v.reshape(1, *v.shape[-2:])
        q, k, v = _aligned(q), _aligned(k), _aligned(v)
        ops.store_kvcache_int4(k, v, codes, scales, context.slot_mapping)
        tables = context.block_tables
        if not context.is_prefill:
            o = ops.paged_attention_int4(q, codes, scales, tables, self.scale,
                                         context_lens=context.context_lens)
            return o.unsqueeze(1)
        n = int(context.max_seqlen_q)
        if tables is not None:
            if self.num_heads // self.num_kv_heads * n <= 32:
                return ops.paged_attention_int4(q, codes, scales, tables, self.scale,
                                                cu_seqlens_k=context.cu_seqlens_k,
                                                cu_seqlens_q=context.cu_seqlens_q, max_seqlen_q=n)
            k, v, tables = _pages_in_16_bits(codes, scales, tables, int(context.max_seqlen_k))
        return ops.prefill_attention(q, k, v, context.cu_seqlens_q, context.cu_seqlens_k, n,
                                     self.scale, block_table=tables)
