"""``RMSNorm`` with the reference's interface (nanovllm/layers/layernorm.py:6-47)
on the HIP kernel ``sd_rmsnorm``: ``forward(x)`` is the plain norm,
``forward(x, residual)`` the fused residual add + norm returning
``(normed, new_residual)``; fp32 arithmetic with the module's bf16 roundings.
``forward_int8`` gives the norm in 8 bits for a linear with ``quant_act_bits = 8``."""
from __future__ import annotations

import torch
from torch import nn

from .. import ops


class RMSNorm(nn.Module):

    def __init__(self, hidden_size: int, eps: float = 1e-6) -> None:
        super().__init__()
        self.eps = eps
        self.weight = nn.Parameter(torch.ones(hidden_size))

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None):
        if residual is None:
            return ops.rmsnorm(x, self.weight, self.eps)
        return ops.rmsnorm(x, self.weight, self.eps, residual=residual)

    def forward_int8(self, x: torch.Tensor, residual: torch.Tensor | None = None):
        """(codes, scale) of the unrounded norm, with ``residual`` ((codes, scale), new_residual)."""
        if residual is None:
            return ops.rmsnorm_int8(x, self.weight, self.eps)
        codes, scale, new = ops.rmsnorm_int8(x, self.weight, self.eps, residual)
        return ops.int8_rows(codes, scale, x.dtype), new
