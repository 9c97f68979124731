"""Serving counterpart of :class:`LoRAOptimizedLinear`: one shared weight, and low-rank adapters of which every row of a batch takes its own
(or none). The reference has the training side only (``deepspeed/linear/optimized_linear.py:76-220``: one adapter for all rows)."""
from __future__ import annotations

from typing import Optional

import torch
import torch.nn as nn

from ..ops.backend import get_ops
from ..ops.plans import AdapterPlan
from .optimized_linear import LoRAOptimizedLinear


class AdapterBank(nn.Module):
    """``n`` adapters of a projection ``input_dim -> output_dim``, of up to ``rank`` each (rounded up to a multiple of 8; smaller ones are padded
    with zeros). An adapter that was never loaded adds nothing. Scales stay fp32 when the bank, or a module that has it, is converted."""

    def __init__(self, n: int, rank: int, input_dim: int, output_dim: int, device=None, dtype=torch.bfloat16):
        super().__init__()
        if n < 1 or rank < 1 or rank > 256 or input_dim % 8 or output_dim % 8:
            raise ValueError("a bank has adapters of rank 1 to 256, between widths that are multiples of 8")
        self.n, self.rank, self.input_dim, self.output_dim = n, -(-rank // 8) * 8, input_dim, output_dim
        self.register_buffer("down", torch.zeros(n, self.rank, input_dim, dtype=dtype, device=device))
        self.register_buffer("up", torch.zeros(n, output_dim, self.rank, dtype=dtype, device=device))
        self.register_buffer("scales", torch.zeros(n, dtype=torch.float32, device=device))

    def _apply(self, fn, recurse=True):
        scales = self.scales
        super()._apply(fn, recurse)
        if self.scales.dtype != torch.float32:
            self.scales = scales.to(self.scales.device)
        return self

    @torch.no_grad()
    def load(self, i: int, down: torch.Tensor, up: torch.Tensor, scale: float) -> None:
        """Adapter ``i`` becomes ``scale * (x @ down.T) @ up.T``: ``down`` [rank, input_dim], ``up`` [output_dim, rank]."""
        r = down.shape[0]
        if not 0 <= i < self.n or r > self.rank or tuple(down.shape) != (r, self.input_dim) or tuple(up.shape) != (self.output_dim, r):
            raise ValueError(f"adapter {i} of {self.n}: down {tuple(down.shape)}, up {tuple(up.shape)} do not fit rank {self.rank}, "
                             f"{self.input_dim} -> {self.output_dim}")
        down, up = down.clone(), up.clone()       # (they may be rows of this bank, its own ones too)
        self.down[i].zero_()
        self.up[i].zero_()
        self.down[i, :r] = down
        self.up[i, :, :r] = up
        self.scales[i] = scale

    def load_linear(self, i: int, linear: LoRAOptimizedLinear) -> None:
        """The adapter of a trained :class:`LoRAOptimizedLinear`."""
        self.load(i, linear.lora_weight_1.weight, linear.lora_weight_2.weight, linear.lora_scaling_factor)

    def plan(self, ids) -> AdapterPlan:
        """``ids[t]``: the adapter of row t, negative for none. One plan serves all layers of a batch whose banks are alike in number and device."""
        return AdapterPlan(ids, self.n, device=self.down.device)


class MultiAdapterLinear(nn.Module):
    """``y[t] = x[t] @ weight.T + bias + (the adapter of row t)(x[t])``, without gradients. ``bank`` may be shared with nothing else than
    projections of the same weight: it holds this projection's adapters."""

    def __init__(self, weight: torch.Tensor, bank: AdapterBank, bias: Optional[torch.Tensor] = None):
        super().__init__()
        if tuple(weight.shape) != (bank.output_dim, bank.input_dim) or weight.dtype != bank.down.dtype:
            raise ValueError(f"weight {tuple(weight.shape)} {weight.dtype} is not the bank's {(bank.output_dim, bank.input_dim)} {bank.down.dtype}")
        self.weight = nn.Parameter(weight, requires_grad=False)
        self.bias = None if bias is None else nn.Parameter(bias, requires_grad=False)
        self.bank = bank

    @torch.no_grad()
    def forward(self, x: torch.Tensor, plan: AdapterPlan) -> torch.Tensor:
        rows = x.reshape(-1, x.shape[-1])
        ops = get_ops(x.device)
        y = torch.empty(rows.shape[0], self.weight.shape[0], dtype=x.dtype, device=x.device)
        if rows.shape[0]:
            ops.gemm(rows, self.weight, y, bias=self.bias)
            ops.adapter_add(y, rows, self.bank.down, self.bank.up, self.bank.scales, plan, out=y)
        return y.view(*x.shape[:-1], self.weight.shape[0])
