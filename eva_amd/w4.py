"""Modules on 4-bit weights with group scales, beside the EXL3 ones: ``W4Linear`` (``ELinear``) and
``W4Experts`` (``ResidentExperts``). Weights are laid out once by ``ops.w4_pack``."""
from __future__ import annotations

import torch

from . import ops

MAX_CALL_ROWS = 65536       # rows per evamx_w4_linear call


class W4Linear:
    """``y = x W^T (+ bias)`` for one packed matrix; x fp16 or bf16 with any leading dimensions."""

    def __init__(self, weight: ops.W4Weight, bias: torch.Tensor | None = None):
        if weight.count != 1:
            raise ValueError(f"a linear takes one matrix, got a stack of {weight.count}")
        if bias is not None and tuple(bias.shape) != (weight.n_out,):
            raise ValueError(f"bias must be [{weight.n_out}], got {tuple(bias.shape)}")
        self.weight, self.bias = weight, bias
        self.in_features, self.out_features = weight.n_in, weight.n_out

    def forward(self, x: torch.Tensor) -> torch.Tensor:
        if x.shape[-1] != self.in_features:
            raise ValueError(f"x has {x.shape[-1]} features, the weight {self.in_features}")
        flat = x.reshape(-1, self.in_features)
        if (flat.shape[1] > 1 and flat.stride(1) != 1) or (flat.shape[0] > 1 and flat.stride(0) < self.in_features):
            flat = flat.contiguous()
        y = torch.empty(flat.shape[0], self.out_features, dtype=x.dtype, device=x.device)
        for r0 in range(0, flat.shape[0], MAX_CALL_ROWS):
            ops.w4_linear(flat[r0:r0 + MAX_CALL_ROWS], self.weight, self.bias, out=y[r0:r0 + MAX_CALL_ROWS])
        return y.reshape(*x.shape[:-1], self.out_features)

    __call__ = forward
