"""Modules on 16-bit weights, beside the quantized ones: ``DenseLinear`` (``W4Linear``) and ``DenseExperts`` (``W4Experts``). They
hold the tensors they are given and can be trained: autograd follows ``ops.linear``, ``ops.sort_tokens``, ``ops.expert_linear`` and
``ops.combine_tokens``."""
from __future__ import annotations

import torch

from . import ops


class DenseLinear:
    """``activation(x W^T + bias) + residual`` for one matrix; x fp16 or bf16 with any leading dimensions (``ops.linear``)."""

    def __init__(self, weight: torch.Tensor, bias: torch.Tensor | None = None, *, activation: str | None = None, limit: float = 0.0):
        if weight.ndim != 2 or (bias is not None and tuple(bias.shape) != (weight.shape[0],)):
            raise ValueError("weight must be [n_out, n_in], bias [n_out]")
        self.weight, self.bias, self.activation, self.limit = weight, bias, activation, limit
        self.in_features = weight.shape[1]
        self.out_features = weight.shape[0] // 2 if activation == "swiglu" else weight.shape[0]

    def forward(self, x: torch.Tensor, residual: torch.Tensor | None = None) -> torch.Tensor:
        if x.shape[-1] != self.in_features:
            raise ValueError(f"x has {x.shape[-1]} features, the weight {self.in_features}")
        shape = (*x.shape[:-1], self.out_features)
        if residual is not None and tuple(residual.shape) != shape:
            raise ValueError(f"residual must be {list(shape)}, got {list(residual.shape)}")
        y = ops.linear(_rows(x), self.weight, self.bias, activation=self.activation, limit=self.limit,
                       residual=None if residual is None else _rows(residual))
        return y.reshape(shape)

    __call__ = forward


class DenseExperts:
    """The experts of an MoE layer: ``gate_up [E, 2 inter, hidden]`` (an expert's gate rows, then its up rows) and ``down [E, hidden,
    inter]``, of the router's indices ``first_expert`` and up (one rank's experts; slots of others add nothing)."""

    def __init__(self, gate_up: torch.Tensor, down: torch.Tensor, *, first_expert: int = 0):
        if gate_up.ndim != 3 or gate_up.shape[1] % 2 or tuple(down.shape) != (gate_up.shape[0], gate_up.shape[2], gate_up.shape[1] // 2):
            raise ValueError("gate_up must be [E, 2 inter, hidden], down [E, hidden, inter]")
        self.gate_up, self.down, self.first_expert = gate_up, down, first_expert
        self.n_local, self.hidden, self.inter = gate_up.shape[0], gate_up.shape[2], gate_up.shape[1] // 2

    def forward(self, x: torch.Tensor, sel: torch.Tensor, weights: torch.Tensor, limit: float = 0.0,
                residual: torch.Tensor | None = None) -> torch.Tensor:
        """Experts of x ``[..., hidden]`` (fp16 or bf16) for routes ``sel`` (integers) and ``weights`` ``[..., topk]``, plus
        ``residual`` of x's shape and type. Hidden activations and each expert's results are rounded to x's type."""
        if x.shape[-1] != self.hidden:
            raise ValueError(f"x has {x.shape[-1]} features, the experts {self.hidden}")
        if residual is not None and residual.shape != x.shape:
            raise ValueError(f"residual must be {list(x.shape)}, got {list(residual.shape)}")
        if sel.dtype.is_floating_point or sel.dtype.is_complex or sel.dtype == torch.bool:
            raise ValueError(f"sel must hold expert indices, got {sel.dtype}")
        flat, topk = _rows(x), sel.shape[-1]
        order = ops.expert_order(sel.reshape(flat.shape[0], topk).to(torch.int64).contiguous(), self.n_local, first_expert=self.first_expert)
        h = ops.expert_linear(ops.sort_tokens(flat, order), self.gate_up, order.starts, activation="swiglu", limit=limit)
        y = ops.expert_linear(h, self.down, order.starts)
        out = ops.combine_tokens(y, order, weights.reshape(flat.shape[0], topk).to(torch.float32).contiguous(),
                                 residual=None if residual is None else _rows(residual))
        return out.reshape(x.shape)

    __call__ = forward


def _rows(x: torch.Tensor) -> torch.Tensor:
    """``x [..., features]`` as rows that are contiguous and do not overlap."""
    return ops._rows_of(x.reshape(-1, x.shape[-1]))
