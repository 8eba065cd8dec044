"""Modules on 4-bit weights with group scales, beside the EXL3 ones: ``W4Linear`` (``ELinear``) and
``W4Experts`` (``ResidentExperts``). Weights are laid out once by ``ops.w4_pack``."""
from __future__ import annotations

import torch

from . import ops

MAX_CALL_ROWS = 65536       # rows per evamx_w4_linear call


def _moe_call_rows(slots: int, hidden: int, inter: int) -> int:
    """Rows of ``slots`` experts each that one evamx_w4_moe_forward call takes (its limits of slots, of x's and of the
    hidden activations' padded values)."""
    pad_hidden, pad_inter, slots = -(-hidden // 128) * 128, -(-inter // 128) * 128, max(slots, 1)
    return max(min(ops._lib.W4_MOE_MAX_SLOTS // slots, (2 ** 31 - 1) // pad_hidden, (2 ** 30 - 1) // (slots * pad_inter)), 1)


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
        if x.ndim == 2 and 0 < x.shape[0] <= MAX_CALL_ROWS and x.is_contiguous():
            return ops.w4_linear(x, self.weight, self.bias)
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


class W4Experts:
    """The experts of an MoE layer: stacks ``gate`` and ``up`` ``[inter, hidden]`` and ``down`` ``[hidden, inter]``,
    of which the last ``n_shared`` are shared experts and the others have the router's indices ``first_expert``
    and up (one rank's experts; slots of others add nothing)."""

    def __init__(self, gate: ops.W4Weight, up: ops.W4Weight, down: ops.W4Weight, *, n_shared: int = 0, first_expert: int = 0):
        shape = (gate.count, gate.n_out, gate.n_in)
        if (up.count, up.n_out, up.n_in) != shape or (down.count, down.n_in, down.n_out) != shape:
            raise ValueError("gate and up must be stacks [inter, hidden], down [hidden, inter], of as many matrices")
        if (up.desc.group, up.scales.dtype, up.zeros is None) != (gate.desc.group, gate.scales.dtype, gate.zeros is None):
            raise ValueError("gate and up must agree in their group size, their scales' type and in having zero points")
        if not 0 <= n_shared <= gate.count:
            raise ValueError(f"{n_shared} shared experts of {gate.count}")
        self.gate, self.up, self.down = gate, up, down
        self.n_shared, self.first_expert = n_shared, first_expert
        self.hidden, self.inter, self.n_local = gate.n_in, gate.n_out, gate.count - n_shared

    def forward(self, x: torch.Tensor, sel: torch.Tensor, weights: torch.Tensor, limit: float = 0.0) -> torch.Tensor:
        """Experts of x ``[..., hidden]`` (fp16 or bf16) for routes ``sel`` (integers) and ``weights`` ``[..., topk]``."""
        if x.shape[-1] != self.hidden:
            raise ValueError(f"x has {x.shape[-1]} features, the experts {self.hidden}")
        flat, topk = x.reshape(-1, self.hidden), sel.shape[-1]
        if (flat.shape[1] > 1 and flat.stride(1) != 1) or (flat.shape[0] > 1 and flat.stride(0) < self.hidden):
            flat = flat.contiguous()
        rows = flat.shape[0]
        sel = sel.reshape(rows, topk).to(torch.int64).contiguous()
        weights = weights.reshape(rows, topk).to(torch.float32).contiguous()
        out = torch.empty(rows, self.hidden, dtype=x.dtype, device=x.device)
        step = _moe_call_rows(topk + self.n_shared, self.hidden, self.inter)
        for r0 in range(0, rows, step):
            part = slice(r0, r0 + step)
            ops.w4_moe_forward(flat[part], self.gate, self.up, self.down, sel[part], weights[part], n_shared=self.n_shared,
                               first_expert=self.first_expert, limit=limit, out=out[part])
        return out.reshape(*x.shape[:-1], self.hidden)

    __call__ = forward
