"""Synthetic 4-bit matrices and their 64-bit values, for the tests of the operators on them."""
from __future__ import annotations

import torch


class Matrix:
    """``count`` matrices [n_out, n_in]: codes as a checkpoint holds them, and W in 64 bits (CPU)."""

    def __init__(self, gen, n_out, n_in, group, *, count=None, zeros=False, dtype=torch.float16, scale=None):
        lead = () if count is None else (count,)
        self.q = torch.randint(0, 16, (*lead, n_out, n_in), generator=gen, dtype=torch.uint8)
        pad = torch.zeros(*lead, n_out, n_in % 2, dtype=torch.uint8)
        full = torch.cat([self.q, pad], -1)
        self.codes = full[..., 0::2] | full[..., 1::2] << 4
        groups = (*lead, n_out, -(-n_in // group))
        s = (torch.rand(groups, generator=gen) + 0.5) * (0.2 * n_in ** -0.5 if scale is None else scale)
        self.scales = s.to(dtype)
        self.zeros = torch.randint(0, 16, groups, generator=gen, dtype=torch.uint8) if zeros else None
        self.n_in, self.group = n_in, group
        at = torch.arange(n_in) // group
        z = 8.0 if self.zeros is None else self.zeros.double()[..., at]
        self.w = (self.q.double() - z) * self.scales.double()[..., at]

    def pack(self, dev):
        from eva_amd import ops
        return ops.w4_pack(self.codes.to(dev), self.scales.to(dev), n_in=self.n_in, group=self.group,
                           zeros=None if self.zeros is None else self.zeros.to(dev))


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def sum_error(n_in):
    """Relative to the sum of magnitudes, what fp32 sums over n_in products in groups of 32 or more may be off:
    a group's products (at most 128 in a row, on matrix cores that may chop: a whole step of 2^-23), then the
    groups and the waves that share a column."""
    return (128 + n_in / 32 + 32) * 2.0 ** -23


def check_linear(y, x, w, bias=None, input_error=0.0):
    """y against x W^T + bias in 64 bits, where w is: half a step of y's type, the sums' error, and inputs off by
    input_error."""
    x64 = x.double().to(w.device)
    ref = x64 @ w.t()
    mag = x64.abs() @ w.abs().t()
    if bias is not None:
        b = bias.double().to(w.device)
        ref, mag = ref + b, mag + b.abs()
    tol = mag * (sum_error(x.shape[-1]) + input_error)
    tol = tol + half_step(y.dtype) * (ref.abs() + tol) + torch.finfo(y.dtype).smallest_normal * half_step(y.dtype)
    off = (y.double().to(w.device) - ref).abs()
    assert (off <= tol).all(), float((off / tol).max())


class Experts:
    """An MoE layer's experts on such matrices."""

    def __init__(self, gen, hidden, inter, count, group, *, zeros=False, dtype=torch.bfloat16, down_group=None, down_zeros=None, scale=None):
        kw = dict(count=count, zeros=zeros, dtype=dtype, scale=scale)
        self.gate, self.up = Matrix(gen, inter, hidden, group, **kw), Matrix(gen, inter, hidden, group, **kw)
        kw["zeros"] = zeros if down_zeros is None else down_zeros
        self.down = Matrix(gen, hidden, inter, group if down_group is None else down_group, **kw)
        self.hidden, self.inter, self.count = hidden, inter, count

    def module(self, dev, **kw):
        from eva_amd.w4 import W4Experts
        return W4Experts(self.gate.pack(dev), self.up.pack(dev), self.down.pack(dev), **kw)

    def reference(self, x, sel, weights, *, n_shared=0, first_expert=0, limit=0.0, dtype=torch.bfloat16):
        """(out, tolerance) in 64 bits on the CPU. The tolerance carries the sums' errors and the hidden
        activations' rounding to fp16 (half a step, relative; the row's factor keeps them from underflow) to the
        output, whose own rounding is half a step of its type."""
        x, weights = x.double().cpu(), weights.double().cpu()
        out, tol = torch.zeros_like(x), torch.zeros_like(x)
        local = self.count - n_shared
        for e in range(self.count):
            if e < local:
                t, k = (sel.cpu() == e + first_expert).nonzero(as_tuple=True)
                w = weights[t, k]
            else:
                t = torch.arange(x.shape[0])
                w = torch.ones(len(t), dtype=torch.float64)
            if not len(t):
                continue
            a, unit = x[t], sum_error(self.hidden)
            g, u = a @ self.gate.w[e].t(), a @ self.up.w[e].t()
            dg, du = unit * (a.abs() @ self.gate.w[e].abs().t()), unit * (a.abs() @ self.up.w[e].abs().t())
            if limit:
                u = u.clamp(-limit, limit)
                if e >= local:
                    g = g.clamp(max=limit)
            s = g * torch.sigmoid(g)
            if limit and e < local:
                s = s.clamp(max=limit)
            h = s * u
            # SiLU's slope is below 1.1; exp and the quotient a few steps of 2^-22 each
            dh = 1.1 * dg * (u.abs() + du) + s.abs() * du + h.abs() * (2.0 ** -20 + half_step(torch.float16))
            dh = dh + h.abs().amax(1, keepdim=True) * 2.0 ** -39
            d = self.down.w[e]
            y, mag = h @ d.t(), h.abs() @ d.abs().t()
            out.index_add_(0, t, w[:, None] * y)
            tol.index_add_(0, t, w.abs()[:, None] * (dh @ d.abs().t() + (sum_error(self.inter) + 2.0 ** -20) * mag))
        return out, tol + half_step(dtype) * (out.abs() + tol) + torch.finfo(dtype).smallest_normal * half_step(dtype)
