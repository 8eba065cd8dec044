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
    """y against x W^T + bias in 64 bits: half a step of y's type, the sums' error, and inputs off by input_error."""
    x64 = x.double().cpu()
    ref = x64 @ w.t()
    mag = x64.abs() @ w.abs().t()
    if bias is not None:
        ref, mag = ref + bias.double().cpu(), mag + bias.double().cpu().abs()
    tol = mag * (sum_error(x.shape[-1]) + input_error)
    tol = tol + half_step(y.dtype) * (ref.abs() + tol) + torch.finfo(y.dtype).smallest_normal * half_step(y.dtype)
    off = (y.double().cpu() - ref).abs()
    assert (off <= tol).all(), float((off / tol).max())
