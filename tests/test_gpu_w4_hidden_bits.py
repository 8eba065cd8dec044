"""The hidden activations between the projections of MoE experts on 4-bit weights keep some 22 bits, whatever the calls' type.

Features come in pairs: the gate's two rows are alike, the up projection's differ by a factor 1 + 2^-7, and an output is
the pair's difference times 1.75. A hidden activation rounded to fp16's 11 bits would be off by up to 2^-12 of itself, which
is 2^-4 of the output; the output's own rounding is 2^-9 (bf16) or 2^-12 (fp16) of it."""
import pytest
import torch

from tests.w4_helpers import Experts, half_step

pytestmark = pytest.mark.gpu


def _set(m, q, scales):
    m.q, m.scales = q, scales
    full = torch.cat([q, torch.zeros(*q.shape[:-1], q.shape[-1] % 2, dtype=torch.uint8)], -1)
    m.codes = full[..., 0::2] | full[..., 1::2] << 4
    m.w = (q.double() - 8.0) * scales.double()[..., torch.arange(m.n_in) // m.group]


def _paired(g, hidden, inter, count, group, dtype):
    ex = Experts(g, hidden, inter, count, group, dtype=dtype)
    pairs, even = inter // 2, torch.arange(inter // 2) * 2
    for m, odd in ((ex.gate, 1.0), (ex.up, 1 + 2.0 ** -7)):
        q, s = m.q.clone(), torch.full_like(m.scales, 0.25)
        q[:, even + 1], s[:, even + 1] = q[:, even], 0.25 * odd
        _set(m, q, s)
    q = torch.full_like(ex.down.q, 8)
    n = torch.arange(hidden)
    p = 2 * (n * 37 % pairs)
    q[:, n, p], q[:, n, p + 1] = 15, 1
    _set(ex.down, q, torch.full_like(ex.down.scales, 0.25))
    return ex, p


def _hidden(ex, x, e):
    a = x.double()
    g, u = a @ ex.gate.w[e].t(), a @ ex.up.w[e].t()
    return g * torch.sigmoid(g) * u


@pytest.mark.parametrize("rows,topk,inter", [(1, 2, 256), (1, 2, 333), (1, 2, 3200), (1, 2, 6272), (1, 8, 4224), (3, 2, 200), (9, 2, 256),
                                             (9, 2, 3200), (16, 2, 6272), (20, 2, 200), (40, 2, 256), (64, 2, 333), (65, 2, 256), (130, 2, 512)])
@pytest.mark.parametrize("group", [32, 128])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_differences_of_hidden_activations(dev, rows, topk, inter, group, dtype):
    hidden = 128
    g = torch.Generator().manual_seed(rows + inter)
    ex, p = _paired(g, hidden, inter, 1, group, dtype)
    x = torch.zeros(rows, hidden, dtype=dtype)               # one value a row: the gate's and the up products are exact
    x[torch.arange(rows), torch.arange(rows) % hidden] = (1 + torch.rand(rows, generator=g)).to(dtype)
    sel = torch.full((rows, topk), 7)
    sel[:, topk - 1] = 0                                     # the other slots are another rank's
    y = ex.module(dev)(x.to(dev), sel.to(dev), torch.ones(rows, topk).to(dev)).double().cpu()
    h = _hidden(ex, x, 0)
    ref, mag = 1.75 * (h[:, p] - h[:, p + 1]), 1.75 * (h[:, p].abs() + h[:, p + 1].abs())
    # SiLU's error (2^-20) is the pair's own and goes with the difference; up's rounding, its product with SiLU and the second half's
    # rounding are 2^-24 + 2^-24 + 2^-22 of a hidden activation, the four products' sum on the matrix cores, which may chop, 4 * 2^-23;
    # the second half's last place is 2^-25 beside a row's largest value of 2^14 or more
    tol = mag * 2.0 ** -20 + 1.75 * 2 * h.abs().amax(1, keepdim=True) * 2.0 ** -39
    tol = tol + ref.abs() * 2.0 ** -19 + half_step(dtype) * (ref.abs() + tol)
    off = (y - ref).abs()
    assert (off <= tol).all(), float((off / tol).max())
