"""Zero points of 4-bit weights above the codes' range: 16 (formats that hold the zero point less one) to 31."""
import pytest
import torch

from eva_amd import ops
from tests.w4_helpers import Experts, Matrix, check_linear

pytestmark = pytest.mark.gpu


def _wide(g, m):
    """m with zero points of the whole range, 16 and 31 among them."""
    m.zeros = torch.randint(0, 32, m.scales.shape, generator=g, dtype=torch.uint8)
    m.zeros.view(-1)[:2] = torch.tensor([16, 31], dtype=torch.uint8)
    m.w = (m.q.double() - m.zeros.double()[..., torch.arange(m.n_in) // m.group]) * m.scales.double()[..., torch.arange(m.n_in) // m.group]
    return m


@pytest.mark.parametrize("group", [32, 64, 128, 96])
@pytest.mark.parametrize("rows", [1, 3, 13, 40, 1100])
def test_linear(dev, group, rows):
    """Each kernel of the linear takes them, and so does the dequantized matrix."""
    g = torch.Generator().manual_seed(group + rows)
    n_out = 4100 if rows > 1000 else 100
    m = _wide(g, Matrix(g, n_out, 389, group, zeros=True))
    w = m.pack(dev)
    assert torch.equal(ops.w4_dequant(w).cpu()[0], m.w.float())
    x = torch.randn(rows, 389, generator=g).half().to(dev)
    check_linear(ops.w4_linear(x, w), x, m.w.to(dev))


@pytest.mark.parametrize("rows", [1, 3, 12, 100])
def test_experts(dev, rows):
    g = torch.Generator().manual_seed(rows)
    ex = Experts(g, 256, 160, 3, 64, zeros=True)
    for m in (ex.gate, ex.up, ex.down):
        _wide(g, m)
    x = torch.randn(rows, 256, generator=g).bfloat16()
    sel, w = torch.randint(0, 3, (rows, 2), generator=g), torch.rand(rows, 2, generator=g)
    ref, tol = ex.reference(x, sel, w)
    off = (ex.module(dev)(x.to(dev), sel.to(dev), w.to(dev)).double().cpu() - ref).abs()
    assert (off <= tol).all(), float((off / tol).max())


def test_larger_ones_are_refused(dev):
    g = torch.Generator().manual_seed(1)
    m = Matrix(g, 32, 64, 32, zeros=True)
    for bad in (32, 255):
        m.zeros[5, 1] = bad
        with pytest.raises(ValueError, match="zero points"):
            m.pack(dev)


@pytest.mark.parametrize("rows", [1, 9, 40])
def test_bytes_an_owner_wrote(dev, rows):
    """A weight whose buffers its owner fills: the products and the dequantized matrix read the same five bits of a byte."""
    g = torch.Generator().manual_seed(rows)
    m = _wide(g, Matrix(g, 48, 160, 32, zeros=True))
    w = m.pack(dev)
    x = torch.randn(rows, 160, generator=g).half().to(dev)
    y, full = ops.w4_linear(x, w), ops.w4_dequant(w)
    w.zeros += torch.randint(0, 8, w.zeros.shape, generator=g, dtype=torch.uint8).to(dev) * 32
    assert torch.equal(ops.w4_linear(x, w), y) and torch.equal(ops.w4_dequant(w), full)
