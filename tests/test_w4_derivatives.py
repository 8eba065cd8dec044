"""The products on 4-bit weights have no derivatives: inputs that carry one, backward or forward, are refused."""
import pytest
import torch
from torch.autograd import forward_ad

from eva_amd import ops
from tests.w4_helpers import Experts, Matrix


def test_inputs_with_derivatives_are_refused():
    x = torch.ones(3)
    ops._no_grad("f", x, None)
    with pytest.raises(ValueError, match="f has no backward"):
        ops._no_grad("f", None, x.clone().requires_grad_())
    with torch.no_grad():
        ops._no_grad("f", x.clone().requires_grad_())
    with forward_ad.dual_level():
        dual = forward_ad.make_dual(x.clone(), torch.ones(3))
        ops._no_grad("f", x, None)
        with pytest.raises(ValueError, match="f has no forward-mode"):
            ops._no_grad("f", x, dual)
        with torch.no_grad(), pytest.raises(ValueError, match="f has no forward-mode"):
            ops._no_grad("f", dual)
        with torch.inference_mode():
            ops._no_grad("f", dual)
        ops._no_grad("f", forward_ad.unpack_dual(dual).primal)
    ops._no_grad("f", x)


@pytest.mark.gpu
def test_products_refuse_tangents(dev):
    g = torch.Generator().manual_seed(1)
    w, b = Matrix(g, 32, 64, 32).pack(dev), torch.zeros(32, dtype=torch.float16, device=dev)
    m = Experts(g, 64, 32, 3, 32, dtype=torch.float16).module(dev)
    x = torch.randn(2, 64, generator=g).half().to(dev)
    sel, weights = torch.zeros(2, 1, dtype=torch.int64, device=dev), torch.ones(2, 1, device=dev)
    y, z = ops.w4_linear(x, w, b), m(x, sel, weights)
    with forward_ad.dual_level():
        def dual(t):
            return forward_ad.make_dual(t.clone(), torch.ones_like(t))

        for call in (lambda: ops.w4_linear(dual(x), w), lambda: ops.w4_linear(x, w, dual(b)), lambda: m(dual(x), sel, weights),
                     lambda: m(x, sel, dual(weights)), lambda: ops.w4_linear(x, w, out=dual(y))):
            with pytest.raises(ValueError, match="forward-mode"):
                call()
        assert torch.equal(ops.w4_linear(x, w, b), y) and torch.equal(m(x, sel, weights), z)
