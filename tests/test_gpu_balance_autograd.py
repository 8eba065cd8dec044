"""The balance loss as a training step meets it: what its backward pass refuses, and the way back to a router's weight."""
import pytest
import torch

from eva_amd import ops

pytestmark = pytest.mark.gpu


def test_a_backward_pass_alone_is_not_captured(dev, monkeypatch):
    """The forward pass ran eagerly, the backward one finds its stream capturing (told so: nothing is captured here)."""
    z = torch.randn(12, 8, generator=torch.Generator().manual_seed(1)).to(dev).requires_grad_()
    loss, _ = ops.balance_loss(z, z.topk(2, 1).indices)
    with monkeypatch.context() as m:
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        with pytest.raises(RuntimeError, match="not captured"):
            torch.autograd.grad(loss.sum(), z, retain_graph=True)
    grad, = torch.autograd.grad(loss.sum(), z)
    assert grad.isfinite().all()
