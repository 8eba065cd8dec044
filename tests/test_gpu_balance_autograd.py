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


@pytest.mark.parametrize("score", ["sigmoid", "sqrt_softplus"])
def test_gradient_of_the_routers_weight(dev, score):
    """Logits from the program's own product, routes from the framework's router, the gradient of the router's weight against
    64 bits; behind ops.router_logits there is no way back, and backward() says so."""
    from tests.test_gpu_balance import _oracle

    g = torch.Generator().manual_seed(9)
    rows, hidden, experts, topk = 300, 256, 40, 4
    x = torch.randn(rows, hidden, generator=g).bfloat16().to(dev)
    w = (torch.randn(experts, hidden, generator=g) / 16).to(dev).requires_grad_()
    starts, gl = [0, 100, 300], torch.tensor([0.5, 2.0])
    logits = x.float() @ w.t()
    sel, _, _ = ops.route_topk(logits.detach(), topk, score)
    loss, counts = ops.balance_loss(logits, sel, score_fn=score, seq_starts=torch.tensor(starts, dtype=torch.int32, device=dev))
    (loss * gl.to(dev)).sum().backward()
    z = logits.detach().cpu().double().requires_grad_()
    ref, ref_counts = _oracle(z, sel.cpu(), score, starts)
    dz, = torch.autograd.grad(ref, z, gl.double())
    x64 = x.cpu().double()
    assert torch.equal(counts.cpu(), ref_counts)
    # a logit's gradient is off by 64 fp32 steps of itself and of its share (below 1/8 here) times the largest count of its
    # sequence, as its factor has it; the product sums 300 rows in fp32
    unit, bound = 2.0 ** -24, torch.zeros(rows, 1, dtype=torch.float64)
    for s, (lo, hi) in enumerate(zip(starts[:-1], starts[1:])):
        bound[lo:hi] = gl[s].double() * experts / (topk * (hi - lo) ** 2) * ref_counts[s].max()
    off_z = bound / 8 * 64 * unit + dz.abs() * 64 * unit
    tol = off_z.expand(rows, experts).t() @ x64.abs() + (rows + 8) * 2 * unit * (dz.abs().t() @ x64.abs())
    off = (w.grad.cpu().double() - dz.t() @ x64).abs()
    assert (off <= tol).all(), float((off / tol).max())
    behind, _ = ops.balance_loss(ops.router_logits(x, w.detach()), sel, score_fn=score)
    with pytest.raises(RuntimeError, match="does not require grad"):
        behind.sum().backward()
