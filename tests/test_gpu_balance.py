"""Expert counts, balance loss and its gradient against their definition in 64 bits."""
import pytest
import torch

from eva_amd import ops

pytestmark = pytest.mark.gpu
SCORES = ["sigmoid", "sqrt_softplus"]


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _oracle(z, sel, score, starts=None, mask=None):
    """(loss, counts) in 64 bits, differentiable in z, from logarithms of the scores (no underflow)."""
    t, e = z.shape
    starts = [0, t] if starts is None else [min(max(int(v), 0), t) for v in starts]
    if score == "sigmoid":
        log_a = torch.nn.functional.logsigmoid(z)
    else:
        # log softplus(z) = z + log(softplus(z) / e^z); far below zero that ratio is 1 - e^z / 2
        soft = torch.nn.functional.softplus(z.clamp(min=-30), threshold=1e9)
        log_a = 0.5 * torch.where(z < -30, z, soft.log())
    empty = (z == float("-inf")).all(1, keepdim=True)
    p = torch.softmax(torch.where(empty, torch.zeros_like(log_a), log_a), 1)
    p = torch.where(empty, torch.zeros_like(p), p)
    losses, counts = [], torch.zeros(len(starts) - 1, e, dtype=torch.int32)
    for s, (lo, hi) in enumerate(zip(starts[:-1], starts[1:])):
        rows = torch.arange(lo, max(lo, hi))
        if mask is not None:
            rows = rows[mask[rows]]
        picks = sel[rows].reshape(-1)
        counts[s] = torch.bincount(picks[(picks >= 0) & (picks < e)], minlength=e).int()
        n = len(rows)
        losses.append((counts[s].double() * p[rows].sum(0)).sum() * (e / (sel.shape[1] * n * n)) if n else p[rows].sum())
    return torch.stack(losses), counts


def _check(dev, z, sel, score, starts=None, mask=None, seed=0):
    """z, sel, starts, mask on the CPU; z of the type under test."""
    z64 = z.double().requires_grad_()
    loss, counts = _oracle(z64, sel, score, starts, mask)
    gl = torch.rand(len(loss), generator=_gen(seed)) + 0.5
    grad, = torch.autograd.grad(loss, z64, gl.double(), allow_unused=True)
    grad = torch.zeros_like(z64) if grad is None else grad
    leaf = z.to(dev).requires_grad_()
    starts_d = None if starts is None else torch.as_tensor(starts, dtype=torch.int32, device=dev)
    mask_d = None if mask is None else mask.to(dev)
    got, got_counts = ops.balance_loss(leaf, sel.to(dev), score_fn=score, seq_starts=starts_d, token_mask=mask_d)
    got_grad, = torch.autograd.grad(got, leaf, gl.to(dev))
    assert torch.equal(got_counts.cpu(), counts)
    # a score and its slope: a few fp32 functions and products, each within 4 steps; shares: a sum over the experts
    # in a tree; the loss: positive terms over the rows, at most rows / 64 + 64 in a row
    unit = 2.0 ** -24
    tol = (64 + z.shape[0] / 16) * unit
    assert ((got.detach().cpu().double() - loss.detach()).abs() <= tol * loss.detach().abs()).all()
    # the gradient: p (c_j - sum c p) loses relative to the sequence's largest count
    e, k = z.shape[1], sel.shape[1]
    bound = torch.zeros(z.shape[0], 1, dtype=torch.float64)
    st = [0, z.shape[0]] if starts is None else [min(max(int(v), 0), z.shape[0]) for v in starts]
    for s, (lo, hi) in enumerate(zip(st[:-1], st[1:])):
        if hi > lo:
            n = hi - lo if mask is None else max(1, int(mask[lo:hi].sum()))
            bound[lo:hi] = gl[s].double() * e / (k * n * n) * counts[s].max()
    p = torch.softmax(torch.nn.functional.logsigmoid(z64.detach()) if score == "sigmoid" else
                      0.5 * torch.where(z64 < -30, z64, torch.nn.functional.softplus(z64.clamp(min=-30), threshold=1e9).log()).detach(), 1)
    p = torch.nan_to_num(p)
    fine = bound * p * 64 * unit + grad.abs() * (torch.finfo(z.dtype).eps / 2 + 64 * unit) + torch.finfo(z.dtype).smallest_normal * torch.finfo(z.dtype).eps
    off = (got_grad.cpu().double() - grad).abs()
    assert (off <= fine).all(), float((off / fine).max())
    return got, got_counts, got_grad


@pytest.mark.parametrize("rows,experts,topk", [(1, 1, 1), (1, 2, 1), (3, 7, 2), (5, 64, 6), (64, 65, 8), (257, 160, 8), (1000, 256, 8),
                                               (333, 384, 6), (130, 512, 32), (5000, 255, 4)])
@pytest.mark.parametrize("score", SCORES)
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16, torch.float16])
def test_one_sequence(dev, rows, experts, topk, score, dtype):
    z = (2 * torch.randn(rows, experts, generator=_gen(rows + experts))).to(dtype)
    _check(dev, z, z.float().topk(topk, 1).indices, score)


@pytest.mark.parametrize("starts", [[0, 10, 10, 64, 200], [0, 0, 0, 200], [5, 60, 190], [0, 1, 2, 3, 200], [200, 200], [0, 64, 128, 192, 200],
                                    [0, 300], [-5, 40]])
@pytest.mark.parametrize("score", SCORES)
def test_sequences_and_masks(dev, starts, score):
    """Empty sequences, rows before the first and behind the last, starts outside the rows, masked rows that hold
    NaN, a sequence whose rows are all masked."""
    g = _gen(len(starts))
    z = torch.randn(200, 96, generator=g)
    sel = z.topk(5, 1).indices
    _check(dev, z, sel, score, starts)
    mask = torch.rand(200, generator=g) < 0.7
    mask[60:130] = False
    _, _, grad = _check(dev, z, sel, score, starts, mask)
    bad = z.clone()
    bad[~mask] = float("nan")
    leaf = bad.to(dev).requires_grad_()
    loss, _ = ops.balance_loss(leaf, sel.to(dev), score_fn=score, seq_starts=torch.tensor(starts, dtype=torch.int32, device=dev),
                               token_mask=mask.to(dev))
    again, = torch.autograd.grad(loss, leaf, torch.rand(len(starts) - 1, generator=_gen(0)).add(0.5).to(dev))
    assert torch.equal(again, grad) and (again.cpu()[~mask] == 0).all()


@pytest.mark.parametrize("rows,sequences", [(5000, 700), (16385, 3), (40000, 64), (300, 4000)])
def test_many_sequences(dev, rows, sequences):
    """Sequences of one token, many to a chunk of rows and many chunks to a sequence."""
    g = _gen(sequences)
    z = torch.randn(rows, 70, generator=g)
    cuts = torch.randint(0, rows + 1, (sequences - 1,), generator=g).sort().values.tolist()
    mask = torch.rand(rows, generator=g) < 0.9
    _check(dev, z, z.topk(3, 1).indices, "sigmoid", [0, *cuts, rows], mask)


@pytest.mark.parametrize("score", SCORES)
def test_far_logits(dev, score):
    """Scores that underflow for a whole row keep their shares; -inf has none; a row of -inf alone has only picks."""
    z = torch.randn(40, 64, generator=_gen(3)) * 3
    z[3] -= 150
    z[4] -= 1000
    z[5, :60] = -float("inf")
    z[6] += 80
    z[7, 9] = 300
    z[8] = -float("inf")
    z[9] = torch.finfo(torch.float32).min
    z[10, 1:] = torch.finfo(torch.float32).min
    z[11] -= 17
    z[12] -= 15
    _check(dev, z, z.topk(4, 1).indices, score)


def test_picks_that_are_none(dev):
    z = torch.randn(30, 16, generator=_gen(4))
    sel = torch.randint(-3, 20, (30, 4), generator=_gen(5))
    sel[0] = 7                                        # the same expert four times
    sel[1, 0], sel[1, 1] = 2 ** 40, -2 ** 40
    _check(dev, z, sel, "sigmoid", [0, 13, 30])


@pytest.mark.parametrize("score", SCORES)
def test_gradient_against_differences(dev, score):
    z = torch.randn(6, 9, generator=_gen(7), dtype=torch.float64)
    sel = z.topk(3, 1).indices
    leaf = z.float().to(dev).requires_grad_()
    loss, _ = ops.balance_loss(leaf, sel.to(dev), score_fn=score)
    loss.sum().backward()
    h = 1e-4
    for i, j in ((0, 0), (2, 5), (5, 8), (3, 3)):
        d = torch.zeros_like(z)
        d[i, j] = h
        num = (_oracle(z + d, sel, score)[0] - _oracle(z - d, sel, score)[0]).item() / (2 * h)
        assert abs(leaf.grad[i, j].item() - num) <= 1e-6 + 1e-5 * abs(num)     # h^2 of the difference, fp32 of the kernel


@pytest.mark.parametrize("rows", [3, 700, 20000])
def test_strides_repeats_and_graph(dev, rows):
    """A slice of wider rows gives the same bits; so does every repeat, and every replay of a captured forward and
    explicit gradient."""
    g = _gen(rows)
    wide = torch.randn(rows, 150, generator=g).to(dev)
    z = wide[:, 7:135]
    sel = z.topk(6, 1).indices
    starts = torch.tensor([0, rows // 3, rows // 3, rows], dtype=torch.int32, device=dev)
    gl = torch.tensor([0.5, 1.0, 2.0], device=dev)

    def step(z, sel):
        loss, counts, tokens = ops.balance_stats(z, sel, seq_starts=starts)
        return loss, counts, tokens, ops.balance_loss_grad(gl, z, counts, tokens, 6, seq_starts=starts)

    ref = step(z, sel)
    assert ref[2].tolist() == [rows // 3, 0, rows - rows // 3]
    for other in (step(z.contiguous(), sel), step(z, sel)):
        assert all(torch.equal(a, b) for a, b in zip(ref, other))
    sz, ssel = z.contiguous().clone(), sel.clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        out = step(sz, ssel)
    for k in range(4):
        sz.copy_(torch.randn(rows, 128, generator=g))
        ssel.copy_(sz.topk(6, 1).indices)
        graph.replay()
        assert all(torch.equal(a, b) for a, b in zip(out, step(sz, ssel))), k
        torch.cuda.synchronize()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = step(z, sel)
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(ref, other))


def test_empty_batch_and_shared_leaf(dev):
    """No rows at all; and logits used twice, whose gradients add."""
    z = torch.zeros(0, 8, device=dev, requires_grad=True)
    loss, counts = ops.balance_loss(z, torch.zeros(0, 2, dtype=torch.int64, device=dev))
    loss.sum().backward()
    assert loss.item() == 0 and counts.sum().item() == 0 and z.grad.shape == (0, 8)
    leaf = torch.randn(9, 8, generator=_gen(1)).to(dev).requires_grad_()
    sel = leaf.topk(2, 1).indices
    one, = torch.autograd.grad(ops.balance_loss(leaf, sel)[0].sum(), leaf)
    two, = torch.autograd.grad(ops.balance_loss(leaf, sel)[0].sum() + 3 * ops.balance_loss(leaf, sel)[0].sum(), leaf)
    assert torch.allclose(two, 4 * one, rtol=1e-6, atol=0)
    through, = torch.autograd.grad(ops.balance_loss(leaf * 2.0, sel)[0], leaf, torch.ones(1, device=dev).expand(1))
    direct, = torch.autograd.grad(ops.balance_loss(x2 := (leaf * 2).detach().requires_grad_(), sel)[0].sum(), x2)
    assert torch.equal(through, 2 * direct)


def test_refusals(dev):
    z = torch.randn(4, 8, device=dev)
    sel = z.topk(2, 1).indices
    for bad in (z.double(), z[0], z.t(), z.cpu()):
        with pytest.raises(ValueError):
            ops.balance_loss(bad, sel)
    for bad in (sel.int(), sel[:3], sel.t(), sel.cpu()):
        with pytest.raises(ValueError):
            ops.balance_loss(z, bad)
    for kw in (dict(score_fn="softmax"), dict(seq_starts=torch.tensor([0, 4], device=dev)), dict(token_mask=torch.ones(4, device=dev)),
               dict(token_mask=torch.ones(3, dtype=torch.bool, device=dev)), dict(seq_starts=torch.zeros(1, dtype=torch.int32, device=dev))):
        with pytest.raises(ValueError):
            ops.balance_loss(z, sel, **kw)
    with pytest.raises(ops._lib.EvamxError):
        ops.balance_loss(torch.randn(2, 513, device=dev), sel[:2])
    with pytest.raises(ops._lib.EvamxError):
        ops.balance_loss(z, torch.zeros(4, 33, dtype=torch.int64, device=dev))
    leaf = z.clone().requires_grad_()
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(ops.balance_loss(leaf, sel)[0].sum(), leaf, create_graph=True)
    with pytest.raises(RuntimeError, match="captured"):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            ops.balance_loss(leaf, sel)


def test_after_the_router(dev):
    """As a router's step uses it: logits and routes from the framework's router, the loss's gradient back to the
    router's weight."""
    g = _gen(9)
    x = torch.randn(300, 256, generator=g).bfloat16().to(dev)
    w = (torch.randn(40, 256, generator=g) / 16).to(dev)
    for score in SCORES:
        z = ops.router_logits(x, w)
        idx, _, _ = ops.route_topk(z, 4, score)
        _, counts, grad = _check(dev, z.cpu(), idx.cpu(), score, [0, 100, 300])
        assert counts.sum(1).tolist() == [400, 800]
