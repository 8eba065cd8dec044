"""Tokens sorted by expert and back (ops.expert_order, sort_tokens, combine_tokens) and their gradients, against 64 bits."""
import pytest
import torch

from eva_amd import ops

pytestmark = pytest.mark.gpu
TYPES = [torch.bfloat16, torch.float16, torch.float32]


def order_of(sel, n, first=0):
    """(starts, position) by a stable sort on the host."""
    e = (sel.cpu() - first).flatten().tolist()
    slots = sorted((s for s in range(len(e)) if 0 <= e[s] < n), key=lambda s: e[s])
    position = torch.full((len(e),), -1, dtype=torch.int32)
    position[torch.tensor(slots, dtype=torch.int64)] = torch.arange(len(slots), dtype=torch.int32)
    starts = torch.tensor([sum(1 for s in slots if e[s] < x) for x in range(n + 1)], dtype=torch.int32)
    return starts, position.view(sel.shape)


def routes(rows, topk, experts, seed, padded=False):
    g = torch.Generator().manual_seed(seed)
    sel = torch.randint(0, experts, (rows, topk), generator=g)
    if padded:
        sel[torch.rand(rows, generator=g) < 0.3] = -1
    return sel


@pytest.mark.parametrize("rows,topk,experts,first,n", [
    (1, 1, 1, 0, 1), (1, 8, 256, 0, 256), (7, 3, 5, 2, 2), (63, 1, 64, 0, 64), (257, 6, 384, 192, 96), (255, 8, 256, 0, 256),
    (256, 8, 256, 0, 256), (2049, 1, 1024, 0, 1024), (3001, 8, 1000, 0, 999), (1000, 32, 7, 0, 7), (70000, 8, 33, 4, 20)])
def test_order(dev, rows, topk, experts, first, n):
    sel = routes(rows, topk, experts, rows + topk, padded=rows > 5)
    got = ops.expert_order(sel.to(dev), n, first_expert=first)
    if rows * topk > 20000:      # the same by torch's stable sort
        e = (sel - first).flatten()
        e = torch.where((e >= 0) & (e < n), e, n)
        by = e.argsort(stable=True)
        position = torch.empty_like(by)
        position[by] = torch.arange(by.numel())
        position = torch.where(e < n, position, -1).int().view(sel.shape)
        starts = torch.searchsorted(e[by], torch.arange(n + 1)).int()
    else:
        starts, position = order_of(sel, n, first)
    assert torch.equal(got.starts.cpu(), starts) and torch.equal(got.position.cpu(), position)


def test_order_of_odd_numbers(dev):
    """The same expert several times for a token, numbers far outside, no token at all."""
    big = 2 ** 63 - 1
    sel = torch.tensor([[3, 3, 3], [big, -big - 1, 0], [4, 3, -1]], device=dev)
    got = ops.expert_order(sel, 4)
    assert got.starts.tolist() == [0, 1, 1, 1, 5] and got.position.tolist() == [[1, 2, 3], [-1, -1, 0], [-1, 4, -1]]
    far = ops.expert_order(torch.tensor([[-big - 1], [big], [5]], device=dev), 3, first_expert=big - 1)
    assert far.starts.tolist() == [0, 0, 1, 1] and far.position.flatten().tolist() == [-1, 0, -1]
    low = ops.expert_order(torch.tensor([[-big - 1], [big], [-big + 1]], device=dev), 3, first_expert=-big - 1)
    assert low.position.flatten().tolist() == [0, -1, 1]
    none = ops.expert_order(torch.empty(0, 8, dtype=torch.int64, device=dev), 5)
    assert none.starts.tolist() == [0] * 6 and none.position.shape == (0, 8)
    x = torch.empty(0, 16, dtype=torch.bfloat16, device=dev)
    assert ops.sort_tokens(x, none).shape == (0, 16) and ops.combine_tokens(x, none).shape == (0, 16)
    dy, dw = ops.combine_tokens_grad(x, x, none, torch.empty(0, 8, device=dev))
    assert dy.shape == (0, 16) and dw.shape == (0, 8)


CASES = [  # rows, hidden, topk, experts, first, n
    (1, 7168, 8, 256, 0, 256), (1, 1, 1, 4, 0, 4), (5, 1001, 3, 8, 0, 8), (40, 640, 3, 40, 11, 13), (129, 520, 9, 24, 0, 24),
    (33, 4100, 32, 64, 5, 40), (300, 63, 6, 384, 0, 384)]


def unit(dtype):
    return torch.finfo(dtype).eps / 2


@pytest.mark.parametrize("dtype", TYPES)
@pytest.mark.parametrize("rows,hidden,topk,experts,first,n", CASES)
@pytest.mark.parametrize("strided", [False, True])
def test_rows_and_gradients(dev, dtype, rows, hidden, topk, experts, first, n, strided):
    sel = routes(rows, topk, experts, 3 * rows + hidden, padded=rows > 4)
    order = ops.expert_order(sel.to(dev), n, first_expert=first)
    position = order.position.cpu().long()
    g = torch.Generator().manual_seed(hidden)

    def make(r, c=hidden):
        t = torch.randn(r, c + (3 if strided else 0), generator=g).to(dtype)
        return t.to(dev)[:, 1:c + 1] if strided else t.to(dev)

    x, gs = make(rows).requires_grad_(), make(rows * topk)
    xs = ops.sort_tokens(x, order)
    dx, = torch.autograd.grad(xs, x, gs)
    here = position >= 0
    x64, gs64 = x.detach().cpu().double(), gs.cpu().double()
    want = torch.zeros(rows * topk, hidden, dtype=torch.float64)
    t, k = here.nonzero(as_tuple=True)
    want[position[t, k]] = x64[t]
    assert torch.equal(xs.detach().cpu().double(), want)                      # copies, and zeros behind the last
    sums, sizes = torch.zeros_like(x64), torch.zeros_like(x64)
    sums.index_add_(0, t, gs64[position[t, k]])
    sizes.index_add_(0, t, gs64[position[t, k]].abs())
    # topk fp32 additions and one rounding
    assert ((dx.cpu().double() - sums).abs() <= topk * 2.0 ** -24 * sizes * 1.01 + unit(dtype) * sums.abs() * 1.01 + 1e-8).all()

    y, gr, res = make(rows * topk).requires_grad_(), make(rows), make(rows).requires_grad_()
    w = torch.rand(rows, topk, generator=g).to(dev).requires_grad_()
    out = ops.combine_tokens(y, order, w, residual=res)
    dy, dw, dres = torch.autograd.grad(out, (y, w, res), gr)
    y64, w64, gr64 = y.detach().cpu().double(), w.detach().cpu().double(), gr.cpu().double()
    sums, sizes = res.detach().cpu().double(), res.detach().cpu().double().abs()
    sums.index_add_(0, t, w64[t, k, None] * y64[position[t, k]])
    sizes.index_add_(0, t, (w64[t, k, None] * y64[position[t, k]]).abs())
    assert ((out.detach().cpu().double() - sums).abs() <= (topk + 1) * 2.0 ** -24 * sizes * 1.01 + unit(dtype) * sums.abs() * 1.01 + 1e-8).all()
    assert torch.equal(dres, gr)
    want = torch.zeros(rows * topk, hidden, dtype=torch.float64)
    want[position[t, k]] = w64[t, k, None] * gr64[t]
    # a product in fp32, then one rounding; fp16 below its normal numbers: half of 2^-24
    assert ((dy.cpu().double() - want).abs() <= (2.0 ** -24 + unit(dtype)) * 1.01 * want.abs() + 2.0 ** -25).all()
    assert not dy[int(order.starts[-1]):].any()
    dots, sizes = torch.zeros(rows, topk, dtype=torch.float64), torch.zeros(rows, topk, dtype=torch.float64)
    dots[t, k] = (gr64[t] * y64[position[t, k]]).sum(1)
    sizes[t, k] = (gr64[t] * y64[position[t, k]]).abs().sum(1)
    # a lane adds hidden / 256 or more values, then six levels
    assert dw.dtype == torch.float32 and ((dw.cpu().double() - dots).abs() <= (hidden / 128 + 16) * 2.0 ** -24 * sizes + 1e-12).all()
    plain = ops.combine_tokens(y.detach(), order)                             # without weights: the sorted rows' gradient's own sums
    assert torch.equal(plain, ops.sort_tokens_grad(y.detach(), order))


def test_fewer_rows_than_slots(dev):
    """Sorted rows cut to those that there are, and to fewer: the others add nothing, and have no gradient."""
    sel = torch.tensor([[0, 5], [1, 0], [7, 1]], device=dev)
    order = ops.expert_order(sel, 2)                                          # 4 rows of 6 slots
    y = torch.arange(1.0, 13.0, device=dev).view(4, 3).requires_grad_()
    out = ops.combine_tokens(y, order)
    assert out.tolist() == [[1, 2, 3], [11, 13, 15], [10, 11, 12]]
    dy, = torch.autograd.grad(out, y, torch.ones_like(out))
    assert dy.tolist() == [[1.0] * 3] * 4
    w = torch.full((3, 2), 2.0, device=dev, requires_grad=True)
    short = y.detach()[:3].requires_grad_()
    out = ops.combine_tokens(short, order, w)
    assert out.tolist() == [[2, 4, 6], [22, 26, 30], [0, 0, 0]]
    dy, dw = torch.autograd.grad(out, (short, w), torch.ones_like(out))
    assert dy.tolist() == [[2.0] * 3] * 3 and dw.tolist() == [[6, 0], [24, 15], [0, 0]]


def test_infinities_and_nan_stay_in_their_rows(dev):
    sel = torch.tensor([[0, 1], [1, 9], [2, 9]], device=dev)
    order = ops.expert_order(sel, 3)
    y = torch.ones(6, 8, dtype=torch.bfloat16, device=dev)
    y[int(order.position[2, 0])] = float("nan")
    y[4:] = float("inf")                                                      # rows of no slot
    w = torch.full((3, 2), 0.5, device=dev)
    w[:, 1][1:] = float("nan")                                                # weights of slots without a row
    out = ops.combine_tokens(y, order, w)
    assert out[0].eq(1).all() and out[1].eq(0.5).all() and out[2].isnan().all()
    dy, dw = ops.combine_tokens_grad(torch.ones(3, 8, dtype=torch.bfloat16, device=dev), y, order, w)
    assert dy[:4].eq(0.5).all() and dy[4:].eq(0).all() and dw[0].tolist() == [8, 8] and dw[1].tolist() == [8, 0] and dw[2, 0].isnan()


def test_garbage_in_an_order_stays_in_bounds(dev):
    """Positions and starts of any content: rows outside of the tensors are neither read nor written."""
    position = torch.tensor([[0, 2 ** 31 - 1], [-7, 3], [4, 100]], dtype=torch.int32, device=dev)
    for last in (-5, 0, 3, 2 ** 31 - 1):
        order = ops.ExpertOrder(torch.tensor([0, last], dtype=torch.int32, device=dev), position)
        x = torch.ones(3, 40, device=dev)
        assert ops.sort_tokens(x, order).shape == (6, 40)
        assert ops.combine_tokens(torch.ones(6, 40, device=dev), order, torch.ones(3, 2, device=dev)).isfinite().all()
        dy, dw = ops.combine_tokens_grad(x, torch.ones(6, 40, device=dev), order, torch.ones(3, 2, device=dev))
        assert dw.tolist() == [[40, 0], [0, 40], [40, 0]]


def test_results_repeat_on_other_streams_and_in_graphs(dev):
    sel = routes(600, 8, 64, 5).to(dev)
    x = torch.randn(600, 1032, generator=torch.Generator().manual_seed(1)).bfloat16().to(dev)
    w = torch.rand(600, 8, generator=torch.Generator().manual_seed(2)).to(dev)

    def run():
        order = ops.expert_order(sel, 40, first_expert=10)
        xs = ops.sort_tokens(x, order)
        out = ops.combine_tokens(xs, order, w, residual=x)
        return [*order, xs, out, *ops.combine_tokens_grad(x, xs, order, w), ops.sort_tokens_grad(xs, order)]

    first = run()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        again = run()
    torch.cuda.current_stream().wait_stream(side)
    assert all(torch.equal(a, b) for a, b in zip(first, again))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for k in range(3):
        x.copy_(torch.randn(600, 1032, generator=torch.Generator().manual_seed(10 + k)).bfloat16())
        sel.copy_(routes(600, 8, 64, 20 + k))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, run())), k


def test_refusals(dev, monkeypatch):
    sel = routes(4, 2, 8, 1).to(dev)
    order = ops.expert_order(sel, 8)
    x, y, w = torch.ones(4, 16, device=dev), torch.ones(8, 16, device=dev), torch.ones(4, 2, device=dev)
    for bad in (lambda: ops.expert_order(sel.int(), 8), lambda: ops.expert_order(sel.cpu(), 8), lambda: ops.expert_order(sel, 0),
                lambda: ops.expert_order(sel, 1025), lambda: ops.expert_order(sel[:, :1], 8),
                lambda: ops.expert_order(torch.zeros(2, 33, dtype=torch.int64, device=dev), 8),
                lambda: ops.sort_tokens(x[:3], order), lambda: ops.sort_tokens(x.double(), order), lambda: ops.sort_tokens(x.t(), order),
                lambda: ops.sort_tokens(x.cpu(), order), lambda: ops.sort_tokens(x, ops.ExpertOrder(order.starts.long(), order.position)),
                lambda: ops.combine_tokens(y, order, w.double()), lambda: ops.combine_tokens(y, order, w[:, :1]),
                lambda: ops.combine_tokens(y, order, w, residual=x.half()), lambda: ops.combine_tokens(y, order, w, residual=y),
                lambda: ops.combine_tokens_grad(x[:2], y, order, w), lambda: ops.combine_tokens_grad(x.half(), y, order, w)):
        with pytest.raises(ValueError):
            bad()
    x.requires_grad_()
    xs = ops.sort_tokens(x, order)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(xs.sum(), x, create_graph=True)
    out = ops.combine_tokens(xs, order, w)
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(out.sum(), x, create_graph=True, retain_graph=True)
    with monkeypatch.context() as m:                      # told that the stream is capturing: nothing is captured here
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        for call in (lambda: ops.sort_tokens(x, order), lambda: ops.combine_tokens(xs, order, w),
                     lambda: torch.autograd.grad(out.sum(), x, retain_graph=True)):
            with pytest.raises(RuntimeError, match="captured"):
                call()
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        dual = fwd.make_dual(x.detach(), torch.ones_like(x))
        with pytest.raises(ValueError, match="forward-mode"):
            ops.sort_tokens(dual, order)


def test_the_most_slots(dev):
    """2^26 slots, more tokens than a launch has workgroups for: copies are exact, and so are sums of one row."""
    rows, hidden, n = 1 << 26, 5, 7
    sel = (torch.arange(rows, device=dev) * 5 + 3).remainder_(n + 1).view(rows, 1) - 1        # 0..n - 1, and -1 in every eighth
    x = torch.arange(rows, device=dev).view(rows, 1).bitwise_and(2047).half().expand(rows, hidden).contiguous()
    order = ops.expert_order(sel, n)
    assert order.starts[-1] == (sel >= 0).sum()
    xs = ops.sort_tokens(x, order)
    at = order.position.view(-1).long()
    here = at >= 0
    assert torch.equal(xs[at[here]], x[here]) and not xs[order.starts[-1]:].any()
    weights = torch.full((rows, 1), 0.5, device=dev)
    out = ops.combine_tokens(xs, order, weights)
    assert torch.equal(out, x * 0.5 * here.view(-1, 1))
    dy, dw = ops.combine_tokens_grad(x, xs, order, weights)
    assert torch.equal(dy, xs * 0.5)
    want = (x[:, :1].float() ** 2 * here.view(-1, 1)) * hidden                                # whole numbers below 2^24.4, the last bits a rounding
    assert ((dw - want).abs() <= 2.0 ** -22 * want).all()


def test_a_gradient_of_other_rows_is_refused(dev):
    order = ops.expert_order(routes(4, 2, 8, 1).to(dev), 8)
    for rows in (7, 9):
        with pytest.raises(ValueError, match="slots"):
            ops.sort_tokens_grad(torch.ones(rows, 16, device=dev), order)
