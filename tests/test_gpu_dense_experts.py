"""The modules on 16-bit weights: a layer's operators together, forward and backward, captured, on other streams; what the operators
refuse; addresses past 32 bits."""
import pytest
import torch

from eva_amd import ops
from eva_amd.dense import DenseExperts, DenseLinear

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def layer(seed, rows, hidden, inter, experts, topk, dtype, dev):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(rows, hidden, generator=g).to(dtype).to(dev)
    gate_up = torch.randn(experts, 2 * inter, hidden, generator=g).mul_(1.5 * hidden ** -0.5).to(dtype).to(dev)
    down = torch.randn(experts, hidden, inter, generator=g).mul_(1.5 * inter ** -0.5).to(dtype).to(dev)
    z = torch.randn(rows, 2 * experts, generator=g).to(dev)
    sel, weights, _ = ops.route_topk(z, topk, "sigmoid")            # the layer holds half of the router's experts
    return x, gate_up, down, sel, weights


@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("rows,hidden,inter,experts,topk", [(1, 256, 128, 4, 2), (5, 1000, 333, 12, 5), (90, 640, 384, 20, 3), (700, 328, 200, 6, 4)])
def test_a_layer(dev, dtype, rows, hidden, inter, experts, topk):
    """Outputs and all gradients against 64 bits. The tolerance follows the roundings (to 16 bits: hidden activations, experts'
    results, the output; backwards the slots' gradients, those of hidden activations, D, the sorted rows', the tokens') through the
    sizes of what they are multiplied with, and counts fp32 sums of n values as n / 2 + 64 units."""
    x, gate_up, down, sel, weights = layer(rows, rows, hidden, inter, experts, topk, dtype, dev)
    first, u, v = experts // 2, torch.finfo(dtype).eps / 2, 2.0 ** -24
    tiny = 2.0 ** -24 if dtype == FP16 else 0.0                     # half of fp16's smallest number, with room
    leaves = [t.detach().requires_grad_() for t in (x, gate_up, down, weights)]
    g = torch.randn(rows, hidden, generator=torch.Generator().manual_seed(1)).to(dtype).to(dev)
    out = DenseExperts(leaves[1], leaves[2], first_expert=first)(leaves[0], sel, leaves[3])
    grads = torch.autograd.grad(out, leaves, g)
    x64, w1, w2, wt, g64, sel = (t.cpu().double() if t.is_floating_point() else t.cpu() for t in (x, gate_up, down, weights, g, sel))
    want = [torch.zeros_like(t) for t in (x64, x64, w1, w2, wt)]     # out, dx, dgate_up, ddown, dweights
    tol = [torch.zeros_like(t) for t in want]

    def n(k):
        return (k / 2 + 64) * v

    for e in range(experts):
        t, k = (sel == first + e).nonzero(as_tuple=True)
        if not t.numel():
            continue
        xe, we, ge = x64[t], wt[t, k][:, None], g64[t]
        pre, pre_off = xe @ w1[e].t(), n(hidden) * (xe.abs() @ w1[e].abs().t())
        gate, up = pre.chunk(2, 1)
        go, uo = pre_off.chunk(2, 1)
        s = torch.sigmoid(gate)
        h, slope = gate * s * up, s * (1 + gate * (1 - s))
        h_off = 1.13 * go * (up.abs() + uo) + (gate.abs() + go) * uo + 16 * v * gate.abs() * up.abs()
        h_off = h_off + u * (h.abs() + h_off) + tiny
        y, y_off = h @ w2[e].t(), n(inter) * (h.abs() @ w2[e].abs().t()) + h_off @ w2[e].abs().t()
        y_off = y_off + u * (y.abs() + y_off) + tiny
        want[0].index_add_(0, t, we * y)
        tol[0].index_add_(0, t, we * (y_off + topk * v * (y.abs() + y_off)))
        want[4][t, k] = (ge * y).sum(1)
        tol[4][t, k] = (ge.abs() * (y_off + n(hidden) * (y.abs() + y_off))).sum(1)
        dy = we * ge
        dy_off = (u + v) * dy.abs() + tiny
        dh, dh_off = dy @ w2[e], n(hidden) * ((dy.abs() + dy_off) @ w2[e].abs()) + dy_off @ w2[e].abs()
        dh_off = dh_off + u * (dh.abs() + dh_off) + tiny
        want[3][e] = dy.t() @ h
        off = (dy.abs() + dy_off).t() @ h_off + dy_off.t() @ h.abs() + n(t.numel()) * ((dy.abs() + dy_off).t() @ (h.abs() + h_off))
        tol[3][e] = off + u * (want[3][e].abs() + off) + tiny
        d = torch.cat((dh * up * slope, dh * gate * s), 1)
        far = dh.abs() + dh_off
        d_off = torch.cat((dh_off * 1.13 * up.abs() + far * (1.2 * go * (up.abs() + uo) + 1.13 * uo),
                           dh_off * gate.abs() + far * 1.13 * go), 1)
        d_off += 32 * v * torch.cat((far * up.abs() * 1.13, far * gate.abs()), 1)
        d_off = d_off + u * (d.abs() + d_off) + tiny
        want[2][e] = d.t() @ xe
        off = d_off.t() @ xe.abs() + n(t.numel()) * ((d.abs() + d_off).t() @ xe.abs())
        tol[2][e] = off + u * (want[2][e].abs() + off) + tiny
        dx = d @ w1[e]
        off = d_off @ w1[e].abs() + n(2 * inter) * ((d.abs() + d_off) @ w1[e].abs())
        off = off + u * (dx.abs() + off) + tiny
        want[1].index_add_(0, t, dx)
        tol[1].index_add_(0, t, off + topk * v * (dx.abs() + off))
    for i in (0, 1):
        tol[i] += u * (want[i].abs() + tol[i]) + tiny
    for name, got, ref, off in zip(("out", "dx", "dgate_up", "ddown", "dweights"), (out.detach(), *grads), want, tol):
        diff = (got.cpu().double() - ref).abs()
        assert (diff <= off).all(), (name, float((diff / off.clamp(min=1e-300)).max()))


def test_leading_dimensions_and_residuals(dev):
    g = torch.Generator().manual_seed(3)
    x = torch.randn(2, 3, 5, 64, generator=g).bfloat16().to(dev)
    w, b = torch.randn(96, 64, generator=g).bfloat16().to(dev), torch.randn(96, generator=g).bfloat16().to(dev)
    residual = torch.randn(2, 3, 5, 48, generator=g).bfloat16().to(dev)
    lin = DenseLinear(w, b, activation="swiglu", limit=2.0)
    y = lin(x, residual)
    assert torch.equal(y.view(30, 48), ops.linear(x.view(30, 64), w, b, activation="swiglu", limit=2.0, residual=residual.view(30, 48)))
    flipped = x.transpose(0, 2)
    assert torch.equal(lin(flipped), lin(flipped.contiguous()))
    held = residual.view(30, 48).clone()                              # the residual's own buffer, through the C entry point's terms
    assert lin(x[:0]).shape == (0, 3, 5, 48) and lin.out_features == 48 and torch.equal(held, residual.view(30, 48))
    x, gate_up, down, sel, weights = layer(8, 12, 64, 32, 6, 2, BF16, dev)
    experts = DenseExperts(gate_up, down, first_expert=2)
    plain, added = experts(x, sel, weights), experts(x.view(3, 4, 64), sel.view(3, 4, 2), weights.view(3, 4, 2), residual=x.view(3, 4, 64))
    away = (added.view(12, 64).double() - plain.double() - x.double()).abs()
    # the sum before its rounding against the one after: a step of each of the two roundings
    assert (away <= 2.0 ** -8 * (plain.double().abs() + added.view(12, 64).double().abs()) * 1.01).all()
    assert experts(x[:0], sel[:0], weights[:0]).shape == (0, 64)
    for bad in (lambda: lin(x[:, :32]), lambda: lin(torch.zeros(4, 64, device=dev).bfloat16(), x[:4]), lambda: DenseLinear(w, b[:5]),
                lambda: DenseExperts(gate_up[:, 1:], down), lambda: DenseExperts(gate_up, down[:, :, 1:]), lambda: experts(x[:, :8], sel, weights),
                lambda: experts(x, sel, weights, residual=x[:4])):
        with pytest.raises(ValueError):
            bad()


def test_no_rows_have_gradients_of_zero(dev):
    x, w, b = (torch.randn(*s, device=dev, dtype=BF16, requires_grad=True) for s in ((0, 40), (3, 24, 40), (3, 24)))
    starts = torch.zeros(4, dtype=torch.int32, device=dev)
    for act in (None, "swiglu"):
        y = ops.expert_linear(x, w, starts, b, activation=act)
        dx, dw, db = torch.autograd.grad(y, (x, w, b), torch.ones_like(y))
        assert dx.shape == (0, 40) and not dw.any() and not db.any() and dw.shape == w.shape and db.shape == b.shape


@pytest.mark.parametrize("rows", [3, 40, 600])
def test_captured_and_on_other_streams(dev, rows):
    """The layer's forward pass and its gradients through the functions for a capture, replayed with other inputs, and two calls at
    once on two streams."""
    x, gate_up, down, sel, weights = layer(rows, rows, 328, 136, 10, 4, BF16, dev)
    grad = torch.randn(rows, 328, generator=torch.Generator().manual_seed(2)).bfloat16().to(dev)

    def run():
        with torch.no_grad():
            order = ops.expert_order(sel, 10, first_expert=4)
            xs = ops.sort_tokens(x, order)
            h, pre = ops.expert_linear(xs, gate_up, order.starts, activation="swiglu", limit=1.0, return_pre=True)
            y = ops.expert_linear(h, down, order.starts)
            out = ops.combine_tokens(y, order, weights, residual=x)
            dy, dweights = ops.combine_tokens_grad(grad, y, order, weights)
            dh, ddown, _ = ops.expert_linear_grad(dy, h, down, order.starts)
            dxs, dgate_up, db = ops.expert_linear_grad(dh, xs, gate_up, order.starts, pre, activation="swiglu", limit=1.0)
            lin, lin_pre = ops.linear(x, gate_up[0], activation="gelu", return_pre=True)
            return [out, dweights, ddown, dgate_up, db, ops.sort_tokens_grad(dxs, order), lin,
                    *ops.linear_grad(lin, x, gate_up[0], lin_pre, activation="gelu")]

    first = run()
    leaves = [t.detach().requires_grad_() for t in (x, gate_up, down, weights)]
    eager = DenseExperts(leaves[1], leaves[2], first_expert=4)(leaves[0], sel, leaves[3], limit=1.0, residual=leaves[0])
    dx, dgate_up, ddown, dweights = torch.autograd.grad(eager, leaves, grad)
    assert torch.equal(eager.detach(), first[0]) and torch.equal(dweights, first[1]) and torch.equal(ddown, first[2])
    assert torch.equal(dgate_up, first[3]) and torch.equal(dx, first[5] + grad)
    streams, both = [torch.cuda.Stream(), torch.cuda.Stream()], []
    for s in streams:
        s.wait_stream(torch.cuda.current_stream())
    for s in streams:
        with torch.cuda.stream(s):
            both.append(run())
    for s in streams:
        torch.cuda.current_stream().wait_stream(s)
    assert all(torch.equal(a, b) for got in both for a, b in zip(first, got))
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        held = run()
    for k in range(3):
        g = torch.Generator().manual_seed(50 + k)
        x.copy_(torch.randn(rows, 328, generator=g).bfloat16())
        sel.copy_(torch.randint(0, 20, sel.shape, generator=g))
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(held, run())), k


def test_any_starts_stay_in_bounds(dev):
    """Tables that fall, are negative or pass the rows: rows of none of the experts, or of some, but no access outside."""
    x, w = torch.ones(300, 64, dtype=BF16, device=dev), torch.ones(3, 48, 64, dtype=BF16, device=dev)
    for rows in (8, 300):
        for table in ([0, -5, 7, 3], [0, 2 ** 31 - 1, 0, 2 ** 31 - 1], [-2 ** 31, 5, 5, 4], [250, 260, 280, 299]):
            starts = torch.tensor(table, dtype=torch.int32, device=dev)
            y = ops.expert_linear(x[:rows], w, starts)
            dx, dw, db = ops.expert_linear_grad(y, x[:rows], w, starts)
            assert y.shape == (rows, 48) and dx.shape == (rows, 64) and dw.shape == w.shape and db.shape == (3, 48)
            torch.cuda.synchronize()


def test_infinities_and_nan(dev):
    """They stay in their rows and columns; a clamp passes a NaN on; rows behind the last are not looked at."""
    x = torch.ones(40, 72, dtype=BF16, device=dev)
    w = torch.full((2, 32, 72), 0.125, dtype=BF16, device=dev)
    x[3], x[7, 5] = float("nan"), float("inf")
    x[30:] = float("nan")
    starts = torch.tensor([0, 10, 30], dtype=torch.int32, device=dev)
    y = ops.expert_linear(x, w, starts, activation="swiglu", limit=2.0)
    assert y[3].isnan().all() and y[7].eq(4).all() and not y[30:].any()
    rest = torch.cat((y[:3], y[4:7], y[8:30]))
    assert rest.eq(rest[0, 0]).all() and rest.isfinite().all()
    for act, want in (("silu", float("inf")), ("gelu", float("inf")), ("relu", float("inf"))):
        z = ops.expert_linear(x, w, starts, activation=act)
        assert z[7].eq(want).all() and z[3].isnan().all() and not z[30:].any()
    w[1, 4] = float("nan")
    y = ops.expert_linear(x, w, starts)
    assert y[:3].isfinite().all() and y[10:30, 4].isnan().all() and y[10:30, :4].isfinite().all()
    grad = torch.ones(40, 32, dtype=BF16, device=dev)
    grad[12] = float("nan")
    w[1, 4] = 0.125
    dx, dw, db = ops.expert_linear_grad(grad, x, w, starts)
    assert dx[12].isnan().all() and dx[:12].isfinite().all() and dx[13:30].isfinite().all() and not dx[30:].any()
    assert dw[1].isnan().all() and db[1].isnan().all() and db[0].eq(10).all()


def test_refusals(dev, monkeypatch):
    x, w, b = (torch.ones(*s, dtype=BF16, device=dev) for s in ((6, 64), (32, 64), (32,)))
    starts, stack = torch.tensor([0, 6], dtype=torch.int32, device=dev), w[None]
    y, pre = ops.linear(x, w, b, activation="silu", return_pre=True)
    assert ops.linear(x, w, return_pre=True)[1] is None
    for bad in (lambda: ops.linear(x.float(), w.float()), lambda: ops.linear(x, w.half()), lambda: ops.linear(x, w.t()), lambda: ops.linear(x, w[:, :32]),
                lambda: ops.linear(x.cpu(), w), lambda: ops.linear(x, w.cpu()), lambda: ops.linear(x, stack), lambda: ops.linear(x, w, b[:5]),
                lambda: ops.linear(x, w, b.float()), lambda: ops.linear(x, w, activation="tanh"), lambda: ops.linear(x, w, limit=1.0),
                lambda: ops.linear(x, w, activation="swiglu", limit=-1.0), lambda: ops.linear(x, w[:31], activation="swiglu"),
                lambda: ops.linear(x, w, residual=x), lambda: ops.linear(x, w, residual=y[:2]), lambda: ops.linear(x.t(), w),
                lambda: ops.linear(x.expand(2, 6, 64), w), lambda: ops.linear(x[:1].expand(6, 64), w),
                lambda: ops.expert_linear(x, w, starts), lambda: ops.expert_linear(x, stack, starts.long()),
                lambda: ops.expert_linear(x, stack, starts[:1]), lambda: ops.expert_linear(x, stack, None),
                lambda: ops.expert_linear(x, w[None].expand(2, 32, 64), torch.zeros(3, dtype=torch.int32, device=dev)),
                lambda: ops.expert_linear(x, stack, starts, b), lambda: ops.linear_grad(y, x, w, activation="silu"),
                lambda: ops.linear_grad(y, x, w, pre[:3], activation="silu"), lambda: ops.linear_grad(y[:3], x, w, pre, activation="silu"),
                lambda: ops.linear_grad(y.half(), x, w), lambda: ops.expert_linear_grad(y, x, w, starts)):
        with pytest.raises(ValueError):
            bad()
    w.requires_grad_()
    y = ops.linear(x, w, b, activation="silu")
    with pytest.raises(RuntimeError, match="once"):
        torch.autograd.grad(y.sum(), w, create_graph=True, retain_graph=True)
    with monkeypatch.context() as m:                      # told that the stream is capturing: nothing is captured here
        m.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
        for call in (lambda: ops.linear(x, w), lambda: ops.expert_linear(x, w[None], starts), lambda: torch.autograd.grad(y.sum(), w, retain_graph=True)):
            with pytest.raises(RuntimeError, match="captured"):
                call()
    dw, = torch.autograd.grad(y.sum(), w)                 # an expanded gradient
    assert dw.isfinite().all() and dw.eq(dw[0]).all()
    import torch.autograd.forward_ad as fwd
    with fwd.dual_level():
        with pytest.raises(ValueError, match="forward-mode"):
            ops.linear(fwd.make_dual(x, torch.ones_like(x)), w.detach())


def test_only_the_wanted_gradients(dev):
    """A frozen matrix, frozen inputs, a bias alone: what is asked for has the same bits."""
    g = torch.Generator().manual_seed(4)
    x, w, b, gr = (torch.randn(*s, generator=g).half().to(dev) for s in ((70, 96), (40, 96), (40,), (70, 40)))
    every = ops.linear_grad(gr, x, w)
    for wanted in ((0,), (1,), (2,), (0, 2), (1, 2)):
        leaves = [t.detach().requires_grad_(i in wanted) for i, t in enumerate((x, w, b))]
        got = torch.autograd.grad(ops.linear(*leaves), [leaves[i] for i in wanted], gr)
        assert all(torch.equal(a, every[i]) for a, i in zip(got, wanted))


def test_past_32_bits(dev):
    """Sorted rows, weights and results whose byte and value offsets pass 2^32 and 2^31: the last rows against the first ones' arithmetic."""
    rows, topk, hidden = 42000, 8, 7168                                       # 336000 sorted rows: 4.8 GB, 2.4e9 values
    sel = torch.zeros(rows, topk, dtype=torch.int64, device=dev)
    sel[:] = torch.arange(topk, device=dev)
    x = torch.randn(rows, hidden, device=dev, dtype=BF16)
    order = ops.expert_order(sel, topk)
    xs = ops.sort_tokens(x, order)
    assert torch.equal(xs[-rows:], x) and torch.equal(xs[:rows], x)
    back = ops.combine_tokens(xs, order, torch.full((rows, topk), 0.125, device=dev))
    assert torch.equal(back, x)                                               # eight exact eighths
    w = torch.randn(topk, 64, hidden, device=dev, dtype=BF16) * 0.01
    y = ops.expert_linear(xs, w, order.starts)
    part = ops.linear(x[-300:], w[-1])
    # the same products, summed in another order: fp32 sums of 7168 values, then a rounding of 2^-8
    size = x[-300:].float().abs() @ w[-1].float().abs().t()
    assert ((y[-300:].float() - part.float()).abs() <= 2 * (7168 / 2 + 64) * 2.0 ** -24 * size + 2.0 ** -7 * part.float().abs()).all()
    dx, dw, _ = ops.expert_linear_grad(y, xs, w, order.starts)
    last = ops.linear_grad(y[-rows:], x, w[-1])
    # each sum in fp32 in another order (dx: 64 products, dw: 42000), then a rounding
    size = y[-300:].float().abs() @ w[-1].float().abs()
    assert ((dx[-300:].float() - last[0][-300:].float()).abs() <= 2 * 96 * 2.0 ** -24 * size + 2.0 ** -7 * last[0][-300:].float().abs()).all()
    size = y[-rows:].float().abs().t() @ x.float().abs()
    assert ((dw[-1].float() - last[1].float()).abs() <= 2 * (42000 / 2 + 64) * 2.0 ** -24 * size + 2.0 ** -7 * last[1].float().abs()).all()
    del xs, y, dx, dw, back
    big = torch.randn(5, 70000, 8192, device=dev, dtype=BF16)                # 5.7 GB of weights, 2.9e9 values
    rows = torch.randn(10, 8192, device=dev, dtype=BF16)
    for count in (2, 30):                                                     # few rows, and tiles
        xs = rows[:2].repeat(5 * count // 2, 1)
        starts = torch.arange(6, device=dev, dtype=torch.int32) * count
        y = ops.expert_linear(xs, big, starts)
        part = ops.linear(rows[:2], big[4])
        size = rows[:2].float().abs() @ big[4].float().abs().t()
        assert ((y[-2:].float() - part.float()).abs() <= 2 * (8192 / 2 + 64) * 2.0 ** -24 * size + 2.0 ** -7 * part.float().abs()).all()


def test_long_copies(dev):
    """Weights of odd rows, 17 GB, which are copied first: the last expert's against a product of its matrix alone."""
    experts, n_out, n_in = 1024, 8256, 1001
    w = torch.randn(experts, n_out, n_in, device=dev, dtype=BF16)
    x = torch.randn(5 * experts, n_in, device=dev, dtype=BF16)
    y = ops.expert_linear(x, w, torch.arange(experts + 1, device=dev, dtype=torch.int32) * 5)
    for e in (0, 511, 1023):
        part = ops.linear(x[5 * e:5 * e + 5], w[e])
        size = x[5 * e:5 * e + 5].float().abs() @ w[e].float().abs().t()
        # fp32 sums of 1001 values in another order, then a rounding of 2^-8 each
        assert ((y[5 * e:5 * e + 5].float() - part.float()).abs() <= 2 * (1001 / 2 + 64) * 2.0 ** -24 * size + 2.0 ** -7 * part.float().abs()).all()


def test_rows_far_apart(dev):
    """Row strides above 2^21 values: copied."""
    stride = (1 << 21) + 8
    flat = torch.randn(80 * stride, device=dev, dtype=BF16)
    x, w = flat.view(80, stride)[:, :64], flat.view(80, stride)[:40, 128:192]
    assert torch.equal(ops.linear(x, w), ops.linear(x.contiguous(), w.contiguous()))
    gr = flat.view(80, stride)[:, 256:296]
    for a, b in zip(ops.linear_grad(gr, x, w), ops.linear_grad(gr.contiguous(), x.contiguous(), w.contiguous())):
        assert torch.equal(a, b)


def test_routes_of_no_indices_are_refused(dev):
    layer = DenseExperts(torch.zeros(4, 16, 8, dtype=BF16, device=dev), torch.zeros(4, 8, 8, dtype=BF16, device=dev))
    x, weights = torch.ones(3, 8, dtype=BF16, device=dev), torch.ones(3, 2, device=dev)
    for dtype in (torch.float32, torch.bool):
        with pytest.raises(ValueError, match="indices"):
            layer(x, torch.ones(3, 2, device=dev).to(dtype), weights)
    assert layer(x, torch.ones(3, 2, dtype=torch.int32, device=dev), weights).shape == x.shape


@pytest.mark.parametrize("act", [None, "swiglu"])
def test_few_rows_beside_many(dev, act):
    """Weights of more than the caches hold, with experts of 0 to some hundred rows: each against a product of its matrix alone."""
    counts = [0, 1, 16, 17, 3, 0, 130, 15, 64, 18, 2, 300]
    n_out, n_in, tail = 4096, 4104, 20
    starts = torch.tensor([0] + counts, dtype=torch.int32).cumsum(0).to(torch.int32).to(dev)
    g = torch.Generator(device=dev).manual_seed(6)
    x, w = (torch.randn(*s, generator=g, device=dev, dtype=BF16) for s in ((sum(counts) + tail, n_in), (len(counts), n_out, n_in)))
    bias = torch.randn(len(counts), n_out, generator=g, device=dev, dtype=BF16)
    w *= n_in ** -0.5
    assert w.numel() * 2 > 256 << 20 and sum(counts) + tail <= 64 * len(counts)
    y, pre = ops.expert_linear(x, w, starts, bias, activation=act, return_pre=True)
    assert not y[sum(counts):].any()
    for e, n in enumerate(counts):
        if n:
            rows = slice(int(starts[e]), int(starts[e]) + n)
            part, z = ops.linear(x[rows], w[e], bias[e], activation=act, return_pre=True)
            # fp32 sums of 4104 values in another order; then an activation whose slope is below 1.1 a factor, and a rounding of 2^-8 each
            size = x[rows].float().abs() @ w[e].float().abs().t() + bias[e].float().abs()
            near = 2 * (4104 / 2 + 64) * 2.0 ** -24 * size
            if act is None:
                assert pre is None and ((y[rows].float() - part.float()).abs() <= near + 2.0 ** -7 * part.float().abs()).all()
                continue
            assert ((pre[rows] - z).abs() <= near).all()
            (ga, gu), (na, nu) = z.chunk(2, 1), near.chunk(2, 1)
            silu = torch.nn.functional.silu(ga)
            near = 1.1 * na * (gu.abs() + nu) + silu.abs() * nu + 2.0 ** -20 * silu.abs() * gu.abs()
            assert ((y[rows].float() - part.float()).abs() <= near + 2.0 ** -7 * part.float().abs()).all()


def test_few_rows_alone_beside_none(dev):
    """Two matrices of more than the caches hold and more rows than four for each, but none that has more than sixteen."""
    w = torch.randn(2, 8704, 8192, device=dev, dtype=BF16) * 0.01
    x = torch.randn(12, 8192, device=dev, dtype=BF16)
    y = ops.expert_linear(x, w, torch.tensor([0, 4, 9], dtype=torch.int32, device=dev))
    assert not y[9:].any()
    for e, rows in ((0, slice(0, 4)), (1, slice(4, 9))):
        part = ops.linear(x[rows], w[e])
        size = x[rows].float().abs() @ w[e].float().abs().t()
        # fp32 sums of 8192 values in another order, then a rounding of 2^-8 each
        assert ((y[rows].float() - part.float()).abs() <= 2 * (8192 / 2 + 64) * 2.0 ** -24 * size + 2.0 ** -7 * part.float().abs()).all()
