"""The MoE experts on 4-bit weights with group scales against their definition in 64 bits."""
import pytest
import torch

from eva_amd import ops
from tests.w4_helpers import Experts

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator().manual_seed(seed)


def _routes(g, rows, experts, topk, skew=False):
    z = torch.randn(rows, experts, generator=g)
    if skew:
        z[:, :2] += 6
    sel = z.topk(topk, 1).indices
    w = torch.sigmoid(z).gather(1, sel)
    return sel, w / w.sum(1, keepdim=True)


def _check(dev, ex, x, sel, w, limit=0.0, **kw):
    ref, tol = ex.reference(x, sel, w, limit=limit, dtype=x.dtype, **kw)
    y = ex.module(dev, **kw)(x.to(dev), sel.to(dev), w.to(dev), limit=limit)
    assert y.dtype == x.dtype and y.shape == x.shape
    off = (y.double().cpu() - ref).abs()
    assert (off <= tol).all(), float((off / tol).max())
    return y


CONFIGS = [  # hidden, inter, experts, topk, shared, group, zeros, dtype
    (128, 128, 4, 2, 0, 128, False, torch.bfloat16),
    (640, 384, 40, 3, 1, 64, True, torch.float16),
    (1000, 333, 24, 5, 2, 32, False, torch.bfloat16),
    (1024, 512, 16, 4, 0, 128, True, torch.bfloat16),
    (33, 17, 7, 7, 0, 32, True, torch.float16),
    (512, 256, 130, 8, 1, 128, False, torch.bfloat16),
]


@pytest.mark.parametrize("config", CONFIGS)
@pytest.mark.parametrize("rows", [1, 2, 3, 9, 16, 33, 100, 260])
def test_layer(dev, config, rows):
    hidden, inter, experts, topk, shared, group, zeros, dtype = config
    g = _gen(rows + hidden)
    ex = Experts(g, hidden, inter, experts + shared, group, zeros=zeros, dtype=dtype)
    x = (1.5 * torch.randn(rows, hidden, generator=g)).to(dtype)
    sel, w = _routes(g, rows, experts, topk, skew=rows % 2 == 0)
    _check(dev, ex, x, sel, w, n_shared=shared, limit=0.0 if rows % 3 else 0.5)


@pytest.mark.parametrize("inter", [700, 2100, 5000])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_one_token_of_wide_experts(dev, inter, dtype):
    """One token whose slots' hidden activations take little of the workgroup's LDS, most of it, or do not fit."""
    g = _gen(inter)
    ex = Experts(g, 192, inter, 11, 64, zeros=True, dtype=dtype)
    x = (1.5 * torch.randn(1, 192, generator=g)).to(dtype)
    sel, w = _routes(g, 1, 10, 9)
    _check(dev, ex, x, sel, w, n_shared=1, limit=3.0)


@pytest.mark.parametrize("rows", [1, 5, 16, 70, 200])
def test_a_rank_of_the_experts(dev, rows):
    """An expert range: slots of other experts add nothing, a token with none of them gets zeros whatever its
    weights hold, and an index may be anything."""
    g = _gen(rows)
    ex = Experts(g, 256, 192, 6, 64, zeros=True)
    x = torch.randn(rows, 256, generator=g).bfloat16()
    sel, w = _routes(g, rows, 30, 4)
    sel[0] = torch.tensor([0, 1, 29, 16])
    w[0] = float("nan")
    if rows > 2:
        sel[1] = torch.tensor([2 ** 40, -2 ** 40, -1, 2 ** 31])
    y = _check(dev, ex, x, sel, w, first_expert=10)
    assert (y[0] == 0).all()


@pytest.mark.parametrize("rows", [1, 6, 20, 90])
def test_repeated_experts_and_weights(dev, rows):
    """The same expert twice in a token, zero and negative weights, all tokens on one expert."""
    g = _gen(rows)
    ex = Experts(g, 320, 160, 5, 32)
    x = torch.randn(rows, 320, generator=g).bfloat16()
    sel = torch.randint(0, 5, (rows, 3), generator=g)
    sel[0] = 2
    w = torch.randn(rows, 3, generator=g)
    w[-1, 1] = 0
    _check(dev, ex, x, sel, w)
    _check(dev, ex, x, torch.full_like(sel, 4), w)


@pytest.mark.parametrize("rows", [1, 4, 24, 150])
def test_clamps(dev, rows):
    """Gates far past the limit on both sides, the routed expert clamped after SiLU and the shared one before; a
    group size and zero points of the down projection's own."""
    g = _gen(rows)
    ex = Experts(g, 256, 128, 5, 64, zeros=True, scale=0.05, down_group=32, down_zeros=False)
    x = (3 * torch.randn(rows, 256, generator=g)).bfloat16()
    sel, w = _routes(g, rows, 4, 2)
    _check(dev, ex, x, sel, w, n_shared=1, limit=1.5)
    _check(dev, ex, x, sel, w, n_shared=1, limit=0.0)


@pytest.mark.parametrize("rows", [1, 3, 40])
@pytest.mark.parametrize("scale", [2.0 ** -40, 2.0 ** 20])
def test_hidden_range(dev, rows, scale):
    """Hidden activations far outside fp16's range (no limit): their row's factor keeps them."""
    g = _gen(rows)
    ex = Experts(g, 256, 200, 4, 128, scale=0.02)
    x = (torch.randn(rows, 256, generator=g) * scale).bfloat16()
    sel, w = _routes(g, rows, 4, 2)
    _check(dev, ex, x, sel, w)


@pytest.mark.parametrize("rows", [2, 16, 60])
def test_inf_and_nan_stay_in_their_rows(dev, rows):
    g = _gen(rows)
    ex = Experts(g, 256, 128, 4, 64)
    m = ex.module(dev)
    x = torch.randn(rows, 256, generator=g).bfloat16()
    sel, w = _routes(g, rows, 4, 2)
    clean = m(x.to(dev), sel.to(dev), w.to(dev), limit=10.0)
    x[0, 3], x[-1, 7] = float("nan"), float("inf")
    y = m(x.to(dev), sel.to(dev), w.to(dev), limit=10.0)
    assert torch.equal(y[1:-1], clean[1:-1])
    assert y[0].isnan().all()


@pytest.mark.parametrize("rows", [1, 2, 9, 40])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_one_infinite_hidden_activation(dev, rows, dtype):
    """One hidden activation overflows fp32: the outputs are infinities of its weights' signs, not NaN."""
    g = _gen(rows)
    ex = Experts(g, 128, 256, 2, 128)
    for m in (ex.gate, ex.up):
        m.q[0, 17] = 15
        m.codes[0, 17] = 255
    ex.up.scales[0, 17] = 3e38
    ex.down.q[0, :, 17] = torch.randint(0, 2, (128,), generator=g, dtype=torch.uint8) * 15
    ex.down.codes[0, :, 8] = ex.down.q[0, :, 16] | ex.down.q[0, :, 17] << 4
    x = torch.ones(rows, 128, dtype=dtype)
    y = ex.module(dev)(x.to(dev), torch.zeros(rows, 1, dtype=torch.int64, device=dev), torch.ones(rows, 1, device=dev)).cpu()
    assert torch.equal(y.float(), torch.where(ex.down.q[0, :, 17] == 15, torch.inf, -torch.inf).expand(rows, 128))


def test_rows_do_not_depend_on_their_batch(dev):
    """Up to 16 rows a token's bits are those it has alone."""
    g = _gen(8)
    ex = Experts(g, 1024, 384, 12, 128)
    m = ex.module(dev, n_shared=1)
    x = torch.randn(16, 1024, generator=g).bfloat16().to(dev)
    sel, w = (t.to(dev) for t in _routes(g, 16, 11, 4, skew=True))
    whole = m(x, sel, w, limit=10.0)
    for rows in (1, 2, 3, 7, 8, 9, 15):
        assert torch.equal(m(x[:rows], sel[:rows], w[:rows], limit=10.0), whole[:rows]), rows
    assert torch.equal(m(x[5:6], sel[5:6], w[5:6], limit=10.0), whole[5:6])


@pytest.mark.parametrize("rows", [1, 4, 16, 80, 300])
def test_strides_graph_and_streams(dev, rows):
    g = _gen(rows)
    ex = Experts(g, 384, 256, 16, 64, zeros=True)
    m = ex.module(dev, n_shared=1)
    wide = torch.randn(rows, 401, generator=g).bfloat16().to(dev)
    sel, w = (t.to(dev) for t in _routes(g, rows, 15, 4))
    x = wide[:, 9:393]
    ref = m(x.contiguous(), sel, w)
    assert torch.equal(m(x, sel, w), ref) and torch.equal(m(x, sel.int(), w.double()), ref)
    assert torch.equal(m(x.reshape(rows, 1, 384), sel.reshape(rows, 1, 4), w.reshape(rows, 1, 4)), ref.reshape(rows, 1, 384))
    assert m(x[:0], sel[:0], w[:0]).shape == (0, 384)
    out = torch.full((rows, 400), 3.0, dtype=torch.bfloat16, device=dev)
    ops.w4_moe_forward(x, m.gate, m.up, m.down, sel, w, n_shared=1, out=out[:, 5:389])
    assert torch.equal(out[:, 5:389], ref) and (out[:, :5] == 3).all() and (out[:, 389:] == 3).all()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = m(x, sel, w)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, ref)
    # two captured graphs that share one workspace, replayed in turn with new inputs and routes
    ws = torch.empty(ops.lib().evamx_w4_moe_workspace_bytes(rows, 4, 1, 384, 256), dtype=torch.uint8, device=dev)
    graphs = []
    for _ in range(2):
        sx, ss, sw = x.contiguous(), sel.clone(), w.clone()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            y = ops.w4_moe_forward(sx, m.gate, m.up, m.down, ss, sw, n_shared=1, workspace=ws)
        graphs.append((graph, sx, ss, sw, y))
    for k in range(5):
        graph, sx, ss, sw, y = graphs[k % 2]
        nsel, nw = _routes(g, rows, 15, 4, skew=k % 2 == 0)
        sx.copy_(torch.randn(rows, 384, generator=g))
        ss.copy_(nsel)
        sw.copy_(nw)
        graph.replay()
        assert torch.equal(y, m(sx, ss, sw)), k
        torch.cuda.synchronize()


@pytest.mark.parametrize("dtype,group,zeros", [(torch.bfloat16, 128, False), (torch.float16, 64, True), (torch.bfloat16, 32, True),
                                               (torch.float16, 128, False)])
def test_expert_loads_at_the_units_edges(dev, dtype, group, zeros):
    """Experts of every number of rows at which the kernels or their units change, in one call: none, 1, 16, 17, up to 257."""
    loads = [0, 1, 16, 17, 31, 0, 32, 33, 48, 49, 63, 64, 65, 80, 81, 96, 97, 127, 128, 129, 0, 257, 15]
    g = _gen(group)
    ex = Experts(g, 320, 200, len(loads), group, zeros=zeros, dtype=dtype)
    sel = torch.cat([torch.full((n,), e) for e, n in enumerate(loads)])
    sel = sel[torch.randperm(len(sel), generator=g)].reshape(-1, 1)
    x = (1.5 * torch.randn(len(sel), 320, generator=g)).to(dtype)
    w = torch.randn(len(sel), 1, generator=g)
    _check(dev, ex, x, sel, w, limit=2.0)


@pytest.mark.parametrize("experts", [200, 1000])
def test_many_experts_few_rows_each(dev, experts):
    """As many units as a call can have: every expert with one more row than a unit holds, or with one."""
    g = _gen(experts)
    ex = Experts(g, 64, 48, experts, 32)
    for per in (1, 16, 17):
        if per * experts > 8000:
            continue
        sel = torch.arange(experts).repeat(per)[torch.randperm(per * experts, generator=g)].reshape(-1, 1)
        x = torch.randn(len(sel), 64, generator=g).bfloat16()
        _check(dev, ex, x, sel, torch.ones(len(sel), 1))


@pytest.mark.parametrize("rows", [1, 3, 12, 100])
def test_workspace_holds_anything(dev, rows):
    g = _gen(rows)
    ex = Experts(g, 256, 160, 9, 64, zeros=True)
    m = ex.module(dev, n_shared=1)
    x = torch.randn(rows, 256, generator=g).bfloat16().to(dev)
    sel, w = (t.to(dev) for t in _routes(g, rows, 8, 3))
    sel[0, 0] = 50                                        # a slot that nobody computes
    ref = m(x, sel, w)
    ws = torch.empty(ops.lib().evamx_w4_moe_workspace_bytes(2 * rows, 3, 1, 256, 160), dtype=torch.uint8, device=dev)
    for fill in (0, 255, 0x7f):
        ws.fill_(fill)
        assert torch.equal(ops.w4_moe_forward(x, m.gate, m.up, m.down, sel, w, n_shared=1, workspace=ws), ref)


def test_router_statistics_and_experts_together(dev):
    """A layer as it is used: the router's logits and routes, its balance, the experts' products."""
    g = _gen(2)
    ex = Experts(g, 512, 256, 33, 128)
    m = ex.module(dev, n_shared=1)
    gate_w = (torch.randn(32, 512, generator=g) / 16).to(dev)
    for rows in (1, 12, 130):
        x = torch.randn(rows, 512, generator=g).bfloat16().to(dev)
        z = ops.router_logits(x, gate_w)
        idx, w, _ = ops.route_topk(z, 4, "sigmoid")
        y = m(x, idx, w, limit=10.0)
        ref, tol = ex.reference(x, idx, w, n_shared=1, limit=10.0)
        assert ((y.double().cpu() - ref).abs() <= tol).all()
        leaf = z.clone().requires_grad_()
        loss, counts = ops.balance_loss(leaf, idx)
        loss.sum().backward()
        assert torch.equal(counts[0].cpu(), torch.bincount(idx.cpu().reshape(-1), minlength=32).int())
        assert leaf.grad.isfinite().all() and abs(float(leaf.grad.sum(1).abs().max())) < 1.0


def test_large_calls_are_split(dev):
    g = _gen(3)
    ex = Experts(g, 64, 32, 3, 32)
    m = ex.module(dev)
    rows = 65536 // 2 + 77
    x = torch.randn(rows, 64, generator=g).bfloat16().to(dev)
    sel, w = (t.to(dev) for t in _routes(g, rows, 3, 2))
    y = m(x, sel, w)
    for lo in (0, 32768 - 20, rows - 40):
        part = slice(lo, lo + 40)
        ref, tol = ex.reference(x[part], sel[part], w[part])
        assert ((y[part].double().cpu() - ref).abs() <= tol).all()


def test_refusals(dev):
    g = _gen(1)
    ex = Experts(g, 64, 32, 3, 32)
    m = ex.module(dev)
    x = torch.randn(4, 64, device=dev).bfloat16()
    sel, w = (t.to(dev) for t in _routes(g, 4, 3, 2))
    call = lambda x=x, sel=sel, w=w, **kw: ops.w4_moe_forward(x, m.gate, m.up, m.down, sel, w, **kw)
    call()
    for kw in (dict(x=x.float()), dict(x=x[:, :32]), dict(x=x[0]), dict(x=x.cpu()), dict(sel=sel.int()), dict(sel=sel[:3]), dict(w=w.half()),
               dict(w=w[:, :1]), dict(out=torch.empty(4, 65, dtype=torch.bfloat16, device=dev)), dict(x=x.detach().requires_grad_()),
               dict(x=x[:0], sel=sel[:0], w=w[:0])):
        with pytest.raises(ValueError):
            call(**kw)
    for kw in (dict(n_shared=4), dict(limit=-1.0), dict(limit=float("nan")), dict(workspace=torch.empty(64, dtype=torch.uint8, device=dev))):
        with pytest.raises(ops._lib.EvamxError):
            call(**kw)
    with pytest.raises(ops._lib.EvamxError, match="fit"):
        ops.w4_moe_forward(x, m.gate, m.up, m.gate, sel, w)
    with pytest.raises(ops._lib.EvamxError, match="scale type"):
        ops.w4_moe_forward(x, m.gate, Experts(g, 64, 32, 3, 32, dtype=torch.float16).up.pack(dev), m.down, sel, w)
    with pytest.raises(ops._lib.EvamxError, match="group size"):
        ops.w4_moe_forward(x, m.gate, Experts(g, 64, 32, 3, 64).up.pack(dev), m.down, sel, w)
