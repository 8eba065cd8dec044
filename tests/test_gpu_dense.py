"""Products on 16-bit weights (ops.linear, ops.expert_linear) and their gradients, against 64 bits."""
import pytest
import torch

from eva_amd import ops

pytestmark = pytest.mark.gpu
BF16, FP16 = torch.bfloat16, torch.float16


def act64(v, act, limit):
    if act is None:
        return v
    if act == "relu":
        return v.clamp(min=0)
    if act == "gelu":
        return v * torch.special.ndtr(v)
    if act == "silu":
        return v * torch.sigmoid(v)
    g, u = v.chunk(2, -1)
    a = g * torch.sigmoid(g)
    return a.clamp(max=limit) * u.clamp(-limit, limit) if limit else a * u


def make(g, dtype, *shape, scale=1.0, strided=False, offset=1):
    """Device rows of this type, or a view whose rows start at odd places."""
    if strided:
        wide = torch.randn(*shape[:-1], shape[-1] + offset + 2, generator=g).mul_(scale).to(dtype).to("cuda")
        return wide[..., offset:offset + shape[-1]]
    return torch.randn(*shape, generator=g).mul_(scale).to(dtype).to("cuda")


def check_product(x, w, bias, residual, starts, act, limit, grad):
    """One call and its gradients against 64 bits. Tolerances: fp32 sums of n products, each of them exact, are off by at most n / 2 +
    64 units (2^-24) of the sum of their sizes: the matrix cores add 32 at a time, the rest is a tree or a chain of n / 32 steps;
    the activation's own functions by 16 units; then one rounding. Gradients see D, rounded to 16 bits, and the error of pre."""
    dtype, u16, u32 = x.dtype, torch.finfo(x.dtype).eps / 2, 2.0 ** -24
    leaves = [t if t is None else t.detach().requires_grad_() for t in (x, w, bias, residual)]
    if starts is None:
        y = ops.linear(leaves[0], leaves[1], leaves[2], activation=act, limit=limit, residual=leaves[3])
    else:
        y = ops.expert_linear(leaves[0], leaves[1], starts, leaves[2], activation=act, limit=limit)
    wanted = [t for t in leaves if t is not None]
    got = torch.autograd.grad(y, wanted, grad)
    dx, dw = got[0], got[1]
    db = got[2] if bias is not None else None
    if residual is not None:
        assert torch.equal(got[-1], grad)
    with torch.no_grad():        # the call that autograd does not follow
        same = ops.linear(x, w, bias, activation=act, limit=limit, residual=residual) if starts is None else \
            ops.expert_linear(x, w, starts, bias, activation=act, limit=limit)
    assert torch.equal(same, y.detach())
    rows, n_in = x.shape
    cuts = [0, rows] if starts is None else starts.tolist()
    w3, b2 = (w[None], None if bias is None else bias[None]) if starts is None else (w, bias)
    dw3 = dw[None] if starts is None else dw
    n_out = w3.shape[1]
    tiny = 2.0 ** -24 if dtype == FP16 else 0.0          # half of the smallest fp16 number, with room
    for e, (lo, hi) in enumerate(zip(cuts[:-1], cuts[1:])):
        xe, we = x[lo:hi].cpu().double(), w3[e].cpu().double()
        if lo == hi:
            assert not dw3[e].any() and (db is None or not (db if starts is None else db[e]).any())
            continue
        pre = xe @ we.t()
        size = xe.abs() @ we.abs().t()
        if b2 is not None:
            pre += b2[e].cpu().double()
            size += b2[e].cpu().double().abs()
        pre_off = (n_in / 2 + 64) * u32 * size
        v = pre.clone().requires_grad_()
        a = act64(v, act, limit)
        if act == "swiglu":
            gate, up = pre.chunk(2, -1)
            go, uo = pre_off.chunk(2, -1)
            a_off = 1.13 * go * (up.abs() + uo) + (gate.abs() + go) * uo
        else:
            a_off = 1.13 * pre_off
        want = a.detach()
        a_off = a_off + 16 * u32 * (want.abs() + (gate.abs() * up.abs() if act == "swiglu" else pre.abs()))
        if residual is not None:
            want = want + residual[lo:hi].cpu().double()
            a_off = a_off + u32 * want.abs()
        off = (y[lo:hi].detach().cpu().double() - want).abs()
        tol = a_off + u16 * (want.abs() + a_off) + tiny
        assert (off <= tol).all(), ("y", e, float((off / tol).max()))
        ge = grad[lo:hi].cpu().double()
        if act is None:
            d, d_off = ge, torch.zeros_like(ge)
        else:
            d, = torch.autograd.grad(a, v, ge)
            # slopes change by at most 1.2 (gelu'' and silu'' are below 1) a unit of pre, twice that for swiglu's products
            if act == "swiglu":
                d_off = torch.cat((ge.abs() * (1.2 * go * (up.abs() + uo) + 1.13 * uo), ge.abs() * 1.13 * go), 1)
                sized = torch.cat((ge.abs() * up.abs() * 1.13, ge.abs() * gate.abs()), 1)
                if limit:        # beside a border either side may be taken
                    a_gate = gate * torch.sigmoid(gate)
                    near = torch.cat(((a_gate - limit).abs() <= 4 * go + 1e-5, (up.abs() - limit).abs() <= 4 * uo + 1e-5), 1)
                    d_off += near * (sized + torch.cat((ge.abs() * limit, ge.abs() * limit), 1))
            else:
                d_off = 1.2 * ge.abs() * pre_off
                sized = ge.abs() * (1.13 + pre.abs() * 0)
                if act == "relu":
                    d_off = d_off + (pre.abs() <= pre_off) * ge.abs()
            d_off = d_off + 32 * u32 * sized
            d_off = d_off + u16 * (d.abs() + d_off) + tiny
        want = d @ we
        tol = (n_out / 2 + 64) * u32 * (d.abs() @ we.abs()) + d_off @ we.abs()
        tol = tol + u16 * (want.abs() + tol) + tiny
        off = (dx[lo:hi].cpu().double() - want).abs()
        assert (off <= tol).all(), ("dx", e, float((off / tol).max()))
        want = d.t() @ xe
        tol = ((hi - lo) / 2 + 64) * u32 * (d.abs().t() @ xe.abs()) + d_off.t() @ xe.abs()
        tol = tol + u16 * (want.abs() + tol) + tiny
        off = (dw3[e].cpu().double() - want).abs()
        assert (off <= tol).all(), ("dw", e, float((off / tol).max()))
        if db is not None:
            want = d.sum(0)
            tol = ((hi - lo) / 2 + 64) * u32 * d.abs().sum(0) + d_off.sum(0)
            tol = tol + u16 * (want.abs() + tol) + tiny
            off = ((db if starts is None else db[e]).cpu().double() - want).abs()
            assert (off <= tol).all(), ("db", e, float((off / tol).max()))
    tail = cuts[-1]
    assert not y[tail:].any() and not dx[tail:].any()


DENSE = [  # rows, n_in, n_out
    (1, 1, 1), (1, 2048, 520), (3, 40, 16), (13, 1001, 303), (16, 128, 64), (17, 264, 48), (33, 72, 200), (64, 520, 130), (65, 64, 128),
    (100, 328, 264), (130, 1000, 250), (256, 512, 512), (300, 777, 90), (513, 1032, 264), (1500, 96, 2000)]


@pytest.mark.parametrize("rows,n_in,n_out", DENSE)
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("act", [None, "silu", "swiglu"])
def test_linear(dev, rows, n_in, n_out, dtype, act):
    g = torch.Generator().manual_seed(rows * 7 + n_in)
    if act == "swiglu":
        n_out += n_out % 2
    cols = n_out // 2 if act == "swiglu" else n_out
    x, w = make(g, dtype, rows, n_in), make(g, dtype, n_out, n_in, scale=2 * n_in ** -0.5)
    bias = make(g, dtype, n_out) if rows % 2 else None
    residual = make(g, dtype, rows, cols) if n_out % 4 == 0 else None
    check_product(x, w, bias, residual, None, act, 1.5 if act == "swiglu" and n_in % 3 else 0.0, make(g, dtype, rows, cols))


@pytest.mark.parametrize("act", ["gelu", "relu"])
@pytest.mark.parametrize("rows", [5, 200])
def test_other_activations(dev, act, rows):
    g = torch.Generator().manual_seed(rows)
    check_product(make(g, BF16, rows, 136), make(g, BF16, 72, 136, scale=0.3), make(g, BF16, 72), None, None, act, 0.0, make(g, BF16, rows, 72))


@pytest.mark.parametrize("rows,n_in,n_out,offset", [(9, 200, 64, 1), (9, 200, 64, 8), (150, 200, 136, 1), (150, 200, 136, 8), (400, 136, 72, 3)])
def test_strides(dev, rows, n_in, n_out, offset):
    g = torch.Generator().manual_seed(rows + offset)
    kw = dict(strided=True, offset=offset)
    check_product(make(g, BF16, rows, n_in, **kw), make(g, BF16, n_out, n_in, scale=0.1, **kw), None, make(g, BF16, rows, n_out, **kw), None, None,
                  0.0, make(g, BF16, rows, n_out, **kw))


GROUPS = [  # rows of each expert, rows behind the last, n_in, n_out
    ([1], 0, 64, 32), ([0, 1, 0, 2, 0], 5, 72, 48), ([3, 0, 17, 1, 40, 70], 2, 136, 96), ([129, 0, 1, 300, 64, 65], 31, 200, 264),
    ([40] * 20, 0, 64, 520), ([257, 511, 2], 0, 520, 130), ([0, 0, 0], 7, 64, 64), ([600, 0, 5, 333], 100, 333, 250), ([2] * 100, 30, 40, 24)]


@pytest.mark.parametrize("counts,tail,n_in,n_out", GROUPS)
@pytest.mark.parametrize("dtype", [BF16, FP16])
@pytest.mark.parametrize("act", [None, "swiglu"])
def test_expert_linear(dev, counts, tail, n_in, n_out, dtype, act):
    g = torch.Generator().manual_seed(sum(counts) + n_in)
    rows, experts = sum(counts) + tail, len(counts)
    cols = n_out // 2 if act == "swiglu" else n_out
    starts = torch.tensor([0] + counts).cumsum(0).int().to(dev)
    x, w = make(g, dtype, rows, n_in), make(g, dtype, experts, n_out, n_in, scale=2 * n_in ** -0.5)
    x[rows - tail:] = float("nan")                                         # not read
    grad = make(g, dtype, rows, cols)
    grad[rows - tail:] = float("nan")
    check_product(x, w, make(g, dtype, experts, n_out) if n_in % 3 else None, None, starts, act, 1.0 if n_out % 16 == 0 and act else 0.0, grad)


@pytest.mark.parametrize("act", [None, "swiglu"])
def test_the_largest_tiles(dev, act):
    """Enough tiles of 256 by 256 for each direction: row tiles of every size, the last column tile cut, a sum that ends inside
    a k-tile."""
    g = torch.Generator().manual_seed(5)
    counts = [1024 + 33, 256, 70, 0, 190, 1024, 1024]
    x, w = make(g, BF16, sum(counts), 1096), make(g, BF16, len(counts), 1608, 1096, scale=0.05)
    starts = torch.tensor([0] + counts).cumsum(0).int().to(dev)
    check_product(x, w, make(g, BF16, len(counts), 1608), None, starts, act, 1.0 if act else 0.0, make(g, BF16, sum(counts), 804 if act else 1608))
    rows = 3333
    check_product(make(g, FP16, rows, 2120), make(g, FP16, 2504, 2120, scale=0.05), None, None, None, act, 0.0,
                  make(g, FP16, rows, 1252 if act else 2504))


@pytest.mark.parametrize("act", [None, "swiglu"])
def test_many_small_tiles(dev, act):
    """More tiles of 128 by 128 than CUs, in each direction, where those of 256 by 256 would leave CUs idle."""
    g = torch.Generator().manual_seed(8)
    counts = [(7 * e + 3) % 31 for e in range(40)] + [150]
    x, w = make(g, BF16, sum(counts), 1016), make(g, BF16, len(counts), 1024, 1016, scale=0.05)
    starts = torch.tensor([0] + counts).cumsum(0).int().to(dev)
    check_product(x, w, make(g, BF16, len(counts), 1024), None, starts, act, 1.0 if act else 0.0, make(g, BF16, sum(counts), 512 if act else 1024))
