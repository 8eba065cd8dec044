"""The linear on 4-bit weights with group scales against its definition in 64 bits."""
import pytest
import torch

from eva_amd import ops
from eva_amd.w4 import W4Linear
from tests.w4_helpers import Matrix, check_linear

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator().manual_seed(seed)


@pytest.mark.parametrize("n_out,n_in,group", [(16, 128, 128), (1, 1, 32), (17, 129, 64), (33, 250, 32), (40, 777, 128), (128, 512, 96),
                                              (31, 1000, 256), (16, 640, 512)])
@pytest.mark.parametrize("zeros", [False, True])
@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_pack_and_dequant(dev, n_out, n_in, group, zeros, dtype):
    """The packed matrix holds every code, scale and zero point: its fp32 values are the 64-bit ones rounded
    once (code - zero and the scale are exact, so the product is)."""
    for count in (None, 3):
        m = Matrix(_gen(n_in), n_out, n_in, group, count=count, zeros=zeros, dtype=dtype)
        got = ops.w4_dequant(m.pack(dev)).cpu()
        assert torch.equal(got, m.w.float().reshape(got.shape))


SHAPES = [(16, 128, 128), (1, 1, 32), (17, 33, 32), (130, 511, 64), (48, 513, 32), (100, 1000, 128), (256, 2048, 128), (512, 640, 64),
          (2048, 1024, 32), (65, 4096, 128)]


@pytest.mark.parametrize("n_out,n_in,group", SHAPES)
@pytest.mark.parametrize("rows", [1, 2, 4, 5, 8, 13, 16, 17, 50, 130])
def test_linear(dev, n_out, n_in, group, rows):
    g = _gen(rows * 1000 + n_in)
    for dtype, zeros, bias in ((torch.bfloat16, False, False), (torch.float16, True, True)):
        m = Matrix(g, n_out, n_in, group, zeros=zeros, dtype=dtype)
        x = torch.randn(rows, n_in, generator=g).to(dtype).to(dev)
        b = torch.randn(n_out, generator=g).to(dtype).to(dev) if bias else None
        check_linear(ops.w4_linear(x, m.pack(dev), b), x, m.w, b)


@pytest.mark.parametrize("n_out,n_in,group,zeros,dtype", [(4096, 512, 128, False, torch.bfloat16), (4100, 517, 64, True, torch.float16),
                                                          (4351, 900, 32, False, torch.float16), (12000, 128, 128, True, torch.bfloat16)])
@pytest.mark.parametrize("rows", [1024, 1025, 1041, 1070, 1087])
def test_many_rows(dev, n_out, n_in, group, zeros, dtype, rows):
    """The tiles of 64 rows by 256 columns: last tiles of every kind (1, 17, 33 rows and more; columns that end inside
    a wave's), one to eight k-tiles, results at any address."""
    g = _gen(rows + n_in)
    m = Matrix(g, n_out, n_in, group, zeros=zeros, dtype=dtype)
    w, w64 = m.pack(dev), m.w.to(dev)
    x = torch.randn(rows, n_in, generator=g).to(dtype).to(dev)
    b = torch.randn(n_out, generator=g).to(dtype).to(dev)
    y = ops.w4_linear(x, w, b)
    check_linear(y, x, w64, b)
    out = torch.full((rows, n_out + 9), 7.0, dtype=dtype, device=dev)
    ops.w4_linear(x, w, b, out=out[:, 3:n_out + 3])
    assert torch.equal(out[:, 3:n_out + 3], y) and (out[:, :3] == 7).all() and (out[:, n_out + 3:] == 7).all()
    if n_in % 128 == 0 and dtype == torch.bfloat16:      # fp16 rows at whole tiles are read as they lie
        half = x.half()
        check_linear(ops.w4_linear(half, w), half, w64)


@pytest.mark.parametrize("rows", [1, 2, 9, 40, 300])
def test_workspace_holds_anything(dev, rows):
    """What a workspace held before does not matter, nor that it is larger than needed, or was used by another call."""
    g = _gen(rows)
    m = Matrix(g, 300, 650, 64, dtype=torch.bfloat16)
    w = m.pack(dev)
    x = torch.randn(rows, 650, generator=g).bfloat16().to(dev)
    ref = ops.w4_linear(x, w)
    ws = torch.empty(ops.lib().evamx_w4_linear_workspace_bytes(2 * rows, 650) + 100, dtype=torch.uint8, device=dev)
    for fill in (0, 255, 0x7f):
        ws.fill_(fill)
        assert torch.equal(ops.w4_linear(x, w, workspace=ws), ref)
    assert torch.equal(ops.w4_linear(x[:1], w, workspace=ws), ops.w4_linear(x[:1], w))


def test_fp16_denormals(dev):
    """fp16 values below 2^-14 keep their bits in the products."""
    g = _gen(4)
    m = Matrix(g, 64, 256, 128, scale=64.0)
    for rows in (1, 5, 40):
        x = (torch.randn(rows, 256, generator=g) * 2.0 ** -18).half().to(dev)
        check_linear(ops.w4_linear(x, m.pack(dev)), x, m.w)


@pytest.mark.parametrize("rows", [1, 3, 16, 40, 200])
def test_strides_and_alignment(dev, rows):
    """Rows that start at odd elements, strides that are no multiple of anything, results into a slice: the same
    bits as contiguous ones, and nothing outside the slice is written."""
    g = _gen(rows)
    m = Matrix(g, 75, 387, 32, zeros=True)
    w = m.pack(dev)
    big = torch.randn(rows, 401, generator=g).half().to(dev)
    x = big[:, 5:392]
    ref = ops.w4_linear(x.contiguous(), w)
    check_linear(ref, x, m.w)
    out = torch.full((rows, 83), 7.0, dtype=torch.float16, device=dev)
    ops.w4_linear(x, w, out=out[:, 3:78])
    assert torch.equal(out[:, 3:78], ref)
    assert (out[:, :3] == 7).all() and (out[:, 78:] == 7).all()


@pytest.mark.parametrize("rows", [1, 7, 16, 64])
def test_scale_type_differs_from_x(dev, rows):
    g = _gen(rows)
    for sd, xd in ((torch.float16, torch.bfloat16), (torch.bfloat16, torch.float16)):
        m = Matrix(g, 96, 384, 64, dtype=sd)
        x = torch.randn(rows, 384, generator=g).to(xd).to(dev)
        check_linear(ops.w4_linear(x, m.pack(dev)), x, m.w)


@pytest.mark.parametrize("rows", [1, 5, 16, 100])
@pytest.mark.parametrize("factor", [2.0 ** -120, 2.0 ** -40, 2.0 ** 30, 2.0 ** 100])
def test_bf16_range(dev, rows, factor):
    """bf16 rows far outside fp16's range, and rows of very different ranges in one call."""
    g = _gen(rows)
    m = Matrix(g, 64, 512, 128, dtype=torch.bfloat16, scale=2.0 ** -6)
    x = torch.randn(rows, 512, generator=g)
    x[rows // 2] *= factor
    x = x.bfloat16().to(dev)
    y = ops.w4_linear(x, m.pack(dev))
    check_linear(y, x, m.w)
    zero = torch.zeros_like(x)
    assert (ops.w4_linear(zero, m.pack(dev)) == 0).all()


@pytest.mark.parametrize("rows", [1, 4, 16, 40, 150])
def test_inf_and_nan_stay_in_their_rows(dev, rows):
    g = _gen(rows)
    m = Matrix(g, 80, 300, 32, dtype=torch.bfloat16)
    x = torch.randn(rows, 300, generator=g).bfloat16()
    clean = ops.w4_linear(x.to(dev), m.pack(dev))
    x[0, 17], x[-1, 299] = float("inf"), float("nan")
    y = ops.w4_linear(x.to(dev), m.pack(dev))
    ref = x.float() @ m.w.float().t()
    assert torch.equal(y[1:-1], clean[1:-1])
    assert y[-1].isnan().all()
    if rows > 1:
        assert torch.equal(y[0].float().cpu().isnan(), ref[0].isnan())
        assert torch.equal(y[0].float().cpu().isposinf(), ref[0].isposinf())


def test_rows_do_not_depend_on_their_batch(dev):
    """Up to 16 rows a row's bits are those it has alone (a verification batch's arithmetic)."""
    g = _gen(5)
    for n_out, n_in in ((300, 1000), (4096, 2048), (512, 7168)):
        m = Matrix(g, n_out, n_in, 128, dtype=torch.bfloat16)
        w = m.pack(dev)
        x = torch.randn(16, n_in, generator=g).bfloat16().to(dev)
        whole = ops.w4_linear(x, w)
        for rows in (1, 2, 3, 5, 8, 9, 15):
            assert torch.equal(ops.w4_linear(x[:rows], w), whole[:rows]), (n_out, n_in, rows)
        assert torch.equal(ops.w4_linear(x[7:8], w), whole[7:8])


@pytest.mark.parametrize("rows", [1, 16, 33, 300])
def test_module_graph_and_streams(dev, rows):
    """Leading dimensions, zero rows, another stream, and a captured call replayed with new inputs."""
    g = _gen(rows)
    m = Matrix(g, 200, 700, 64, zeros=True, dtype=torch.bfloat16)
    b = torch.randn(200, generator=g).bfloat16().to(dev)
    lin = W4Linear(m.pack(dev), b)
    x = torch.randn(rows, 700, generator=g).bfloat16().to(dev)
    ref = lin(x)
    check_linear(ref, x, m.w, b)
    assert torch.equal(lin(x.reshape(rows, 1, 700)), ref.reshape(rows, 1, 200))
    assert lin(x[:0]).shape == (0, 200)
    assert torch.equal(lin(x.t().contiguous().t()), ref)
    assert torch.equal(lin(x[:1].expand(3, 700)), ref[:1].expand(3, 200)) or rows > 16
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = lin(x)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(other, ref)
    graph = torch.cuda.CUDAGraph()
    static = x.clone()
    with torch.cuda.graph(graph):
        y = lin(static)
    for k in range(4):
        new = torch.randn(rows, 700, generator=g).bfloat16().to(dev)
        static.copy_(new)
        graph.replay()
        assert torch.equal(y, lin(new)), k
        torch.cuda.synchronize()


def test_a_weight_filled_by_its_owner(dev):
    """A weight made without w4_pack (its buffers read from a file, say), on a device named without an index."""
    g = torch.Generator().manual_seed(5)
    m = Matrix(g, 48, 160, 32, zeros=True)
    packed = m.pack(dev)
    w = ops.W4Weight(1, 48, 160, 32, torch.float16, True, "cuda")
    for a, b in ((w.codes, packed.codes), (w.scales, packed.scales), (w.zeros, packed.zeros)):
        a.copy_(b)
    x = torch.randn(3, 160, generator=g).half().to(dev)
    assert torch.equal(ops.w4_dequant(w), ops.w4_dequant(packed))
    assert torch.equal(ops.w4_linear(x, w), ops.w4_linear(x, packed))


def test_refusals(dev):
    g = _gen(1)
    m = Matrix(g, 32, 64, 32)
    w = m.pack(dev)
    x = torch.randn(2, 64, device=dev, dtype=torch.float16)
    for bad in (x.float(), x[:, :32], x.t(), x[0], x.cpu(), x[:0]):
        with pytest.raises(ValueError):
            ops.w4_linear(bad, w)
    with pytest.raises(ValueError):
        ops.w4_linear(x, Matrix(g, 32, 64, 32, count=2).pack(dev))
    with pytest.raises(ValueError):
        ops.w4_linear(x, w, bias=torch.zeros(31, device=dev, dtype=torch.float16))
    with pytest.raises(ValueError):
        ops.w4_linear(x, w, bias=torch.zeros(32, device=dev, dtype=torch.bfloat16))
    with pytest.raises(ValueError):
        ops.w4_linear(x, w, out=torch.zeros(2, 33, device=dev, dtype=torch.float16))
    with pytest.raises(ValueError, match="backward"):
        ops.w4_linear(x.detach().requires_grad_(), w)
    with pytest.raises(ops._lib.EvamxError, match="workspace"):
        ops.w4_linear(x, w, workspace=torch.empty(16, dtype=torch.uint8, device=dev))
    c, s = m.codes.to(dev), m.scales.to(dev)
    for kw in (dict(n_in=64, group=48), dict(n_in=64, group=0), dict(n_in=66, group=32), dict(n_in=64, group=64)):
        with pytest.raises(ValueError):
            ops.w4_pack(c, s, **kw)
    with pytest.raises(ValueError):
        ops.w4_pack(c, s.float(), n_in=64, group=32)
    with pytest.raises(ValueError):
        ops.w4_pack(c, s, n_in=64, group=32, zeros=torch.zeros(32, 1, dtype=torch.uint8, device=dev))
