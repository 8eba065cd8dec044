"""The products on 4-bit weights at the sizes where their kernels split, widen or read twice: rows long enough to be cut over the
waves of a workgroup, column groups that end inside one, inputs and hidden activations of more than 2^31 bytes."""
import pytest
import torch

from eva_amd import ops
from eva_amd.w4 import W4Linear
from tests.test_gpu_w4_moe import _check, _routes
from tests.w4_helpers import Experts, Matrix, check_linear

pytestmark = pytest.mark.gpu


def _gen(seed):
    return torch.Generator().manual_seed(seed)


# hidden, inter: gate and up in one part, two (from 24 k-tiles) and four (from 48), and down likewise
SPLITS = [(3200, 210), (6200, 130), (200, 3210), (130, 6300), (3130, 3210), (6272, 64)]


@pytest.mark.parametrize("hidden,inter", SPLITS)
@pytest.mark.parametrize("rows", [1, 2, 4, 9, 16, 40])
@pytest.mark.parametrize("dtype,group,zeros", [(torch.bfloat16, 128, False), (torch.float16, 32, True)])
def test_layers_whose_rows_are_split(dev, hidden, inter, rows, dtype, group, zeros):
    g = _gen(rows + hidden)
    ex = Experts(g, hidden, inter, 4, group, zeros=zeros, dtype=dtype)
    x = (1.5 * torch.randn(rows, hidden, generator=g)).to(dtype)
    sel, w = _routes(g, rows, 3, 2)
    _check(dev, ex, x, sel, w, n_shared=1, limit=2.0)


@pytest.mark.parametrize("hidden,inter", SPLITS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_split_rows_do_not_depend_on_their_batch(dev, hidden, inter, dtype):
    """Up to 16 tokens a token's bits are those it has alone, through one token's kernels, those of a few and of 16-row units."""
    g = _gen(inter)
    m = Experts(g, hidden, inter, 6, 64, dtype=dtype).module(dev, n_shared=1)
    x = torch.randn(16, hidden, generator=g).to(dtype).to(dev)
    sel, w = (t.to(dev) for t in _routes(g, 16, 5, 3, skew=True))
    whole = m(x, sel, w, limit=10.0)
    for rows in (1, 2, 3, 4, 5, 9):
        assert torch.equal(m(x[:rows], sel[:rows], w[:rows], limit=10.0), whole[:rows]), rows
    assert torch.equal(m(x[7:8], sel[7:8], w[7:8], limit=10.0), whole[7:8])


@pytest.mark.parametrize("rows", [1, 3, 12, 40, 100])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_hidden_activations_read_twice(dev, rows, dtype):
    """More hidden activations than a workgroup keeps in registers when it makes them ready (8192)."""
    g = _gen(rows)
    ex = Experts(g, 64, 8300, 2, 64, dtype=dtype)
    x = torch.randn(rows, 64, generator=g).to(dtype)
    _check(dev, ex, x, torch.randint(0, 2, (rows, 1), generator=g), torch.rand(rows, 1, generator=g))


@pytest.mark.parametrize("n_out", [8200, 16384, 16400, 18437])
@pytest.mark.parametrize("dtype,group,zeros", [(torch.bfloat16, 64, True), (torch.float16, 128, False)])
def test_wide_matrices(dev, n_out, dtype, group, zeros):
    """32 columns a workgroup on one block of rows (from 1024 column tiles), and 16 below: the same bits a row has alone."""
    g = _gen(n_out)
    for n_in in (200, 1100):
        m = Matrix(g, n_out, n_in, group, zeros=zeros, dtype=dtype)
        w, w64 = m.pack(dev), m.w.to(dev)
        x = torch.randn(16, n_in, generator=g).to(dtype).to(dev)
        whole = ops.w4_linear(x, w)
        check_linear(whole, x, w64)
        for rows in (1, 2, 5, 13):
            assert torch.equal(ops.w4_linear(x[:rows], w), whole[:rows]), (n_in, rows)


@pytest.mark.parametrize("n_out", [2040, 2111, 2303])
@pytest.mark.parametrize("rows", [17, 130, 161, 200, 300])
@pytest.mark.parametrize("dtype,group,zeros", [(torch.float16, 128, True), (torch.bfloat16, 64, False), (torch.bfloat16, 128, False),
                                               (torch.float16, 64, True)])
def test_middle_calls(dev, n_out, rows, dtype, group, zeros):
    """32 rows by 32 and by 64 columns, with columns that end inside a workgroup's or a tile."""
    g = _gen(rows + n_out)
    for n_in in (300, 1300):
        m = Matrix(g, n_out, n_in, group, zeros=zeros, dtype=dtype)
        x = torch.randn(rows, n_in, generator=g).to(dtype).to(dev)
        b = torch.randn(n_out, generator=g).to(dtype).to(dev)
        check_linear(ops.w4_linear(x, m.pack(dev), b), x, m.w.to(dev), b)


@pytest.mark.parametrize("n_in", [8200, 8999])
@pytest.mark.parametrize("rows", [1, 9, 40, 140])
def test_rows_read_twice(dev, n_in, rows):
    """Rows of more values than a workgroup keeps in registers (8192), aligned bf16 ones and fp16 ones that start anywhere."""
    g = _gen(n_in + rows)
    for dtype, off in ((torch.bfloat16, 0), (torch.float16, 3)):
        m = Matrix(g, 130, n_in, 128, dtype=dtype)
        x = torch.randn(rows, n_in + 5, generator=g).to(dtype).to(dev)[:, off:n_in + off]
        check_linear(ops.w4_linear(x, m.pack(dev)), x, m.w)


@pytest.mark.parametrize("rows", [1, 16, 33, 300])
def test_expanded_rows(dev, rows):
    """Rows that are one row in memory give what as many copies give, at every number of rows."""
    g = _gen(rows)
    lin = W4Linear(Matrix(g, 200, 700, 64, zeros=True, dtype=torch.bfloat16).pack(dev))
    x = torch.randn(1, 700, generator=g).bfloat16().to(dev)
    assert torch.equal(lin(x.expand(rows, 700)), lin(x.repeat(rows, 1)))
    assert torch.equal(lin(x.expand(3, 700)), lin(x).expand(3, 200))


def _some(rows, at):
    return torch.tensor(sorted({0, 1, 63, 64, rows // 2, at - 1, at, at + 1, rows - 65, rows - 2, rows - 1}))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_inputs_of_almost_4_gib(dev, dtype):
    """The experts' inputs, made ready and as they lie, reach past 2^31 bytes: rows on both sides of it and the last ones."""
    rows, hidden = 32500, 66048
    g = _gen(3)
    ex = Experts(g, hidden, 32, 2, 128, dtype=dtype)
    x = torch.empty(rows, hidden, dtype=dtype, device=dev).normal_(generator=torch.Generator(dev).manual_seed(1))
    sel = (torch.arange(rows) % 2).reshape(rows, 1)
    w = torch.rand(rows, 1, generator=g)
    y = ex.module(dev)(x, sel.to(dev), w.to(dev))
    some = _some(rows, 2 ** 30 // hidden)
    ref, tol = ex.reference(x[some.to(dev)], sel[some], w[some], dtype=dtype)
    off = (y[some.to(dev)].double().cpu() - ref).abs()
    assert (off <= tol).all(), float((off / tol).max())
    assert y.isfinite().all()


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_hidden_activations_of_almost_4_gib(dev, dtype):
    """65000 slots of 16500 hidden activations, two halves each."""
    rows, inter = 32500, 16500
    g = _gen(4)
    ex = Experts(g, 64, inter, 3, 64, dtype=dtype)
    x = torch.randn(rows, 64, generator=g).to(dtype)
    sel = torch.stack([torch.arange(rows) % 3, (torch.arange(rows) + 1) % 3], 1)
    w = torch.rand(rows, 2, generator=g)
    y = ex.module(dev)(x.to(dev), sel.to(dev), w.to(dev))
    some = _some(rows, rows // 2)
    ref, tol = ex.reference(x[some], sel[some], w[some], dtype=dtype)
    off = (y[some.to(dev)].double().cpu() - ref).abs()
    assert (off <= tol).all(), float((off / tol).max())
    assert y.isfinite().all()


def test_a_linear_of_more_than_4_gib(dev):
    """65536 rows of 33000 bf16 values."""
    rows, n_in = 65536, 33000
    g = _gen(5)
    m = Matrix(g, 40, n_in, 128, dtype=torch.bfloat16)
    x = torch.empty(rows, n_in, dtype=torch.bfloat16, device=dev).normal_(generator=torch.Generator(dev).manual_seed(2))
    y = ops.w4_linear(x, m.pack(dev))
    some = _some(rows, 2 ** 31 // n_in).to(dev)
    check_linear(y[some], x[some], m.w)
    assert y.isfinite().all()


@pytest.mark.parametrize("inter", [3968, 3970])
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
def test_one_token_at_the_most_lds(dev, inter, dtype):
    """Eight slots' hidden activations that just fit one workgroup's LDS, and that just do not."""
    g = _gen(inter)
    ex = Experts(g, 200, inter, 9, 64, dtype=dtype)
    x = torch.randn(1, 200, generator=g).to(dtype)
    sel, w = _routes(g, 1, 9, 8)
    _check(dev, ex, x, sel, w, limit=5.0)
