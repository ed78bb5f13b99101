"""The token embedding against indexing and sums in 64 bits.

Lookup: one product in fp32 and one rounding to the type (scale 1: the same bits).  Gradient: an fp32 sum of n
terms in any order is off by at most n U sum|.|, U = 2^-24, the product with the scale by one unit more, and a
bf16 result by 2^-8 of its size."""
import pytest
import torch

from hdcmamba_b200 import _lib, ops, training

pytestmark = pytest.mark.gpu
F32, BF16 = torch.float32, torch.bfloat16
U = 2.0 ** -24


def check_grad(got, dy, ids, rows, scale, skip=None):
    D = dy.shape[-1]
    i, d = ids.reshape(-1).cpu().long(), dy.reshape(-1, D).double().cpu()
    if skip is not None:
        keep = i != skip
        i, d = i[keep], d[keep]
    ref = torch.zeros(rows, D, dtype=torch.float64).index_add_(0, i, d) * scale
    size = torch.zeros(rows, D, dtype=torch.float64).index_add_(0, i, d.abs()) * abs(scale)
    n = torch.bincount(i, minlength=rows).double()[:, None]
    most = (n + 2) * U * size + (2 ** -8 * ref.abs() if got.dtype == BF16 else 0)
    err = (got.double().cpu() - ref).abs()
    assert (err <= most).all(), float((err / (most + 1e-300)).max())
    assert (got.cpu()[n[:, 0] == 0] == 0).all()


def make_ids(kind, N, rows, g):
    if kind == "one":
        return torch.full((N,), rows - 1)
    if kind == "two":
        return torch.randint(0, 2, (N,), generator=g) * (rows - 1)
    if kind == "sorted":
        return torch.randint(0, rows, (N,), generator=g).sort().values
    if kind == "skewed":
        return (torch.rand(N, generator=g) ** 8 * rows).long().clamp(max=rows - 1)
    return torch.randint(0, rows, (N,), generator=g)


CASES = [(0, 5, 16), (1, 1, 1), (1, 3, 8), (3, 700, 24), (31, 17, 33), (32, 32, 64), (33, 511, 256), (255, 512, 264), (256, 513, 7),
         (1023, 40, 128), (1024, 5000, 40), (1025, 262143, 16), (2500, 262144, 8), (5000, 1, 72), (3000, 2, 520),
         (70000, 300, 16), (140000, 1000, 8)]


@pytest.mark.parametrize("dtype", [F32, BF16])
@pytest.mark.parametrize("kind", ["any", "one", "two", "sorted", "skewed"])
@pytest.mark.parametrize("N,rows,D", CASES)
def test_lookup_and_gradient(dtype, kind, N, rows, D):
    g = torch.Generator().manual_seed(N + rows)
    ids = make_ids(kind, N, rows, g).cuda()
    if D % 2:
        ids = ids.int()
    w = torch.randn(rows, D, generator=g).to(dtype).cuda().requires_grad_()
    y = training.embedding(ids, w)
    assert torch.equal(y, w.detach()[ids.long()])
    dy = torch.randn(N, D, generator=g).to(dtype).cuda()
    (dw,) = torch.autograd.grad(y, [w], dy)
    check_grad(dw, dy, ids, rows, 1.0)
    scaled = ops.embedding(ids, w.detach(), scale=5.5)
    assert torch.equal(scaled, (5.5 * w.detach()[ids.long()].float()).to(dtype))
    check_grad(ops.embedding_bwd(dy, ids, rows, 5.5), dy, ids, rows, 5.5)


@pytest.mark.parametrize("dtype", [F32, BF16])
def test_shapes_views_and_padding(dtype):
    g = torch.Generator().manual_seed(3)
    table = torch.randn(100, 200, generator=g).to(dtype).cuda()
    ids = torch.randint(0, 100, (4, 3, 70), generator=g).cuda()
    for w in (table[:, 8:72], table[:, 1:66], table[::2, :65]):
        i = ids % w.shape[0]
        assert torch.equal(ops.embedding(i, w), w[i])
    i = ids.transpose(0, 2)  # ids in another order of memory
    assert torch.equal(ops.embedding(i, table), table[i])
    out = torch.empty(4, 3, 70, 200, device="cuda", dtype=dtype)
    assert ops.embedding(ids, table, out=out) is out and torch.equal(out, table[ids])
    # gradients: strided, expanded, permuted
    for dy in (torch.randn(4, 3, 70, 128, generator=g).to(dtype).cuda()[..., 3:67],
               torch.randn(64, 4, 3, 70, generator=g).to(dtype).cuda().permute(1, 2, 3, 0),
               torch.randn(4, 1, 1, 64, generator=g).to(dtype).cuda().expand(4, 3, 70, 64)):
        check_grad(ops.embedding_bwd(dy, ids, 100), dy, ids, 100, 1.0)
    dy = torch.randn(4, 3, 70, 64, generator=g).to(dtype).cuda()
    check_grad(ops.embedding_bwd(dy, ids, 100, padding_idx=7), dy, ids, 100, 1.0, skip=7)
    buf = torch.full((102, 80), 3.0, device="cuda", dtype=dtype)
    ops.embedding_bwd(dy, ids, 100, out=buf[1:101, 8:72])
    check_grad(buf[1:101, 8:72], dy, ids, 100, 1.0)
    buf[1:101, 8:72] = 3
    assert (buf == 3).all()
    w = table[:, :64].detach().clone().requires_grad_()
    y = training.embedding(ids, w, scale=2.0, padding_idx=0)
    assert torch.equal(y, (2 * w.detach().float()).to(dtype)[ids])
    check_grad(torch.autograd.grad(y, [w], dy)[0], dy, ids, 100, 2.0, skip=0)


def test_wide_rows_and_many_columns():
    g = torch.Generator().manual_seed(4)
    for D in (4096, 8200, 5001):
        w = torch.randn(50, D, generator=g).to(BF16).cuda()
        ids = torch.randint(0, 50, (300,), generator=g).cuda()
        assert torch.equal(ops.embedding(ids, w), w[ids])
        dy = torch.randn(300, D, generator=g).to(BF16).cuda()
        check_grad(ops.embedding_bwd(dy, ids, 50), dy, ids, 50, 1.0)


def test_non_finite_gradients_stay_in_their_rows():
    ids = torch.tensor([3, 1, 3, 2, 1], device="cuda")
    dy = torch.ones(5, 64, device="cuda", dtype=BF16)
    dy[0, 5], dy[3, 6] = float("inf"), float("nan")
    dw = ops.embedding_bwd(dy, ids, 5)
    assert dw[3, 5] == float("inf") and torch.isnan(dw[2, 6])
    dw[3, 5] = dw[2, 6] = 0
    assert torch.isfinite(dw).all() and (dw[1] == 2).all() and (dw[0] == 0).all() and (dw[4] == 0).all()


def test_an_id_outside_the_table_is_reported():
    w = torch.randn(10, 64, device="cuda").to(BF16)
    ids = torch.tensor([1, 10, 2, -1, 3], device="cuda")
    y = ops.embedding(ids, w)
    assert torch.isnan(y[1]).all() and torch.isnan(y[3]).all() and torch.equal(y[[0, 2, 4]], w[[1, 2, 3]])
    with pytest.raises(_lib.HdcError, match="71"):
        ops.check_device()
    dw = ops.embedding_bwd(torch.ones(5, 64, device="cuda", dtype=BF16), ids, 10)
    assert (dw[1:4] == 1).all() and (dw[0] == 0).all() and (dw[4:] == 0).all()
    with pytest.raises(_lib.HdcError, match="71"):
        ops.check_device()
    ops.check_device()


def test_same_bits_again_and_from_graphs():
    g = torch.Generator().manual_seed(5)
    ids = make_ids("skewed", 20000, 3000, g).cuda()
    dy = torch.randn(20000, 96, generator=g).cuda()
    first = ops.embedding_bwd(dy, ids, 3000)
    assert torch.equal(first, ops.embedding_bwd(dy, ids, 3000))
    graphs = []
    for _ in range(2):
        gr = torch.cuda.CUDAGraph()
        with torch.cuda.graph(gr):
            out = ops.embedding_bwd(dy, ids, 3000)
        graphs.append((gr, out))
    for _ in range(2):
        for gr, out in graphs:
            out.fill_(1)
            gr.replay()
        assert all(torch.equal(first, out) for _, out in graphs)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        other = ops.embedding_bwd(dy, ids, 3000)
    torch.cuda.current_stream().wait_stream(side)
    assert torch.equal(first, other)
