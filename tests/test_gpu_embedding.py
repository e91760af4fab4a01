"""GPU: rows of an embedding table and the table's gradient (ops.embedding, ops.embedding_grad) against the definition in 64 bits.

Tolerances.  A row is one fp32 product and one rounding to its type: off by half a step of each, relative.  A gradient is a sum in
fp32: an addend passes through at most min(m, stretch + groups + blocks) additions, each off by 2^-24 of a partial sum that is no
larger than the sum of the addends' magnitudes; then one product and one rounding to its type."""
import math

import pytest
import torch

from neuradar_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def indices(n, rows, order, seed, dtype=torch.int64):
    g = torch.Generator().manual_seed(seed)
    if order == "one":
        idx = torch.full((n,), rows // 2)
    elif order == "runs":
        idx = torch.randint(0, rows, (n // 7 + 1,), generator=g).repeat_interleave(7)[:n]
    elif order == "skewed":
        idx = ((rows + 1.0) ** torch.rand(n, generator=g, dtype=torch.float64) - 1).long().clamp(0, rows - 1)
    elif order == "sorted":
        idx = torch.randint(0, rows, (n,), generator=g).sort().values
    else:
        idx = torch.randint(0, rows, (n,), generator=g)
    return idx.to(dtype)


def check_rows(out, table, idx, scale):
    want = table.double().cpu()[idx.long().cpu()] * scale
    got = out.double().cpu()
    tol = want.abs() * (half_step(out.dtype) * (1 + 2.0 ** -20) + 2.0 ** -24) + torch.finfo(out.dtype).smallest_normal * half_step(out.dtype)
    assert got.shape == want.shape and bool(((got - want).abs() <= tol).all()), float((got - want).abs().max())


def gradient64(grad, idx, rows, scale, padding):
    grad, idx = grad.double().cpu(), idx.long().cpu()
    keep = (idx >= 0) & (idx < rows)
    if padding is not None:
        keep &= idx != padding % rows
    grad, idx = grad[keep], idx[keep]
    total = torch.zeros(rows, grad.shape[1], dtype=torch.float64).index_add_(0, idx, grad) * scale
    size = torch.zeros(rows, grad.shape[1], dtype=torch.float64).index_add_(0, idx, grad.abs()) * abs(scale)
    return total, size, torch.bincount(idx, minlength=rows)


def check_gradient(got, grad, idx, rows, scale=1.0, padding=None, before=None):
    total, size, count = gradient64(grad, idx, rows, scale, padding)
    if before is not None:
        total, size = total + before.double().cpu(), size + before.double().cpu().abs()
    n = idx.numel()
    adds = torch.minimum(count, torch.tensor(64 + 256 + n // 256 + 2))[:, None].double() + 2
    tol = size * adds * 2.0 ** -24 + total.abs() * half_step(got.dtype) * (1 + 2.0 ** -20) + torch.finfo(got.dtype).smallest_normal * half_step(got.dtype)
    err = (got.double().cpu() - total).abs()
    assert bool((err <= tol).all()), float((err - tol).max())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,rows,dim", [(1, 1, 1), (1, 5, 16), (64, 60, 16), (65, 3, 33), (1000, 257, 7), (513, 70000, 48), (4097, 1000, 1024),
                                        (33, 9, 2500), (3, 2, 65536)])
def test_rows(dtype, n, rows, dim):
    table = (torch.randn(rows, dim, generator=torch.Generator().manual_seed(n)) * 0.5).to(dtype).to(DEV)
    for itype, scale in ((torch.int64, 1.0), (torch.int32, math.sqrt(dim))):
        idx = indices(n, rows, "uniform", 3, itype).to(DEV)
        check_rows(ops.embedding(table, idx, scale), table, idx, scale)
    assert torch.equal(ops.embedding(table, idx), table[idx.long()])  # (a scale of 1 is a copy)


def test_rows_shapes_strides_and_far_indices():
    wide = torch.randn(50, 96, device=DEV)
    table = wide[:, 13:46]  # rows 96 apart, starting off any 16-byte address
    idx = torch.tensor([[0, 49, -1], [50, 7, 7]], device=DEV)
    out = ops.embedding(table, idx, 2.0)
    assert out.shape == (2, 3, 33) and out.is_contiguous()
    for a, b in ((0, 0), (0, 1), (1, 1), (1, 2)):
        assert torch.equal(out[a, b], table[idx[a, b]] * 2.0)
    assert bool(torch.isnan(out[0, 2]).all()) and bool(torch.isnan(out[1, 0]).all())
    assert torch.equal(ops.embedding(wide.t(), torch.tensor([95, 0], device=DEV)), wide.t()[[95, 0]])  # columns apart: copied
    assert torch.equal(ops.embedding(wide, idx[:, 1].to(torch.int32)[::1])[1], wide[7])
    assert ops.embedding(wide, torch.empty(0, 4, dtype=torch.int64, device=DEV)).shape == (0, 4, 96)
    assert ops.embedding(wide[:, :0], idx).shape == (2, 3, 0)
    assert bool(torch.isnan(ops.embedding(wide[:0], torch.zeros(3, dtype=torch.int64, device=DEV))).all())


@pytest.mark.parametrize("dtype", [F32, BF16, F16])
@pytest.mark.parametrize("n,rows,dim,order", [
    (1, 1, 1, "one"), (1, 4, 16, "one"), (2, 1, 3, "one"), (64, 64, 8, "uniform"), (65, 60, 16, "runs"), (1000, 7, 33, "uniform"),
    (2047, 2047, 16, "uniform"), (2048, 2048, 5, "skewed"), (2049, 4096, 48, "sorted"), (16384, 60, 16, "runs"), (16385, 1, 20, "one"),
    (5000, 3, 257, "skewed"), (4096, 100003, 12, "uniform"), (777, 50, 1030, "skewed"), (300, 5, 2500, "uniform"),
    (20000, 300000, 2, "skewed"), (12289, 2, 1, "uniform"), (40000, 5000000, 3, "uniform"), (70001, 513, 24, "skewed")])
def test_gradient(dtype, n, rows, dim, order):
    g = (torch.randn(n, dim, generator=torch.Generator().manual_seed(n + dim)) / 8).to(dtype).to(DEV)
    for itype, scale, padding in ((torch.int64, 1.0, None), (torch.int32, 0.37, -1)):
        idx = indices(n, rows, order, 5, itype).to(DEV)
        got = ops.embedding_grad(g, idx, rows, scale, padding)
        assert got.dtype == dtype
        check_gradient(got, g, idx, rows, scale, padding)
        assert torch.equal(got, ops.embedding_grad(g, idx, rows, scale, padding))  # the same bits again


@pytest.mark.parametrize("dim", [1, 16, 33, 130])
def test_gradient_into_other_types_and_onto_a_buffer(dim):
    n, rows = 3001, 97
    idx = indices(n, rows - 5, "skewed", 1).to(DEV)  # the last rows are named by no index
    g = torch.randn(n, dim, device=DEV) / 8
    for gtype in (F32, BF16, F16):
        for ttype in (F32, BF16, F16):
            x = g.to(gtype)
            check_gradient(ops.embedding_grad(x, idx, rows, dtype=ttype), x, idx, rows)
            before = torch.randn(rows, dim, device=DEV).to(ttype)
            out = before.clone()
            assert ops.embedding_grad(x, idx, rows, 0.5, 3, out=out, accumulate=True) is out
            check_gradient(out, x, idx, rows, 0.5, 3, before)
            assert torch.equal(out[rows - 5:], before[rows - 5:]) and torch.equal(out[3], before[3])
            out = torch.full((rows, dim), float("nan"), device=DEV, dtype=ttype)
            check_gradient(ops.embedding_grad(x, idx, rows, out=out), x, idx, rows)
    room = torch.randn(rows * dim + 1, device=DEV).to(BF16)  # a result that starts off any 16-byte address
    check_gradient(ops.embedding_grad(g, idx, rows, out=room[1:].view(rows, dim)), g, idx, rows)


def test_gradient_of_strided_broadcast_and_shaped_input():
    idx = indices(600, 40, "uniform", 2).to(DEV).view(20, 30)
    wide = torch.randn(20, 30, 64, device=DEV)
    for g in (wide[..., 5:38], wide[:, :, ::2], wide.permute(1, 0, 2).contiguous().permute(1, 0, 2)):
        check_gradient(ops.embedding_grad(g, idx, 40), g.reshape(600, -1), idx.view(-1), 40)
    one = torch.randn(16, device=DEV).expand(600, 16)  # (the gradient of a sum over rows: one row for all)
    check_gradient(ops.embedding_grad(one, idx.view(-1), 40), one, idx.view(-1), 40)
    ones = torch.ones((), device=DEV).expand(20, 30, 8)
    check_gradient(ops.embedding_grad(ones, idx, 40), ones.reshape(600, 8), idx.view(-1), 40)


def test_gradient_far_indices_padding_only_and_nothing():
    rows, dim = 11, 9
    idx = torch.tensor([3, -1, 11, 2 ** 40, 3, -2 ** 40, 10], device=DEV)
    g = torch.randn(7, dim, device=DEV)
    g[[1, 2, 3, 5]] = float("nan")  # what no row takes is not in any row
    got = ops.embedding_grad(g, idx, rows)
    check_gradient(got, torch.nan_to_num(g), idx, rows)
    assert not bool(torch.isnan(got).any())
    assert not bool(ops.embedding_grad(g, torch.full((7,), 4, device=DEV), rows, padding_idx=4).any())
    g[0] = float("inf")  # infinities stay in their row
    got = ops.embedding_grad(g, idx, rows)
    assert bool(torch.isinf(got[3]).all()) and bool(torch.isfinite(got[torch.arange(rows) != 3]).all())
    none = torch.empty(0, dtype=torch.int64, device=DEV)
    assert not bool(ops.embedding_grad(torch.empty(0, dim, device=DEV), none, rows).any())
    kept = torch.randn(rows, dim, device=DEV)
    assert torch.equal(ops.embedding_grad(torch.empty(0, dim, device=DEV), none, rows, out=kept.clone(), accumulate=True), kept)
    assert ops.embedding_grad(torch.empty(3, 0, device=DEV), idx[:3], rows).shape == (rows, 0)
    assert ops.embedding_grad(g, idx, 0).shape == (0, dim)


def test_autograd_against_the_formula_and_differences():
    torch.manual_seed(0)
    table = torch.randn(30, 12, device=DEV, requires_grad=True)
    idx = torch.randint(0, 30, (5, 40), device=DEV)
    w = torch.randn(5, 40, 12, device=DEV)
    loss = (ops.embedding(table, idx, 1.5, padding_idx=4).square() * w).sum()
    loss.backward()
    grad_out = (2 * 1.5 * table.detach()[idx] * w).view(200, 12)
    # (the incoming gradient is itself formed in fp32: 2^-22 of its size on top)
    total, size, _ = gradient64(grad_out, idx.view(-1), 30, 1.5, 4)
    assert bool(((table.grad.double().cpu() - total).abs() <= size * 40 * 2.0 ** -24).all())
    # central differences of a quadratic in one entry are exact up to rounding: 2^-24 of the loss's terms over the step
    def value(t):
        return float((t.double().cpu()[idx.cpu()].mul(1.5).square() * w.double().cpu()).sum())
    for row, col in ((7, 0), (0, 11)):
        up, down = table.detach().clone(), table.detach().clone()
        up[row, col] += 0.5
        down[row, col] -= 0.5
        step = float(up[row, col]) - float(down[row, col])
        assert abs((value(up) - value(down)) / step - float(table.grad[row, col])) <= 1e-4 * float(size[row, col])
    assert not bool(table.grad[4].any())
    bf = torch.randn(9, 8, device=DEV, dtype=BF16, requires_grad=True)
    ops.embedding(bf, torch.tensor([1, 1, 8], device=DEV)).sum().backward()  # (a broadcast gradient)
    assert bf.grad.dtype == BF16 and bf.grad[:, 0].tolist() == [0, 2, 0, 0, 0, 0, 0, 0, 1]


def test_direct_gradient_adds_to_the_buffer():
    table = torch.nn.Parameter(torch.randn(12, 5, device=DEV))
    table.grad = torch.ones(12, 5, device=DEV)
    kept = table.grad
    with ops.direct_param_grads():
        ops.embedding(table, torch.tensor([2, 2, 9], device=DEV)).sum().backward()
    assert table.grad is kept and table.grad[:, 0].tolist() == [1, 1, 3, 1, 1, 1, 1, 1, 1, 2, 1, 1]


def test_other_stream_and_replayed_graph():
    n, rows, dim = 20000, 300, 16
    table, g = torch.randn(rows, dim, device=DEV), torch.randn(n, dim, device=DEV)
    idx = indices(n, rows, "skewed", 9).to(DEV)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        out, grad = ops.embedding(table, idx, 3.0), ops.embedding_grad(g, idx, rows, 3.0)
    torch.cuda.current_stream().wait_stream(s)
    check_rows(out, table, idx, 3.0)
    check_gradient(grad, g, idx, rows, 3.0)
    graphs = []
    for _ in range(2):  # two graphs with workspaces of their own, replayed in turn with eager calls between
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            graphs.append((graph, ops.embedding(table, idx, 3.0), ops.embedding_grad(g, idx, rows, 3.0)))
    for k in range(4):
        g.copy_(torch.randn(n, dim, device=DEV))
        idx.copy_(indices(n, rows, ("skewed", "uniform", "one", "runs")[k], k))
        eager = ops.embedding_grad(g, idx, rows, 3.0)
        for graph, out, grad in graphs:
            graph.replay()
            torch.cuda.synchronize()
            assert torch.equal(out, table[idx] * 3.0) and torch.equal(grad, eager)


def test_refusals():
    table, idx = torch.zeros(4, 2, device=DEV), torch.zeros(3, dtype=torch.int64, device=DEV)
    g = torch.zeros(3, 2, device=DEV)
    for call, what in ((lambda: ops.embedding(table.double(), idx), "float32, bfloat16 or float16"), (lambda: ops.embedding(table[0], idx), "rows, dim"),
                       (lambda: ops.embedding(table, idx.to(torch.int16)), "int64 or int32"), (lambda: ops.embedding(table, idx.cpu()), "device"),
                       (lambda: ops.embedding(table, idx, padding_idx=4), "not a row"), (lambda: ops.embedding(table, idx, padding_idx=-5), "not a row"),
                       (lambda: ops.embedding_grad(g, idx.cpu(), 4), "device"), (lambda: ops.embedding_grad(g, idx, 4, accumulate=True), "give it"),
                       (lambda: ops.embedding_grad(g, idx, 4, out=table[:3]), "contiguous"), (lambda: ops.embedding_grad(g, idx, 4, dtype=torch.float64), "dtype"),
                       (lambda: ops.embedding_grad(g, idx, 4, out=torch.zeros(4, 4, device=DEV)[:, :2]), "contiguous"),
                       (lambda: ops.embedding_grad(g, idx, 4, out=table, dtype=BF16), "contiguous"), (lambda: ops.embedding_grad(g, idx, 4, padding_idx=9), "not a row"),
                       (lambda: ops.embedding_grad(g, idx, 2 ** 31), "out of range"), (lambda: ops.embedding_grad(g, idx, 3, out=g), "must not be grad"), (lambda: ops.embedding_grad(g[:2], idx, 4), "does not fit")):
        with pytest.raises(RuntimeError, match=what):
            call()


def test_far_offsets():
    """Tables and gradients of more than 2^31 elements: every offset in 64 bits, in each of the three ways to the gradient."""
    rows, dim = 2_200_000, 1024
    table = torch.zeros(rows, dim, device=DEV, dtype=BF16)
    idx = torch.tensor([rows - 1, 0, rows - 2, rows - 1], device=DEV)
    table[-2:] = torch.randn(2, dim, device=DEV).to(BF16)
    assert torch.equal(ops.embedding(table, idx), table[idx])
    g = torch.randn(4, dim, device=DEV).to(BF16)
    out = ops.embedding_grad(g, idx, rows, out=table)  # one launch
    assert torch.equal(out[-2], g[2]) and torch.equal(out[0], g[1]) and float(out[1:-2].abs().max()) == 0.0
    assert torch.equal(out[-1], (g[0].float() + g[3].float()).to(BF16))
    many = torch.full((20000,), rows - 1, device=DEV)
    many[::2] = rows - 2
    ones = torch.ones(1, dim, device=DEV, dtype=BF16).expand(20000, dim)
    out = ops.embedding_grad(ones, many, rows, out=table)  # sorted: the tables of two chunks would not be small
    assert bool((out[-2:] == torch.tensor(10000.0, device=DEV).to(BF16)).all()) and float(out[:-2].abs().max()) == 0.0
    del out, table
    grad = torch.zeros(rows, dim, device=DEV, dtype=BF16)
    grad[-3:] = 1.0
    got = ops.embedding_grad(grad, torch.arange(rows, device=DEV) % 7, 7)  # chunks into small tables
    want = torch.zeros(7, dim, device=DEV, dtype=BF16)
    want[[(rows - k) % 7 for k in (1, 2, 3)]] = 1.0
    assert torch.equal(got, want)


def test_two_streams_at_once_and_no_second_derivative():
    sets = []
    for k, (n, rows, dim) in enumerate(((3000, 40, 16), (30000, 900, 24), (30000, 700000, 40))):
        sets.append((torch.randn(n, dim, device=DEV), indices(n, rows, "skewed", k).to(DEV), rows))
    alone = [ops.embedding_grad(*s) for s in sets]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in sets]
    got = []
    for s, st in zip(sets, streams):
        with torch.cuda.stream(st):
            got.append([ops.embedding_grad(*s) for _ in range(5)])
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, bs in zip(alone, got) for b in bs)
    table = torch.randn(5, 3, device=DEV, requires_grad=True)
    (first,) = torch.autograd.grad(ops.embedding(table, torch.tensor([1, 2], device=DEV)).square().sum(), table, create_graph=True)
    with pytest.raises(RuntimeError, match="once_differentiable|does not require grad|differentiable"):
        first.sum().backward()


def test_rows_beyond_the_caches():
    """More than 256 MB of rows leave past the caches: whole and odd widths, the last vector of a row among them."""
    for dim in (257, 512):
        table = (torch.randn(5000, dim, generator=torch.Generator().manual_seed(dim)) * 0.5).to(BF16).to(DEV)
        idx = torch.randint(0, 5000, (300_000_000 // (2 * dim),), device=DEV)
        assert torch.equal(ops.embedding(table, idx, 3.0), (table.float() * 3.0).to(BF16)[idx])


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
def test_row_ends_of_every_width(dtype):
    """A row's last vector is read and written over the one before: widths around the vectors' own, rows that start one element off,
    NaN before and behind every row, all three ways of the gradient, added to what is there too.  Small whole numbers: exact in
    every type (a row's sum: at most 20 * 2 + 3 < 2^8), so nothing may differ at all."""
    gen = torch.Generator().manual_seed(41)
    for dim in [*range(1, 20), 31, 33, 63, 65]:
        for n, rows in ((5, 3), (500, 90), (17000, 6000), (17000, 900000)):
            idx = torch.randint(0, rows, (n,), generator=gen)
            idx = idx[torch.bincount(idx, minlength=rows)[idx] <= 20]
            n = len(idx)
            wide = torch.full((n + 1, dim + 3), float("nan"), dtype=dtype)
            wide[:n, 1:dim + 1] = torch.randint(-2, 3, (n, dim), generator=gen).to(dtype)
            grad = wide.to(DEV)[:n, 1:dim + 1]
            want = torch.zeros(rows, dim).index_add_(0, idx, wide[:n, 1:dim + 1].float())
            got = ops.embedding_grad(grad, idx.to(DEV), rows)
            assert torch.equal(got.float().cpu(), want), (dim, n, rows)
            out = torch.full((rows, dim), 3.0, dtype=dtype, device=DEV)
            ops.embedding_grad(grad, idx.to(DEV), rows, out=out, accumulate=True)
            assert torch.equal(out.float().cpu(), want + 3.0), (dim, n, rows)
            back = torch.randint(0, n, (n + 7,), generator=gen)
            assert torch.equal(ops.embedding(grad, back.to(DEV)).cpu(), wide[:n, 1:dim + 1][back]), (dim, n)
