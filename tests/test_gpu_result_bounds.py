"""GPU: the embedding, norm and clipping kernels write their results and nothing beside them.  Every result lies inside a larger buffer of a
known value, at offsets off any 16-byte address; what surrounds it has to hold that value afterwards.  Workspaces too: exactly the
bytes that the query asks for, with the known value behind them."""
import pytest
import torch

from neuradar_amd import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
KNOWN, ROOM = 77.0, 300  # exact in all three types; elements before and behind (more than a wave's vector stores)


def place(count, dtype, off):
    """(buffer, its part of `count` elements that starts ROOM + off elements in)."""
    buf = torch.full((count + 2 * ROOM + 8,), KNOWN, device=DEV, dtype=dtype)
    return buf, buf[ROOM + off:ROOM + off + count]


def untouched(buf, part):
    at = (part.data_ptr() - buf.data_ptr()) // buf.element_size()
    return bool((buf[:at] == KNOWN).all()) and bool((buf[at + part.numel():] == KNOWN).all())


def indices(n, rows, gen):
    return (((rows + 1.0) ** torch.rand(n, generator=gen, dtype=torch.float64)).long() - 1).clamp_(0, rows - 1).to(DEV)


# (one launch; chunks and a merge; sorted)
WAYS = [(5, 3), (500, 90), (16000, 300000), (17000, 60), (40000, 6000), (17000, 900000)]


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
@pytest.mark.parametrize("n,rows", WAYS, ids=lambda v: str(v))
def test_embedding_gradient(n, rows, dtype):
    gen = torch.Generator().manual_seed(n + rows)
    for k, dim in enumerate((1, 2, 3, 5, 7, 8, 9, 15, 17, 31, 33) + ((63, 65, 130, 513) if rows < 10000 else ())):
        idx = indices(n, rows, gen)
        grad = torch.randint(-2, 3, (n, dim), generator=gen).to(dtype).to(DEV)
        for ttype in (dtype, F32 if dtype != F32 else BF16):
            buf, part = place(rows * dim, ttype, k % 5)
            out = part.view(rows, dim)
            ops.embedding_grad(grad, idx, rows, out=out)
            assert untouched(buf, part), (dim, ttype)
            assert torch.equal(out, ops.embedding_grad(grad, idx, rows, dtype=ttype)), (dim, ttype)
            part.fill_(KNOWN)
            ops.embedding_grad(grad, idx, rows, out=out, accumulate=True)
            assert untouched(buf, part), (dim, ttype)
            names = torch.zeros(rows, dtype=torch.bool, device=DEV)
            names[idx] = True
            assert bool((out[~names] == KNOWN).all()), (dim, ttype)


@pytest.mark.parametrize("grad_dtype", [F32, BF16], ids=str)
def test_embedding_gradient_workspace(grad_dtype):
    """The C entry point with a workspace of exactly the bytes asked for, its contents beforehand whatever they are."""
    lib, gen = _lib.lib(), torch.Generator().manual_seed(3)
    code = _lib.NR_DTYPES[str(grad_dtype)[6:]]
    _lib.ensure_device(0)
    used = 0
    for n, rows, dim in ((17000, 60, 33), (40000, 6000, 7), (113000, 1999, 32), (17000, 900000, 5), (17001, 900000, 24), (130001, 70000, 130), (20000, 3, 2500)):
        need = lib.nr_embedding_bwd_workspace_bytes(rows, dim, n, code)
        used += need > 0
        behind = 4096
        ws = torch.full((need + behind,), 0xA5, device=DEV, dtype=torch.uint8)
        assert ws.data_ptr() % 256 == 0
        idx, grad = indices(n, rows, gen), torch.randn(n, dim, device=DEV).to(grad_dtype)
        out = torch.empty(rows, dim, device=DEV, dtype=grad_dtype)
        assert lib.nr_embedding_bwd(grad.data_ptr(), code, dim, idx.data_ptr(), 8, n, rows, dim, 1.0, -1, out.data_ptr(), code, 0, ws.data_ptr(),
                                    torch.cuda.current_stream().cuda_stream) == 0
        assert bool((ws[need:] == 0xA5).all()), (n, rows, dim)
        assert torch.equal(out, ops.embedding_grad(grad, idx, rows)), (n, rows, dim)
    assert used >= 5


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
def test_rows_apart(dtype):
    """nr_embedding_fwd into rows that lie apart: what is between them stays (the last vector of a row is whole, over the one before)."""
    lib, code = _lib.lib(), _lib.NR_DTYPES[str(dtype)[6:]]
    _lib.ensure_device(0)
    gen = torch.Generator().manual_seed(9)
    for n, rows in ((1, 1), (77, 10), (3000, 500)):
        for dim in (1, 2, 3, 4, 5, 7, 8, 9, 12, 15, 16, 17, 31, 33, 63, 65, 130, 513):
            for gap in (0, 1, 6):
                table = torch.randn(rows, dim, device=DEV).to(dtype)
                idx = indices(n, rows, gen)
                buf, part = place(n * (dim + gap), dtype, dim % 5)
                assert lib.nr_embedding_fwd(table.data_ptr(), code, rows, dim, dim, idx.data_ptr(), 8, n, 1.0, part.data_ptr(), dim + gap,
                                            torch.cuda.current_stream().cuda_stream) == 0
                out = part.view(n, dim + gap)
                assert untouched(buf, part) and bool((out[:, dim:] == KNOWN).all()), (n, dim, gap)
                assert torch.equal(out[:, :dim], table[idx]), (n, dim, gap)


@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
def test_clipped_places(dtype):
    """Lists whose places lie in one bucket, a few elements apart: the elements between them stay."""
    sizes = [1, 2, 3, 5, 7, 8, 9, 15, 17, 255, 2047, 2048, 2049, 8191, 8193, 100003] + [3 + k % 11 for k in range(90)]
    for otype in (F32, BF16, F16):
        grads = [(torch.randn(s + 1, device=DEV) / 8).to(dtype)[1:] for s in sizes]
        gaps = [1 + k % 7 for k in range(len(sizes))]
        buf, part = place(sum(sizes) + sum(gaps), otype, 1)
        outs, mask, at = [], torch.ones(part.numel(), dtype=torch.bool, device=DEV), 0
        for s, gap in zip(sizes, gaps):
            outs.append(part[at:at + s])
            mask[at:at + s] = False
            at += s + gap
        for norm_type in (2.0, float("inf")):
            part.fill_(KNOWN)
            _, f = ops.clip_factor(grads, 0.5, norm_type)
            ops.clip_grads(grads, 0.5, norm_type, out=outs)
            assert untouched(buf, part) and bool((part[mask] == KNOWN).all()), otype
            assert all(torch.equal(o, (g.float() * f).to(otype)) for o, g in zip(outs, grads))
        if otype == dtype:  # in place
            part.fill_(KNOWN)
            ops.clip_grads(outs, 1.0)
            assert untouched(buf, part) and bool((part[mask] == KNOWN).all())


def test_norm_workspace_and_result():
    lib = _lib.lib()
    _lib.ensure_device(0)
    for sizes in ([1], [5, 0, 70000], [7] * 300, [40_000_000, 3]):
        grads = [torch.randn(s, device=DEV) for s in sizes]
        lst = ops._GradList(grads, "gradients")
        need = lib.nr_grad_norm_workspace_bytes(lst.arrays[1], lst.count)
        ws = torch.full((need + 4096,), 0xA5, device=DEV, dtype=torch.uint8)
        buf, result = place(2, F32, 1)
        for scaled in (False, True):
            outs = ops._GradList([torch.empty_like(g) for g in grads], "out")
            st = torch.cuda.current_stream().cuda_stream
            if scaled:
                rc = lib.nr_grad_clip(lst.arrays[0], outs.arrays[0], lst.arrays[1], lst.arrays[2], outs.arrays[2], lst.count, 2, 0.5, result.data_ptr(),
                                      ws.data_ptr(), st)
            else:
                rc = lib.nr_grad_norm(lst.arrays[0], lst.arrays[1], lst.arrays[2], lst.count, 2, 0.5, result.data_ptr(), ws.data_ptr(), st)
            assert rc == 0 and untouched(buf, result) and bool((ws[need:] == 0xA5).all()), sizes
            assert torch.equal(result[0], ops.grad_norm(grads)), sizes


@pytest.mark.parametrize("dtype", [F32, BF16], ids=str)
@pytest.mark.parametrize("n,rows", [(20, 3), (17000, 2), (17000, 700)])
def test_widest_rows(n, rows, dtype):
    """65 536 columns, the widest row there is, in each of the three ways; one row of gradient stands for all (stride 0), whole numbers."""
    gen = torch.Generator().manual_seed(n)
    idx, row = indices(n, rows, gen), torch.randint(-2, 3, (1, 65536), generator=gen).to(dtype).to(DEV)
    buf, part = place(rows * 65536, F32, 3)
    ops.embedding_grad(row.expand(n, 65536), idx, rows, out=part.view(rows, 65536))
    assert untouched(buf, part)
    assert torch.equal(part.view(rows, 65536), torch.bincount(idx, minlength=rows)[:, None].float() * row.float())


@pytest.mark.parametrize("n,rows", [(16, 5), (3000, 70000), (17000, 60), (17000, 900000)])
def test_indices_at_the_ends_of_their_types(n, rows):
    """The lowest and highest values of the index types lie in no table: rows of NaN, and nothing of theirs in a gradient."""
    gen = torch.Generator().manual_seed(n)
    for itype in (torch.int32, torch.int64):
        ends, inside = torch.iinfo(itype), torch.randint(0, rows, (n,), generator=gen)
        idx = inside.to(itype)
        far = torch.rand(n, generator=gen) < 0.3
        values = torch.tensor([ends.min, ends.min + 1, ends.max, ends.max - 1, -1, rows], dtype=itype)
        idx[far] = values[torch.randint(0, 6, (int(far.sum()),), generator=gen)]
        grad = torch.randint(-2, 3, (n, 24), generator=gen).float()
        want = torch.zeros(rows, 24).index_add_(0, inside[~far], grad[~far])
        assert torch.equal(ops.embedding_grad(grad.to(DEV), idx.to(DEV), rows).cpu(), want), itype
        table = torch.randn(rows, 24, generator=gen)
        got = ops.embedding(table.to(DEV), idx.to(DEV)).cpu()
        assert torch.equal(got[~far], table[inside[~far]]) and bool(torch.isnan(got[far]).all()), itype


def test_norm_and_clip_of_a_tensor_beyond_32_bits():
    x = torch.zeros((1 << 31) + 70001, device=DEV, dtype=BF16)
    tail = torch.tensor([12.0], device=DEV)
    x[0], x[-1] = -4.0, 3.0
    assert float(ops.grad_norm([x, tail])) == 13.0 and float(ops.grad_norm([x], 1.0)) == 7.0 and float(ops.grad_norm([x], float("inf"))) == 4.0
    out = torch.full((x.numel() + 1,), KNOWN, device=DEV, dtype=BF16)
    ops.clip_grads([x, tail], 6.5, out=[out[:-1], torch.empty_like(tail)])
    assert float(out[0]) == -2.0 and float(out[-2]) == 1.5 and float(out[-1]) == KNOWN and int(torch.count_nonzero(out[:-1])) == 2
    ops.clip_grads([x, tail], 6.5)
    assert float(x[0]) == -2.0 and float(x[-1]) == 1.5
    assert abs(float(tail) - 6.0) <= 6.0 * (1e-6 / 13.0 + 2.0 ** -23)  # (the factor is 6.5 / (13 + 1e-6), rounded once, and its product once)
