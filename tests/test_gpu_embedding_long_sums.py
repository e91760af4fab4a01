"""GPU: an embedding gradient's long sums keep fp32's precision.  Sums are held in 64 bits; they are rounded to fp32 where they leave a block
for the workspace and once for the result, and, for 16-bit rows, where they pass between the groups of a block.

Tolerances, for addends that are not negative (no cancellation, so every rounding is relative to the total): without a workspace
2^-24, the result's own rounding; with one (chunks of the indices, of 16 000 on one row too, or the sort) 2 * 2^-24; 16-bit rows another log2 of 1 024 groups, a tail and a head: 13 * 2^-24 more.  In fp32 alone thousands of
addends are off by several 2^-24 of their sum (this is what the test is for)."""
import pytest
import torch

from neuradar_amd import _lib, ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16


@pytest.mark.parametrize("n,rows,dim", [(16000, 1, 33), (16000, 3, 16), (16000, 300, 16), (100003, 7, 257), (100003, 1, 8), (262144, 5, 30), (70001, 500000, 40)])
@pytest.mark.parametrize("dtype", [F32, BF16, F16], ids=str)
def test_long_sums(n, rows, dim, dtype):
    gen = torch.Generator().manual_seed(n + rows)
    grad = (torch.rand(n, dim, generator=gen) + 2.0 ** -6).to(dtype)
    idx = torch.randint(0, rows, (n,), generator=gen)
    if rows > 1000:
        idx[torch.rand(n, generator=gen) < 0.9] = rows // 2  # one row has nearly all of them: it crosses every block of the sort
    want = torch.zeros(rows, dim, dtype=torch.float64).index_add_(0, idx, grad.double())
    got = ops.embedding_grad(grad.to(DEV), idx.to(DEV), rows, dtype=F32).double().cpu()
    roundings = 1 if _lib.lib().nr_embedding_bwd_workspace_bytes(rows, dim, n, _lib.NR_DTYPES[str(dtype)[6:]]) == 0 else 2
    half_steps = roundings + (0 if dtype == F32 else 13)
    worst = float(((got - want).abs() / want.clamp_min(1e-30)).max()) * 2.0 ** 24
    assert worst <= half_steps * (1 + 2.0 ** -20), worst
    before = torch.rand(rows, dim, generator=gen)
    out = before.to(DEV)
    ops.embedding_grad(grad.to(DEV), idx.to(DEV), rows, 0.75, out=out, accumulate=True)
    want = want * 0.75 + before.double()
    worst = float(((out.double().cpu() - want).abs() / want.clamp_min(1e-30)).max()) * 2.0 ** 24
    assert worst <= (half_steps + 1) * (1 + 2.0 ** -20), worst  # (rounded once more: added to what is there in fp32)
