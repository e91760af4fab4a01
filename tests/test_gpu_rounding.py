"""GPU: what an element becomes does not depend on where in its tensor it lies -- in a whole vector, in a tensor's end, in a row's."""
import numpy as np
import pytest
import torch

from neuradar_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def between(factor, count, seed):
    """fp32 values whose product with `factor` (fp32), rounded to fp32 and then to fp16, is another one than rounded to fp16 at once."""
    rng, found = np.random.default_rng(seed), []
    while sum(len(f) for f in found) < count:
        x = rng.uniform(0.5, 900.0, 1 << 22).astype(np.float32)
        exact = x.astype(np.float64) * np.float64(factor)  # (48 bits: exact)
        found.append(x[exact.astype(np.float32).astype(np.float16) != exact.astype(np.float16)])
    return torch.from_numpy(np.concatenate(found)[:count])


def test_clipped_to_fp16():
    """The factor of the largest magnitude, 1 024 in a tensor of its own, does not depend on the other values."""
    top = torch.full((1,), 1024.0, device=DEV)
    factor = ops.clip_factor([top], 333.25, float("inf"))[1]
    x = between(np.float32(float(factor)), 3000, 0)
    want = (x * float(factor)).to(torch.float16)  # (torch multiplies in fp32 and rounds the product)
    assert torch.equal(want.float(), (x.to(DEV) * factor).to(torch.float16).float().cpu())
    for size in (1, 3, 4, 7, 100, 3000):
        grads = [top, *x.to(DEV).split(size)]
        out = [torch.empty(len(g), device=DEV, dtype=torch.float16) for g in grads]
        ops.clip_grads(grads, 333.25, float("inf"), out=out)
        assert torch.equal(torch.cat(out[1:]).cpu(), want), size


@pytest.mark.parametrize("accumulate", [False, True])
def test_gradient_rows_in_fp16(accumulate):
    scale = np.float32(0.3271)
    x = between(scale, 3000, 1)
    want = (x * float(scale)).to(torch.float16)
    for dim in (1, 3, 4, 5, 8, 12, 100):
        n = 3000 // dim
        idx = torch.arange(n, device=DEV)
        out = torch.zeros(n, dim, device=DEV, dtype=torch.float16) if accumulate else None
        got = ops.embedding_grad(x[:n * dim].view(n, dim).to(DEV), idx, n, float(scale), out=out, accumulate=accumulate, dtype=torch.float16)
        assert torch.equal(got.cpu().view(-1), want[:n * dim]), dim
