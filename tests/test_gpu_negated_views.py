"""GPU: a view that holds its values negated (the imaginary part of a conjugate is one) is read and written as what it stands for."""
import pytest
import torch

from neuradar_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def views():
    """(view, its values): contiguous and with holes."""
    base = torch.randn(6, 8, device=DEV)
    z = torch.randn(6, 8, device=DEV, dtype=torch.complex64)
    return [(torch._neg_view(base), -base), (z.conj().imag, -z.imag.clone())]


def test_rows_and_gradient():
    idx = torch.tensor([5, 0, 0, 3, 2, 0], device=DEV)
    for view, values in views():
        assert view.is_neg() and not values.is_neg()
        assert torch.equal(ops.embedding(view, idx, 2.0), values[idx] * 2.0)
        assert torch.equal(ops.embedding_grad(view, idx, 7), ops.embedding_grad(values.contiguous(), idx, 7))
    with pytest.raises(RuntimeError, match="contiguous"):
        ops.embedding_grad(torch.ones(6, 8, device=DEV), idx, 6, out=views()[0][0])


def test_norm_and_clipping():
    for view, values in views():
        values = values.contiguous()
        factor = float(ops.clip_factor([values], 0.5)[1])
        assert torch.equal(ops.grad_norm([view]), ops.grad_norm([values]))
        out = torch.empty(6, 8, device=DEV)
        ops.clip_grads([view], 0.5, out=[out])
        assert torch.equal(out, values * factor)
        place = torch._neg_view(torch.empty(6, 8, device=DEV))
        ops.clip_grads([values], 0.5, out=[place])
        assert torch.equal(place.resolve_neg(), values * factor)
        ops.clip_grads([view], 0.5)  # in place
        assert torch.equal(view.resolve_neg(), values * factor)
