"""GPU: a tensor written by clipping or by a gradient into `out` is a write in place to autograd, and nothing that it follows is taken."""
import pytest
import torch
from torch.autograd import forward_ad

from neuradar_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"


def test_a_saved_gradient_that_was_clipped_raises():
    """(g of create_graph is saved by g * g: clipped in place, its product's backward would use other values than it was formed of)"""
    for clip in (lambda p, g: ops.clip_grad_norm_([p], 0.1), lambda p, g: ops.clip_grads([g], 0.1), lambda p, g: ops.clip_grads([g.detach()], 0.1),
                 lambda p, g: ops.clip_grads([torch.ones_like(g)], 0.1, out=[g])):
        leaf = torch.nn.Parameter(torch.randn(7, 5, device=DEV))
        (g,) = torch.autograd.grad((leaf ** 3).sum(), leaf, create_graph=True)
        leaf.grad = g
        z = (g * g).sum()
        with torch.no_grad():
            clip(leaf, g)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            z.backward()
    x = torch.randn(4, 6, device=DEV)  # holes: clipped through a copy
    before = x._version
    ops.clip_grads([x[:, ::2]], 0.1)
    assert x._version > before


def test_counters_go_up_for_what_is_written_only():
    g, out = [torch.randn(5, device=DEV), torch.randn(3, device=DEV)], [torch.empty(5, device=DEV), torch.empty(3, device=DEV)]
    read, written = [t._version for t in g], [t._version for t in out]
    ops.grad_norm(g)
    ops.clip_factor(g, 1.0)
    ops.clip_grads(g, 1.0, out=out)
    assert [t._version for t in g] == read and all(t._version > v for t, v in zip(out, written))
    grad, idx, table = torch.randn(9, 4, device=DEV), torch.randint(0, 6, (9,), device=DEV), torch.zeros(6, 4, device=DEV)
    before = table._version, grad._version
    ops.embedding_grad(grad, idx, 6, out=table)
    assert table._version > before[0] and grad._version == before[1]


def test_followed_tensors_are_refused():
    leaf, plain, idx = torch.randn(3, 2, device=DEV, requires_grad=True), torch.randn(3, 2, device=DEV), torch.tensor([0, 1, 1], device=DEV)
    kept = plain.clone()
    calls = [lambda x: ops.grad_norm([plain, x]), lambda x: ops.clip_factor([plain, x], 1.0), lambda x: ops.clip_grads([plain, x], 1.0),
             lambda x: ops.clip_grads([x], 1.0, out=[plain]), lambda x: ops.clip_grads([plain], 1.0, out=[x]), lambda x: ops.embedding_grad(x, idx, 4),
             lambda x: ops.embedding_grad(plain, idx, 3, out=x)]
    for call in calls:
        for x in (leaf, leaf * 2.0):
            with pytest.raises(RuntimeError, match="derivative"):
                call(x)
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="derivative"):
            call(forward_ad.make_dual(plain.clone(), torch.ones(3, 2, device=DEV)))
    assert torch.equal(plain, kept)
    with torch.no_grad():
        assert float(ops.grad_norm([leaf])) > 0.0 and ops.embedding_grad(leaf, idx, 4).shape == (4, 2)
    with forward_ad.dual_level(), pytest.raises(NotImplementedError):
        ops.embedding(forward_ad.make_dual(plain.clone(), torch.ones(3, 2, device=DEV)), idx)
