"""CPU (no GPU): no derivative through the embedding, norm and clipping entry points is lost without an error."""
import pytest
import torch
from torch.autograd import forward_ad

from neuradar_amd import _lib, ops


@pytest.fixture
def rows_on_the_cpu(monkeypatch):
    """ops.embedding with its launch replaced by torch on detached values (what the kernel does: it sees addresses)."""
    monkeypatch.setattr(ops, "_float_rows", lambda t, what: t)
    monkeypatch.setattr(ops, "_row_index", lambda idx, device: idx)
    monkeypatch.setattr(ops, "_embedding_rows", lambda table, idx, scale: forward_ad.unpack_dual(table).primal.detach()[idx] * scale)


def test_a_tangent_is_not_dropped(rows_on_the_cpu):
    table, idx = torch.randn(4, 3), torch.tensor([1, 1, 3])
    for requires_grad in (False, True):
        with forward_ad.dual_level():
            dual = forward_ad.make_dual(table.clone().requires_grad_(requires_grad), torch.ones(4, 3))
            with pytest.raises(NotImplementedError):
                ops.embedding(dual, idx, 2.0)
            with torch.no_grad(), pytest.raises(NotImplementedError):  # (forward mode goes on under no_grad)
                ops.embedding(dual, idx, 2.0)
            assert torch.equal(ops.embedding(table, idx, 2.0), table[idx] * 2.0)  # a tensor without a tangent
    assert ops.embedding(table, idx).grad_fn is None
    leaf = table.clone().requires_grad_()
    assert ops.embedding(leaf, idx).grad_fn is not None
    with torch.no_grad():
        assert ops.embedding(leaf, idx).grad_fn is None


def test_calls_without_a_derivative_refuse_tensors_that_autograd_follows():
    leaf, plain, idx = torch.randn(3, 2, requires_grad=True), torch.randn(3, 2), torch.tensor([0, 1, 1])
    calls = [lambda x: ops.grad_norm([x, plain]), lambda x: ops.clip_factor([x], 1.0), lambda x: ops.clip_grads([x], 1.0),
             lambda x: ops.clip_grads([x], 1.0, out=[plain]), lambda x: ops.embedding_grad(x, idx, 4),
             lambda x: ops.embedding_grad(plain, idx, 3, out=x)]
    for call in calls:
        for x in (leaf, leaf * 2.0):
            with pytest.raises(RuntimeError, match="derivative"):
                call(x)
        with forward_ad.dual_level(), pytest.raises(RuntimeError, match="derivative"):
            call(forward_ad.make_dual(plain.clone(), torch.ones(3, 2)))
        with torch.no_grad(), pytest.raises(RuntimeError, match="no CPU path"):  # (not followed: on to the next check)
            call(leaf)


def test_written_tensors_are_marked():
    x, y = torch.randn(3), torch.randn(2)
    before = x._version, y._version
    with torch.inference_mode():
        inferred = torch.randn(2)  # (has no counter)
    assert _lib.tensors().nr_mark_written([x, inferred, y]) == 0
    assert x._version > before[0] and y._version > before[1]
    leaf = torch.randn(3, requires_grad=True)
    (g,) = torch.autograd.grad((leaf ** 3).sum(), leaf, create_graph=True)
    z = (g * g).sum()  # saves g
    _lib.tensors().nr_mark_written([g])
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        z.backward()
