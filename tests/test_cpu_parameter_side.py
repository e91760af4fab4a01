"""CPU (no GPU): what the embedding, gradient-norm and clipping entry points refuse before anything is launched."""
from array import array

import pytest
import torch

from neuradar_amd import _lib, ops

E = _lib.NR_EINVAL
BIG = 1 << 20  # any non-null, aligned address: refused before it is read


def test_embedding_entry_points_refuse_bad_arguments():
    lib = _lib.lib()

    def fwd(table=BIG, dtype=0, rows=10, dim=8, stride=8, idx=BIG, idx_bytes=8, n=4, out=BIG, out_stride=8):
        return lib.nr_embedding_fwd(table, dtype, rows, dim, stride, idx, idx_bytes, n, 1.0, out, out_stride, None)

    def bwd(grad=BIG, dtype=0, stride=8, idx=BIG, idx_bytes=8, n=20000, rows=10, dim=8, out=BIG, out_dtype=0, workspace=BIG):
        return lib.nr_embedding_bwd(grad, dtype, stride, idx, idx_bytes, n, rows, dim, 1.0, -1, out, out_dtype, 1, workspace, None)

    for kw in (dict(dtype=3), dict(dtype=-1), dict(rows=-1), dict(rows=0x7FFFFFFF), dict(dim=-1), dict(dim=65537), dict(idx_bytes=2), dict(n=-1),
               dict(n=0x80000000), dict(idx=None), dict(out=None), dict(table=None), dict(out_stride=7), dict(stride=-1),
               dict(n=0x7FFFFFFF, dim=65536, out_stride=65536),
               dict(idx=BIG + 4), dict(table=BIG + 2), dict(out=BIG + 1)):
        assert fwd(**kw) == E, kw
    assert fwd(n=0) == 0 and fwd(dim=0, out_stride=0) == 0
    for kw in (dict(dtype=3), dict(out_dtype=7), dict(rows=-1), dict(rows=0x7FFFFFFF), dict(dim=-1), dict(dim=65537), dict(idx_bytes=1), dict(n=-1),
               dict(n=0x80000000), dict(grad=None), dict(idx=None), dict(out=None), dict(workspace=None), dict(workspace=BIG + 8), dict(stride=-1),
               dict(out=BIG + 2), dict(grad=BIG + 2), dict(idx=BIG + 4)):
        assert bwd(**kw) == E, kw
    assert bwd(rows=0) == 0 and bwd(dim=0) == 0 and bwd(n=0) == 0
    assert lib.nr_embedding_bwd_workspace_bytes(10, 8, -1, 0) == E and lib.nr_embedding_bwd_workspace_bytes(10, 8, 4, 5) == E
    assert lib.nr_embedding_bwd_workspace_bytes(10, 8, 0, 0) == 0 and lib.nr_embedding_bwd_workspace_bytes(10, 8, 20000, 0) > 0


def test_norm_entry_points_refuse_bad_arguments():
    lib = _lib.lib()
    ptrs, numel, dtypes = array("q", [BIG, BIG]), array("q", [4, 4]), array("i", [0, 1])

    def at(a):
        return a.buffer_info()[0]

    def norm(p=ptrs, n=numel, d=dtypes, count=2, kind=2, max_norm=1.0, result=BIG, workspace=BIG):
        return lib.nr_grad_norm(p and at(p), n and at(n), d and at(d), count, kind, max_norm, result, workspace, None)

    def scale(p=ptrs, o=ptrs, d=dtypes, od=dtypes, n=numel, result=BIG):
        return lib.nr_grad_scale(at(p), o and at(o), at(n), at(d), od and at(od), 2, result, None)

    for kw in (dict(p=None), dict(n=None), dict(d=None), dict(count=-1), dict(kind=3), dict(kind=-1), dict(max_norm=-1.0),
               dict(max_norm=float("nan")), dict(result=None), dict(workspace=None), dict(workspace=BIG + 4), dict(p=array("q", [BIG, 0])),
               dict(p=array("q", [BIG + 2, BIG])), dict(d=array("i", [0, 9])), dict(n=array("q", [4, -1]))):
        assert norm(**kw) == E, kw
    for kw in (dict(o=None), dict(od=None), dict(result=None), dict(o=array("q", [0, BIG])), dict(o=array("q", [BIG, BIG + 1]))):
        assert scale(**kw) == E, kw
    def clip(o=ptrs, od=dtypes, kind=2, max_norm=1.0, result=BIG, workspace=BIG):
        return lib.nr_grad_clip(at(ptrs), o and at(o), at(numel), at(dtypes), od and at(od), 2, kind, max_norm, result, workspace, None)

    for kw in (dict(o=None), dict(od=None), dict(kind=5), dict(max_norm=-2.0), dict(result=None), dict(workspace=None), dict(o=array("q", [BIG, BIG + 1]))):
        assert clip(**kw) == E, kw
    assert lib.nr_grad_norm_workspace_bytes(at(numel), -1) == E and lib.nr_grad_norm_workspace_bytes(at(array("q", [-5])), 1) == E
    assert lib.nr_grad_norm_workspace_bytes(None, 0) == 0 and lib.nr_grad_norm_workspace_bytes(at(numel), 2) == 16


def test_cpu_tensors_are_refused():
    table, idx = torch.zeros(4, 2), torch.zeros(3, dtype=torch.int64)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.embedding(table, idx)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.embedding_grad(torch.zeros(3, 2), idx, 4)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.grad_norm([table])
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.clip_grads([table], 1.0)
    p = torch.nn.Parameter(torch.zeros(3))
    assert float(ops.clip_grad_norm_([p], 1.0)) == 0.0  # (no gradient: nothing to do)
    p.grad = torch.ones(3)
    with pytest.raises(RuntimeError, match="no CPU path"):
        ops.clip_grad_norm_([p], 1.0)
    with pytest.raises(RuntimeError, match="does not fit"):
        ops.embedding_grad(torch.zeros(2, 2), idx, 4)
    with pytest.raises(RuntimeError, match="float32, bfloat16 or float16"):
        ops.grad_norm([table.double()])


def test_clipping_needs_the_whole_group():
    from neuradar_amd.step import FlatAdam

    p = torch.nn.Parameter(torch.ones(8))
    for bad in (-1.0, float("nan")):
        with pytest.raises(ValueError, match="max_norm"):
            FlatAdam([p], lr=1e-2, max_norm=bad)
    opt = FlatAdam([p], lr=1e-2, max_norm=1.0)
    with pytest.raises(RuntimeError, match="whole group"):
        opt.step_buffer(0)
    with pytest.raises(RuntimeError, match="whole group"):
        opt.step_buffer_split(0, 1, None)
    with pytest.raises(RuntimeError, match="shard"):
        opt.shard_buffer(0, 0, 2)
    with pytest.raises(RuntimeError, match="no gradients"):
        ops.clip_factor([], 1.0)


def test_embedding_module_mirrors_the_reference():
    from neuradar_amd.encodings import Embedding

    emb = Embedding(7, 3)
    assert list(emb.state_dict()) == ["embedding.weight"] and emb.get_out_dim() == 3 and emb.in_dim == 7
    assert torch.equal(emb.mean(dim=0), emb.embedding.weight.mean(0))
    assert not bool(Embedding(7, 3, padding_idx=2).embedding.weight[2].any())
    with pytest.raises(RuntimeError, match="no CPU path"):
        emb(torch.tensor([1, 2]))
