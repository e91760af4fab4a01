"""GPU: the global norm of many gradients and their clipping (ops.grad_norm, clip_grads, clip_grad_norm_) against 64 bits and torch.

Tolerances.  Sums are in fp64 (nothing at fp32's scale); the norm is rounded to fp32 once: 2^-24 relative.  The factor is rounded
once and multiplied once in fp32, the product rounded to its type: 2^-23 and half a step of the type."""
import math

import pytest
import torch

from neuradar_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
F32, BF16, F16 = torch.float32, torch.bfloat16, torch.float16
INF = float("inf")


def half_step(dtype):
    return torch.finfo(dtype).eps / 2


def norm64(grads, p):
    x = torch.cat([g.detach().double().cpu().reshape(-1) for g in grads])
    if p == INF:
        return float(x.abs().max()) if x.numel() else 0.0
    return float(x.abs().sum()) if p == 1 else float(x.square().sum().sqrt())


def ragged(sizes, dtypes, seed=0):
    gen = torch.Generator().manual_seed(seed)
    return [(torch.randn(s, generator=gen) * 10.0 ** (-(k % 4))).to(dtypes[k % len(dtypes)]).to(DEV) for k, s in enumerate(sizes)]


def check_clip(out, grads, max_norm, p, norm):
    n64 = norm64(grads, p)
    assert abs(float(norm) - n64) <= n64 * 2.0 ** -23, (float(norm), n64)
    f = min(1.0, max_norm / (n64 + 1e-6))
    for o, g in zip(out, grads):
        want = g.double().cpu() * f
        tol = want.abs() * (half_step(o.dtype) * (1 + 2.0 ** -20) + 2.0 ** -23) + torch.finfo(o.dtype).smallest_normal * half_step(o.dtype)
        assert bool(((o.double().cpu() - want).abs() <= tol).all())


SIZES = [[1], [7], [8], [2048], [2049], [100003], [0, 5, 0, 1], [3] * 95, [3] * 96, [17] * 97, [1 + 13 * k for k in range(290)],
         [3000001, 1, 64, 4099]]


@pytest.mark.parametrize("sizes", SIZES, ids=lambda s: f"{len(s)}x{s[0]}")
@pytest.mark.parametrize("dtypes", [(F32,), (BF16,), (F16,), (F32, BF16, F16)], ids=["f32", "bf16", "f16", "mixed"])
def test_norm_and_clip(sizes, dtypes):
    grads = ragged(sizes, dtypes)
    for p in (2.0, 1.0, INF):
        n64 = norm64(grads, p)
        norm = ops.grad_norm(grads, p)
        assert norm.shape == () and norm.dtype == F32 and abs(float(norm) - n64) <= n64 * 2.0 ** -23
        assert torch.equal(norm, ops.grad_norm(grads, p))
        for ratio in (0.3, 2.0):
            out = [torch.full_like(g, 9.0) for g in grads]
            check_clip(out, grads, ratio * n64, p, ops.clip_grads(grads, ratio * n64, p, out=out))
            mine = [g.clone() for g in grads]
            assert torch.equal(norm, ops.clip_grads(mine, ratio * n64, p))  # (with the factor formed in the scaling launch as well)
            assert all(torch.equal(a, b) for a, b in zip(mine, out)) and (ratio < 1 or all(torch.equal(a, b) for a, b in zip(mine, grads)))


def test_matches_torch_on_parameters():
    torch.manual_seed(1)
    params = [torch.nn.Parameter(torch.randn(*s, device=DEV)) for s in ((32, 32), (32,), (3, 5, 7), (1,), (32, 32, 7, 7))]
    params.append(torch.nn.Parameter(torch.randn(4, device=DEV)))  # has no gradient
    params[4].data = params[4].data.contiguous(memory_format=torch.channels_last)
    for p in params[:-1]:
        p.grad = torch.randn_like(p)
    assert not params[4].grad.is_contiguous()
    want = [p.grad.clone() for p in params[:-1]]
    n64 = norm64(want, 2.0)
    norm = ops.clip_grad_norm_(iter(params), 1.25, error_if_nonfinite=True)
    check_clip([p.grad for p in params[:-1]], want, 1.25, 2.0, norm)
    for p, g in zip(params, want):
        p.grad = g.clone()
    ref = torch.nn.utils.clip_grad_norm_(params, 1.25)
    assert abs(float(ref) - n64) <= 1e-5 * n64 and params[-1].grad is None
    assert float(ops.clip_grad_norm_(params[-1:], 1.0)) == 0.0
    lone = params[0]
    before = lone.grad.clone()
    check_clip([lone.grad], [before], 0.1, 2.0, ops.clip_grad_norm_([lone, lone], 0.1))  # listed twice: counted once


def test_layouts():
    base = torch.randn(40, 50, device=DEV)
    holes, turned, off = base[:, 3:20], torch.randn(6, 9, device=DEV).t(), torch.randn(101, device=DEV)[1:]
    grads = [holes, turned, off]
    kept = [g.clone() for g in grads]
    edge = base[:, 20:].clone()
    check_clip(grads, kept, 0.7, 2.0, ops.clip_grads(grads, 0.7))
    assert torch.equal(base[:, 20:], edge)
    out = [torch.empty(40, 34, device=DEV, dtype=BF16)[:, ::2], torch.empty(9, 6, device=DEV), torch.empty(205, device=DEV, dtype=F16)[5:105]]
    now = [g.clone() for g in grads]
    check_clip(out, now, 0.2, 1.0, ops.clip_grads(grads, 0.2, 1.0, out=out))
    scalar = torch.tensor(-3.0, device=DEV)
    assert float(ops.grad_norm(scalar)) == 3.0 and float(ops.grad_norm([torch.empty(0, device=DEV)])) == 0.0


def test_extreme_values():
    big, small = torch.full((1000,), 3e38, device=DEV), torch.full((1000,), 1e-40, device=DEV)
    assert float(ops.grad_norm(big[:1])) == float(big[0])  # a square that fp32 does not hold
    assert float(ops.grad_norm(big)) == INF  # (the norm itself is beyond fp32)
    n = float(ops.grad_norm(small))
    assert abs(n - norm64([small], 2.0)) <= 2.0 ** -149
    for p in (2.0, 1.0, INF):
        bad = [torch.ones(5000, device=DEV), torch.ones(300, device=DEV, dtype=BF16)]
        bad[1][299] = INF
        assert float(ops.grad_norm(bad, p)) == INF
        out = [g.clone() for g in bad]
        ops.clip_grads(out, 1.0, p)  # factor 0: zeros, and inf * 0
        assert not bool(out[0].any()) and bool(torch.isnan(out[1][299])) and not bool(out[1][:299].any())
        bad[0][4999] = float("nan")
        assert math.isnan(float(ops.grad_norm(bad, p)))
        ops.clip_grads(bad, 1.0, p)
        assert bool(torch.isnan(bad[0]).all()) and bool(torch.isnan(bad[1]).all())
    with pytest.raises(RuntimeError, match="not finite"):
        q = torch.nn.Parameter(torch.ones(3, device=DEV))
        q.grad = torch.full((3,), INF, device=DEV)
        ops.clip_grad_norm_([q], 1.0, error_if_nonfinite=True)
    assert bool(torch.isinf(q.grad).all())
    zero = [torch.zeros(10, device=DEV)]
    assert float(ops.clip_grads(zero, 0.0)) == 0.0 and not bool(zero[0].any())
    one = [torch.ones(4, device=DEV)]
    ops.clip_grads(one, INF)
    assert bool((one[0] == 1).all())


def test_other_stream_and_replayed_graphs():
    grads = ragged([5000, 33, 70000] + [11] * 120, (F32, BF16))
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        norm = ops.grad_norm(grads)
    torch.cuda.current_stream().wait_stream(s)
    n64 = norm64(grads, 2.0)
    assert abs(float(norm) - n64) <= n64 * 2.0 ** -23
    graphs = []
    for ratio in (0.5, 0.25):
        out = [torch.empty_like(g) for g in grads]
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            norm = ops.clip_grads(grads, ratio, out=out)
        graphs.append((graph, ratio, out, norm))
    for k in range(3):
        for g, v in zip(grads, ragged([g.numel() for g in grads], (F32, BF16), seed=k + 5)):
            g.copy_(v)
        for graph, ratio, out, norm in graphs:
            graph.replay()
            torch.cuda.synchronize()
            eager = [torch.empty_like(g) for g in grads]
            n = ops.clip_grads(grads, ratio, out=eager)
            assert torch.equal(n, norm) and all(torch.equal(a, b) for a, b in zip(out, eager))
        check_clip(eager, grads, ratio, 2.0, n)


def test_refusals():
    g = torch.ones(6, device=DEV)
    for call, what in ((lambda: ops.grad_norm([g], 3.0), "norm_type"), (lambda: ops.clip_grads([g], -1.0), "max_norm"),
                       (lambda: ops.clip_grads([g], float("nan")), "max_norm"), (lambda: ops.clip_grads([g, g], 1.0), "listed twice"),
                       (lambda: ops.clip_grads([g, g + 1], 1.0, out=[g, g]), "listed twice"), (lambda: ops.clip_grads([g], 1.0, out=[g[:5]]), "same size"),
                       (lambda: ops.clip_grads([g], 1.0, out=[g, g + 1]), "same size"), (lambda: ops.clip_grads([g], 1.0, out=[g.double()]), "float32"),
                       (lambda: ops.grad_norm([g, torch.ones(2)]), "one device"), (lambda: ops.grad_norm([g.to_sparse()]), "."),
                       (lambda: ops.clip_grads([g.view(2, 3).t()], 1.0, out=[g.clone()]), "shapes")):
        with pytest.raises(RuntimeError, match=what):
            call()
    assert bool((g == 1).all())


def test_norm_and_scale_as_separate_calls():
    """The C entry points one after the other (a caller that keeps the factor): the same bits as in one call."""
    from neuradar_amd import _lib

    for sizes in ((5000, 7, 123457), (40000000, 3), (75000001, 5)):  # (few partial results, thousands, results beyond the caches)
        grads = ragged(sizes, (F32, BF16))
        lst = ops._GradList(grads, "gradients")
        outs = [torch.empty_like(g) for g in grads]
        dst = ops._GradList(outs, "out")
        result = ops._norm_and_factor(lst, 0.5, 2.0, grads[0].device)
        lib = _lib.lib()
        assert lib.nr_grad_scale(lst.arrays[0], dst.arrays[0], lst.arrays[1], lst.arrays[2], dst.arrays[2], 2 if len(sizes) == 2 else 3, result.data_ptr(),
                                 torch.cuda.current_stream().cuda_stream) == 0
        other = [torch.empty_like(g) for g in grads]
        assert torch.equal(ops.clip_grads(grads, 0.5, out=other), result[0])
        assert all(torch.equal(a, b) and torch.equal(a, (g.float() * result[1]).to(g.dtype)) for a, b, g in zip(outs, other, grads))
