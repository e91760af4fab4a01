"""GPU: results that share memory with what is read are refused before anything is launched; the calls next to those are not."""
import pytest
import torch

from neuradar_amd import ops

pytestmark = pytest.mark.gpu
DEV = "cuda:0"
BF16 = torch.bfloat16


def test_clipping_refuses_shared_memory():
    buf = torch.randn(4000, device=DEV)
    kept, a, b = buf.clone(), buf[:1000], buf[2000:3000]
    as_bf16 = buf.view(BF16)
    for grads, out, what in (([a], [as_bf16[:1000]], "a gradient"), ([a], [as_bf16[1000:2000]], "a gradient"), ([a], [buf[1:1001]], "a gradient"),
                             ([a], [buf[999:1999]], "a gradient"), ([as_bf16[:1000]], [buf[:1000]], "a gradient"), ([a, b], [b, a], "a gradient"),
                             ([a, b], [buf[3000:], a], "a gradient"), ([a, b], [buf[3000:], buf[3000:]], "listed twice"),
                             ([a, b], [buf[1000:2000], buf[1999:2999]], "listed twice"), ([a, buf[500:1500]], None, "listed twice"),
                             ([buf[:10:2], buf[:10:2]], None, "listed twice"), ([a], [buf[3000:3001].expand(1000)], "in one place"),
                             ([a[:1].expand(5)], None, "in one place")):
        for ratio in (0.01, 1e9):
            with pytest.raises(RuntimeError, match=what):
                ops.clip_grads(grads, ratio, out=out)
    assert torch.equal(buf, kept)


def test_clipping_beside_and_in_place():
    buf = torch.randn(4000, device=DEV)
    a, b, behind = buf[:1000], buf[2000:3000], buf[1000:2000]
    want = buf.clone()
    f = float(ops.clip_factor([a, b], 0.5)[1])
    want[1000:2000], want[2000:3000] = want[:1000] * f, want[2000:3000] * f
    ops.clip_grads([a, b], 0.5, out=[behind, b])  # right behind a gradient; one of two in place
    assert torch.equal(buf, want)
    halves = torch.randn(6, 8, device=DEV)
    want = halves * float(ops.clip_factor([halves], 0.5)[1])
    ops.clip_grads([halves[:, ::2], halves[:, 1::2]], 0.5)  # interleaved: every element once
    assert torch.allclose(halves, want, rtol=2.0 ** -21, atol=0)
    empty = torch.empty(0, device=DEV)
    assert float(ops.clip_grads([empty, empty], 1.0)) == 0.0


def test_embedding_gradient_refuses_shared_memory():
    idx = torch.tensor([0, 1, 1, 3], device=DEV)
    buf = torch.randn(4 * 20, device=DEV)
    kept = buf.clone()
    wide = buf.view(4, 20)
    grad = wide[:, :8]
    for out in (buf[:32].view(4, 8), buf[30:62].view(4, 8), buf[40:72].view(4, 8), buf.view(BF16)[:32].view(4, 8)):
        for accumulate in (False, True):
            with pytest.raises(RuntimeError, match="share memory"):
                ops.embedding_grad(grad, idx, 4, out=out, accumulate=accumulate)
    with pytest.raises(RuntimeError, match="share memory"):
        ops.embedding_grad(torch.ones(4, 1, device=DEV), idx, 8, out=idx.view(torch.float32).view(8, 1))
    assert torch.equal(buf, kept)
    room = buf[8:16].view(1, 8)  # between two rows of grad
    want = (grad[idx == 0].sum(0), wide[1:].clone())
    ops.embedding_grad(grad, idx, 1, out=room)
    assert torch.equal(room[0], want[0]) and torch.equal(wide[1:], want[1]) and torch.equal(wide[0, :8], kept[:8])
