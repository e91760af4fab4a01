"""CPU (no GPU): what the clipping and the embedding gradient refuse because it shares memory, on addresses alone."""
from array import array

import pytest
import torch

from neuradar_amd import _lib, ops

BASE = 1 << 30
F32, BF16, F16 = 0, 1, 2
APART, TWICE, READ = 0, 1, 2


def shared(src, dst):
    """src, dst: (first byte behind BASE, type, elements) each."""
    cols = [array("q", [BASE + s[0] for s in src]), array("i", [s[1] for s in src]), array("q", [BASE + d[0] for d in dst]),
            array("i", [d[1] for d in dst]), array("q", [s[2] for s in src])]
    return _lib.tensors().nr_shared_memory(*(c.buffer_info()[0] for c in cols), len(src))


def by_bytes(src, dst):
    """The definition: which bytes are written, and by whom read."""
    size = lambda t: 4 if t == F32 else 2  # noqa: E731
    span = lambda t: set(range(t[0], t[0] + t[2] * size(t[1])))  # noqa: E731
    for i, d in enumerate(dst):
        if any(span(d) & span(e) for e in dst[:i]):
            return TWICE
    for i, s in enumerate(src):
        for j, d in enumerate(dst):
            if span(s) & span(d) and not (i == j and s == d):
                return READ
    return APART


@pytest.mark.parametrize("src,dst,want", [
    ([(0, F32, 8)], [(0, F32, 8)], APART),  # in place
    ([(0, F32, 8)], [(32, F32, 8)], APART),  # right behind it
    ([(0, F32, 8)], [(0, BF16, 8)], READ),  # a 16-bit view of the gradient's own memory
    ([(0, F32, 8)], [(16, BF16, 8)], READ),  # its second half
    ([(0, F32, 8)], [(4, F32, 8)], READ),  # one element off
    ([(32, BF16, 8)], [(0, F32, 8)], APART), ([(31 * 2, BF16, 8)], [(32, F32, 8)], READ),
    ([(0, F32, 8), (64, F32, 8)], [(0, F32, 8), (64, F32, 8)], APART), ([(0, F32, 8), (16, F32, 8)], [(0, F32, 8), (16, F32, 8)], TWICE),
    ([(0, F32, 8), (64, F32, 8)], [(64, F32, 8), (0, F32, 8)], READ),  # swapped
    ([(0, F32, 8), (64, F32, 8)], [(200, F32, 8), (200, F32, 8)], TWICE), ([(0, F32, 8), (64, F32, 8)], [(200, F32, 8), (228, F32, 8)], TWICE),
    ([(0, F32, 8), (64, F32, 8)], [(0, F32, 8), (200, F32, 8)], APART),  # one of two in place
    ([(0, F32, 8), (64, F32, 8)], [(200, F32, 8), (0, F32, 8)], READ), ([(0, F32, 0), (64, F32, 8)], [(64, F32, 0), (64, F32, 8)], APART)])
def test_lists(src, dst, want):
    assert shared(src, dst) == want == by_bytes(src, dst)
    assert shared(src[::-1], dst[::-1]) == want


def test_lists_against_the_definition():
    gen = torch.Generator().manual_seed(0)
    seen = set()
    for _ in range(4000):
        n = int(torch.randint(1, 5, (1,), generator=gen))
        draw = torch.randint(0, 40, (n, 2), generator=gen).tolist()
        kinds, sizes = torch.randint(0, 3, (n, 2), generator=gen).tolist(), torch.randint(0, 4, (n,), generator=gen).tolist()
        src = [(4 * d[0], k[0], z) for d, k, z in zip(draw, kinds, sizes)]
        dst = [s if d[1] < 20 else (4 * d[1], k[1], s[2]) for s, d, k in zip(src, draw, kinds)]
        got = shared(src, dst)
        assert got == by_bytes(src, dst), (src, dst)
        seen.add(got)
    assert seen == {APART, TWICE, READ}


def test_rows_and_a_result():
    """Rows of a wide buffer against a contiguous place anywhere in it: the bytes of both, compared as sets."""
    base = torch.arange(240, dtype=torch.float32)
    cells = lambda t: {t.data_ptr() + 4 * (sum(i * s for i, s in zip(at, t.stride()))) for at in [  # noqa: E731
        (i, j) for i in range(t.shape[0]) for j in range(t.shape[1])]}
    found = set()
    for n, dim, stride, at in ((5, 4, 10, 30), (5, 10, 10, 3), (1, 4, 0, 50), (6, 4, 0, 50), (4, 6, 3, 20), (3, 1, 40, 100), (0, 4, 10, 0), (3, 0, 10, 0)):
        rows = base.as_strided((n, dim), (stride, 1), at)
        for place in range(0, 200, 1):
            for shape in ((1, 3), (2, 3), (1, 0), (3, 13)):
                out = base[place:place + shape[0] * shape[1]].view(shape)
                want = bool(cells(rows) & cells(out))
                assert ops._shares_memory(rows, stride, out) == want, (n, dim, stride, at, place, shape)
                found.add(want)
    assert found == {True, False}


def test_c_entry_points_refuse_in_place_in_another_type():
    lib = _lib.lib()
    ptrs, numel, f32, bf16 = array("q", [BASE]), array("q", [8]), array("i", [F32]), array("i", [BF16])
    p, n, a, b = (x.buffer_info()[0] for x in (ptrs, numel, f32, bf16))
    assert lib.nr_grad_scale(p, p, n, a, b, 1, BASE, None) == _lib.NR_EINVAL
    assert lib.nr_grad_clip(p, p, n, b, a, 1, 2, 1.0, BASE, BASE, None) == _lib.NR_EINVAL
