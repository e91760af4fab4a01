"""CPU (no GPU): where the guard allocator and the red-zone harness put a buffer in its region.  What they find rests on two facts: nothing
is mapped behind a region (the runtime's), and a buffer ends with its region (this arithmetic)."""
import ctypes

import pytest

import test_gpu_redzone as redzone

GRANULE = 2 << 20
SIZES = [1, 2, 15, 16, 17, 4096, 8192 + 2, GRANULE - 512, GRANULE - 511, GRANULE - 64, GRANULE - 63, GRANULE - 1, GRANULE, GRANULE + 1, 5 * GRANULE + 4]


@pytest.mark.parametrize("size", SIZES)
def test_a_guarded_tensor_ends_with_its_region(size):
    redzone._ensure_guard_so()
    guard = ctypes.CDLL(redzone.GUARD_SO)
    region, offset, span = (ctypes.c_size_t() for _ in range(3))
    guard.guard_layout.argtypes = [ctypes.c_size_t] + [ctypes.POINTER(ctypes.c_size_t)] * 3
    guard.guard_layout.restype = None
    guard.guard_layout(size, ctypes.byref(region), ctypes.byref(offset), ctypes.byref(span))
    region, offset, span = region.value, offset.value, span.value
    assert offset + span == region and region % GRANULE == 0 and region - span < GRANULE + 64
    assert size <= span < size + 16 and offset % 16 == 0  # (the slack behind an odd size is less than a vector)
    assert offset >= 64  # (the canary)


@pytest.mark.parametrize("size", [0] + SIZES)
def test_a_red_zone_buffer_ends_with_its_region(size):
    region, offset = redzone.place(size)
    assert region % GRANULE == 0 and offset % 16 == 0 and 0 <= region - (offset + size) < 16
    assert offset >= 256  # (the canaries in front that are compared)


def test_no_helper_tells_a_kernel_of_elements_that_its_buffer_lacks():
    assert "lie" not in redzone._case.__code__.co_varnames and "overrun" not in redzone._guarded_cnn_leg.__code__.co_varnames
