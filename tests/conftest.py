"""Test-session plumbing.

* `gpu` marker; gpu tests are skipped (not failed) on a box without a GPU.
* ORDER: the golden parity of the hot path runs FIRST, the heavy multi-stream / full-size /
  subprocess tests LAST, so that one failure under `-x` cannot erase the parity evidence (round 4: a crash in test #128 of 314 left
  187 tests, all of test_gpu_parity.py among them, unreported).
* CRASH CONTAINMENT: on a GPU box the session runs its tests in ONE pytest-xdist worker process (`-n 1` semantics, set here because
  the driver's command line is fixed).  A worker that dies (SIGABRT from the ROCr fault handler, SIGSEGV, ...) is reported by the
  controller as an ordinary FAILED test carrying the test's node id, a new worker takes the remaining tests, and the summary line
  is printed as usual.  NR_TEST_XDIST=0 turns it off (then the node id of every test is written to the real stderr before it
  starts, see pytest_runtest_logstart, so an abort's tail still names the test)."""
import os
import sys

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
if ROOT not in sys.path:
    sys.path.insert(0, ROOT)

# the hot path's golden parity first ...
FIRST = ("test_gpu_parity.py", "test_gpu_lp.py", "test_gpu_renderers.py", "test_gpu_fullsize.py", "test_gpu_fused_actors.py")
# ... and the multi-stream / full-size / subprocess tests last (~90 of 361: >= 270 tests are reported before the first of them)
LAST = ("test_gpu_amp.py", "test_gpu_full_step.py", "test_gpu_graph_replay.py", "test_gpu_dp.py", "test_gpu_bench_line.py",
        "test_gpu_convergence.py", "test_gpu_adam_split.py", "test_bench_launcher.py", "test_gpu_redzone.py")  # (the last two: an opt-in kernel, test tooling)


def _gpu_visible() -> bool:
    if os.environ.get("NR_TEST_ASSUME_GPU") == "1":  # (exercising this file's GPU-session plumbing on a CPU box)
        return True
    import torch

    return torch.cuda.is_available()


def _is_worker(config) -> bool:
    return hasattr(config, "workerinput")


def pytest_configure(config):
    global _CONFIG
    _CONFIG = config
    config.addinivalue_line("markers", "gpu: needs a real MI355X (run with -m gpu on the GPU box)")
    # the tests' reference legs run channels-last convolution backwards through MIOpen (torch.autocast CNNs): the explicit
    # workaround for MIOpen 3.5.0's overrunning NHWC backward-data kernels, inherited by every child process the tests start
    import neuradar_amd

    neuradar_amd.apply_miopen_workaround()
    _c_level_stderr_to_the_log(config)
    want = os.environ.get("NR_TEST_XDIST", "auto")
    if want == "0" or _is_worker(config) or not config.pluginmanager.hasplugin("xdist"):
        return
    if getattr(config.option, "numprocesses", None) or getattr(config.option, "tx", None):
        return  # the command line asked for its own distribution
    if getattr(config.option, "usepdb", False) or getattr(config.option, "capture", "fd") == "no" and want != "1":
        return  # -s / --pdb sessions stay in-process (the worker's output would not be shown)
    if want == "1" or _gpu_visible():
        # what `-n 1` sets up in xdist's pytest_cmdline_main; its (trylast) pytest_configure then creates the session
        config.option.numprocesses = 1
        config.option.dist = "load"
        config.option.tx = ["popen"]


def _c_level_stderr_to_the_log(config) -> None:
    """On a GPU box: python-level capture only (`--capture=sys` semantics) instead of pytest's default fd capture, in the
    controller and in every xdist worker.  What C code writes to fd 2 -- the ROCr runtime's "Memory access fault by GPU node ...",
    glibc's "free(): invalid pointer", a HIP `guarantee` -- then reaches the session's log at once, next to the node id of the
    crashed test; under fd capture it dies with the process inside pytest's temporary file (round 4: two aborts, no message)."""
    if os.environ.get("NR_TEST_CAPTURE", "sys") != "sys" or getattr(config.option, "capture", "fd") != "fd" or not _gpu_visible():
        return
    capman = config.pluginmanager.getplugin("capturemanager")
    if capman is None or getattr(capman, "_method", None) != "fd":
        return
    try:
        capman.stop_global_capturing()
        capman._method = "sys"
        capman.start_global_capturing()
        capman.suspend_global_capture()  # (the state pytest is in at this point: suspended until a test runs; the terminal reporter
        #                                   created after this hook must get the REAL sys.stdout)
    except Exception:  # noqa: BLE001 -- a pytest whose capture manager looks different: keep its default
        pass


def _rank(item) -> int:
    name = os.path.basename(str(item.fspath))
    if name in FIRST:
        return FIRST.index(name)
    if name in LAST:
        return 1000 + LAST.index(name)
    return 100


def pytest_collection_modifyitems(config, items):
    items.sort(key=_rank)  # (stable: the order inside a file and among the unranked files stays as collected)
    if _gpu_visible():
        return
    skip = pytest.mark.skip(reason="no GPU visible")
    for item in items:
        if "gpu" in item.keywords:
            item.add_marker(skip)


_CONFIG = None


def _real_stderr_fd() -> int:
    """fd of the terminal / log behind pytest's fd capture (the capture plugin keeps a dup of the original fd 2)."""
    capman = _CONFIG.pluginmanager.getplugin("capturemanager") if _CONFIG is not None else None
    err = getattr(getattr(capman, "_global_capturing", None), "err", None)
    return getattr(err, "targetfd_save", 2)


def pytest_runtest_logstart(nodeid, location):
    """Without the worker process (NR_TEST_XDIST=0): the node id goes to the REAL stderr, so that the last line in front of a
    fatal signal's dump names the test that was running."""
    if os.environ.get("NR_TEST_XDIST", "auto") != "0" or os.environ.get("NR_TEST_LOGSTART", "1") == "0":
        return
    try:
        os.write(_real_stderr_fd(), f"\n[start] {nodeid}\n".encode())
    except OSError:
        pass
