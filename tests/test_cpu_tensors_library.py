"""CPU (no GPU): the library that reads tensors where they lie is taken only beside the torch and the Python it was compiled for."""
import os
import subprocess
import sys

import pytest
import torch

from neuradar_amd import _lib


def test_it_is_built_for_this_process():
    assert _lib.tensors().nr_built_for().decode() == _lib.built_for() == f"torch {torch.__version__} python {sys.version_info[0]}.{sys.version_info[1]}"
    assert not _lib._other_torch()


@pytest.mark.parametrize("version", ["2.10.0", "2.10.0+rocm7", "2.11.0+rocm7.0"])
def test_another_torch_is_refused_and_built_for_again(monkeypatch, version):
    monkeypatch.setattr(torch, "__version__", version)
    monkeypatch.setattr(_lib, "_tensors", None)
    with pytest.raises(RuntimeError, match="was built for"):
        _lib.tensors()
    assert _lib._other_torch() and _lib._stale()
    calls = []
    monkeypatch.setattr(subprocess, "check_call", lambda cmd, **kw: calls.append(cmd))
    _lib.build()
    assert "-B" in calls[1] and "-B" not in calls[0]  # (its source has not changed)


def test_the_kernels_build_without_torch():
    """(what make would run, with an interpreter that has nothing)"""
    r = subprocess.run(["make", "-C", _lib.CSRC, "-n", "-B", "PYTHON=/bin/false", "libneuradar_hip.so"], capture_output=True, text=True)
    assert r.returncode == 0 and "tensor_list" not in r.stdout and "embedding.hip" in r.stdout


def test_build_takes_the_running_interpreter(monkeypatch):
    calls = []
    monkeypatch.setattr(subprocess, "check_call", lambda cmd, **kw: calls.append(cmd))
    _lib.build(force=True)
    assert [c[-2] for c in calls] == ["libneuradar_hip.so", "libneuradar_tensors.so"]
    assert all(f"PYTHON={sys.executable}" in c and c[-1] == "-B" for c in calls)
    assert os.path.isabs(sys.executable)
