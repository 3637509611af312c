"""The Python module over torch's headers is built for the torch that it runs with."""

from __future__ import annotations

import os
import re
import subprocess

import pytest
import torch

from kempnerforge_amd import _lib

CSRC = os.path.join(os.path.dirname(os.path.abspath(_lib.__file__)), "csrc")


def _make(tmp_path, **variables):
    """What make would run to bring the module in ``tmp_path`` up to date."""
    got = subprocess.run(["make", "-n", "-C", CSRC, f"BUILD={tmp_path}/obj", f"PYMOD={tmp_path}/m.so",
                          *(f"{k}={v}" for k, v in variables.items()), f"{tmp_path}/m.so"],
                         capture_output=True, text=True)
    assert got.returncode == 0, got.stderr
    return got.stdout


def _stamp(tmp_path, **variables):
    got = subprocess.run(["make", "-C", CSRC, f"BUILD={tmp_path}/obj",
                          *(f"{k}={v}" for k, v in variables.items()), f"{tmp_path}/obj/torch.id"],
                         capture_output=True, text=True)
    assert got.returncode == 0, got.stderr


def test_another_torch_builds_the_module_again(tmp_path):
    _stamp(tmp_path)
    assert torch.__version__ in (tmp_path / "obj" / "torch.id").read_text()
    (tmp_path / "m.so").write_text("")  # newer than the stamp and the sources
    _stamp(tmp_path)  # the same torch: the stamp stays as it is
    assert os.path.getmtime(tmp_path / "obj" / "torch.id") <= os.path.getmtime(tmp_path / "m.so")
    os.utime(tmp_path / "m.so", (0, 0))
    _stamp(tmp_path, TORCH_ID="/elsewhere 9.9.9")
    assert "9.9.9" in (tmp_path / "obj" / "torch.id").read_text()
    line = _make(tmp_path, TORCH_ID="/elsewhere 9.9.9")
    assert "kf_torch.cpp" in line and "compiled_with_cxx11_abi" in line
    assert "CXX11_ABI=1" not in line  # asked of torch, not fixed


def test_a_module_for_another_torch_is_refused(monkeypatch):
    if not os.path.exists(_lib.LIB_PATH):
        pytest.skip("library not built")
    version = torch.__version__
    assert _lib.native().torch_version in version
    monkeypatch.setattr(_lib, "_native", None)
    monkeypatch.setattr(torch, "__version__", "9.9.9+rocm7.0")
    with pytest.raises(RuntimeError, match="was built for torch"):
        _lib.native()
    # (what follows the numbers is a build's name)
    monkeypatch.setattr(torch, "__version__", re.match(r"[\d.]+\d", version)[0] + "a0+git1")
    assert _lib.native().torch_version in version
