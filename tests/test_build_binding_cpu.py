"""The build of the policy operators' torch binding (ur3e_amd/_build.py): left out where torch is missing, made again where torch or
the command is another one."""
import os
import sys
import time

import pytest

from ur3e_amd import _build


@pytest.fixture
def runs(tmp_path, monkeypatch):
    """the commands that the build would run, with a binding that is newer than its sources"""
    out = []

    def run(cmd, check):
        out.append(cmd)
        (tmp_path / "ur3e_policy_torch.so").touch()
    monkeypatch.setattr(_build, "OBJ", str(tmp_path))
    monkeypatch.setattr(_build, "TORCH_LIB", str(tmp_path / "ur3e_policy_torch.so"))
    monkeypatch.setattr(_build.subprocess, "run", run)
    return out


def test_without_torch_the_binding_is_left_out(runs, monkeypatch, capsys):
    monkeypatch.setitem(sys.modules, "torch", None)
    _build._build_torch(True, True)
    assert runs == [] and "not built" in capsys.readouterr().out


def test_another_torch_is_another_binding(runs, monkeypatch):
    import torch
    _build._build_torch(False, False)
    assert len(runs) == 1
    new = time.time() + 60
    os.utime(_build.TORCH_LIB, (new, new))
    _build._build_torch(False, False)
    assert len(runs) == 1  # nothing has changed
    monkeypatch.setattr(torch, "__version__", "0.0")
    _build._build_torch(False, False)
    assert len(runs) == 2
