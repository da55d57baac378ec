"""The host module has the object layouts of one PyTorch compiled in: it is
rebuilt for another, and refused by another."""

from __future__ import annotations

import importlib.util
import subprocess
import types

import pytest
import torch

import build_native
from src import _native as nat


def test_rebuilt_for_another_pytorch(tmp_path, monkeypatch):
    lib, stamp = tmp_path / "m3_host.so", tmp_path / "m3_host.torch"
    monkeypatch.setattr(build_native, "HOST_LIB", str(lib))
    monkeypatch.setattr(build_native, "HOST_STAMP", str(stamp))
    built = []

    def run(cmd, **kw):
        built.append(cmd)
        with open(cmd[cmd.index("-o") + 1], "w") as f:
            f.write("module")
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")
    monkeypatch.setattr(subprocess, "run", run)
    monkeypatch.setattr(build_native.shutil, "which", lambda name: "/usr/bin/" + name)
    nvcc = "/usr/local/cuda/bin/nvcc"
    for version, times in ((str(torch.__version__), 1), (str(torch.__version__), 1), ("2.99.0", 2), ("2.99.0", 2)):
        monkeypatch.setattr(torch, "__version__", version)
        assert build_native.build_host(nvcc) is True and len(built) == times
        assert f'-DM3_TORCH_VERSION="{version}"' in built[-1]
    stamp.unlink()  # of a build that did not note it
    assert build_native.build_host(nvcc) is True and len(built) == 3


def test_refused_by_another_pytorch(monkeypatch):
    spec = importlib.util.spec_from_file_location("m3_host", nat.HOST_PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    assert module.torch_version == str(torch.__version__)
    monkeypatch.setattr(nat, "_host", None)
    assert nat.host_entry("linear_w4") is not nat._no_host
    monkeypatch.setattr(nat, "_host", None)
    monkeypatch.setattr(torch, "__version__", "2.99.0")
    with pytest.raises(RuntimeError, match="--force"):
        nat.host_entry("linear_w4")
    assert nat._host is None
    with pytest.raises(ImportError):  # a module from before versions were noted
        nat._check_host(types.ModuleType("m3_host"))
