"""The build of the host module: what it needs, and what happens without."""

from __future__ import annotations

import os
import shutil
import sys

import pytest

import build_native


@pytest.fixture
def place(tmp_path, monkeypatch):
    """A library folder of its own."""
    monkeypatch.setattr(build_native, "HOST_LIB", str(tmp_path / "m3_host.so"))
    return tmp_path / "m3_host.so"


def _without_torch(monkeypatch, tmp_path):
    monkeypatch.setitem(sys.modules, "torch", None)  # import raises


def _without_compiler(monkeypatch, tmp_path):
    which = shutil.which
    monkeypatch.setattr(shutil, "which", lambda name, *a, **k: None if name == "g++" else which(name, *a, **k))


def _without_headers(monkeypatch, tmp_path):
    import torch
    monkeypatch.setattr(torch, "__file__", str(tmp_path / "torch" / "__init__.py"))


@pytest.mark.parametrize("without", [_without_torch, _without_compiler, _without_headers])
@pytest.mark.parametrize("stale", [False, True])
def test_left_out_where_something_is_missing(without, stale, place, tmp_path, monkeypatch, capsys):
    if stale:  # a module of older sources would not fit the library
        place.write_bytes(b"")
        os.utime(place, (1, 1))
    without(monkeypatch, tmp_path)
    assert build_native.build_host("/usr/local/cuda/bin/nvcc") is False
    assert not place.exists() and "left out" in capsys.readouterr().err


def test_current_module_is_kept_without_a_compiler(place, tmp_path, monkeypatch):
    place.write_bytes(b"")
    _without_compiler(monkeypatch, tmp_path)
    assert build_native.build_host("/usr/local/cuda/bin/nvcc") is True and place.exists()
