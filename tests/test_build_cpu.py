"""The build on machines without a torch that has CUDA: the library needs none, so nothing may fail."""
import importlib.machinery

import pytest

from pufferlean_b200 import build


@pytest.fixture
def commands(monkeypatch):
    ran = []
    monkeypatch.setattr(build.subprocess, "check_call", lambda cmd, **_: ran.append(cmd))
    monkeypatch.setattr(build, "TORCH_EXT", "/nonexistent/pl_torch.so")
    return ran


def _torch_at(monkeypatch, path):
    spec = importlib.machinery.ModuleSpec("torch", None, is_package=True)
    spec.submodule_search_locations = [str(path)]
    monkeypatch.setattr(build.importlib.util, "find_spec", lambda name: spec)


def test_torch_without_cuda_is_left_out(tmp_path, monkeypatch, commands):
    (tmp_path / "lib").mkdir()
    (tmp_path / "lib" / "libc10.so").touch()
    _torch_at(monkeypatch, tmp_path)
    build._torch_ext(False)
    assert not commands


def test_torch_with_cuda_is_built_for(tmp_path, monkeypatch, commands):
    (tmp_path / "lib").mkdir()
    (tmp_path / "lib" / "libc10_cuda.so").touch()
    _torch_at(monkeypatch, tmp_path)
    build._torch_ext(False)
    assert len(commands) == 1 and "-lc10_cuda" in commands[0]


def test_no_torch(monkeypatch, commands):
    monkeypatch.setattr(build.importlib.util, "find_spec", lambda name: None)
    build._torch_ext(False)
    assert not commands
