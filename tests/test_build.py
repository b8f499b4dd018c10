"""The build's order and what it needs (no compiler is started)."""

import importlib.util
import os
import subprocess
import sys

import pytest

import torch

from scacchi_b200 import _build, _lib

PATH = _build.__file__


@pytest.fixture
def build(monkeypatch):
    """The module by itself, with every command recorded in place of running."""
    spec = importlib.util.spec_from_file_location("build_alone", PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    commands = []

    class Done:
        def wait(self):
            return 0

    def record(cmd, **kw):
        commands.append(cmd)
        return Done()

    class Commands:
        run = Popen = staticmethod(record)

    monkeypatch.setattr(module, "subprocess", Commands)
    monkeypatch.setattr(module.os, "makedirs", lambda *a, **kw: None)
    module.commands = commands
    return module


def test_the_library_is_built_first_and_without_the_extension(build, monkeypatch):
    def fails(force=False):
        build.commands.append("extension")
        raise ModuleNotFoundError("No module named 'torch'")

    monkeypatch.setattr(build, "build_host", fails)
    monkeypatch.setattr(build, "stale", lambda: True)
    with pytest.warns(RuntimeWarning, match="extension module was not built.*torch"):
        assert build.build() == build.LIB
    assert len(build.commands) == len(build.UNITS) + 2 and build.commands[-1] == "extension"
    assert build.commands[-2][-len(build.UNITS) - 1] == build.LIB


def test_another_library_takes_no_extension(build, monkeypatch):
    monkeypatch.setattr(build, "build_host", lambda force=False: 1 / 0)
    assert build.build(out="/tmp/other.so") == "/tmp/other.so"
    assert len(build.commands) == len(build.UNITS) + 1


def test_build_works_where_torch_is_absent():
    code = f"""
import importlib.util, sys, warnings
sys.modules["torch"] = None
spec = importlib.util.spec_from_file_location("build_alone", {PATH!r})
b = importlib.util.module_from_spec(spec)
spec.loader.exec_module(b)
b._build_library = lambda *a: print("library")
with warnings.catch_warnings(record=True) as seen:
    warnings.simplefilter("always")
    assert b.build(force=True) == b.LIB
assert len(seen) == 1 and "torch" in str(seen[0].message)
"""
    out = subprocess.run([sys.executable, "-c", code], capture_output=True, text=True,
                         env={**os.environ, "PYTHONPATH": ""}, timeout=120)
    assert out.returncode == 0 and out.stdout == "library\n", out.stderr


def test_the_extension_names_what_it_was_built_against(monkeypatch):
    path = _build.host_path()
    assert sys.implementation.cache_tag in path and torch.__version__.replace("+", ".") in path
    monkeypatch.setattr(torch, "__version__", "99.0")
    assert _build.host_path() != path and "99.0" in _build.host_path()


def _declines(module):
    return all(getattr(module, n)(1, 2) is None for n in (
        "log_probs", "log_probs_gradient", "gradient_norm", "adamw_step", "adamw_moments"))


def test_without_a_compiler_calls_go_through_python(monkeypatch, tmp_path):
    def fails(force=False):
        raise FileNotFoundError("g++")

    monkeypatch.setattr(_build, "host_path", lambda: str(tmp_path / "none.so"))
    monkeypatch.setattr(_build, "build_host", fails)
    with pytest.warns(RuntimeWarning, match="cannot be used.*g\\+\\+"):
        assert _declines(_lib.host.__wrapped__())


def test_an_extension_that_does_not_load_is_passed_over(monkeypatch, tmp_path):
    broken = tmp_path / "broken.so"
    broken.write_bytes(b"\x7fELF and no more")
    monkeypatch.setattr(_build, "host_path", lambda: str(broken))
    with pytest.warns(RuntimeWarning, match="cannot be used"):
        assert _declines(_lib.host.__wrapped__())


def test_the_extension_itself_loads():
    assert _lib.host() is not _lib.PythonCalls
    assert _lib.host().__name__ == "scacchi_b200._host"
