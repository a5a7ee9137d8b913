"""The build of the native calls' module: what makes it stale, and what refuses a stale one."""

from __future__ import annotations

import os

import pytest
import torch

from pagedserve_b200 import _native, build


class _Compiled(Exception):
    pass


@pytest.fixture
def commands(monkeypatch, tmp_path):
    """The compiler commands _build_calls would run, beside a module that is up to date."""
    seen = []
    monkeypatch.setattr(build, "BUILD", str(tmp_path))
    monkeypatch.setattr(build, "CALLS", str(tmp_path / "_calls.so"))
    (tmp_path / "_calls.so").touch()
    (tmp_path / "calls.key").write_text("\n".join(build._calls_command()))

    def run(cmd, **kw):
        seen.append(cmd)
        raise _Compiled

    monkeypatch.setattr(build.subprocess, "run", run)
    return seen


def test_calls_are_current(commands):
    build._build_calls(False)
    assert commands == []


@pytest.mark.parametrize("what", ["torch", "python", "compiler"])
def test_calls_are_rebuilt_for_another_torch_python_or_compiler(commands, monkeypatch, what):
    if what == "torch":
        monkeypatch.setattr(torch, "__version__", "0.0.1")
    elif what == "python":
        monkeypatch.setattr("sysconfig.get_config_var", lambda name: ".cpython-1-none.so")
    else:
        monkeypatch.setenv("CXX", "another-c++")
    with pytest.raises(_Compiled):
        build._build_calls(False)
    assert len(commands) == 1


def test_two_builds_do_not_share_a_file(commands, monkeypatch):
    for pid in (11, 12):
        monkeypatch.setattr(os, "getpid", lambda: pid)
        with pytest.raises(_Compiled):
            build._build_calls(True)
    first, second = (c[c.index("-o") + 1] for c in commands)
    assert first != second and os.path.dirname(first) == os.path.dirname(second) == build.BUILD


def test_a_module_built_for_another_torch_is_refused(monkeypatch):
    assert _native.calls() is not None
    monkeypatch.setattr(_native, "_calls", None)
    monkeypatch.setattr(torch, "__version__", "0.0.1")
    with pytest.raises(RuntimeError, match="built for"):
        _native.calls()
