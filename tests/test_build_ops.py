"""The extension module of the int8 operators belongs to one torch and one Python, and processes that
build at once take turns (no GPU and no compiler needed)."""

from __future__ import annotations

import os
import stat
import subprocess
import sys
import sysconfig

import pytest
import torch

from tests.conftest import ROOT


def _compiler(tmp_path, body=""):
    """A stand-in for g++: logs a line and writes its output in two steps."""
    cc = tmp_path / "cxx"
    cc.write_text(f"""#!/bin/sh
echo run >> {tmp_path}/log
while [ "$1" != "-o" ]; do shift; done
printf half > "$2"; {body}
printf whole >> "$2"
""")
    cc.chmod(cc.stat().st_mode | stat.S_IXUSR)
    return str(cc)


@pytest.fixture
def tree(tmp_path, monkeypatch):
    from strands_decider_b200 import build

    monkeypatch.setattr(build, "LIBDIR", str(tmp_path / "lib"))
    monkeypatch.setattr(build, "OBJDIR", str(tmp_path / "obj"))
    monkeypatch.setenv("CXX", _compiler(tmp_path))
    return lambda: (tmp_path / "log").read_text().count("run")


def test_another_torch_or_python_gets_a_module_of_its_own(tree, monkeypatch):
    from strands_decider_b200 import build

    first = build.build_ops()
    assert open(first).read() == "halfwhole" and tree() == 1
    assert build.build_ops() == first and tree() == 1
    seen = {first}
    suffix = sysconfig.get_config_var("EXT_SUFFIX")
    for patch in (lambda: monkeypatch.setattr(torch, "__version__", "2.99.0"),
                  lambda: monkeypatch.setattr(torch.version, "git_version", "0" * 40),
                  lambda: monkeypatch.setattr(torch, "compiled_with_cxx11_abi", lambda: False),
                  lambda: monkeypatch.setattr(sysconfig, "get_config_var", lambda n: ".cpython-399" + suffix)):
        patch()
        path = build.build_ops()
        assert path not in seen and open(path).read() == "halfwhole"
        seen.add(path)
    assert tree() == 5
    build.build_ops(force=True)
    assert tree() == 6


def test_a_module_of_another_torch_is_not_loaded(monkeypatch):
    from strands_decider_b200 import _lib, build

    build.build()
    monkeypatch.setattr(_lib, "_int8_ops", None)
    monkeypatch.setattr(torch, "__version__", "2.99.0")
    with pytest.raises(RuntimeError, match="strands_decider_b200.build"):
        _lib.int8_ops()


def test_processes_that_build_at_once_take_turns(tmp_path):
    child = ("import sys; from strands_decider_b200 import build as b; "
             "b.LIBDIR, b.OBJDIR = sys.argv[1] + '/lib', sys.argv[1] + '/obj'; print(open(b.build_ops()).read())")
    env = {**os.environ, "CXX": _compiler(tmp_path, "sleep 2"), "PYTHONPATH": ROOT}
    runs = [subprocess.Popen([sys.executable, "-c", child, str(tmp_path)], env=env, cwd=ROOT, stdout=subprocess.PIPE,
                             text=True) for _ in range(3)]
    assert [r.communicate(timeout=300)[0].strip() for r in runs] == ["halfwhole"] * 3
    assert (tmp_path / "log").read_text().count("run") == 1
    assert len(os.listdir(tmp_path / "lib")) == 1
