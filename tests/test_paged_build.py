"""The build of the library and of the torch binding beside it."""
import os

import pytest

from rcutetts_b200 import build

if not (os.path.exists(build.LIB) and os.path.exists(build.EXT)):
    build.build()


@pytest.fixture
def built(monkeypatch):
    """A library that is up to date, so that build() gets to the binding at once."""
    monkeypatch.setattr(build, "_compile", lambda src, hdr, verbose: build.LIB)


def hide(monkeypatch, module):
    monkeypatch.setitem(__import__("sys").modules, module, None)


def test_library_builds_without_torch(built, monkeypatch, tmp_path, capsys):
    hide(monkeypatch, "torch")
    monkeypatch.setattr(build, "EXT", str(tmp_path / "_paged_ext.so"))
    assert build.build() == build.LIB
    assert not os.path.exists(build.EXT)
    assert "torch" in capsys.readouterr().err


def fake_compiler(monkeypatch):
    """The compiler calls of build_ext(): each is noted and leaves its output."""
    import subprocess

    calls = []

    def run(cmd, **kw):
        calls.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return subprocess.CompletedProcess(cmd, 0, "", "")

    monkeypatch.setattr(build.subprocess, "run", run)
    return calls


@pytest.mark.parametrize("what", ["torch", "python"])
def test_binding_is_built_again_for_another_torch_or_python(built, monkeypatch, tmp_path, what):
    import sysconfig

    import torch

    monkeypatch.setattr(build, "EXT", str(tmp_path / "_paged_ext.so"))
    monkeypatch.setattr(build, "BUILD", str(tmp_path))
    calls = fake_compiler(monkeypatch)
    build.build_ext()
    build.build_ext()
    assert len(calls) == 1  # up to date
    if what == "torch":
        monkeypatch.setattr(torch, "__version__", "0.0.1")
    else:
        old = sysconfig.get_config_var
        monkeypatch.setattr(sysconfig, "get_config_var", lambda name: "cpython-39-none" if name == "SOABI" else old(name))
    build.build_ext()
    assert len(calls) == 2
    build.build_ext()
    assert len(calls) == 2


def test_binding_of_another_torch_is_refused(monkeypatch):
    """It uses torch's C++ classes, whose layout goes with the version: import says so instead of running on it."""
    import subprocess
    import sys

    code = "import torch; torch.__version__ = '0.0.1'; from rcutetts_b200 import paged"
    r = subprocess.run([sys.executable, "-c", code], cwd=build.ROOT, capture_output=True, text=True)
    assert r.returncode and "ImportError" in r.stderr and "0.0.1" in r.stderr and "python -m rcutetts_b200.build" in r.stderr


@pytest.mark.parametrize("gone", ["torch", "binding"])
def test_star_import_without_the_binding(gone):
    """`from rcutetts_b200 import *` needs neither torch nor the binding: then it comes without the paged operators."""
    import subprocess
    import sys

    hide = {"torch": "sys.modules['torch'] = None", "binding": "import os.path; e = os.path.exists; "
            "os.path.exists = lambda p: '_paged_ext' not in str(p) and e(p); sys.modules['rcutetts_b200._paged_ext'] = None"}[gone]
    code = f"import sys; {hide}\nfrom rcutetts_b200 import *\nLMConfig(); FrameEngine; assert 'paged_plan' not in globals()"
    r = subprocess.run([sys.executable, "-c", code], cwd=build.ROOT, capture_output=True, text=True)
    assert r.returncode == 0, r.stderr


def test_star_import_has_the_paged_operators():
    names = {}
    exec("from rcutetts_b200 import *", names)
    assert {"LMConfig", "QwenW", "PagedStep", "paged_plan", "paged_append", "paged_attention", "paged_attention_workspace"} <= set(names)
