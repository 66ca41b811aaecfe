"""The build of the library and of the torch binding beside it."""
import os

import pytest

from rcutetts_b200 import build


@pytest.fixture
def built(monkeypatch):
    """A library that is up to date, so that build() gets to the binding at once."""
    if not os.path.exists(build.LIB):
        build.build()
    monkeypatch.setattr(build, "_compile", lambda src, hdr, verbose: build.LIB)


def hide(monkeypatch, module):
    monkeypatch.setitem(__import__("sys").modules, module, None)


def test_library_builds_without_torch(built, monkeypatch, tmp_path, capsys):
    hide(monkeypatch, "torch")
    monkeypatch.setattr(build, "EXT", str(tmp_path / "_paged_ext.so"))
    assert build.build() == build.LIB
    assert not os.path.exists(build.EXT)
    assert "torch" in capsys.readouterr().err
