"""What the build needs and what it does without."""
import os
import sys

import pytest

from dolittle_b200 import build


def without_torch(monkeypatch):
    monkeypatch.setitem(sys.modules, "torch", None)


def without_a_compiler(monkeypatch):
    monkeypatch.setenv("CXX", "no-such-compiler")


def without_headers(monkeypatch):
    real = os.path.exists
    monkeypatch.setattr(os.path, "exists", lambda p: real(p) and not str(p).endswith("ATen.h"))


@pytest.mark.parametrize("absent", [without_torch, without_a_compiler, without_headers])
def test_the_library_builds_without_what_only_the_torch_calls_need(absent, monkeypatch, tmp_path, capsys):
    """The C ABI has no use for torch, its headers or g++: the module is left out, with a message."""
    monkeypatch.setattr(build, "TORCH_OUT", str(tmp_path / "_torch_shared.so"))
    absent(monkeypatch)
    assert build.build() == build.OUT
    assert not (tmp_path / "_torch_shared.so").exists()
    assert "torch calls" in capsys.readouterr().err
