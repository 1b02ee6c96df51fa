"""What the build needs and what it does without."""
import importlib.util
import os
import sys
import types

import pytest

from dolittle_b200 import _lib, build, shared


def without_torch(monkeypatch):
    monkeypatch.setitem(sys.modules, "torch", None)


def with_a_folder_called_torch(monkeypatch):
    monkeypatch.setattr(importlib.util, "find_spec", lambda name: types.SimpleNamespace(origin=None))


def without_a_compiler(monkeypatch):
    monkeypatch.setenv("CXX", "no-such-compiler")


def without_headers(monkeypatch):
    real = os.path.exists
    monkeypatch.setattr(os.path, "exists", lambda p: real(p) and not str(p).endswith("ATen.h"))


@pytest.mark.parametrize("absent", [without_torch, with_a_folder_called_torch, without_a_compiler,
                                     without_headers])
def test_the_library_builds_without_what_only_the_torch_calls_need(absent, monkeypatch, tmp_path, capsys):
    """The C ABI has no use for torch, its headers or g++: the module is left out, with a message."""
    monkeypatch.setattr(_lib, "HERE", str(tmp_path))
    absent(monkeypatch)
    assert build.build() == build.OUT
    assert not list(tmp_path.iterdir())
    assert "torch calls" in capsys.readouterr().err


def a_torch(folder, version="2.11.0", library=b"x" * 100):
    """The files of a torch build that name it."""
    (folder / "lib").mkdir(parents=True)
    (folder / "version.py").write_text(f"__version__ = '{version}'\n")
    (folder / "lib" / "libtorch_python.so").write_bytes(library)
    return types.SimpleNamespace(origin=str(folder / "__init__.py"))


def test_each_torch_and_python_has_a_module_of_its_own(monkeypatch, tmp_path):
    specs = [a_torch(tmp_path / "a"), a_torch(tmp_path / "b"), a_torch(tmp_path / "c", version="2.12.0"),
             a_torch(tmp_path / "d", library=b"x" * 101)]
    paths = []
    for spec in specs:
        monkeypatch.setattr(importlib.util, "find_spec", lambda name, spec=spec: spec)
        paths.append(_lib.torch_calls_path())
    monkeypatch.setattr(_lib.sysconfig, "get_config_var", lambda name: "cpython-399-other")
    paths.append(_lib.torch_calls_path())
    assert paths[0] == paths[1] and len(set(paths)) == 4


def test_a_module_of_another_torch_is_left_alone(monkeypatch, tmp_path):
    other = tmp_path / "_torch_shared.so"
    other.write_bytes(b"of another torch")
    monkeypatch.setattr(_lib, "HERE", str(tmp_path))
    monkeypatch.setattr(shared, "_calls", None)
    with pytest.raises(ImportError, match="dolittle_b200.build"):
        shared._extension()
    made = build.build_torch_calls()
    assert os.path.dirname(made) == str(tmp_path) and other.read_bytes() == b"of another torch"
    assert build.build_torch_calls() == made  # up to date
    shared._extension()
