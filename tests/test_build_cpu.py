"""The build script: the library comes without torch, what is up to date is not made again, and an extension for another torch is none."""
import importlib.util
import os
import subprocess
import types

import pytest

from et_b200 import build as b


class Compilers:
    """Stand-ins that leave the file that they were asked for, or fail."""

    def __init__(self, folder):
        self.folder, self.calls, self.fails, self.missing = str(folder), [], set(), set()

    def __call__(self, cmd, **_):
        self.calls.append(cmd[0])
        if cmd[0] in self.missing:
            raise FileNotFoundError(2, "No such file or directory", cmd[0])
        if cmd[0] in self.fails:
            return types.SimpleNamespace(returncode=1, stdout="", stderr="no such header\n")
        path = cmd[cmd.index("-o") + 1]
        assert os.path.dirname(path) == self.folder
        with open(path, "w"):
            pass
        return types.SimpleNamespace(returncode=0, stdout="", stderr="")

    def take(self):
        calls, self.calls = self.calls, []
        return calls


@pytest.fixture
def compilers(monkeypatch, tmp_path):
    made = tmp_path / "made"
    made.mkdir()
    c = Compilers(made)
    monkeypatch.setattr(subprocess, "run", c)
    monkeypatch.setattr(b, "HERE", str(made))
    monkeypatch.setattr(b, "LIB", str(made / "libet_b200.so"))
    monkeypatch.setattr(b, "BINDING", str(made / "_binding.so"), raising=False)
    return c


@pytest.fixture
def torch_is(monkeypatch, tmp_path):
    """Makes the torch that is found one of a given version, or none."""
    find = importlib.util.find_spec

    def set_to(version):
        spec = None
        if version is not None:
            folder = tmp_path / version / "torch"
            folder.mkdir(parents=True, exist_ok=True)
            (folder / "__init__.py").write_text("")
            (folder / "version.py").write_text(f"__all__ = ['__version__']\n__version__ = '{version}'\ndebug = False\n")
            spec = types.SimpleNamespace(origin=str(folder / "__init__.py"))
        monkeypatch.setattr(importlib.util, "find_spec", lambda name, *a: spec if name == "torch" else find(name, *a))
    return set_to


def extensions(c):
    return sorted(f for f in os.listdir(c.folder) if f.startswith("_binding"))


def test_without_torch_the_library_is_all(compilers, torch_is):
    torch_is(None)
    assert b.build() == b.LIB and compilers.take() == ["nvcc"] and not extensions(compilers)
    assert not b.needs_build() and b.build() == b.LIB and compilers.take() == []


def test_what_is_there_is_not_made_again(compilers, torch_is):
    torch_is("2.11.0+cu128")
    b.build()
    assert compilers.take() == ["nvcc", "g++"] and len(extensions(compilers)) == 1 and not b.needs_build()
    b.build()
    assert compilers.take() == []
    b.build(force=True)
    assert compilers.take() == ["nvcc", "g++"]


def test_another_torch_needs_another_extension(compilers, torch_is):
    torch_is("2.11.0+cu128")
    b.build()
    first = extensions(compilers)
    compilers.take()
    torch_is("2.12.0")
    assert b.needs_build()
    b.build()
    assert compilers.take() == ["g++"] and len(extensions(compilers)) == 1 and extensions(compilers) != first and not b.needs_build()


@pytest.mark.parametrize("how", ["fails", "missing"])
def test_an_extension_that_does_not_compile_ends_no_build(compilers, torch_is, how, capsys):
    torch_is("2.11.0+cu128")
    getattr(compilers, how).add("g++")
    assert b.build() == b.LIB and "checked in Python" in capsys.readouterr().err and not extensions(compilers)
    assert b.build() == b.LIB and compilers.take() == ["nvcc", "g++", "g++"]   # (the library is not compiled again)


def test_a_library_that_does_not_compile_does(compilers, torch_is):
    torch_is("2.11.0+cu128")
    compilers.fails.add("nvcc")
    with pytest.raises(RuntimeError):
        b.build()


def test_only_the_extension_of_this_torch_is_loaded(monkeypatch, tmp_path):
    """One that is missing, or is not for this Python, leaves the checks in Python."""
    from et_b200 import ops
    for path in (None, str(tmp_path / "none.so"), str(tmp_path / "broken.so")):
        (tmp_path / "broken.so").write_bytes(b"not a library")
        monkeypatch.setattr(ops, "binding_path", lambda path=path: path)
        monkeypatch.setattr(ops, "_fast", None)
        assert ops._load_fast() is False
