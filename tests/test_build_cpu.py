"""The build's two steps: the library (nvcc), and the module of its calls on tensors (g++, PyTorch's headers).  No GPU is needed."""
import os

import pytest

from orca_b200 import _lib, build


@pytest.fixture
def steps(monkeypatch):
    """The steps that build() takes from here on, by name; the library's does nothing, for it is there."""
    build.build()
    taken = []
    monkeypatch.setattr(build, "_build_library", lambda verbose: taken.append("library"), raising=False)
    return taken


def test_the_library_is_whole_without_the_module(steps, monkeypatch, tmp_path, capsys):
    """A module that cannot be built is said, fails nobody who does not use it, and does not make the next call start from the beginning."""
    monkeypatch.setattr(build, "ROWS", str(tmp_path / "_rows.so"))
    for command in (["false"], [str(tmp_path / "no-such-compiler")]):
        monkeypatch.setattr(build, "_rows_command", lambda: command)
        assert build.build() == build.LIB
        assert "_rows.so" in capsys.readouterr().err
    assert steps == [] and not os.path.exists(build.ROWS)


def test_a_module_of_an_earlier_source_does_not_stay(steps, monkeypatch, tmp_path):
    at = tmp_path / "_rows.so"
    at.write_bytes(b"an earlier one")
    os.utime(at, (1, 1))
    monkeypatch.setattr(build, "ROWS", str(at))
    monkeypatch.setattr(build, "_rows_command", lambda: ["false"])
    build.build()
    assert steps == [] and not at.exists()


def test_each_step_follows_its_own_sources(steps, monkeypatch, tmp_path):
    at = tmp_path / "_rows.so"
    monkeypatch.setattr(build, "ROWS", str(at))
    monkeypatch.setattr(build, "_build_rows", lambda: steps.append("module"))
    build.build()
    assert steps == ["module"]
    steps.clear()
    monkeypatch.setattr(build, "LIB", str(tmp_path / "lib.so"))
    build.build()
    assert steps == ["library", "module"]
    steps.clear()
    build.build(force=True)
    assert steps == ["library", "module"]


@pytest.mark.parametrize("other", ["PyTorch", "Python", "interface"])
def test_a_module_of_another_pytorch_is_refused_and_built_again(steps, monkeypatch, other):
    """It derives from PyTorch's classes: one that was made for another version may load and fail in any way."""
    assert build.rows_fit() and _lib.rows().made_for == build.rows_made_for()
    monkeypatch.setattr(build, "_build_rows", lambda: steps.append("module"))
    build.build()
    assert steps == []
    if other == "PyTorch":
        import torch
        monkeypatch.setattr(torch, "__version__", torch.__version__ + "1")
    elif other == "Python":
        monkeypatch.setattr(build.sysconfig, "get_config_var", lambda name: "cpython-0")
    else:
        monkeypatch.setattr(_lib, "VERSION", _lib.VERSION + 1)
        monkeypatch.setattr(_lib, "lib", lambda: None)
    monkeypatch.setattr(_lib, "_rows", None)
    with pytest.raises(ImportError, match="orca_b200.build"):
        _lib.rows()
    build.build()
    assert steps == ["module"]
