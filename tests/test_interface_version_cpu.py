"""What a host that was written for an earlier build of the library finds.  No GPU is needed."""
import os
import re

import pytest

from orca_b200 import _lib, build

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_the_version_names_the_layout_of_prepared_operands():
    """One line a layout in the header, the last one's number the version: entry points added beside the others change no operand, and a
    host that compares the version it was written for goes on."""
    build.build()
    text = open(os.path.join(ROOT, "include", "orca_b200.h")).read()
    version = int(re.search(r"#define ORCA_VERSION (\d+)", text).group(1))
    lines = re.findall(r"^ \* (\d+): (.*)$", text[:text.index("#define ORCA_VERSION")], re.M)
    assert [int(n) for n, _ in lines] == list(range(1, version + 1))
    assert all("img" in what for _, what in lines)
    assert _lib.lib().orca_version() == version


def test_a_library_without_an_entry_point_is_refused(monkeypatch):
    build.build()
    monkeypatch.setitem(_lib.SYMBOLS, "orca_not_there", (None, []))
    monkeypatch.setattr(_lib, "_lib", None)
    with pytest.raises(ImportError, match="orca_not_there"):
        _lib.lib()
