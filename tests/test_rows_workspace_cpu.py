"""How much workspace attention over the last interactions of lists asks for.  No GPU is needed."""
import ctypes as C

import pytest

from orca_b200 import _lib, build


@pytest.fixture(scope="module")
def L():
    build.build()
    return _lib.lib()


@pytest.mark.parametrize("rows", [1, 64, 65, 200, 600, 6000])
def test_lists_that_are_never_cut_have_no_results_of_parts(L, rows):
    """Ten interactions are one part; a part's results are 4160 bytes."""
    for last in (1, 10, 16):
        assert 0 < L.orca_packed_attend_last_workspace_bytes(rows, last) <= 20 * rows + 6 * 256 + 4
    assert L.orca_packed_attend_last_workspace_bytes(rows, 100) >= 4160 * 2


@pytest.mark.parametrize("rows", [1, 64, 65, 6000, 1 << 24])
def test_any_list_fits_the_whole_workspace(L, rows):
    most = L.orca_packed_attend_lists_workspace_bytes(rows)
    assert L.orca_packed_attend_last_workspace_bytes(rows, 0) == most
    sizes = [L.orca_packed_attend_last_workspace_bytes(rows, last) for last in (1, 10, 64, 65, 1000, 1 << 20, 1 << 40, (1 << 63) - 1)]
    assert sizes == sorted(sizes) and sizes[-1] == most


def test_refusals(L):
    for args in ((-1, 10), (-1, 0), (10, -1)):
        assert L.orca_packed_attend_last_workspace_bytes(*args) == -1
    keep = (C.c_char * (1 << 12))()
    p = (C.addressof(keep) + 255) & ~255
    for last, n in ((10, 40), (0, 40), (300, 70)):
        need = L.orca_packed_attend_last_workspace_bytes(n, last)
        assert L.orca_packed_attend_lists(p, p, 10, p, 10, 1, p, p, p, p, p, 10, p, p, last, n, p, p, None, p, need - 1, None) == 1
        assert b"too small" in L.orca_last_error()
