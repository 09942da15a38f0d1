"""What device code has to keep to on its failure paths, held against its source: a wait of a kernel on its own copies cannot be
made to run out on a GPU that works (a look at a barrier suspends the thread for longer than a copy takes: with a limit of one
clock none of 300 launches gave up)."""
import ctypes
import os
import re
import subprocess

import pytest

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "orca_b200", "csrc")


def _source(name):
    text = open(os.path.join(CSRC, name)).read()
    return re.sub(r"//[^\n]*|/\*.*?\*/", "", text, flags=re.S)


@pytest.mark.parametrize("name,done", [("attn_query.cu", "accfull"), ("attn_out.cu", "acc2"), ("gru_rows.cu", "accfull"),
                                       ("score_rows.cu", "accfull")])
def test_a_warp_that_gives_up_stops_and_waits_for_what_it_has_in_flight(name, done):
    """A copy thread whose slot is not handed back issues no further copy into it (nor arrives twice on its barrier), the
    products stop likewise, and copies and products are waited for before shared and tensor memory are given up."""
    text = _source(name)
    copies, rest = text.split("if (warp == 0) {", 1)[1].split("} else if (warp == 1) {", 1)
    products = rest.split("} else {", 1)[0]
    at = [copies.index(x) for x in ("; alive && ", "mbar_wait(empty(", "if (!alive) break;", "mbar_expect_tx(full(", "mbar_settle(full(")]
    assert at == sorted(at)
    assert "if (alive) mma_commit(empty(s));" in products and re.search(r"[^(] mma_commit\(empty", products.replace("if (alive) ", "(")) is None
    assert products.rindex(f"mma_commit({done})") < products.index(f"mbar_settle({done}, (t - 1) & 1)")


def test_a_query_that_did_not_come_is_waited_for():
    text = _source("attention.cu")
    at = [text.index(x) for x in ("mbar_wait(qbar, phase", "phase ^= alive;", "if (!alive) tc::mbar_settle(qbar, phase);")]
    assert at == sorted(at)


def test_no_entry_point_drops_the_status_word_it_is_given():
    """Every entry point that takes one hands it to what it launches: its kernels have nothing else to say that rows are wrong."""
    for name in os.listdir(CSRC):
        assert name.endswith((".cu", ".cuh")) is False or "(void)d_status" not in _source(name), name


def test_rows_at_the_ends_of_an_array_are_known(tmp_path):
    """Rows between borders are read by pieces of memory: each whose first begins before the array, or whose last ends behind it, is one of `edge_rows` from either
    end, whatever lies between rows (nothing: the same row again)."""
    body = re.search(r"int64_t edge_rows\(int vb, const Rows &r\) \{[^}]*\}", _source("norm.cu")).group(0)
    code = "#include <algorithm>\n#include <cstdint>\nusing std::max;\nstruct Rows { const char *p; int64_t stride; };\n" + body + \
        '\nextern "C" int64_t edge(int vb, int64_t stride) { return edge_rows(vb, Rows{nullptr, stride}); }\n'
    (tmp_path / "edge.cpp").write_text(code)
    subprocess.check_call(["g++", "-std=c++17", "-shared", "-fPIC", str(tmp_path / "edge.cpp"), "-o", str(tmp_path / "edge.so")])
    lib = ctypes.CDLL(str(tmp_path / "edge.so"))
    lib.edge.restype, lib.edge.argtypes = ctypes.c_int64, [ctypes.c_int, ctypes.c_int64]
    for size in (2, 4):
        vb = 4 * size
        for begin in range(0, vb, size):
            for width in (1, 2, 3, 5, 33, 172):
                for stride in (0, size, 2 * size, 3 * size, 5 * size, vb, width * size, (width + 4) * size):
                    edge = lib.edge(vb, stride)
                    for rows in (1, 2, 17, 40, 90):
                        end = begin + (rows - 1) * stride + width * size
                        for row in range(rows):
                            at = begin + row * stride
                            if at // vb * vb < begin or -(-(at + width * size) // vb) * vb > end:
                                assert row < edge or row >= rows - edge, (size, begin, width, stride, rows, row)


def test_codes_are_shifted_where_the_compiler_cannot_fold_it():
    """A shift in C++ before the selection of codes' bytes was lost for every other value (nvcc 12.9): neither of the two stands there."""
    body = _source("optim.cu").split("void codes_of(", 1)[1].split("\ntemplate", 1)[0].split("\n}", 1)[0]
    assert "<< 4" not in body and body.count("four_left(") == 2
