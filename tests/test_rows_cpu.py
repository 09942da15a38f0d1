"""Refusals of the calls on packed rows and of lookups, and the plain forms that the GPU tests compare with.  No GPU is needed."""
import ctypes as C
from fractions import Fraction

import numpy as np
import pytest
import torch

import rows_reference as ref
from orca_b200 import _lib, build


@pytest.fixture(scope="module")
def L():
    build.build()
    return _lib.lib()


def test_the_plain_format():
    """Offset, step and codes of the plain form against their definition in exact fractions."""
    rs = np.random.RandomState(0)
    x = np.concatenate([rs.randn(6, 172), rs.randn(3, 172) * 1e-20 + 5, rs.randint(0, 31, (3, 172)) * 0.5]).astype(np.float32)
    for row, w in zip(x, ref.pack(x)):
        for g, c in enumerate((slice(0, 128), slice(128, 172))):
            v = [Fraction(float(a)) for a in row[c]]
            bits = int(w[g])
            f = lambda b: Fraction(float(np.array(b & 0xffffffff, np.uint32).view(np.float32)))
            off, step = f(bits & 0xffff0000), f(bits << 16)
            up = f((bits & 0xffff0000) - 0x10000 if off < 0 else (bits & 0xffff0000) + 0x10000) if off != 0 else None
            assert off <= min(v) and (up is None or up > min(v))
            want = (max(v) - off) / 15
            assert step >= want and (step == 0 or f((bits << 16) - 0x10000) < want)
            for j, a in enumerate(v):
                col = j + (128 if g else 0)
                code = int(w[2 + col // 8]) >> (4 * (col % 8)) & 15
                assert step == 0 and code == 0 or abs(a - off - step * code) <= step / 2
    assert np.array_equal(ref.pack(ref.unpack(ref.pack(np.zeros((1, 172))))), np.zeros((1, 24), np.uint32))


def _buffer(n=1 << 16):
    b = (C.c_char * (n + 256))()
    return b, (C.addressof(b) + 255) & ~255


BAD = 1
UNSUPPORTED = 2


def test_push_and_pull_refuse(L):
    keep, p = _buffer()
    push = dict(words=p, rows=10, x=p, type=0, stride=172, ids=p, n=4, record=p, status=None, stream=None)
    bad = [dict(words=None), dict(rows=0), dict(x=None), dict(n=-1), dict(stride=171), dict(ids=None), dict(record=None), dict(words=p + 4),
           dict(ids=None, record=None, n=11)]
    for b in bad:
        assert L.orca_packed_push(*{**push, **b}.values()) == BAD, b
        assert b"orca_packed_push" in L.orca_last_error()
    assert L.orca_packed_push(*{**push, "type": 3}.values()) == UNSUPPORTED
    assert L.orca_packed_push(*{**push, "n": 0}.values()) == 0
    pull = dict(words=p, rows=10, ids=p, n=4, out=p, status=None, stream=None)
    for b in [dict(words=None), dict(rows=0), dict(ids=None), dict(n=-1), dict(out=None), dict(out=p + 4), dict(words=p + 8)]:
        assert L.orca_packed_pull(*{**pull, **b}.values()) == BAD, b
    assert L.orca_packed_pull(*{**pull, "n": 0}.values()) == 0
    del keep


def test_attend_refuses(L):
    keep, p = _buffer()
    a = dict(qt=p, words=p, rows=10, edges=p, n_edges=10, packed=1, w=p, nbr=p, eid=p, delta=p, k=10, n=4, ctx=p, valid=p, status=None,
             ws=p, ws_bytes=1 << 40, stream=None)
    for b in [dict(qt=None), dict(words=None), dict(rows=0), dict(edges=None), dict(n_edges=0), dict(packed=2), dict(w=None), dict(nbr=None),
              dict(eid=None), dict(delta=None), dict(k=-1), dict(n=-1), dict(ctx=None), dict(valid=None), dict(qt=p + 4), dict(words=p + 4),
              dict(edges=p + 4), dict(ctx=p + 4), dict(k=1000, ws=None), dict(k=1000, ws=p + 16), dict(k=1000, ws_bytes=100),
              dict(rows=1 << 31), dict(n_edges=1 << 31), dict(k=(1 << 30) + 1)]:
        assert L.orca_packed_attend(*{**a, **b}.values()) == BAD, b
    assert L.orca_packed_attend(*{**a, "n": 0}.values()) == 0
    a = dict(qt=p, words=p, rows=10, edges=p, n_edges=10, packed=1, w=p, indptr=p, nbr=p, eid=p, ts=p, nodes_of=10, nodes=p, times=p, last=0,
             n=4, ctx=p, valid=p, status=None, ws=p, ws_bytes=1 << 40, stream=None)
    for b in [dict(qt=None), dict(indptr=None), dict(nbr=None), dict(eid=None), dict(ts=None), dict(nodes_of=0), dict(nodes=None),
              dict(times=None), dict(last=-1), dict(n=-1), dict(ws=None), dict(ws=p + 8), dict(ws_bytes=1000), dict(ctx=p + 8)]:
        assert L.orca_packed_attend_lists(*{**a, **b}.values()) == BAD, b
    assert L.orca_packed_attend_lists(*{**a, "n": 0}.values()) == 0
    assert L.orca_packed_attend_workspace_bytes(-1, 10) == -1 and L.orca_packed_attend_workspace_bytes(10, -1) == -1
    assert L.orca_packed_attend_lists_workspace_bytes(-1) == -1
    del keep


def test_lookup_refuses(L):
    keep, p = _buffer()
    a = dict(table=p, rows=10, stride=172, width=172, type=0, ids=p, ids64=0, n=4, scale=1.0, out=p, status=None, stream=None)
    for b in [dict(table=None), dict(rows=-1), dict(stride=171), dict(width=0), dict(ids=None), dict(n=-1), dict(out=None), dict(table=p + 2),
              dict(out=p + 2), dict(ids=p + 4, ids64=1), dict(rows=1 << 31), dict(width=(1 << 24) + 1, stride=1 << 25)]:
        assert L.orca_rows_lookup(*{**a, **b}.values()) == BAD, b
    assert L.orca_rows_lookup(*{**a, "type": 7}.values()) == UNSUPPORTED
    assert L.orca_rows_lookup(*{**a, "n": 0}.values()) == 0
    a = dict(g=p, stride=172, width=172, type=0, ids=p, ids64=0, n=4, rows=10, scale=1.0, padding=-1, grad=p, status=None, ws=p,
             ws_bytes=1 << 40, stream=None)
    for b in [dict(g=None), dict(stride=171), dict(width=0), dict(ids=None), dict(n=-1), dict(rows=-1), dict(grad=None), dict(g=p + 2),
              dict(grad=p + 1), dict(ids=p + 4, ids64=1), dict(n=1 << 31), dict(n=5000, ws=None), dict(n=5000, ws=p + 8), dict(n=5000, ws_bytes=8)]:
        assert L.orca_rows_grad(*{**a, **b}.values()) == BAD, b
    assert L.orca_rows_grad(*{**a, "type": -1}.values()) == UNSUPPORTED
    assert L.orca_rows_grad(*{**a, "n": 0, "rows": 0}.values()) == 0
    for args in ((-1, 10, 172), (10, 10, (1 << 24) + 1), (1 << 31, 10, 172), (10, -1, 172), (10, 1 << 31, 172), (10, 10, 0)):
        assert L.orca_rows_grad_workspace_bytes(*args) == -1
    assert L.orca_rows_grad_workspace_bytes(0, 0, 172) >= 0
    del keep


def test_python_refuses():
    from orca_b200.lookup import _scale_of, lookup_rows
    from orca_b200.packed import PackedHistory, PackedRows, _host_ids
    for make in (lambda: PackedRows(10, "cpu"), lambda: PackedHistory(10, 172, "cpu")):
        with pytest.raises(RuntimeError):
            make()
    for bad in (torch.zeros(3, 24, dtype=torch.int32), np.zeros((3, 24), np.int32), None):
        with pytest.raises(ValueError):
            PackedRows.from_words(bad)
    for bad in (0, -1, 1 << 31):
        with pytest.raises(ValueError):
            PackedRows(bad, "cuda")
    with pytest.raises(ValueError):
        lookup_rows(torch.zeros(3, 4), [0])
    for bad in (float("inf"), float("nan"), 1e39):
        with pytest.raises(ValueError):
            _scale_of(bad)
    for bad in ([3], [-1], [0, 1 << 40]):
        with pytest.raises(_lib.OrcaError):
            _host_ids(bad, 3, "ids")
    with pytest.raises(TypeError):
        _host_ids([0.5], 3, "ids")


def test_the_compiled_calls_check_what_they_get():
    m = _lib.rows()
    for name in ("lookup", "grad", "attend", "attend_lists", "push", "pull"):
        with pytest.raises(RuntimeError):
            getattr(m, name)()                         # (the number of arguments)
    for call in (lambda: m.pull(1, 2, 3), lambda: m.push(None, None, None, None, None), lambda: m.attend(*[None] * 8),
                 lambda: m.attend_lists(*[None] * 13)):
        with pytest.raises(TypeError):
            call()
    words, status, qt = torch.zeros(3, 24, dtype=torch.int32), torch.zeros(4, dtype=torch.int32), torch.zeros(2, 1056)
    edges, w, nbr, delta = torch.zeros(5, 172), torch.zeros(172), torch.zeros(2, 4, dtype=torch.int32), torch.zeros(2, 4)
    for i, bad in ((2, qt[:, :1032]), (3, edges.half()), (3, edges[:0]), (4, w[:9]), (5, nbr.long()), (6, nbr[:, :3]), (7, delta.double())):
        args = [words, status, qt, edges, w, nbr, nbr, delta]
        args[i] = bad
        with pytest.raises(ValueError):
            m.attend(*args)
