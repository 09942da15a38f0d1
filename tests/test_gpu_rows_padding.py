"""Padding of the tables that attention reads: neighbour 0 is no slot, whatever stands beside it."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("edge", ["packed", "float32"])
@pytest.mark.parametrize("rows,k", [(1, 10), (50, 20), (3, 300), (200, 33)])
def test_padding_slots_carry_any_edge(edge, rows, k):
    """The same bits as with edge 0 beside them, and nothing is reported."""
    from orca_b200.packed import PackedRows
    dev = torch.device("cuda:0")
    rs = np.random.RandomState(rows + k)
    up = lambda a: torch.from_numpy(a).to(dev)
    p = PackedRows.of(up(rs.randn(60, 172).astype(np.float32)))
    edges = up(rs.randn(70, 172).astype(np.float32))
    edges = PackedRows.of(edges) if edge == "packed" else edges
    nbr = np.where(rs.rand(rows, k) < 0.5, 0, rs.randint(1, 60, (rows, k))).astype(np.int32)
    eid = np.where(nbr == 0, 0, rs.randint(0, 70, (rows, k))).astype(np.int32)
    delta = np.where(nbr == 0, 0, rs.uniform(0, 1e6, (rows, k))).astype(np.float32)
    qt, w = up(rs.randn(rows, 1056).astype(np.float32)), up((1 / 10 ** np.linspace(0, 9, 172)).astype(np.float32))
    want = p.attend(qt, up(nbr), up(eid), up(delta), edges, w)
    for pad in (-1, 70, -2 ** 31, 2 ** 31 - 1):
        got = p.attend(qt, up(nbr), up(np.where(nbr == 0, pad, eid).astype(np.int32)), up(np.where(nbr == 0, np.nan, delta).astype(np.float32)),
                       edges, w)
        assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
        p.check_status()
