"""The workspace of attention over the last interactions of lists: as much as is asked for is enough, and no more is taken."""
from types import SimpleNamespace

import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu

GUARD = 1 << 16


def _case(rows, slots, n=40):
    """Queries that all have whole lists of `slots` interactions."""
    from orca_b200.packed import PackedRows
    dev = torch.device("cuda:0")
    rs = np.random.RandomState(rows + slots)
    up = lambda a: torch.from_numpy(a).to(dev)
    lists = 7
    a = SimpleNamespace(n_nodes=lists, indptr=up(np.arange(lists + 1, dtype=np.int64) * slots), adj_nbr=up(rs.randint(1, n, lists * slots).astype(np.int32)),
                        adj_eid=up(rs.randint(0, n, lists * slots).astype(np.int32)), adj_ts=up(np.tile(np.arange(slots) * 1000.0, lists)))
    table = PackedRows.of(up(rs.randn(n, 172).astype(np.float32)))
    return dict(p=table, a=a, qt=up(rs.randn(rows, 1056).astype(np.float32)), nodes=up(rs.randint(0, lists, rows).astype(np.int32)),
                times=up(np.full(rows, 1e9)), w=up((1 / 10 ** np.linspace(0, 9, 172)).astype(np.float32)))


@pytest.mark.parametrize("rows", [1, 64, 65, 600])
@pytest.mark.parametrize("last", [1, 10, 16, 17, 64, 65, 129, 1000])
def test_what_is_asked_for_is_enough(rows, last):
    """Nothing behind it is written; the same bits as with the workspace for lists of any length."""
    from orca_b200 import _lib
    L = _lib.lib()
    c = _case(rows, 1000)
    p, a, dev = c["p"], c["a"], c["qt"].device
    need, most = L.orca_packed_attend_last_workspace_bytes(rows, last), L.orca_packed_attend_lists_workspace_bytes(rows)
    assert need <= most

    def run(nbytes):
        ws = torch.full((nbytes + GUARD,), 0xab, dtype=torch.uint8, device=dev)
        ctx, valid = torch.empty(rows, 1032, device=dev), torch.empty(rows, dtype=torch.uint8, device=dev)
        _lib.check(L.orca_packed_attend_lists(c["qt"].data_ptr(), p.words.data_ptr(), 40, p.words.data_ptr(), 40, 1, c["w"].data_ptr(),
                                              a.indptr.data_ptr(), a.adj_nbr.data_ptr(), a.adj_eid.data_ptr(), a.adj_ts.data_ptr(), 7,
                                              c["nodes"].data_ptr(), c["times"].data_ptr(), last, rows, ctx.data_ptr(), valid.data_ptr(),
                                              p.status.data_ptr(), ws.data_ptr(), nbytes, _lib.stream_ptr(dev)))
        assert bool((ws[nbytes:] == 0xab).all()) and bool(valid.all())
        return ctx

    assert torch.equal(run(need), run(most))
    p.check_status()


@pytest.mark.parametrize("rows", [65, 600, 6000])
def test_the_last_ten_take_little_memory(rows):
    c = _case(rows, 50)
    call = lambda: c["p"].attend_lists(c["qt"], c["a"], c["nodes"], c["times"], c["p"], c["w"], last=10)
    ctx, _ = call()
    torch.cuda.synchronize()
    torch.cuda.reset_peak_memory_stats()
    before = torch.cuda.memory_allocated()
    again, _ = call()
    # what it returns, each rounded up to 512 bytes, and 20 bytes a row beside it (blocks of the allocator: 2 MB at most)
    assert torch.cuda.max_memory_allocated() - before <= rows * (1032 * 4 + 1 + 20) + (2 << 20)
    assert torch.equal(ctx, again)
