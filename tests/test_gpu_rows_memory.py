"""What tables of rows in 4 bits take on the device."""
import numpy as np
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_a_packed_history_is_its_rows_flags_and_record():
    """96 bytes a row, 4 for the last position of a pushed id, 1 for its flag; 4 more where the budget is all rows."""
    from orca_b200.history import History
    from orca_b200.packed import PackedHistory
    dev = torch.device("cuda:0")
    n, sizes = 500_000, {}
    # (bytes that were asked for: the allocator hands out blocks that are up to 1 MB larger)
    asked = lambda: torch.cuda.memory_stats()["requested_bytes.all.current"]
    x, ids = torch.ones(2000, 172, device=dev), torch.arange(2000, device=dev)
    for name, make in (("packed", lambda: PackedHistory(n, 172, dev, 10)), ("all", lambda: PackedHistory(n, 172, dev)), ("fp32", lambda: History(n, 172, dev))):
        before = asked()
        h = make()
        h.push(x, ids)
        assert bool((h.pull(ids) == 1).all())
        torch.cuda.synchronize()
        sizes[name] = asked() - before
        del h
    assert sizes["packed"] <= 101 * n + 16 * 512 and sizes["all"] <= 105 * n + 16 * 512
    assert sizes["fp32"] >= 6.6 * sizes["all"]


def test_a_history_in_fp32_keeps_the_last_of_equal_ids():
    from orca_b200.history import History
    dev = torch.device("cuda:0")
    h = History(50, 172, dev)
    rs = np.random.RandomState(0)
    for _ in range(3):
        x, ids = rs.randn(40, 172).astype(np.float32), rs.randint(0, 50, 40)
        want = h.emb.cpu().numpy().copy()
        for i, row in zip(ids, x):
            want[i] = row
        h.push(torch.from_numpy(x).to(dev), ids)
        assert np.array_equal(h.emb.cpu().numpy(), want)
