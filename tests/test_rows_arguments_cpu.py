"""What the calls on rows refuse before anything is launched.  No GPU is needed: the checks come before the device is asked for."""
from types import SimpleNamespace

import pytest
import torch

from orca_b200 import _lib


def _lists(n_nodes=9, slots=40):
    """Arguments of the compiled attend_lists, on the CPU."""
    words, status, qt = torch.zeros(3, 24, dtype=torch.int32), torch.zeros(4, dtype=torch.int32), torch.zeros(2, 1056)
    edges, w = torch.zeros(5, 172), torch.zeros(172)
    ids = torch.zeros(slots, dtype=torch.int32)
    return dict(words=words, status=status, qt=qt, edges=edges, w=w, indptr=torch.zeros(n_nodes + 1, dtype=torch.int64), adj_nbr=ids,
                adj_eid=ids, adj_ts=torch.zeros(slots, dtype=torch.float64), n_nodes=n_nodes, nodes=torch.zeros(2, dtype=torch.int32),
                times=torch.zeros(2, dtype=torch.float64), last=0)


@pytest.mark.parametrize("name", ["indptr", "adj_nbr", "adj_eid", "adj_ts"])
@pytest.mark.parametrize("how", ["column", "expanded", "turned"])
def test_an_adjacency_of_views_is_refused(name, how):
    """The kernel reads these arrays as they lie in memory: a column's values lie elsewhere, an expanded one's storage ends early."""
    a = _lists()
    t = a[name]
    a[name] = {"column": lambda: t[:, None].repeat(1, 3)[:, 1], "expanded": lambda: t[:1].expand(len(t)), "turned": lambda: t.repeat(2)[::2]}[how]()
    assert a[name].shape == t.shape
    with pytest.raises(ValueError, match="contiguous"):
        _lib.rows().attend_lists(*a.values())


@pytest.mark.parametrize("kind", ["rows", "history"])
def test_embeddings_refuse_a_history_of_another_device(monkeypatch, kind):
    """Its rows would be handed to kernels on the model's device."""
    from orca_b200.packed import PackedHistory, PackedRows
    from orca_b200.tgn import TGN
    rows = PackedRows.__new__(PackedRows)
    rows.device = torch.device("cuda:1")
    monkeypatch.setattr(PackedRows, "pull", lambda *a: pytest.fail("it was read"))
    model = SimpleNamespace(device=torch.device("cuda:0"), edge_raw_features=SimpleNamespace(device=torch.device("cuda:0")), n_layers=2)
    history = rows
    if kind == "history":
        history = PackedHistory.__new__(PackedHistory)
        torch.nn.Module.__init__(history)
        history.rows = rows
    with pytest.raises(ValueError, match="cuda:1"):
        TGN.packed_embeddings(model, history, [1], [0.0])


def test_embeddings_refuse_what_is_not_packed(monkeypatch):
    from orca_b200.history import History
    from orca_b200.tgn import TGN
    history = History.__new__(History)
    torch.nn.Module.__init__(history)
    monkeypatch.setattr(History, "pull", lambda *a: pytest.fail("it was read"))
    model = SimpleNamespace(device=torch.device("cuda:0"), edge_raw_features=SimpleNamespace(device=torch.device("cuda:0")), n_layers=2)
    for other in (history, torch.zeros(3, 172), None):
        with pytest.raises(TypeError, match="PackedRows"):
            TGN.packed_embeddings(model, other, [1], [0.0])
