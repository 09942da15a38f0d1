"""Derivatives that the calls on rows do not have: each is refused where it is asked for, none is left out in silence."""
import pytest
import torch
from torch.autograd import forward_ad as fw

pytestmark = pytest.mark.gpu


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def test_a_tangent_in_a_lookups_backward_pass(dev):
    """Forward over reverse: the gradient would carry the tangent of what stands behind the lookup."""
    from orca_b200.lookup import lookup_rows
    table = torch.randn(50, 172, device=dev, requires_grad=True)
    ids = torch.randint(0, 50, (7,), device=dev)
    w = torch.randn(7, 172, device=dev)
    with fw.dual_level():
        y = (lookup_rows(table, ids) * fw.make_dual(w, torch.ones_like(w))).sum()
        with pytest.raises(NotImplementedError, match="forward derivative"):
            torch.autograd.grad(y, table)
    (g,) = torch.autograd.grad((lookup_rows(table, ids) * w).sum(), table)       # (without one, as before)
    want = torch.zeros_like(table).index_add_(0, ids, w)
    # (seven addends at most on either side: six roundings of a sum of seven times the largest)
    assert (g - want).abs().max() <= 2 * 6 * 2.0 ** -24 * 7 * w.abs().max()


def test_derivatives_of_lookup_grad(dev):
    from orca_b200.lookup import lookup_grad
    ids = torch.randint(0, 50, (7,), device=dev)
    g = torch.randn(7, 172, device=dev)
    want = lookup_grad(g, ids, 50)
    with fw.dual_level():
        with pytest.raises(NotImplementedError, match="forward derivative"):
            lookup_grad(fw.make_dual(g, torch.ones_like(g)), ids, 50)
    g.requires_grad_(True)
    out = lookup_grad(g, ids, 50)
    assert torch.equal(out, want)
    with pytest.raises(RuntimeError, match="no derivative"):
        out.sum().backward()
    with torch.no_grad():
        assert not lookup_grad(g, ids, 50).requires_grad
    assert not lookup_grad(g.detach(), ids, 50).requires_grad


def _attention(dev):
    """A packed table, an adjacency, and arguments of both forms of attention."""
    from types import SimpleNamespace
    from orca_b200.packed import PackedRows
    rows = PackedRows.of(torch.randn(30, 172, device=dev))
    ids = lambda *s: torch.randint(1, 30, s, dtype=torch.int32, device=dev)
    adjacency = SimpleNamespace(n_nodes=3, indptr=torch.tensor([0, 0, 5, 12], device=dev), adj_nbr=ids(12), adj_eid=ids(12),
                                adj_ts=torch.arange(12, dtype=torch.float64, device=dev))
    both = dict(qt=torch.randn(2, 1056, device=dev), edges=torch.randn(30, 172, device=dev), time_w=torch.rand(172, device=dev))
    table = dict(both, nbr=ids(2, 4), eid=ids(2, 4), delta=torch.rand(2, 4, device=dev))
    lists = dict(both, finder=adjacency, nodes=torch.tensor([1, 2], device=dev), timestamps=torch.full((2,), 50.0, device=dev))
    return rows, table, lists


@pytest.mark.parametrize("name", ["qt", "edges", "time_w", "delta", "timestamps"])
def test_attention_refuses_inputs_that_ask_for_a_derivative(dev, name):
    rows, table, lists = _attention(dev)
    for call, args in ((rows.attend, table), (rows.attend_lists, lists)):
        if name not in args:
            continue
        want = call(**args)[0]
        leaf = args[name].clone().requires_grad_(True)
        with pytest.raises(NotImplementedError, match="no gradient"):
            call(**{**args, name: leaf})
        with torch.no_grad():
            assert torch.equal(call(**{**args, name: leaf})[0], want)
        with fw.dual_level():
            with pytest.raises(NotImplementedError, match="no gradient"):
                call(**{**args, name: fw.make_dual(args[name], torch.ones_like(args[name]))})


def test_embeddings_over_packed_rows_refuse_edges_that_ask_for_a_derivative(dev):
    from helpers import graph
    from orca_b200.packed import PackedHistory
    from test_gpu_model import make_model
    g = graph("t_nb2")
    tgn = make_model(g)
    h = PackedHistory(g.n_nodes, 172, dev)
    nodes, times = g.sources[-20:], g.timestamps[-20:]
    want = tgn.packed_embeddings(h, nodes, times, 10)
    edges = tgn.edge_raw_features.clone().requires_grad_(True)
    with pytest.raises(NotImplementedError, match="no gradient"):
        tgn.packed_embeddings(h, nodes, times, 10, edges)
    with torch.no_grad():
        assert torch.equal(tgn.packed_embeddings(h, nodes, times, 10, edges), want)


class Watched(torch.Tensor):
    """A tensor whose operators are its own."""
    @classmethod
    def __torch_dispatch__(cls, func, types, args=(), kwargs=None):
        raise AssertionError("not asked")


def test_traces_and_tensors_that_stand_for_others(dev):
    """A trace would keep outputs that nothing fills; vmap and torch.func hand over tensors without memory: refused, by the calls on rows as by those of a training step."""
    from orca_b200.lookup import lookup_grad, lookup_rows
    from orca_b200.norm import layer_norm, layer_norm_grad
    x, g = torch.randn(5, 7, 172, device=dev), torch.randn(5, 7, 172, device=dev)
    ids = torch.randint(0, 7, (9,), device=dev)
    for f, args in ((layer_norm, (x,)), (layer_norm_grad, (g, x)), (lambda t: lookup_rows(t, ids), (x[0],)), (lambda t: lookup_grad(t, ids, 9), (torch.randn(9, 172, device=dev),))):
        want = f(*args)
        with pytest.raises(NotImplementedError, match="traced"):
            torch.jit.trace(f, args)
        got = f(*args)
        assert all(torch.equal(a, b) for a, b in (zip(want, got) if isinstance(want, tuple) else ((want, got),)))
    for call in (lambda: torch.func.vmap(layer_norm)(x), lambda: torch.func.grad(lambda t: layer_norm(t).sum())(x), lambda: torch.func.vmap(lambda t: lookup_rows(t, ids))(x),
                 lambda: layer_norm(torch.Tensor._make_subclass(Watched, x)), lambda: torch.func.vmap(lambda w: layer_norm(x[0], w))(x[0])):
        with pytest.raises(NotImplementedError, match="memory"):
            call()
    assert torch.equal(layer_norm(torch.nn.Parameter(x)), layer_norm(x))
