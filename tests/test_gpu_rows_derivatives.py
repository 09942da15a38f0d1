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
