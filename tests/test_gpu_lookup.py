"""Lookups of trained rows and their gradient on the GPU, against 64 bits.

A looked-up value is scale * row rounded once in fp32 and once to the table's type.  A gradient sums cnt contributions in fp32: cnt
roundings of the sum of magnitudes at most, the scale's, and the type's."""
import numpy as np
import pytest
import torch

import rows_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _half(t):
    return torch.finfo(t).eps / 2


def _tiny(t):
    return torch.finfo(t).smallest_normal * torch.finfo(t).eps      # a step below the normal values


def _check_rows(out, table, ids, scale):
    t = table.detach().double().cpu().numpy()
    inside = (ids >= 0) & (ids < len(t))
    want = np.where(inside[..., None], t[np.where(inside, ids, 0)] * np.float64(np.float32(scale)), 0.0)
    got = out.detach().double().cpu().numpy()
    assert got.shape == want.shape
    assert (np.abs(got - want) <= (_half(out.dtype) + ref.EPS) * np.abs(want) + _tiny(out.dtype)).all()


def _check_grad(got, g, ids, n, scale, padding, dtype):
    want, mag, cnt = ref.lookup_grad(g.double().cpu().numpy().reshape(ids.size, g.shape[-1]), ids.reshape(-1), n, float(np.float32(scale)), padding)
    got = got.double().cpu().numpy()
    assert (np.abs(got - want) <= _half(dtype) * np.abs(want) + ref.EPS * (cnt[:, None] + 1) * (1 + 2.0 ** -7) * mag + _tiny(dtype)).all()
    assert not got[cnt == 0].any()


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("m,n,width,ids", [(1, 1, 1, "same"), (1, 7, 172, "any"), (31, 4, 172, "any"), (600, 9228, 172, "any"),
                                           (2049, 300, 33, "any"), (5000, 70000, 172, "skewed"), (20011, 50, 7, "skewed"),
                                           (9000, 12, 172, "same"), (33, 10, 600, "any"), (2048, 40, 172, "skewed"), (66001, 3, 5, "same"), (700, 300, 1031, "any"), (70001, 66000, 20, "any")])
def test_lookup_and_gradient(dev, dtype, m, n, width, ids):
    from orca_b200.lookup import lookup_rows
    rs = np.random.RandomState(m + width)
    table = torch.from_numpy(rs.randn(n, width).astype(np.float32)).to(dev, dtype).requires_grad_(True)
    at = {"any": lambda: rs.randint(0, n, m), "same": lambda: np.full(m, n - 1), "skewed": lambda: (rs.rand(m) ** 4 * n).astype(np.int64)}[ids]()
    g = torch.from_numpy(rs.randn(m, width).astype(np.float32)).to(dev, dtype)
    grads = []
    for wide, scale, padding in ((torch.int64, 1.0, None), (torch.int32, 1.0, None), (torch.int32, -2.7, int(at[0]))):
        d = torch.from_numpy(at).to(dev, wide)
        out = lookup_rows(table, d, scale, padding)
        _check_rows(out, table, at, scale)
        (grad,) = torch.autograd.grad(out, table, g)
        assert grad.dtype == dtype
        _check_grad(grad, g, at, n, scale, padding, dtype)
        grads.append(grad)
    assert torch.equal(grads[0], grads[1])


def test_gradient_against_differences(dev):
    """The directional derivative of a sum of squares from the gradient, and from values of the function in 64 bits."""
    from orca_b200.lookup import lookup_rows
    rs = np.random.RandomState(3)
    start, way, ids = rs.randn(40, 172), rs.randn(40, 172), rs.randint(0, 40, 333)
    table = torch.from_numpy(start.astype(np.float32)).to(dev).requires_grad_(True)
    (lookup_rows(table, ids, 1.5) ** 2).sum().backward()
    f = lambda t: ((1.5 * t[ids]) ** 2).sum()
    h = 1e-4
    slope = (f(start + h * way) - f(start - h * way)) / (2 * h)          # (of a square: exact but for 64-bit roundings)
    got = float((table.grad.double().cpu().numpy() * way).sum())
    mag = (np.abs(4.5 * start[ids]) * np.abs(way[ids])).sum()
    assert abs(got - slope) <= ref.EPS * 30 * mag


def test_shapes_strides_and_expanded_gradients(dev):
    from orca_b200.lookup import lookup_rows, lookup_grad
    rs = np.random.RandomState(5)
    big = torch.from_numpy(rs.randn(30, 400).astype(np.float32)).to(dev)
    for table in (big[:, 3:175], big[::2, :172], big[:, ::2], big.t()[:172].contiguous().t(), big[:1, :9], big[:, 4:6]):
        for shape in ((), (0,), (5,), (2, 3, 4), (7, 0)):
            ids = rs.randint(0, table.shape[0], shape)
            t = table.detach().requires_grad_(True)
            d = torch.from_numpy(np.asarray(ids)).to(dev)
            out = lookup_rows(t, d, 0.5)
            _check_rows(out, t, np.asarray(ids), 0.5)
            out.sum().backward()                                        # (an expanded gradient)
            _check_grad(t.grad, torch.ones(max(ids.size, 0) if shape else 1, table.shape[1]), np.asarray(ids), table.shape[0], 0.5, None,
                        torch.float32)
    d = torch.from_numpy(rs.randint(0, 30, (6, 10))).to(dev)
    wide = torch.from_numpy(rs.randn(6, 10, 50).astype(np.float32)).to(dev)
    for g in (wide[..., 1:34], wide.transpose(0, 1).contiguous().transpose(0, 1), wide[:, :1].expand(6, 10, 50), wide[..., ::3]):
        _check_grad(lookup_grad(g, d, 30), g, d.cpu().numpy(), 30, 1.0, None, torch.float32)
    turned = d.t()
    assert torch.equal(lookup_rows(big, turned), big[turned])


def test_ids_outside_the_table(dev):
    from orca_b200 import _lib
    from orca_b200.lookup import lookup_grad, lookup_rows
    rs = np.random.RandomState(6)
    table = torch.from_numpy(rs.randn(20, 172).astype(np.float32)).to(dev)
    ids = np.array([3, 20, -1, 19, 1 << 40, -(1 << 40) + 3, 0])
    d, status = torch.from_numpy(ids).to(dev), torch.zeros(4, dtype=torch.int32, device=dev)
    _check_rows(lookup_rows(table, d, 1.0, status=status), table, ids, 1.0)
    assert int(status[0]) == _lib.E_BOUNDS
    status.zero_()
    g = torch.from_numpy(rs.randn(7, 172).astype(np.float32)).to(dev)
    _check_grad(lookup_grad(g, d, 20, status=status), g, ids, 20, 1.0, None, torch.float32)
    assert int(status[0]) == _lib.E_BOUNDS
    _check_rows(lookup_rows(table, d), table, ids, 1.0)            # (without a status they are left out all the same)
    for bad in (ids, [20], np.array([-1])):
        with pytest.raises(_lib.OrcaError):
            lookup_rows(table, bad)
    empty = torch.zeros(0, 5, device=dev)
    assert not lookup_rows(empty, torch.tensor([0, 3], device=dev)).any()
    assert lookup_grad(torch.ones(2, 5, device=dev), torch.tensor([0, 3], device=dev), 0).shape == (0, 5)


def test_values_that_are_not_numbers_stay_in_their_rows(dev):
    from orca_b200.lookup import lookup_grad
    rs = np.random.RandomState(7)
    ids = rs.randint(1, 50, 4000)
    g = rs.randn(4000, 172).astype(np.float32)
    bad = np.flatnonzero(ids == 7)[3]
    g[bad, 11], g[np.flatnonzero(ids == 9)[0], 0] = np.nan, np.inf
    got = lookup_grad(torch.from_numpy(g).to(dev), torch.from_numpy(ids).to(dev), 50).cpu().numpy()
    assert np.isnan(got[7, 11]) and np.isposinf(got[9, 0]) and np.isfinite(got).sum() == got.size - 2


def test_streams_and_a_captured_gradient(dev):
    """The gradient from a graph, replayed with other ids, while an eager graph of the same table lives; two streams at once."""
    from orca_b200.lookup import lookup_grad, lookup_rows
    rs = np.random.RandomState(8)
    table = torch.from_numpy(rs.randn(500, 172).astype(np.float32)).to(dev).requires_grad_(True)
    at = [torch.from_numpy(rs.randint(0, 500, 3001)).to(dev) for _ in range(3)]
    g = torch.from_numpy(rs.randn(3001, 172).astype(np.float32)).to(dev)
    want = [lookup_grad(g, i, 500, 0.3) for i in at]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [None, None]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = lookup_grad(g, at[i], 500, 0.3)
    torch.cuda.synchronize()
    assert torch.equal(got[0], want[0]) and torch.equal(got[1], want[1])
    alive = lookup_rows(table, at[0], 0.3)
    ids = at[0].clone()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rows, out = lookup_rows(table.detach(), ids, 0.3), lookup_grad(g, ids, 500, 0.3)
    for i in (1, 2, 0):
        ids.copy_(at[i])
        graph.replay()
        assert torch.equal(out, want[i]) and torch.equal(rows, lookup_rows(table.detach(), at[i], 0.3))
    alive.backward(g)
    assert torch.equal(table.grad, want[0])


def test_second_derivatives_are_refused(dev):
    from orca_b200.lookup import lookup_rows
    table = torch.randn(5, 4, device=dev, requires_grad=True)
    (g,) = torch.autograd.grad((lookup_rows(table, [1, 2]) ** 2).sum(), table, create_graph=True)
    with pytest.raises(RuntimeError):
        torch.autograd.grad(g.sum(), table)


def test_what_the_node_refuses(dev):
    from orca_b200.lookup import lookup_grad, lookup_rows
    table = torch.randn(50, 172, device=dev, requires_grad=True)
    ids = torch.randint(0, 50, (7,), device=dev)
    out = lookup_rows(table, ids)
    out.sum().backward()
    with pytest.raises(RuntimeError):
        out.sum().backward()                  # (no second pass without retain_graph)
    out = lookup_rows(table, ids)
    ids.add_(0)
    with pytest.raises(RuntimeError):
        out.sum().backward()                  # (its ids were written in place)
    with pytest.raises(NotImplementedError):
        with torch.autograd.forward_ad.dual_level():
            lookup_rows(torch.autograd.forward_ad.make_dual(table.detach(), torch.ones_like(table)), ids)
    for bad in (float("inf"), 1e39):
        with pytest.raises(ValueError):
            lookup_rows(table, ids, bad)
        with pytest.raises(ValueError):
            lookup_grad(out.detach(), ids, 50, bad)
    for call in (lambda: lookup_rows(table, ids, padding=50), lambda: lookup_rows(table, ids, status=torch.zeros(4, device=dev)),
                 lambda: lookup_rows(table[:, :0], ids), lambda: lookup_grad(out.detach(), ids[:3], 50), lambda: lookup_grad(out.sum(), ids, 50)):
        with pytest.raises(ValueError):
            call()
    with pytest.raises(TypeError):
        lookup_rows(table, ids.short())
    from orca_b200._lib import OrcaError
    long = torch.empty(0x7fffffff, 1, dtype=torch.bfloat16, device=dev)
    with pytest.raises(OrcaError):
        lookup_rows(long, ids)                # (more rows than the library takes)


def test_graphs_of_a_lookup(dev):
    """retain_graph, two lookups of one table, a table that is not a leaf, no graph where none is wanted, a single id without a shape."""
    from orca_b200.lookup import lookup_rows
    table = torch.randn(50, 172, device=dev, requires_grad=True)
    ids = torch.randint(0, 50, (7, 3), device=dev)
    out = lookup_rows(table, ids)
    (a,) = torch.autograd.grad(out.sum(), table, retain_graph=True)
    (b,) = torch.autograd.grad(out.sum(), table)
    assert torch.equal(a, b) and torch.equal(a.sum(1) / 172, torch.bincount(ids.reshape(-1), minlength=50).float())
    (c,) = torch.autograd.grad((lookup_rows(table, ids) + lookup_rows(table, ids.int())).sum(), table)
    assert torch.equal(c, 2 * a)
    (d,) = torch.autograd.grad(lookup_rows(2 * table, ids).sum(), table)
    assert torch.equal(d, 2 * a)
    assert lookup_rows(table.detach(), ids).grad_fn is None
    with torch.no_grad():
        assert not lookup_rows(table, ids).requires_grad
    for one in (3, np.int64(3), torch.tensor(3), torch.tensor(3, device=dev)):
        assert torch.equal(lookup_rows(table, one), table[3])


def test_offsets_past_32_bits(dev):
    """A table and a gradient of more than 2^32 bytes."""
    from orca_b200.lookup import lookup_grad, lookup_rows
    rs = np.random.RandomState(33)
    m = 6_300_000
    table = torch.zeros(m, 172, device=dev)
    x = torch.from_numpy(rs.randn(60, 172).astype(np.float32)).to(dev)
    table[m - 60:] = x
    for n in (50, 3000):                    # (few ids, and ids that are sorted)
        at = torch.from_numpy(rs.randint(0, 60, n)).to(dev)
        assert torch.equal(lookup_rows(table, at + m - 60, 2.0), 2 * x[at])
        g = torch.from_numpy(rs.randn(n, 172).astype(np.float32)).to(dev)
        grad = lookup_grad(g, at + m - 60, m)
        want, mag, cnt = ref.lookup_grad(g.cpu().numpy(), at.cpu().numpy(), 60, 1.0)
        assert (np.abs(grad[m - 60:].cpu().numpy() - want) <= ref.EPS * (cnt[:, None] + 1) * mag).all()
        assert not grad[:m - 60].any()


def test_captured_backward_pass(dev):
    """Replayed with other ids; refused while an eager graph of the same table lives, whose stream it would end on."""
    from orca_b200.lookup import lookup_grad, lookup_rows
    table = torch.randn(50, 172, device=dev, requires_grad=True)
    g = torch.randn(40, 172, device=dev)
    at = [torch.randint(0, 50, (40,), device=dev) for _ in range(3)]
    ids = at[0].clone()
    alive = lookup_rows(table, ids)
    with pytest.raises(RuntimeError, match="lookup_grad"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            out = lookup_rows(table, ids)
            torch.autograd.grad(out, table, g)
    del out
    torch.cuda.synchronize()
    alive.backward(g)
    assert torch.equal(table.grad, lookup_grad(g, ids, 50))
    del alive
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        (grad,) = torch.autograd.grad(lookup_rows(table, ids), table, g)
    for a in at[1:]:
        ids.copy_(a)
        graph.replay()
        assert torch.equal(grad, lookup_grad(g, a, 50))
