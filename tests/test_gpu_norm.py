"""Layer norm and its gradients on the GPU, against 64 bits: bounds of train_reference.py and half a step of the output's type."""
import numpy as np
import pytest
import torch

import train_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
EPS = 1e-5


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _np(t):
    return t.detach().double().cpu().numpy()


def _within(got, want, off):
    got, half = _np(got), torch.finfo(got.dtype).eps / 2
    tiny = torch.finfo(torch.float32).smallest_normal * 2.0 ** -23 if half < 2.0 ** -20 else 2.0 ** -24      # (a step below the normal values of fp16)
    assert got.shape == want.shape
    far = np.abs(got - want) - (half * (np.abs(want) + off) + off + tiny)
    assert (far <= 0).all(), (np.unravel_index(far.argmax(), far.shape), far.max())


def _tensors(dev, rows, width, dtype, weight_dtype, seed=0, spread=1.0, offset=0.5):
    rs = np.random.RandomState(seed + rows + width)
    t = lambda a, d=dtype: torch.from_numpy(np.asarray(a, dtype=np.float32)).to(dev, d)
    x = t(rs.randn(rows, width) * spread + offset * rs.randn(rows, 1))
    return x, t(1 + 0.2 * rs.randn(width), weight_dtype), t(0.3 * rs.randn(width), weight_dtype), t(rs.randn(rows, width))


def _check(x, w, b, g, out, grads, eps=EPS):
    width = x.shape[-1]
    x, g = _np(x).reshape(-1, width), None if g is None else _np(g).reshape(-1, width)
    w64, b64 = np.ones(width) if w is None else _np(w), np.zeros(width) if b is None else _np(b)
    y, *_, off = ref.norm(x, w64, b64, float(np.float32(eps)))
    _within(out.reshape(-1, width), y, off)
    if grads is not None:
        want = ref.norm_grad(g, x, w64, float(np.float32(eps)))
        for got, value, bound in zip(grads, want[:3], want[3:]):
            if got is not None:
                _within(got.reshape(value.shape), value, bound)


def _run(x, w, b, g, eps=EPS):
    from orca_b200.norm import layer_norm
    leaves = [t.detach().requires_grad_(True) if t is not None else None for t in (x, w, b)]
    out = layer_norm(*leaves, eps)
    assert out.dtype == x.dtype and out.shape == x.shape
    there = [t for t in leaves if t is not None]
    grads = list(torch.autograd.grad(out, there, g))
    for t, d in zip(there, grads):
        assert d.dtype == t.dtype and d.shape == t.shape
    return out, [grads.pop(0) if t is not None else None for t in leaves]


WIDTHS = [1, 2, 3, 5, 8, 31, 32, 33, 64, 100, 127, 128, 172, 192, 256, 260, 344, 512, 515, 516, 640, 688, 1000, 1023, 1024, 1032, 2048, 2051, 4096, 4104, 8192, 8200,
          16384, 16392, 20001, 40000]


@pytest.mark.parametrize("dtype,weights", [(t, w) for t in TYPES for w in dict.fromkeys((t, torch.float32))], ids=str)
@pytest.mark.parametrize("width", WIDTHS)
def test_widths(dev, width, dtype, weights):
    for rows in (1, 2, 7, 67) if width <= 8200 else (1, 5):
        x, w, b, g = _tensors(dev, rows, width, dtype, weights)
        out, grads = _run(x, w, b, g)
        _check(x, w, b, g, out, grads)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,width", [(600, 172), (6000, 172), (70001, 172), (100003, 8), (30011, 33), (4001, 688), (5003, 515), (900, 4096), (300, 8192), (257, 10000),
                                        (200001, 1), (2500, 2051)])
def test_many_rows(dev, rows, width, dtype):
    x, w, b, g = _tensors(dev, rows, width, dtype, dtype)
    out, grads = _run(x, w, b, g)
    _check(x, w, b, g, out, grads)
    again, same = _run(x, w, b, g)
    assert torch.equal(out, again) and all(torch.equal(p, q) for p, q in zip(grads, same))


@pytest.mark.parametrize("width", [172, 688, 8192, 40000])
@pytest.mark.parametrize("offset", [1e4, 1e6])
def test_rows_far_from_zero(dev, width, offset):
    """A mean of ten thousand, or a million, times the spread: its rounding to fp32 is as large as the values around it."""
    x, w, b, g = _tensors(dev, 40, width, torch.float32, torch.float32, offset=offset)
    out, grads = _run(x, w, b, g)
    _check(x, w, b, g, out, grads)


def test_few_values_and_constant_rows(dev):
    from orca_b200.norm import layer_norm, layer_norm_grad
    for dtype in TYPES:
        for width in (1, 172, 8192, 20000):
            x = torch.full((3, width), 2.5, device=dev, dtype=dtype)
            w, b = torch.full((width,), 3.0, device=dev, dtype=dtype), torch.full((width,), 0.25, device=dev, dtype=dtype)
            assert torch.equal(layer_norm(x, w, b), b.expand(3, width))           # nothing varies: the bias
            dx, dw, db = layer_norm_grad(torch.ones_like(x), x, w)
            assert not dw.any() and (db == 3).all() and torch.isfinite(dx).all()
            assert layer_norm(x, w, b, eps=0.0).isnan().all()                     # 0 / 0, as the formula has it


@pytest.mark.parametrize("width", [33, 172, 1024, 8192, 20000])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_without_weight_or_bias(dev, width, dtype):
    for other in dict.fromkeys((dtype, torch.float32)):
        x, w, b, g = _tensors(dev, 19, width, dtype, other)
        for weight, bias in ((None, None), (w, None), (None, b)):
            out, grads = _run(x, weight, bias, g)
            _check(x, weight, bias, g, out, grads)


@pytest.mark.parametrize("width", [7, 172, 688, 8192, 20000])
def test_what_is_not_a_number_stays_in_its_row(dev, width):
    for value in (float("nan"), float("inf"), -float("inf")):
        x, w, b, g = _tensors(dev, 70, width, torch.float32, torch.float32)
        x[11, width // 2] = value
        out, (dx, dw, db) = _run(x, w, b, g)
        assert out[11].isnan().all() and dx[11].isnan().all() and dw.isnan().all() and torch.isfinite(db).all()
        rest = [i for i in range(70) if i != 11]
        _check(x[rest], w, b, g[rest], out[rest], [dx[rest], None, None])


@pytest.mark.parametrize("width", [6, 172, 688, 8192])
def test_shapes_and_strides(dev, width):
    """Rows that lie apart, turned, shifted by an element, repeated; gradients likewise."""
    rs = np.random.RandomState(4)
    new = lambda *s: torch.from_numpy(rs.randn(*s).astype(np.float32)).to(dev)
    w, b = new(width + 1)[1:], new(width + 3)[3:]
    wide = new(9, 2 * width + 5)
    flat = new(5 * width + 1)[1:].view(5, width)
    views = [wide[:, :width], wide[:, 3:3 + width], wide[::2, 4:4 + width], new(width, 7).t(), new(7, 2 * width)[:, ::2], flat, new(2, 3, 4, width), new(2, 3, width).transpose(0, 1),
             new(3, 1, width).expand(3, 5, width), new(width), new(1, width), new(0, width), new(4, 0, width), new(6, 8, width)[:, 2:5]]
    for x in views:
        for dtype in (torch.float32, torch.bfloat16):
            x_ = x if dtype == torch.float32 else x.to(dtype)        # (keeps strides that fill memory)
            g = new(*x.shape).to(dtype)
            for g_ in (g, g[..., :1].expand(x.shape), torch.zeros(1, device=dev, dtype=dtype).add_(0.5).expand(x.shape)):
                out, grads = _run(x_, w, b, g_)
                _check(x_, w, b, g_, out, grads)
    for shape in ((0, width), (2, 0, width)):
        _, (dx, dw, db) = _run(torch.zeros(shape, device=dev), w, b, torch.zeros(shape, device=dev))
        assert dx.shape == shape and not dw.any() and not db.any()


@pytest.mark.parametrize("width", [172, 2048, 20000])
def test_only_what_is_wanted(dev, width):
    from orca_b200.norm import layer_norm, layer_norm_grad
    x, w, b, g = _tensors(dev, 300, width, torch.float32, torch.float32)
    want = layer_norm_grad(g, x, w)
    for which in ((1, 0, 0), (0, 1, 0), (0, 0, 1), (1, 0, 1), (0, 1, 1)):
        leaves = [t.detach().requires_grad_(bool(k)) for t, k in zip((x, w, b), which)]
        (layer_norm(*leaves) * g).sum().backward()
        for t, d, k in zip(leaves, want, which):
            assert (t.grad is not None) == bool(k) and (t.grad is None or torch.equal(t.grad, d))
    assert not layer_norm(x, w, b).requires_grad
    with torch.no_grad():
        assert not layer_norm(x.requires_grad_(True), w, b).requires_grad


def test_gradients_against_differences(dev):
    """The slope of a sum of squares along a direction, from the gradients and from values of the function in 64 bits.  Differences of a smooth
    function err by h^2 / 6 of its third derivative: ten thousand times less than the bound here."""
    rs = np.random.RandomState(3)
    x, w, b = rs.randn(30, 172), 1 + 0.1 * rs.randn(172), 0.1 * rs.randn(172)
    x, w, b = (a.astype(np.float32).astype(np.float64) for a in (x, w, b))
    ways = [rs.randn(*a.shape) for a in (x, w, b)]
    f = lambda x, w, b: (ref.norm(x, w, b, float(np.float32(EPS)))[0] ** 2).sum()
    from orca_b200.norm import layer_norm
    leaves = [torch.from_numpy(a.astype(np.float32)).to(dev).requires_grad_(True) for a in (x, w, b)]
    (layer_norm(*leaves) ** 2).sum().backward()
    y, *_, off_y = ref.norm(x, w, b, float(np.float32(EPS)))
    *_, off_x, off_w, off_b = ref.norm_grad(2 * y, x, w, float(np.float32(EPS)))
    # (2 y is off itself by twice the forward pass's bound: another such share of each gradient's terms)
    more = ref.norm_grad(2 * off_y + 2 * ref.U * np.abs(y), x, np.abs(w), float(np.float32(EPS)))
    _, h, r, *_ = ref.norm(x, w, b, float(np.float32(EPS)))
    d = (2 * off_y + 2 * ref.U * np.abs(y))
    off_x = off_x + r * (d * np.abs(w) + (d * np.abs(w)).mean(1, keepdims=True) + np.abs(h) * (d * np.abs(w * h)).mean(1, keepdims=True))
    off_w, off_b = off_w + (d * np.abs(h)).sum(0), off_b + d.sum(0)
    del more
    step = 1e-4
    for i, (leaf, way, off) in enumerate(zip(leaves, ways, (off_x, off_w, off_b))):
        moved = lambda s: [a + s * way if k == i else a for k, a in enumerate((x, w, b))]
        slope = (f(*moved(step)) - f(*moved(-step))) / (2 * step)
        got = (_np(leaf.grad) * way).sum()
        bound = (off * np.abs(way)).sum() + ref.U * np.abs(_np(leaf.grad) * way).sum() + 1e-6 * abs(slope)
        assert abs(got - slope) <= bound, (i, got, slope, bound)


def test_streams_and_a_captured_step(dev):
    """Two streams at once; forward pass and gradients from a graph that is replayed with other rows."""
    from orca_b200.norm import layer_norm, layer_norm_grad
    inputs = [_tensors(dev, 3001, 172, torch.float32, torch.float32, seed=s) for s in range(3)]
    want = [(layer_norm(x, w, b), *layer_norm_grad(g, x, w)) for x, w, b, g in inputs]
    torch.cuda.synchronize()
    streams, got = [torch.cuda.Stream() for _ in range(2)], [None, None]
    for _ in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                x, w, b, g = inputs[i]
                got[i] = (layer_norm(x, w, b), *layer_norm_grad(g, x, w))
    torch.cuda.synchronize()
    for a, c in zip(got, want):
        assert all(torch.equal(p, q) for p, q in zip(a, c))
    held = [t.clone() for t in inputs[0]]
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        x, w, b, g = held
        out = (layer_norm(x, w, b), *layer_norm_grad(g, x, w))
    for given, c in list(zip(inputs, want))[::-1]:
        for h, t in zip(held, given):
            h.copy_(t)
        graph.replay()
        assert all(torch.equal(p, q) for p, q in zip(out, c))


def test_a_captured_backward_pass(dev):
    """As a user captures a whole step; with an older graph of the same leaves alive it is refused and the process lives."""
    from orca_b200.norm import layer_norm
    x, w, b, g = _tensors(dev, 700, 172, torch.float32, torch.float32)
    want = _run(x, w, b, g)[1]
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        torch.autograd.grad(layer_norm(*leaves), leaves, g)
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        grads = torch.autograd.grad(layer_norm(*leaves), leaves, g)
    graph.replay()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for p, q in zip(grads, want))
    older = layer_norm(*leaves)          # on the default stream
    second = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="layer_norm_grad"):
        with torch.cuda.graph(second, stream=side):
            torch.autograd.grad(layer_norm(*leaves), leaves, g)
    torch.cuda.synchronize()
    assert torch.equal(older, layer_norm(*leaves))


def test_no_second_and_no_forward_derivatives(dev):
    import torch.autograd.forward_ad as fw
    from orca_b200.norm import layer_norm, layer_norm_grad
    x, w, b, g = _tensors(dev, 20, 172, torch.float32, torch.float32)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    out = layer_norm(*leaves)
    grads = torch.autograd.grad(out, leaves, g, create_graph=True)
    for d in grads:
        with pytest.raises(RuntimeError, match="no derivative"):
            d.sum().backward(retain_graph=True)
    with pytest.raises(RuntimeError, match="second time"):
        out2 = layer_norm(*leaves)
        out2.sum().backward()
        out2.sum().backward()
    with fw.dual_level():
        for k in range(3):
            args = [fw.make_dual(t, torch.ones_like(t)) if i == k else t for i, t in enumerate((x, w, b))]
            with pytest.raises(NotImplementedError):
                layer_norm(*args)
        for args in ((fw.make_dual(g, g), x, w), (g, fw.make_dual(x, x), w), (g, x, fw.make_dual(w, w))):
            with pytest.raises(NotImplementedError):
                layer_norm_grad(*args)


def test_inputs_changed_before_the_backward_pass_are_noticed(dev):
    from orca_b200.norm import layer_norm
    x, w, b, g = _tensors(dev, 20, 172, torch.float32, torch.float32)
    leaves = [t.detach().requires_grad_(True) for t in (x, w, b)]
    for changed in (0, 1):
        out = layer_norm(*leaves)
        with torch.no_grad():
            leaves[changed].add_(1.0)
        with pytest.raises(RuntimeError, match="modified by an inplace operation"):
            out.sum().backward()


def test_refusals(dev):
    from orca_b200.norm import layer_norm, layer_norm_grad
    x, w, b, g = _tensors(dev, 4, 172, torch.float32, torch.float32)
    for call, error in ((lambda: layer_norm(x.double()), TypeError), (lambda: layer_norm(x, w.double()), TypeError), (lambda: layer_norm(x, w.half()), TypeError),
                        (lambda: layer_norm(x.half(), w.half(), b), TypeError), (lambda: layer_norm(x, w[:-1]), ValueError), (lambda: layer_norm(x, w[None]), ValueError),
                        (lambda: layer_norm(x, w.cpu()), ValueError), (lambda: layer_norm(x, w, b.cpu()), ValueError), (lambda: layer_norm(x.cpu()), TypeError),
                        (lambda: layer_norm(torch.tensor(1.0, device=dev)), ValueError), (lambda: layer_norm(x[:, :0]), ValueError), (lambda: layer_norm(x.to_sparse()), TypeError),
                        (lambda: layer_norm_grad(g.half(), x, w), ValueError), (lambda: layer_norm_grad(g[:3], x, w), ValueError), (lambda: layer_norm_grad(g.cpu(), x, w), ValueError)):
        with pytest.raises(error):
            call()
    assert torch.equal(layer_norm(x, w, b), layer_norm(x, w, b))


def _to_c(dev, rows, width, dtype, off, extra=0):
    """Rows `off` elements behind a border of 512 bytes, `extra` elements between them; what lies around them is kept."""
    rs = np.random.RandomState(rows + width + off)
    whole = torch.from_numpy(rs.randn(off + rows * (width + extra) + 40).astype(np.float32)).to(dev, dtype)
    return whole, whole[off:off + rows * (width + extra)].view(rows, width + extra)[:, :width]


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,width", [(1, 1), (3, 2), (9, 5), (40, 33), (37, 172), (21, 515), (5, 4097), (3, 8191)])
def test_rows_that_begin_between_borders(dev, dtype, rows, width):
    """Inputs and outputs of the C calls off a border by the same number of elements: wide loads begin before a row and end behind it, and nothing
    around the rows is changed."""
    from orca_b200 import _lib
    L, code = _lib.lib(), _lib.TYPES[dtype]
    for off in (1, 2, 3, 5):
        (_, x), (_, g), (out_all, out), (dx_all, dx) = (_to_c(dev, rows, width, dtype, off) for _ in range(4))
        _, w, b, _ = _tensors(dev, 2, width, dtype, dtype)
        around = out_all.clone(), dx_all.clone()
        stream = torch.cuda.current_stream().cuda_stream
        _lib.check(L.orca_layer_norm(x.data_ptr(), width, rows, width, code, w.data_ptr(), b.data_ptr(), code, EPS, out.data_ptr(), stream))
        ws = torch.empty(L.orca_layer_norm_grad_workspace_bytes(rows, width), dtype=torch.uint8, device=dev)
        dw, db = torch.empty_like(w), torch.empty_like(b)
        _lib.check(L.orca_layer_norm_grad(g.data_ptr(), width, x.data_ptr(), width, rows, width, code, w.data_ptr(), code, EPS, dx.data_ptr(), dw.data_ptr(),
                                          db.data_ptr(), ws.data_ptr(), ws.numel(), stream))
        _check(x, w, b, g, out, [dx, dw, db])
        for now, was in zip((out_all, dx_all), around):
            assert torch.equal(now[:off], was[:off]) and torch.equal(now[off + rows * width:], was[off + rows * width:])


def test_strided_weights(dev):
    x, w, b, g = _tensors(dev, 50, 344, torch.float32, torch.float32)
    out, grads = _run(x[:, :172], w[::2], b[1::2], g[:, :172])
    _check(x[:, :172].contiguous(), w[::2].contiguous(), b[1::2].contiguous(), g[:, :172].contiguous(), out, grads)


def test_more_than_32_bits_of_elements(dev):
    """The last rows of 4.3 GB; sums over rows with gradients in the first and last rows alone."""
    from orca_b200.norm import layer_norm, layer_norm_grad
    rows, width = 12500007, 172
    x = torch.randn(rows, width, device=dev, dtype=torch.bfloat16)
    assert x.numel() > 1 << 31
    _, w, b, _ = _tensors(dev, 2, width, torch.bfloat16, torch.float32)
    g = torch.zeros_like(x)
    ends = list(range(70)) + list(range(rows - 70, rows))
    g[:70].normal_()
    g[-70:].normal_()
    out = layer_norm(x, w, b)
    dx, dw, db = layer_norm_grad(g, x, w)
    _check(x[ends], w, b, g[ends], out[ends], [dx[ends], dw, db])
    assert not dx[70:-70].any()


@pytest.mark.parametrize("width", [33, 172, 515, 2048, 20000])
def test_one_row_for_all(dev, width):
    """Rows, or their gradients, that are one row many times over (no memory lies between them)."""
    for dtype in (torch.float32, torch.bfloat16):
        x, w, b, g = _tensors(dev, 90, width, dtype, dtype)
        for x_, g_ in ((x[:1].expand(90, width), g), (x, g[3:4].expand(90, width)), (x[:1].expand(90, width), g[:1].expand(90, width))):
            out, grads = _run(x_, w, b, g_)
            _check(x_, w, b, g_, out, grads)


def test_inference_mode(dev):
    from orca_b200.norm import layer_norm, layer_norm_grad
    x, w, b, g = _tensors(dev, 90, 172, torch.float32, torch.float32)
    want = layer_norm(x, w, b), *layer_norm_grad(g, x, w)
    with torch.inference_mode():
        got = layer_norm(x, w, b), *layer_norm_grad(g, x, w)
    assert all(torch.equal(p, q) for p, q in zip(got, want))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,width", [(700, 24), (300, 33), (2000, 64), (300, 172), (300, 344), (200, 515), (100, 688), (100, 1000), (70, 1024), (70, 2051), (50, 4096), (40, 8192), (20, 16384)])
def test_rows_whose_values_are_unlike_each_other(dev, rows, width, dtype):
    """Some values, at the beginning, spread over the row or in pieces of 16 bytes that are, lie 3 to 1000 deviations from the rest: what a row's sums are taken
    around may be far from its mean.

    What the arithmetic may be off by where it is not, in steps U = 2^-24 of a value h, whose mean square is one, with the mean at most one and a half deviations
    away: differences 2.5, their mean 2.5, its product 1.5, sum 1, the root 4, a variance that twenty sums lead to 3.6: 16 in the mean over a row.  A gradient d has
    the same again for each h that it is made with and 24 of its own size.  Sums over rows have twice the mean for a single value."""
    rs = np.random.RandomState(width)
    x = rs.randn(rows, width)
    way = np.arange(rows) % 4
    shift = np.array([0, 3, 10, 30, 100, 1000])[np.arange(rows) % 6] * np.where(np.arange(rows) % 5 == 0, -1.0, 1.0)
    column = np.arange(width)
    front, spread, one, pieces = column < max(1, min(32, width // 3)), (column < width // 2) & (column % 4 < 2), column < 1, column < 0
    for values in (2, 4, 8) if width >= 100 else ():
        for k in range(32 // values):
            at = width // values * (2 * k + 1) // (64 // values) * values
            pieces |= (column >= at) & (column < at + values)
    x += shift[:, None] * np.stack([front, spread, one, pieces])[way]
    up = lambda a, t: torch.from_numpy(a.astype(np.float32)).to(dev, t)
    x, g, w, b = up(x, dtype), up(rs.randn(rows, width), dtype), up(1 + 0.1 * rs.randn(width), torch.float32), up(np.zeros(width), torch.float32)
    out, (dx, dw, db) = _run(x, w, b, g)
    again, same = _run(x, w, b, g)
    assert torch.equal(out, again) and all(torch.equal(p, q) for p, q in zip((dx, dw, db), same))
    x, g, w = _np(x), _np(g), _np(w)
    y, h, r, *_ = ref.norm(x, w, 0.0, float(np.float32(EPS)))
    want, want_w, want_b, *_ = ref.norm_grad(g, x, w, float(np.float32(EPS)))
    d = g * w
    rms = lambda a: np.sqrt((a * a).mean(1, keepdims=True))
    size = r * (40 * rms(d) + 16 * np.abs((d * h).mean(1, keepdims=True)))
    if dtype == torch.float32:
        assert (rms(_np(out) - y) <= 16 * ref.U * 1.5).all(), (rms(_np(out) - y) / ref.U).max()
        assert (rms(_np(dx) - want) <= ref.U * size).all(), (rms(_np(dx) - want) / (ref.U * size)).max()
    else:
        _within(out, y, 32 * ref.U * (1 + np.abs(h)) * np.abs(w))
        _within(dx, want, 2 * ref.U * size * (1 + np.abs(h)))
    off = (np.abs(g) * (32 * (1 + np.abs(h)) + (rows + 60) * np.abs(h))).sum(0) * ref.U
    assert (np.abs(_np(dw) - want_w) <= off).all(), (np.abs(_np(dw) - want_w) / off).max()


@pytest.mark.parametrize("width", [7, 172, 344, 688, 2051, 8192, 20000])
@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
def test_rows_whose_squares_leave_the_range(dev, dtype, width):
    """Such a row is NaN, with its gradients, whatever else it would look like; rows up to there are right."""
    x, w, b, g = _tensors(dev, 70, width, dtype, torch.float32)
    signs = torch.where(torch.arange(width, device=dev) % 2 == 0, 1.0, -1.0)
    x[11], x[12], x[40] = (1e20 * signs).to(dtype), (1e30 * x[12].float()).to(dtype), (3e19 * (1 + signs)).to(dtype)
    x[50], x[51] = (1e16 * x[50].float()).to(dtype), (1e-16 * x[51].float()).to(dtype)
    out, (dx, dw, db) = _run(x, w, b, g)
    lost = [11, 12, 40]
    assert out[lost].isnan().all() and dx[lost].isnan().all() and dw.isnan().all() and torch.isfinite(db).all()
    rest = [i for i in range(70) if i not in lost]
    _check(x[rest], w, b, g[rest], out[rest], [dx[rest], None, None])


@pytest.mark.parametrize("dtype", TYPES, ids=str)
@pytest.mark.parametrize("rows,width", [(1, 172), (17, 172), (90, 172), (90, 64), (700, 1024), (40, 8188)])
def test_the_same_row_again_between_borders(dev, dtype, rows, width):
    """A stride of zero in the C calls, for x, for gradients and for both, all of them off a border by the same number of elements."""
    from orca_b200 import _lib
    L, code = _lib.lib(), _lib.TYPES[dtype]
    for off in (1, 2, 3):
        (_, x), (_, g), (out_all, out), (dx_all, dx) = (_to_c(dev, rows, width, dtype, off) for _ in range(4))
        g.mul_(0.5)
        _, w, b, _ = _tensors(dev, 2, width, dtype, dtype)
        around = out_all.clone(), dx_all.clone()
        stream = torch.cuda.current_stream().cuda_stream
        for x_stride, g_stride in ((0, 0), (0, width), (width, 0)):
            x_, g_ = (t if stride else t[:1].expand(rows, width) for t, stride in ((x, x_stride), (g, g_stride)))
            _lib.check(L.orca_layer_norm(x.data_ptr(), x_stride, rows, width, code, w.data_ptr(), b.data_ptr(), code, EPS, out.data_ptr(), stream))
            ws = torch.empty(L.orca_layer_norm_grad_workspace_bytes(rows, width), dtype=torch.uint8, device=dev)
            dw, db = torch.empty_like(w), torch.empty_like(b)
            _lib.check(L.orca_layer_norm_grad(g.data_ptr(), g_stride, x.data_ptr(), x_stride, rows, width, code, w.data_ptr(), code, EPS, dx.data_ptr(), dw.data_ptr(),
                                              db.data_ptr(), ws.data_ptr(), ws.numel(), stream))
            _check(x_, w, b, g_, out, [dx, dw, db])
            for now, was in zip((out_all, dx_all), around):
                assert torch.equal(now[:off], was[:off]) and torch.equal(now[off + rows * width:], was[off + rows * width:])


@pytest.mark.parametrize("dtype,widths", [(torch.float32, [2, 33, 172, 515, 1000, 2051, 4098, 8190, 8191, 8192, 8200, 12288, 16384, 20001]), (torch.bfloat16, [33, 172, 515, 2051, 7001, 8192, 8200, 16392]),
                                          (torch.float16, [172, 515, 8190, 12289])], ids=str)
@pytest.mark.parametrize("rows", [140, 2000])
def test_every_value_counts(dev, dtype, widths, rows):
    """Each value of a row is the only one that is not zero in one row, and so is its gradient: a sum without it, of a row or over rows, is far off (few rows of
    many values are shared by clusters).  What the arithmetic may be off by: 32 steps U of a value and of a deviation (sums are taken around a number up to one and a half of
    them away), in dx of r times the value that is not zero, or of the mean of squares of all."""
    from orca_b200.norm import layer_norm, layer_norm_grad
    a, half = 100.0, torch.finfo(dtype).eps / 2
    for width in widths:
        here, else_, dx_here, dx_else = ref.one_apart(width, a, float(np.float32(EPS)))
        w = torch.ones(width, device=dev, dtype=dtype)
        r = 1 / np.sqrt(a * a * (width - 1) / width / width + EPS)
        for first in range(0, width, rows):
            n = min(rows, width - first)
            at = torch.arange(first, first + n, device=dev)
            one = torch.zeros(n, width, device=dev, dtype=dtype)
            one[torch.arange(n, device=dev), at] = 1
            out, (dx, dw, db) = layer_norm(one * a, w), layer_norm_grad(one, one * a, w)
            for got, there, other, size, size_other in ((out, here, else_, 1, 1), (dx, dx_here, dx_else, 2 * r, 2 * r / np.sqrt(width))):
                off, off_other = (32 * ref.U * (abs(v) + s) + half * abs(v) * (1 + 2.0 ** -10) + 2.0 ** -25 * (dtype == torch.float16) for v, s in ((there, size), (other, size_other)))
                mine = got[torch.arange(n, device=dev), at].double()
                assert (mine - there).abs().max() <= off, (width, first, float((mine - there).abs().max()), off)
                rest = got.double()
                rest[torch.arange(n, device=dev), at] = other
                assert (rest - other).abs().max() <= off_other, (width, first, float((rest - other).abs().max()), off_other)
            want = torch.zeros(width, device=dev, dtype=torch.float64)
            want[at] = here
            assert ((dw.double() - want).abs() <= (32 * ref.U + half * (1 + 2.0 ** -10)) * want.abs() + 2.0 ** -25 * (dtype == torch.float16)).all(), (width, first)
            want[at] = 1
            assert torch.equal(db.double(), want)


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_rows_of_one_value(dev, dtype):
    """Of any value: the bias, and with an eps of 0 not a number; with another value in one place, a step away, that is the only one that differs."""
    from orca_b200.norm import layer_norm, layer_norm_grad
    for width in (2, 3, 5, 24, 33, 50, 64, 100, 171, 172, 344, 509, 512, 515, 1000, 2051, 8192):
        x = torch.tensor([0.1, -1 / 3, 7.3e3, 1e-4, 0.7, -6e4, 3.1], device=dev).to(dtype)[:, None].expand(7, width).contiguous()
        w, b = torch.full((width,), 3.0, device=dev, dtype=dtype), torch.full((width,), 0.25, device=dev, dtype=dtype)
        assert torch.equal(layer_norm(x, w, b), b.expand(7, width)), width
        assert layer_norm(x, w, b, eps=0.0).isnan().all(), width
        dx, dw, db = layer_norm_grad(torch.ones_like(x), x, w)
        assert not dw.any() and torch.isfinite(dx).all()
        assert layer_norm_grad(torch.ones_like(x), x, w, eps=0.0)[0].isnan().all(), width
        # one value a step of its type away: it is sqrt(width - 1) deviations off, the others 1 / sqrt(width - 1) the other way
        at = torch.arange(7, device=dev) % width
        y = x.clone()
        y.view(torch.int32 if dtype == torch.float32 else torch.int16)[torch.arange(7, device=dev), at] += 1
        got, n = layer_norm(y, None, None, eps=0.0).double(), width
        sign = torch.sign(x[:, 0].double())
        want = (-sign / (n - 1) ** 0.5)[:, None].expand(7, n).clone()
        want[torch.arange(7, device=dev), at] = sign * (n - 1) ** 0.5
        # (the pivot, the mean of up to 8192 values added up in steps, is up to 24 steps away, the values' distance to it rounded: 2^-19 of a step of 16 bits, and of fp32
        # a deviation, 1 / sqrt(n) steps, does not come out of differences that are whole steps off; only that it is not taken for one value there)
        if dtype == torch.float32:
            assert torch.isfinite(got).all() and (got[torch.arange(7, device=dev), at] * sign > 0).all()
        else:
            assert ((got - want).abs() <= (torch.finfo(dtype).eps / 2 + 2.0 ** -10) * want.abs() + 2.0 ** -10).all(), (width, float((got - want).abs().max()))
