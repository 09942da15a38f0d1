"""What the calls of a training step refuse before anything is launched, and the format of moments in 8 bits.  No GPU is needed."""
import ctypes as C

import numpy as np
import pytest
import torch

import train_reference as ref
from orca_b200 import _lib, build


@pytest.fixture(scope="module")
def L():
    build.build()
    return _lib.lib()


@pytest.mark.parametrize("change", [dict(rows=-1), dict(width=0), dict(width=(1 << 24) + 1), dict(x=None), dict(out=None), dict(x=2), dict(type=3), dict(type=7),
                                    dict(weight_type=1), dict(eps=-1.0), dict(eps=float("nan")), dict(eps=float("inf")), dict(weight=66), dict(stride=-4)])
def test_layer_norm_refuses(L, change):
    a = dict(dict(x=64, stride=8, rows=4, width=8, type=0, weight=64, bias=64, weight_type=0, eps=1e-5, out=64), **change)
    assert L.orca_layer_norm(*[a[k] for k in ("x", "stride", "rows", "width", "type", "weight", "bias", "weight_type", "eps", "out")], None) in (1, 2)
    g = dict(a, g=a["x"], dx=a["out"])
    rc = L.orca_layer_norm_grad(*[g[k] for k in ("g", "stride", "x", "stride", "rows", "width", "type", "weight", "weight_type", "eps", "dx")], None, None, None, 0, None)
    assert rc in (1, 2) or change == dict(out=None)          # (nothing is wanted: nothing is done)


def test_layer_norm_grad_refuses_a_small_workspace(L):
    need = L.orca_layer_norm_grad_workspace_bytes(1000, 172)
    assert need > 0 and L.orca_layer_norm_grad_workspace_bytes(-1, 172) == -1 and L.orca_layer_norm_grad_workspace_bytes(5, 0) == -1
    for ws, size in ((256, need - 1), (None, need), (260, need)):
        assert L.orca_layer_norm_grad(64, 172, 64, 172, 1000, 172, 0, 64, 0, 1e-5, 64, 64, 64, ws, size, None) == 1


@pytest.mark.parametrize("change", [dict(n=-1), dict(type=3), dict(group=1), dict(group=-1), dict(param=None), dict(grad=None), dict(mean=None), dict(square=None),
                                    dict(step=None), dict(param=66), dict(mean=66), dict(step=66), dict(n=1 << 62)])
def test_adamw_refuses_a_tensor(L, change):
    t = dict(dict(param=64, grad=64, mean=64, square=64, exponents=None, step=64, n=5, type=0, group=0), **change)
    tensors, groups = (_lib.AdamwTensorT * 1)(_lib.AdamwTensorT(**t)), (_lib.AdamwGroupT * 1)(_lib.AdamwGroupT(1e-3, .9, .999, 1e-8, 0.0, None))
    assert L.orca_adamw_step(tensors, 1, groups, 1, 32, -1.0, None, 64, None) in (1, 2)


@pytest.mark.parametrize("change", [dict(beta1=1.0), dict(beta2=-0.1), dict(eps=-1.0), dict(eps=1e-40), dict(eps=float("inf")), dict(beta1=float("nan")), dict(d_lr=2)])
def test_adamw_refuses_a_group(L, change):
    t = _lib.AdamwTensorT(64, 64, 64, 64, None, 64, 5, 0, 0)
    g = _lib.AdamwGroupT(**dict(dict(lr=1e-3, beta1=.9, beta2=.999, eps=1e-8, weight_decay=0.0, d_lr=None), **change))
    assert L.orca_adamw_step((_lib.AdamwTensorT * 1)(t), 1, (_lib.AdamwGroupT * 1)(g), 1, 32, -1.0, None, 64, None) == 1


def test_adamw_refuses(L):
    tensors, groups = (_lib.AdamwTensorT * 1)(_lib.AdamwTensorT(64, 64, 64, 64, None, 64, 5, 0, 0)), (_lib.AdamwGroupT * 1)()
    for args in ((None, 1, groups, 1, 32, -1.0, None, 64), (tensors, 1, None, 1, 32, -1.0, None, 64), (tensors, -1, groups, 1, 32, -1.0, None, 64),
                 (tensors, 1, groups, 1, 16, -1.0, None, 64), (tensors, 1, groups, 1, 8, -1.0, None, 64), (tensors, 1, groups, 1, 32, 1.0, None, 64),
                 (tensors, 1, groups, 1, 32, -1.0, None, None), (tensors, 1, groups, 1, 32, -1.0, None, 32), (tensors, 1, groups, 1, 32, float("nan"), 64, 64), (tensors, 1, groups, 1, 32, 1.0, 66, 64)):
        assert L.orca_adamw_step(*args, None) == 1
    assert L.orca_adamw_moments(None, 1, None) == 1 and L.orca_adamw_moments(tensors, 1, None) == 1
    assert C.sizeof(_lib.AdamwTensorT) == 64 and C.sizeof(_lib.AdamwGroupT) == 48


def test_rows_of_another_kind_are_refused():
    from orca_b200.norm import layer_norm, layer_norm_grad
    x = torch.zeros(3, 4)
    for call in (lambda: layer_norm(x), lambda: layer_norm(x.double()), lambda: layer_norm_grad(x, x), lambda: layer_norm(x.int())):
        with pytest.raises(TypeError, match="CUDA"):
            call()
    for eps in (-1e-5, float("nan"), float("inf")):
        with pytest.raises(ValueError, match="eps"):
            layer_norm(x, eps=eps)
    with pytest.raises(TypeError):
        layer_norm([1.0, 2.0])


def test_parameters_of_another_kind_are_refused():
    from orca_b200.optim import AdamW
    p = torch.nn.Parameter(torch.zeros(3))
    with pytest.raises(RuntimeError, match="CUDA"):
        AdamW([p])
    with pytest.raises(TypeError):
        AdamW([torch.nn.Parameter(torch.zeros(3, dtype=torch.float64))])
    for bad in (dict(bits=16), dict(max_norm=-1.0), dict(max_norm=float("nan")), dict(lr=-1.0), dict(lr=float("nan")), dict(betas=(0.9, 1.0)), dict(betas=(0.9,)),
                dict(eps=-1.0), dict(weight_decay=-0.1)):
        with pytest.raises(ValueError):
            AdamW([p], **bad)


def test_dithering_is_even():
    """Means and variances of sixteen bins over places and steps, and products of neighbours: within five deviations of those of even numbers."""
    n, steps = 4096, 64
    for second in (False, True):
        u = np.stack([ref.dither(n, t, second) for t in range(1, steps + 1)])
        counts = np.bincount((u.ravel() // 65536).astype(int), minlength=16)
        total = n * steps
        assert (np.abs(counts - total / 16) < 5 * np.sqrt(total / 16)).all()
        z = (u + 0.5) / 2 ** 20 - 0.5
        for a, b in ((z[:, 1:], z[:, :-1]), (z[:, 8:], z[:, :-8]), (z[1:], z[:-1]), (z[:, 1:], z[:, :-1])):
            assert abs((a * b).sum()) < 5 * np.sqrt(a.size) / 12
        # each place on its own, over the steps
        assert (np.abs(z.sum(0)) < 5.5 * np.sqrt(steps / 12)).all()
    first, second = (np.stack([ref.dither(n, t, s) for t in range(1, steps + 1)]) / 2 ** 20 - 0.5 for s in (False, True))
    assert abs((first * second).sum()) < 5 * np.sqrt(n * steps) / 12


def test_moments_are_right_on_average():
    """Values over all exponents, held at many steps: the mean of what is held is the value, and a square is never lost: one below the smallest
    code is held as that code every time."""
    rs = np.random.RandomState(1)
    x = (rs.randn(256) * 2.0 ** rs.randint(-14, 1, 256)).astype(np.float32).astype(np.float64)
    for top, square, v in ((14, False, x), (30, True, x * x)):
        v = v.astype(np.float32).astype(np.float64)
        steps = 400
        all_held = np.stack([ref.held(v, t, top, square)[0] for t in range(1, steps + 1)])
        # each is one of the two neighbours on the scale; a step of it is an eighth of its binade, or the smallest one of the block
        step = np.maximum(2.0 ** (np.floor(np.log2(np.abs(v))) - 3), 2.0 ** (np.floor(np.log2(np.abs(v).max())) - top - 2))
        assert (np.abs(all_held - v) < step).all()
        smallest = 2.0 ** (np.floor(np.log2(np.abs(v).max())) - top - 2)
        want = np.maximum(v, smallest) if square else v
        assert (np.abs(all_held.mean(0) - want) < 5.5 * step / 2 / np.sqrt(steps)).all()
        assert not square or (all_held >= smallest).all()


def test_sums_of_squares():
    """A thread's sum in 32 bits is off by 2^-40 of it at most: values in any order, of one size and of many, rising and falling."""
    rs = np.random.RandomState(0)
    n = 20000
    rising = np.sort(np.abs(rs.randn(n, 16)), 1)
    for x in (rs.randn(n, 16), rs.randn(n, 16) * 10.0 ** rs.uniform(-4, 1, (n, 16)), rising, rising[:, ::-1], 2.0 ** np.arange(16) * (1 + rs.rand(n, 16)),
              2.0 ** -np.arange(16) * (1 + rs.rand(n, 16)), np.repeat(1 + rs.rand(n, 1), 16, 1), rs.randn(n, 16) * (rs.rand(n, 16) < 0.1) + 1e-9):
        x = np.ascontiguousarray(x).astype(np.float32)
        want = (x.astype(np.longdouble) ** 2).sum(1)
        assert (np.abs(ref.squares(x) - want) <= 2.0 ** -40 * want).all()


@pytest.mark.parametrize("n", [2, 33, 172, 515, 1000, 2051, 4098, 8190, 8191, 8192, 8200, 12288, 16384, 20001, 40000])
def test_a_value_that_is_left_out_is_seen(n):
    """Rows that are zero but for one value: what a sum is without it is outside of the bounds of the tests on such rows, by a factor of a hundred."""
    a, eps = 100.0, 1e-5
    here, else_, dx, dx_else = ref.one_apart(n, a, eps)
    h, r, d = np.full(n, else_), 1 / np.sqrt(a * a * (n - 1) / n / n + eps), np.zeros(n)
    h[n // 2], d[n // 2] = here, 1
    assert np.allclose(h, ref.norm(np.eye(n)[n // 2:n // 2 + 1] * a, np.ones(n), 0.0, eps)[1][0], rtol=1e-12)
    want = r * (d - d.mean() - h * (d * h).mean())
    assert np.allclose(want[[n // 2, 0]], [dx, dx_else], rtol=1e-9, atol=1e-15)
    far = lambda got, value, size: abs(got - value) / (32 * ref.U * (abs(value) + size))
    # left out of the mean, of the variance
    for mean, var in ((0.0, a * a / n), (a / n, (n - 1) * (a / n) ** 2 / n)):
        r2 = 1 / np.sqrt(var + eps)
        assert max(far((a - mean) * r2, here, 1), far(-mean * r2, else_, 1)) > 100
    # left out of the mean of d, of that of d h
    for c1, c2 in ((0.0, here / n), (1 / n, 0.0)):
        assert max(far(r * (1 - c1 - here * c2), dx, 2 * r), far(r * (-c1 - else_ * c2), dx_else, 2 * r / np.sqrt(n))) > 100


@pytest.mark.parametrize("bits", [32, 8])
def test_groups_without_parameters(bits):
    """As PyTorch's optimisers have them, to which parameters come later: a step does nothing."""
    from orca_b200.optim import AdamW
    opt = AdamW([dict(params=[])], max_norm=1.0, bits=bits)
    assert opt.step(lambda: 3) == 3 and opt.step() is None
    assert [list(x) for x in opt.moments()] == [[], []]
    opt.load_state_dict(opt.state_dict())
    opt.zero_grad()
