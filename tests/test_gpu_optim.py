"""AdamW over many tensors on the GPU, against 64 bits: bounds of train_reference.py and half a step of the parameters' type; moments in 8 bits
are those of the format, every one."""
import copy
import io

import numpy as np
import pytest
import torch

import train_reference as ref

pytestmark = pytest.mark.gpu

TYPES = [torch.float32, torch.bfloat16, torch.float16]
LR, BETAS, EPS, DECAY = 3e-3, (0.9, 0.999), 1e-8, 0.02


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _np(t):
    return t.detach().double().cpu().numpy().ravel()


def _values(rs, n, scale=1.0):
    """Over four orders of magnitude, some of them zero."""
    return (scale * rs.randn(n) * 10.0 ** rs.uniform(-3, 1, n) * (rs.rand(n) > 0.1)).astype(np.float32)


def _params(dev, sizes, dtypes, seed=0):
    rs = np.random.RandomState(seed)
    return [torch.nn.Parameter(torch.from_numpy(_values(rs, n)).to(dev, t)) for n, t in zip(sizes, dtypes)], rs


def _give(params, rs, scale=0.1):
    for p in params:
        p.grad = torch.from_numpy(_values(rs, p.numel(), scale)).to(p.device, p.dtype).view(p.shape)


def _within(got, want, off):
    half = torch.finfo(got.dtype).eps / 2
    tiny = 2.0 ** -149 if got.dtype == torch.float32 else 2.0 ** -133 if got.dtype == torch.bfloat16 else 2.0 ** -25
    got = _np(got)
    far = np.abs(got - want) - (half * (np.abs(want) + off) + off + tiny)
    assert (far <= 0).all(), (int(far.argmax()), float(far.max()), got[far.argmax()], want[far.argmax()])


def _step_and_check(opt, settings=None):
    """One step of it against the reference, from the state that it has."""
    groups, with_grad = opt.param_groups, [p for g in opt.param_groups for p in g["params"] if p.grad is not None]
    eight = opt.bits == 8
    values = dict(zip([p for g in groups for p in g["params"]], zip(*opt.moments())))
    before = {p: (_np(p), _np(p.grad), *(_np(m) for m in values[p]), int(opt.state[p]["step"])) for p in with_grad}
    idle = {p: (p.clone(), {k: v.clone() for k, v in opt.state[p].items()}) for g in groups for p in g["params"] if p.grad is None}
    norm, f = ref.factor([b[1] for b in before.values()], opt.max_norm) if opt.max_norm is not None else (None, 1.0)
    opt.step()
    if norm is not None:
        assert abs(float(opt.grad_norm) - norm) <= 1.01 * ref.U * norm
    values = dict(zip([p for g in groups for p in g["params"]], zip(*opt.moments())))
    for g in groups:
        for p in g["params"]:
            if p not in before:
                assert torch.equal(p, idle[p][0]) and all(torch.equal(v, opt.state[p][k]) for k, v in idle[p][1].items())
                continue
            x, d, m, v, t = before[p]
            assert int(opt.state[p]["step"]) == t + 1
            new, m, v, off, off_m, off_v = ref.adamw(x, d, m, v, t + 1, float(g["lr"]), g["betas"], g["eps"], g["weight_decay"], f, eight)
            _within(p, new, off)
            got_m, got_v = values[p]
            if eight:
                for got, want, top, square in ((got_m, m, 14, False), (got_v, v, 30, True)):
                    held, e = ref.held(want, t + 1, top, square)
                    assert np.array_equal(_np(got), held)
                    assert np.array_equal(opt.state[p]["exponents"][:, int(square)].cpu().numpy(), e)
            else:
                _within(got_m, m, off_m)
                _within(got_v, v, off_v)


SIZES = [1, 2, 7, 8, 31, 255, 256, 257, 511, 2047, 2048, 2049, 4095, 4096, 4097, 8191, 8200, 12288, 70001, 300000]


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("max_norm", [None, 1.0, 1e9])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_sizes(dev, dtype, max_norm, bits):
    from orca_b200.optim import AdamW
    params, rs = _params(dev, SIZES, [dtype] * len(SIZES))
    opt = AdamW(params, LR, BETAS, EPS, DECAY, max_norm, bits)
    for _ in range(4):
        _give(params, rs)
        _step_and_check(opt)


@pytest.mark.parametrize("bits", [32, 8])
def test_types_groups_and_parameters_without_a_gradient(dev, bits):
    from orca_b200.optim import AdamW
    sizes = [513, 0, 1000, 77, 4096, 5, 172 * 31, 900, 256, 33, 3000, 1]
    params, rs = _params(dev, sizes, (TYPES * 4)[:len(sizes)])
    groups = [dict(params=[p], lr=10.0 ** -(i % 5 + 1), betas=(0.5 + 0.04 * i, 0.9 + 0.008 * i), eps=10.0 ** -(i + 2), weight_decay=0.01 * i) for i, p in enumerate(params)]
    opt = AdamW(groups, max_norm=0.7, bits=bits)
    assert len(opt.param_groups) > 8
    for step in range(4):
        _give(params, rs)
        for i, p in enumerate(params):
            if (i + step) % 3 == 0:
                p.grad = None
        if step == 2:
            opt.param_groups[4]["lr"], opt.param_groups[4]["betas"] = 0.5, (0.0, 0.0)
        _step_and_check(opt)
    for p in params:
        p.grad = None
    _step_and_check(opt)
    assert float(opt.grad_norm) == 0.0


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [47, 48, 49, 480, 481, 1201])
def test_many_tensors(dev, count, bits):
    from orca_b200.optim import AdamW
    sizes = [1 + (37 * i) % 600 for i in range(count)]
    params, rs = _params(dev, sizes, ([torch.float32] * 5 + [torch.bfloat16]) * count)
    opt = AdamW(params, LR, BETAS, EPS, DECAY, 1.0, bits)
    for _ in range(2):
        _give(params, rs)
        _step_and_check(opt)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_where_tensors_lie(dev, dtype, bits):
    """Parameters, gradients and moments off by an element, turned, in other orders; gradients that are views."""
    from orca_b200.optim import AdamW
    rs = np.random.RandomState(3)
    new = lambda *s: torch.from_numpy(_values(rs, int(np.prod(s)))).to(dev, dtype).view(*s)
    datas = [new(5001)[1:], new(5003)[3:], new(40, 30).t(), new(2, 3, 5, 7).to(memory_format=torch.channels_last), new(700), new(64, 64), new(900), new(5008)[8:], new(1, 300, 1)]
    params = [torch.nn.Parameter(d) for d in datas]
    opt = AdamW(params, LR, BETAS, EPS, DECAY, 1.0, bits)
    off = torch.zeros(1 + 700, dtype=opt.state[params[4]]["exp_avg"].dtype, device=dev)
    opt.state[params[4]]["exp_avg"] = off[1:]
    one = new(1)
    for step in range(3):
        grads = [new(5000), new(5004)[4:], new(40, 30).t(), new(2, 3, 5, 7), new(1400)[::2], new(64, 64).t(), one.expand(900), new(5001)[1:], new(1, 300, 1)]
        for p, g in zip(params, grads):
            p.grad = g
        flat = [g.contiguous() if p.is_contiguous() else torch.empty_like(p).copy_(g) for p, g in zip(params, grads)]
        # the reference walks memory in the order of the parameter's elements
        order = [p.detach().as_strided((p.numel(),), (1,)) for p in params]
        before = [(_np(o), _np(f.as_strided((f.numel(),), (1,)))) for o, f in zip(order, flat)]
        lists = [[_np(m.as_strided((m.numel(),), (1,))) for m in ms] for ms in opt.moments()]
        _, f = ref.factor([b[1] for b in before], 1.0)
        opt.step()
        for p, o, (x, g), m, v in zip(params, order, before, *lists):
            want, m, v, off_p, *_ = ref.adamw(x, g, m, v, step + 1, LR, BETAS, EPS, DECAY, f, bits == 8)
            _within(o, want, off_p)


def test_zero_norms_and_norms_that_are_not_finite(dev):
    from orca_b200.optim import AdamW
    for bits in (32, 8):
        params, rs = _params(dev, [700, 5000], [torch.float32, torch.bfloat16])
        opt = AdamW(params, LR, BETAS, EPS, DECAY, 0.5, bits)
        _give(params, rs)
        _step_and_check(opt)
        for p in params:
            p.grad = torch.zeros_like(p)
        _step_and_check(opt)
        kept = [p.clone() for p in params], copy.deepcopy(opt.state_dict()["state"])
        for bad in (float("nan"), float("inf")):
            _give(params, rs)
            params[1].grad[77] = bad
            opt.step()
            assert not torch.isfinite(opt.grad_norm)
            assert all(torch.equal(p, k) for p, k in zip(params, kept[0]))
            assert all(torch.equal(opt.state_dict()["state"][i][k], v) for i, s in kept[1].items() for k, v in s.items())
        _give(params, rs)
        _step_and_check(opt)
    # none of it is used up: everything is cut away
    opt = AdamW(params, LR, BETAS, EPS, 0.0, 0.0, 32)
    _give(params, rs)
    _step_and_check(opt)
    opt = AdamW(params, LR, BETAS, EPS, DECAY, float("inf"))
    _give(params, rs)
    _step_and_check(opt)
    assert AdamW(params).grad_norm is None


def test_large_and_small_gradients(dev):
    """Squares over the whole range of fp32; blocks of 8 bits at either end of theirs."""
    from orca_b200.optim import AdamW
    for bits in (32, 8):
        for scale in (1e-30, 1e-19, 1e-12, 1e-4, 1e3, 1e8, 1e17):
            params, rs = _params(dev, [3000, 256], [torch.float32] * 2)
            opt = AdamW(params, LR, BETAS, EPS, DECAY, None, bits)
            for _ in range(2):
                _give(params, rs, scale)
                _step_and_check(opt)


def test_values_that_are_not_numbers(dev):
    """With 32 bits they stay where they are, with 8 in their blocks."""
    from orca_b200.optim import AdamW
    for bits, lost in ((32, 1), (8, 256)):
        params, rs = _params(dev, [2000], [torch.float32])
        opt = AdamW(params, LR, BETAS, EPS, DECAY, None, bits)
        for step in range(3):
            _give(params, rs)
            if step == 0:
                params[0].grad[300] = float("nan")
            opt.step()
        (m,), (v,) = opt.moments()
        for t in (m, v):
            assert int(t.isnan().sum()) == lost and t[256:512].isnan().any()
        assert int(params[0].isnan().sum()) == lost


def test_a_captured_step(dev):
    """Replayed with other gradients and another rate it is what steps one after the other are; a first step, too."""
    from orca_b200.optim import AdamW
    for bits in (32, 8):
        lr = torch.tensor(LR, device=dev)
        a, rs = _params(dev, [5000, 172, 33, 700], [torch.float32, torch.float32, torch.bfloat16, torch.float16])
        b = [torch.nn.Parameter(p.detach().clone()) for p in a]
        _give(a, rs)
        for p, q in zip(a, b):
            q.grad = p.grad.clone()
        one, two = AdamW(a, lr, BETAS, EPS, DECAY, 1.0, bits), AdamW(b, lr, BETAS, EPS, DECAY, 1.0, bits)
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            one.step()
        for rate in (LR, 0.1, 0.001):
            lr.fill_(rate)
            for p, q in zip(a, b):
                g = torch.from_numpy(_values(rs, p.numel())).to(dev, p.dtype)
                p.grad.copy_(g), q.grad.copy_(g)
            graph.replay()
            two.step()
            assert all(torch.equal(p, q) for p, q in zip(a, b)) and torch.equal(one.grad_norm, two.grad_norm)
        assert int(one.state[a[0]]["step"]) == 3
        for x, y in zip(one.moments(), two.moments()):
            assert all(torch.equal(p, q) for p, q in zip(x, y))


def test_streams(dev):
    """Two optimisers on two streams at once are what they are one after the other."""
    from orca_b200.optim import AdamW

    def make(seed):
        params, rs = _params(dev, [40000, 300, 5], [torch.float32] * 3, seed)
        return params, AdamW(params, LR, BETAS, EPS, DECAY, 1.0, 8), rs
    want = []
    for seed in range(2):
        params, opt, rs = make(seed)
        for _ in range(5):
            _give(params, rs)
            opt.step()
        want.append(params)
    both, streams = [make(s) for s in range(2)], [torch.cuda.Stream() for _ in range(2)]
    torch.cuda.synchronize()
    for _ in range(5):
        for (params, opt, rs), s in zip(both, streams):
            with torch.cuda.stream(s):
                _give(params, rs)
                opt.step()
    torch.cuda.synchronize()
    assert all(torch.equal(p, q) for (params, _, _), w in zip(both, want) for p, q in zip(params, w))


@pytest.mark.parametrize("bits", [32, 8])
def test_state_goes_elsewhere_and_comes_back(dev, bits):
    from orca_b200.optim import AdamW
    params, rs = _params(dev, [700, 300, 1000], [torch.float32, torch.bfloat16, torch.float32])
    opt = AdamW([dict(params=params[:2]), dict(params=params[2:], lr=0.1)], LR, BETAS, EPS, DECAY, 1.0, bits)
    for _ in range(2):
        _give(params, rs)
        opt.step()
    file = io.BytesIO()
    torch.save(opt.state_dict(), file)
    file.seek(0)
    others = [torch.nn.Parameter(p.detach().clone()) for p in params]
    for p, q in zip(params, others):
        q.grad = p.grad.clone()
    second = AdamW([dict(params=others[:2]), dict(params=others[2:])], 1.0, max_norm=1.0, bits=bits)
    second.load_state_dict(torch.load(file))
    assert second.param_groups[1]["lr"] == 0.1 and second.param_groups[0]["betas"] == BETAS
    third = copy.deepcopy(second)
    for p, q in zip(params, [p for g in third.param_groups for p in g["params"]]):
        q.grad = p.grad.clone()
    opt.step(), second.step(), third.step()
    assert all(torch.equal(p, q) for p, q in zip(params, others))
    assert all(torch.equal(p, q) for p, q in zip(params, [p for g in third.param_groups for p in g["params"]]))
    for x, y in zip(opt.moments(), second.moments()):
        assert all(torch.equal(p, q) for p, q in zip(x, y))
    with pytest.raises(ValueError):
        AdamW(others, bits=bits).load_state_dict(opt.state_dict())
    with pytest.raises(ValueError):
        AdamW([dict(params=others[:2]), dict(params=others[2:])], bits=40 - bits).load_state_dict(opt.state_dict())


def test_a_checkpoint_of_pytorch(dev):
    from orca_b200.optim import AdamW
    params, rs = _params(dev, [700, 300], [torch.float32] * 2)
    theirs = torch.optim.AdamW(params, LR, BETAS, EPS, DECAY)
    for _ in range(3):
        _give(params, rs)
        theirs.step()
    opt = AdamW(params)
    opt.load_state_dict(theirs.state_dict())
    assert int(opt.state[params[0]]["step"]) == 3 and opt.param_groups[0]["lr"] == LR
    _give(params, rs)
    _step_and_check(opt)


def test_closures_schedulers_and_versions(dev):
    from orca_b200.optim import AdamW
    params, rs = _params(dev, [700], [torch.float32])
    opt = AdamW(params, 1.0)
    plan = torch.optim.lr_scheduler.ExponentialLR(opt, 0.5)

    def closure():
        opt.zero_grad()
        loss = (params[0] ** 2).sum()
        loss.backward()
        return loss
    was = params[0].detach().clone()
    assert float(opt.step(closure).detach()) > 0 and not torch.equal(params[0], was)
    plan.step()
    assert opt.param_groups[0]["lr"] == 0.5
    # a parameter that a graph has kept is not changed under it unnoticed
    out = (params[0] ** 2).sum()
    opt.step()
    with pytest.raises(RuntimeError, match="modified by an inplace operation"):
        out.backward()


def test_refusals(dev):
    from orca_b200.optim import AdamW
    flat = torch.randn(300, device=dev)
    P = torch.nn.Parameter
    for params, error in (([P(flat[:200]), P(flat[100:])], ValueError), ([P(flat[::2])], ValueError), ([P(flat.double())], TypeError), ([P(flat), P(torch.zeros(3))], (RuntimeError, ValueError)),
                          ([P(flat[:1].expand(5))], ValueError)):
        with pytest.raises(error):
            AdamW(params)
    with pytest.raises(ValueError):
        AdamW([P(flat)], lr=torch.tensor(1.0, device=dev, dtype=torch.float64))
    p = P(flat)
    opt = AdamW([p])
    with pytest.raises(ValueError):
        opt.add_param_group(dict(params=[P(flat[7:])]))
    with pytest.raises(ValueError):
        opt.add_param_group(dict(params=[P(torch.zeros(5, device=dev))], betas=(1.0, 0.5)))
    assert len(opt.param_groups) == 1 and len(opt.state) == 1
    opt.add_param_group(dict(params=[P(torch.zeros(5, device=dev))]))
    p.grad = torch.ones_like(p).to_sparse()
    with pytest.raises(ValueError, match="dense"):
        opt.step()
    p.grad = torch.ones_like(p)
    kept = p.detach().clone()
    for k, bad in (("exp_avg", torch.zeros(299, device=dev)), ("exp_avg_sq", torch.zeros(300)), ("step", torch.zeros(1, device=dev)), ("exp_avg", torch.zeros(600, device=dev)[::2])):
        good = opt.state[p][k]
        opt.state[p][k] = bad
        with pytest.raises(ValueError):
            opt.step()
        opt.state[p][k] = good
    for k, bad in (("lr", -1.0), ("betas", (0.9, 1.0)), ("betas", 0.9), ("eps", -1.0), ("lr", torch.zeros(2, device=dev))):
        good = opt.param_groups[0][k]
        opt.param_groups[0][k] = bad
        with pytest.raises((ValueError, TypeError)):
            opt.step()
        opt.param_groups[0][k] = good
    q = opt.param_groups[0]["params"].pop()
    with pytest.raises(ValueError):
        opt.step()
    opt.param_groups[0]["params"].append(q)
    assert torch.equal(p, kept)
    opt.step()
    assert not torch.equal(p, kept)


def test_a_training_step_on_looked_up_rows(dev):
    """Lookup, layer norm, a sum of squares, its gradients, a step that cuts them: all of it against 64 bits, with gradients as the first test of each has them."""
    from orca_b200.lookup import lookup_rows
    from orca_b200.norm import layer_norm
    from orca_b200.optim import AdamW
    rs = np.random.RandomState(5)
    ids = rs.randint(0, 500, 700)
    params, _ = _params(dev, [500 * 172, 172, 172], [torch.float32] * 3)
    table, w, b = params
    table.data = table.data.view(500, 172)
    for bits in (32, 8):
        opt = AdamW(params, LR, BETAS, EPS, DECAY, 0.5, bits)
        for _ in range(3):
            opt.zero_grad()
            x = lookup_rows(table, ids, 0.7, padding=int(ids[0]))
            y = layer_norm(x, w, b)
            (0.5 * (y ** 2).sum()).backward()
            # gradients of the whole chain: those of the norm at the rows that the lookup gave, added up by id
            x64, w64, g64 = (a.detach().double().cpu().numpy() for a in (x, w, y))
            dx, dw, db, off, off_w, off_b = ref.norm_grad(g64, x64, w64, float(np.float32(1e-5)))
            keep = (ids != ids[0])[:, None]
            count = np.bincount(ids, minlength=500)[:, None]
            want, size, far = (np.zeros((500, 172)) for _ in range(3))
            for total, part in ((want, dx), (size, np.abs(dx)), (far, off + ref.U * np.abs(dx))):
                np.add.at(total, ids, float(np.float32(0.7)) * part * keep)
            got = table.grad.double().cpu().numpy()
            assert (np.abs(got - want) <= far + ref.MORE * ref.U * (count + 2) * size + 2.0 ** -149).all()
            assert (np.abs(w.grad.double().cpu().numpy() - dw) <= off_w + ref.U * np.abs(dw)).all()
            assert (np.abs(b.grad.double().cpu().numpy() - db) <= off_b + ref.U * np.abs(db)).all()
            _step_and_check(opt)


def test_norms_of_tiny_and_huge_gradients(dev):
    """Squares that leave the range of 32 bits, alone and beside others: the norm is that of 64 bits."""
    from orca_b200.optim import AdamW
    for scales in ((1e-30,), (1e-22,), (1e-38, 1e-44), (1e20,), (1e30,), (1e-25, 1.0, 1e15)):
        rs = np.random.RandomState(2)
        params = [torch.nn.Parameter(torch.zeros(3000, device=dev)) for _ in scales]
        opt = AdamW(params, max_norm=float("inf"))
        for p, scale in zip(params, scales):
            p.grad = torch.from_numpy((scale * rs.randn(3000)).astype(np.float32)).to(dev)
        norm, _ = ref.factor([_np(p.grad) for p in params], float("inf"))
        opt.step()
        assert abs(float(opt.grad_norm) - norm) <= 1.01 * ref.U * norm + 2.0 ** -150, scales


def test_more_than_32_bits_of_elements(dev):
    """The first and the last blocks of a parameter with more than 2^31 elements, moments in 8 bits."""
    from orca_b200.optim import AdamW
    n = (1 << 31) + 4096 + 261
    p = torch.nn.Parameter(torch.zeros(n, device=dev, dtype=torch.bfloat16))
    p.grad = torch.zeros_like(p)
    rs = np.random.RandomState(9)
    spans = [(0, 4096), ((1 << 31) - 4096, n)]
    for a, b in spans:
        p.data[a:b] = torch.from_numpy(_values(rs, b - a)).to(dev, torch.bfloat16)
    opt = AdamW([p], LR, BETAS, EPS, DECAY, 1.0, 8)
    state = {a: (np.zeros(b - a), np.zeros(b - a)) for a, b in spans}
    for t in (1, 2):
        for a, b in spans:
            p.grad[a:b] = torch.from_numpy(_values(rs, b - a, 0.1)).to(dev, torch.bfloat16)
        before = [(_np(p[a:b]), _np(p.grad[a:b])) for a, b in spans]
        _, f = ref.factor([g for _, g in before], 1.0)
        opt.step()
        (m,), (v,) = opt.moments()
        for (a, b), (x, g) in zip(spans, before):
            want, m64, v64, off, *_ = ref.adamw(x, g, *state[a], t, LR, BETAS, EPS, DECAY, f, True)
            _within(p[a:b], want, off)
            state[a] = ref.held(m64, t, 14, False, a)[0], ref.held(v64, t, 30, True, a)[0]
            assert np.array_equal(_np(m[a:b]), state[a][0]) and np.array_equal(_np(v[a:b]), state[a][1])
        del m, v
    assert not p[4096:(1 << 31) - 4096].any()


def test_a_rate_on_the_device_stays_where_it_is(dev):
    """Loading a state sets it; a step that was captured goes on with what was loaded."""
    from orca_b200.optim import AdamW
    params, rs = _params(dev, [700], [torch.float32])
    lr = torch.tensor(0.5, device=dev)
    opt = AdamW(params, lr)
    _give(params, rs)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        opt.step()
    saved = opt.state_dict()
    saved["param_groups"][0]["lr"] = 0.0
    opt.load_state_dict(saved)
    assert opt.param_groups[0]["lr"] is lr
    opt.param_groups[0]["weight_decay"] = 0.0
    was = params[0].detach().clone()
    graph.replay()          # (weight decay, too, is lr's)
    assert torch.equal(params[0], was) and int(opt.state[params[0]]["step"]) == 1


def test_made_on_one_stream_and_stepped_on_another(dev):
    """State is there whichever stream takes the first step; an optimiser that is made inside a capture is refused."""
    from orca_b200.optim import AdamW
    params, rs = _params(dev, [1 << 22], [torch.float32])
    _give(params, rs)
    copies = [torch.nn.Parameter(p.detach().clone()) for p in params]
    copies[0].grad = params[0].grad.clone()
    torch.cuda.synchronize()
    stream = torch.cuda.Stream()
    busy = torch.randn(4096, 4096, device=dev)
    for _ in range(20):
        busy = busy @ busy * 0.01          # (what is enqueued behind it comes late)
    opt = AdamW(params)
    with torch.cuda.stream(stream):
        opt.step()
    other = AdamW(copies)
    other.step()
    torch.cuda.synchronize()
    assert torch.equal(params[0], copies[0])
    graph = torch.cuda.CUDAGraph()
    with pytest.raises(RuntimeError, match="replay"):
        with torch.cuda.graph(graph):
            AdamW(copies)


def test_inference_mode_and_one_gradient_for_two(dev):
    """A step where nothing is recorded; two parameters that have the same tensor as their gradient; a gradient that is its parameter."""
    from orca_b200.optim import AdamW
    for bits in (32, 8):
        params, rs = _params(dev, [3000, 3000, 3000], [torch.float32] * 3)
        opt = AdamW(params, LR, BETAS, EPS, DECAY, 1.0, bits)
        _give(params, rs)
        params[1].grad = params[0].grad
        params[2].grad = params[2].detach()
        with torch.inference_mode():
            _step_and_check(opt)


def test_a_state_that_does_not_fit_changes_nothing(dev):
    """Settings are looked at before anything is taken over, and nothing is shared with where they come from."""
    from orca_b200.optim import AdamW
    params, rs = _params(dev, [700, 30], [torch.float32] * 2)
    opt = AdamW(params, torch.tensor(LR, device=dev))
    _give(params, rs)
    opt.step()
    kept = copy.deepcopy(opt.state_dict())
    for change in (dict(betas=(1.0, 0.5)), dict(lr=-1.0), dict(eps=1e-40)):
        bad = copy.deepcopy(kept)
        bad["param_groups"][0].update(change)
        for state in bad["state"].values():
            state["exp_avg"].zero_()
        with pytest.raises(ValueError):
            opt.load_state_dict(bad)
    short = copy.deepcopy(kept)
    short["state"][1]["exp_avg_sq"] = short["state"][1]["exp_avg_sq"][:-1]
    with pytest.raises(ValueError):
        opt.load_state_dict(short)
    now = opt.state_dict()
    assert now["param_groups"][0]["betas"] == kept["param_groups"][0]["betas"] and float(now["param_groups"][0]["lr"]) == float(kept["param_groups"][0]["lr"])
    assert all(torch.equal(now["state"][i][k], v) for i, state in kept["state"].items() for k, v in state.items())
    second = AdamW([torch.nn.Parameter(p.detach().clone()) for p in params], 1.0)
    second.load_state_dict(opt.state_dict())
    assert isinstance(second.param_groups[0]["lr"], float)
    assert all(second.state[p][k] is not opt.state[q][k] for p, q in zip(second.param_groups[0]["params"], params) for k in ("exp_avg", "step"))


@pytest.mark.parametrize("dtype", TYPES, ids=str)
def test_the_norm_is_that_of_64_bits(dev, dtype):
    """As it is rounded once: a thread's sum is off by 2^-40 of it at most, so the root by 2^-41, 2^-16 of half a step of fp32 (2^-25 at least); the
    factor and the codes that follow from it, every one, at many small sizes and orders."""
    from orca_b200.optim import AdamW
    rs = np.random.RandomState(11)
    sizes = [2, 7, 16, 16, 16, 33, 160, 160, 1000, 4096, 5000] * 12
    for i, n in enumerate(sizes):
        x = rs.randn(n)
        x = np.sort(np.abs(x)) if i % 3 == 1 else x * 10.0 ** rs.uniform(-2, 1, n) if i % 3 == 2 else x
        p = torch.nn.Parameter(torch.from_numpy(rs.randn(n).astype(np.float32)).to(dev, dtype))
        p.grad = torch.from_numpy(x.astype(np.float32)).to(dev, dtype)
        opt = AdamW([p], LR, BETAS, EPS, DECAY, 0.1, 8)
        norm, _ = ref.factor([_np(p.grad)], 0.1)
        _step_and_check(opt)
        got = np.float32(float(opt.grad_norm))
        assert abs(float(got) - norm) <= 0.5 * float(np.spacing(got)) * (1 + 2.0 ** -14), (i, n)


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("eps", [0.0, 1e-30, 1e-20, 1e-13, 2e-10])
def test_small_gradients_beside_a_small_eps(dev, eps, bits):
    """Squares that are subnormal in fp32 count as what they are: an update is off by 18 steps (root 2, that of the correction 4, their product and sum 2, inverse 2,
    three products 3, the rate and its correction 3, moments 2), and by a step of the parameter."""
    from orca_b200.optim import AdamW
    rs = np.random.RandomState(4)
    p = torch.nn.Parameter(torch.zeros(5000, device=dev))
    opt = AdamW([p], LR, BETAS, eps, 0.0, None, bits)
    for t in range(1, 4):
        g = (10.0 ** rs.uniform(-20, -16, 5000) * np.where(rs.rand(5000) < 0.5, -1, 1)).astype(np.float32)
        (m,), (v,) = ([_np(x) for x in xs] for xs in opt.moments())
        was = _np(p)
        p.grad = torch.from_numpy(g).to(dev)
        opt.step()
        near = lambda x: x.astype(np.float32).astype(np.float64)
        f32, g = ref.f32, g.astype(np.float64)
        m = near(f32(BETAS[0]) * m + near(f32(1 - BETAS[0]) * g))
        v = near(f32(BETAS[1]) * v + near(f32(1 - BETAS[1]) * near(g * g)))
        assert (v[v > 0] < 2.0 ** -126).any() and (v > 0).all()
        by = LR / (1 - BETAS[0] ** t) * m / (np.sqrt(v) / np.sqrt(1 - BETAS[1] ** t) + eps)
        assert (np.abs(_np(p) - (was - by)) <= ref.U * (18 * np.abs(by) + 2 * np.abs(was))).all()


def test_checkpoints_of_another_optimiser_are_refused(dev):
    """What PyTorch's optimisers do that this one does not is no state of it: nothing is changed."""
    from orca_b200.optim import AdamW
    params, rs = _params(dev, [700], [torch.float32])
    _give(params, rs)
    for make in (lambda: torch.optim.AdamW(params, maximize=True), lambda: torch.optim.AdamW(params, amsgrad=True), lambda: torch.optim.Adam(params, weight_decay=0.1)):
        theirs = make()
        theirs.step()
        opt = AdamW(params)
        kept = copy.deepcopy(opt.state_dict())
        with pytest.raises(ValueError):
            opt.load_state_dict(theirs.state_dict())
        now = opt.state_dict()
        assert now["param_groups"] == kept["param_groups"]
        assert all(torch.equal(now["state"][0][k], v) for k, v in kept["state"][0].items())
    theirs = torch.optim.Adam(params, LR)          # (without weight decay it is the same)
    theirs.step()
    opt = AdamW(params)
    opt.load_state_dict(theirs.state_dict())
    _give(params, rs)
    _step_and_check(opt)
    for more in (dict(maximize=True), dict(amsgrad=True)):
        with pytest.raises(ValueError):
            AdamW([dict(params=[torch.nn.Parameter(torch.zeros(5, device=dev))], **more)])


def test_a_step_that_does_not_fit_changes_nothing(dev):
    from orca_b200.optim import AdamW
    params, rs = _params(dev, [700, 30], [torch.float32] * 2)
    opt = AdamW(params)
    _give(params, rs)
    opt.step()
    kept = copy.deepcopy(opt.state_dict())
    for bad in (None, "missing", "many", -1, float("nan"), float("inf"), 1.5, 2 ** 31, torch.tensor(-3), torch.tensor([1, 2]), torch.tensor(float("nan"))):
        given = copy.deepcopy(kept)
        for state in given["state"].values():
            state["exp_avg"].zero_()
        if isinstance(bad, str) and bad == "missing":
            del given["state"][1]["step"]
        else:
            given["state"][1]["step"] = bad
        with pytest.raises(ValueError, match="step"):
            opt.load_state_dict(given)
        assert all(torch.equal(opt.state_dict()["state"][i][k], v) for i, s in kept["state"].items() for k, v in s.items())
    for step in (7, 7.0, torch.tensor(7.0), torch.tensor([7], dtype=torch.int32, device=dev)):
        given = copy.deepcopy(kept)
        given["state"][0]["step"] = step
        opt.load_state_dict(given)
        assert [int(opt.state[p]["step"]) for p in params] == [7, 1]


@pytest.mark.parametrize("bits", [32, 8])
def test_checkpoints_of_parameters_that_lie_otherwise(dev, bits):
    """Moments are those of a parameter's elements, wherever they lie: a checkpoint of one that lies otherwise is taken with 32 bits, and with 8, whose blocks are those
    of memory, refused; states whose tensors are flat go by memory."""
    from orca_b200.optim import AdamW
    rs = np.random.RandomState(8)
    x, g = (torch.from_numpy(_values(rs, 40 * 30)).to(dev).view(40, 30) for _ in range(2))

    def made(turned, flat=False):
        p = torch.nn.Parameter((x.t().contiguous().t() if turned else x).clone(memory_format=torch.preserve_format))
        assert p.is_contiguous() != turned
        opt = AdamW([p], LR, BETAS, EPS, DECAY, None, bits)
        if flat:
            for name in ("exp_avg", "exp_avg_sq"):
                opt.state[p][name] = torch.zeros(1200, device=dev, dtype=opt.state[p][name].dtype)
        p.grad = g.clone()
        return p, opt
    for source in (False, True):
        for target in (False, True):
            for flat in (False, True):
                p, opt = made(source)
                opt.step()
                saved = copy.deepcopy(opt.state_dict())
                q, other = made(target, flat)
                if bits == 8 and source != target:
                    kept = copy.deepcopy(other.state_dict())
                    with pytest.raises(ValueError, match="order"):
                        other.load_state_dict(saved)
                    assert all(torch.equal(other.state_dict()["state"][0][k], v) for k, v in kept["state"][0].items())
                    continue
                other.load_state_dict(saved)
                with torch.no_grad():
                    q.copy_(p)
                opt.step(), other.step()
                assert torch.equal(p, q)
                for a, b in zip(opt.moments(), other.moments()):
                    assert torch.equal(a[0], b[0] if b[0].shape == q.shape else b[0].as_strided(q.shape, q.stride()))
                good, other.state[q]["exp_avg"] = other.state[q]["exp_avg"], torch.zeros(2400, device=dev, dtype=other.state[q]["exp_avg"].dtype)[::2]
                with pytest.raises(ValueError):
                    other.load_state_dict(saved)
                other.state[q]["exp_avg"] = good
                # and flat ones go to where they came from
                if flat and target:
                    r, third = made(True)
                    third.load_state_dict(copy.deepcopy(other.state_dict()))
                    with torch.no_grad():
                        r.copy_(q)
                    third.step(), other.step()
                    assert torch.equal(r, q)


def test_hooks_of_loading(dev):
    """A hook before sees the state dict and may give another; one behind sees what was taken over; both of a copy, too, and none once it is removed."""
    from orca_b200.optim import AdamW
    params, rs = _params(dev, [30], [torch.float32])
    opt = AdamW(params)
    saved, seen = opt.state_dict(), []

    def other(optimizer, state_dict):
        seen.append("before")
        groups = [dict(g, lr=0.25) for g in state_dict["param_groups"]]
        state_dict["param_groups"] = None          # (the caller's is another dict)
        return dict(state_dict, param_groups=groups)
    first = opt.register_load_state_dict_pre_hook(other)
    second = opt.register_load_state_dict_post_hook(lambda optimizer: seen.append(optimizer.param_groups[0]["lr"]))
    opt.load_state_dict(saved)
    assert seen == ["before", 0.25] and saved["param_groups"] is not None
    first.remove()
    opt.load_state_dict(saved)
    assert seen == ["before", 0.25, saved["param_groups"][0]["lr"]]
    second.remove()

    def in_place(optimizer, state_dict):
        seen.append(len(state_dict["state"]))
        state_dict["param_groups"] = [dict(g, lr=0.125) for g in state_dict["param_groups"]]
    watch = opt.register_load_state_dict_pre_hook(in_place)
    opt.load_state_dict(saved)
    assert seen[3:] == [1] and opt.param_groups[0]["lr"] == 0.125 and saved["param_groups"][0]["lr"] != 0.125
    watch.remove()
    copy.deepcopy(opt).load_state_dict(saved)
    assert len(seen) == 4


@pytest.mark.parametrize("bits", [32, 8])
@pytest.mark.parametrize("count", [1, 31, 32, 33, 127, 128, 129, 319, 320, 321, 641])
def test_as_many_tensors_as_a_launch_takes(dev, count, bits):
    """Counts at the borders between the kernels for few, some and many tensors, and of a launch and the next, which goes on with the norm and the steps."""
    from orca_b200.optim import AdamW
    params, rs = _params(dev, [1 + (37 * i) % 300 if i % 50 else 5000 for i in range(count)], [torch.float32] * count)
    opt = AdamW(params, LR, BETAS, EPS, DECAY, 1.0, bits)
    for _ in range(2):
        _give(params, rs)
        _step_and_check(opt)


@pytest.mark.parametrize("bits", [32, 8])
def test_more_tensors_of_each_type_than_a_launch_takes(dev, bits):
    from orca_b200.optim import AdamW
    params, rs = _params(dev, [1 + (37 * i) % 300 for i in range(1000)], TYPES * 334)
    groups = [dict(params=params[i::10], lr=10.0 ** -(i % 4 + 1), weight_decay=0.01 * i) for i in range(10)]
    opt = AdamW(groups, LR, BETAS, EPS, DECAY, 1.0, bits)
    for _ in range(2):
        _give(params, rs)
        _step_and_check(opt)


@pytest.mark.parametrize("bits", [32, 8])
def test_state_that_is_exchanged(dev, bits):
    """A step goes by what stands in ``state``: by a dict that replaces another, whatever the order of parameters there; without one it is refused."""
    from orca_b200.optim import AdamW
    params, rs = _params(dev, [700, 30, 300], [torch.float32] * 3)
    opt = AdamW(params, LR, BETAS, EPS, DECAY, 1.0, bits)
    _give(params, rs)
    _step_and_check(opt)
    fresh = AdamW([torch.nn.Parameter(p.detach().clone()) for p in params], bits=bits)
    for p, q in list(zip(params, fresh.param_groups[0]["params"]))[1:]:
        opt.state[p] = fresh.state[q]
    _give(params, rs)
    _step_and_check(opt)
    assert [int(opt.state[p]["step"]) for p in params] == [2, 1, 1]
    kept = dict(opt.state)
    opt.state.clear()
    with pytest.raises(ValueError, match="state"):
        opt.step()
    for p in params[::-1]:
        opt.state[p] = kept[p]
    _give(params, rs)
    _step_and_check(opt)
    assert [int(opt.state[p]["step"]) for p in params] == [3, 2, 2]
    opt.state["other"] = {}
    _give(params, rs)
    _step_and_check(opt)
    opt.state[fresh.param_groups[0]["params"][0]] = {}
    with pytest.raises(ValueError, match="groups"):
        opt.step()


def test_a_step_that_two_parameters_have(dev):
    """It would be counted twice: refused, as long as both have a gradient."""
    from orca_b200.optim import AdamW
    params, rs = _params(dev, [700, 30, 5], [torch.float32, torch.bfloat16, torch.float32])
    opt = AdamW([dict(params=params[:1]), dict(params=params[1:])], LR, BETAS, EPS, DECAY)
    _give(params, rs)
    own, opt.state[params[2]]["step"] = opt.state[params[2]]["step"], opt.state[params[0]]["step"]
    kept = [p.detach().clone() for p in params]
    with pytest.raises(ValueError, match="of its own"):
        opt.step()
    assert all(torch.equal(p, k) for p, k in zip(params, kept)) and int(opt.state[params[0]]["step"]) == 0
    params[2].grad = None
    opt.step()
    assert [int(opt.state[p]["step"]) for p in params] == [1, 1, 1]
    opt.state[params[2]]["step"] = own
    _give(params, rs)
    _step_and_check(opt)


def test_parameters_made_in_inference_mode(dev):
    """Outside of it they are not changed, as by any other call: refused before anything is enqueued."""
    from orca_b200.optim import AdamW
    with torch.inference_mode():
        p = torch.nn.Parameter(torch.randn(300, device=dev))
        p.grad = torch.randn(300, device=dev)
        opt = AdamW([p], max_norm=1.0)
        opt.step()
        kept = p.clone(), opt.state[p]["step"].clone()
    with pytest.raises(RuntimeError, match="inference mode"):
        opt.step()
    assert torch.equal(p, kept[0]) and torch.equal(opt.state[p]["step"], kept[1])


@pytest.mark.parametrize("bits", [32, 8])
def test_parameters_that_come_later(dev, bits):
    from orca_b200.optim import AdamW
    opt = AdamW([dict(params=[])], LR, BETAS, EPS, DECAY, 1.0, bits)
    opt.step()
    params, rs = _params(dev, [700, 30], [torch.float32, torch.bfloat16])
    for p in params:
        opt.add_param_group(dict(params=[p]))
        _give(params, rs)
        _step_and_check(opt)
    assert [int(opt.state[p]["step"]) for p in params] == [2, 1]


@pytest.mark.parametrize("bits", [32, 8])
def test_state_that_was_taken_out_is_loaded_again(dev, bits):
    from orca_b200.optim import AdamW
    params, rs = _params(dev, [700, 30], [torch.float32, torch.bfloat16])
    opt = AdamW(params, LR, BETAS, EPS, DECAY, None, bits)
    _give(params, rs)
    opt.step()
    saved = copy.deepcopy(opt.state_dict())
    for taken in (params[:1], params):
        for p in taken:
            del opt.state[p]
        opt.load_state_dict(saved)
        assert [int(opt.state[p]["step"]) for p in params] == [1, 1]
        now = opt.state_dict()["state"]
        assert all(torch.equal(now[i][k], v) for i, s in saved["state"].items() for k, v in s.items())
    _give(params, rs)
    _step_and_check(opt)
