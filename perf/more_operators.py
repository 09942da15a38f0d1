"""A training step next to trained rows: layer norm with its gradients, AdamW over many tensors with states in 32 or 8 bits.

What a user who trains on rows of node tables (``orca_b200.lookup``) goes on with:

``norm``    Layer norm over the last dimension, and where the case has it the gradients of rows, weight and bias (``layer_norm``).
``adamw``   One step of AdamW over all tensors, gradients cut to a norm over all of them where the case has it (``AdamW``).
``adamw8``  The same with both moments in 8 bits, which are read afterwards, as a program that watches its training does
            (``AdamW(bits=8)``, ``moments``).

AdamW with g' = g * f, f = min(1, max_norm / norm) in 32 bits, t steps with this one:
  m' = b1 m + (1 - b1) g',  v' = b2 v + (1 - b2) g'^2,  p' = p (1 - lr wd) - lr / (1 - b1^t) m' / (sqrt(v' / (1 - b2^t)) + eps).

Moments in 8 bits are held by blocks of 256 of a tensor.  A block's exponent E is the exponent field of its largest magnitude as fp32, 33 at
least.  The mean has a sign, 4 bits of exponent and 3 of mantissa; exponent 14 is the binade that E names, 0 the subnormal one.  The square
has 5 bits of exponent (30 is that binade) and 3 of mantissa.  What is held is the moment in 32 bits (products by the coefficients and the
factor rounded, the last product and sum together, once): its position on the scale of codes, to 20 bits behind the point (ties to even), plus u,
rounded down; u are 20 bits that follow from the step and the element's place in its tensor (``_dither``).  A square that is not zero has code 1 at least.

Sizes are those of the model and of the synthetic workloads in ``orca_b200/synthetic.py`` (rows of 172 and 688, batches of 200 to 2000 edges, up
to 1,140,149 nodes) and ranges around them.
"""
import math
import types

import torch

own = False

D = 172
BLOCK = 256            # elements of a tensor that share an exponent
STEPS = 1000           # that the moments have behind them
LR, BETAS, EPS, DECAY = 1e-4, (0.9, 0.999), 1e-8, 0.01
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}
SIZE = {"float32": 4, "bfloat16": 2, "float16": 2}


# ---------------------------------------------------------------------------------------------- the cases
def listed():
    return [
        # one embedding is normalised as it is asked for
        dict(name="norm_one", op="norm", rows=1, width=172, type="float32", weight="float32", grad=False),
        # a training step's rows of a batch of 200 edges
        dict(name="norm_batch", op="norm", rows=600, width=172, type="float32", weight="float32", grad=True),
        # messages of a batch of 2000 edges in 16 bits, weights in 32
        dict(name="norm_messages", op="norm", rows=4001, width=688, type="bfloat16", weight="float32", grad=True),
        # a large batch and its neighbours
        dict(name="norm_group", op="norm", rows=66001, width=172, type="bfloat16", weight="bfloat16", grad=True),
        # an odd width: no row begins where a wide load could
        dict(name="norm_odd", op="norm", rows=20011, width=515, type="float16", weight="float16", grad=True),
        # all nodes of the largest graph
        dict(name="norm_nodes", op="norm", rows=1140150, width=172, type="float32", weight="float32", grad=True),
        # wide rows of other models
        dict(name="norm_wide", op="norm", rows=8191, width=8192, type="bfloat16", weight="bfloat16", grad=True),
        # the two-layer model's own parameters, gradients cut
        dict(name="adamw_model", op="adamw", layers=2, table=0, tensors=0, largest=0, type="float32", clip=True),
        # many tensors of all sizes
        dict(name="adamw_many", op="adamw", layers=0, table=0, tensors=293, largest=400001, type="float32", clip=False),
        # a trained table of the largest graph's nodes beside the model
        dict(name="adamw_table", op="adamw", layers=2, table=1140150, tensors=0, largest=0, type="float32", clip=False),
        # the one-layer model, moments in 8 bits
        dict(name="adamw8_model", op="adamw8", layers=1, table=0, tensors=0, largest=0, type="float32", clip=True),
        # the table in 16 bits, its moments in 8
        dict(name="adamw8_table", op="adamw8", layers=0, table=1140150, tensors=0, largest=0, type="bfloat16", clip=True),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    op = rng.choice(["norm", "norm", "adamw", "adamw8"])
    t = rng.choice(list(TYPES))
    if op == "norm":
        width = rng.choice([172, 172, 344, 516, 688, _log(rng, 1, 8192), _log(rng, 1, 8192)])
        return dict(op=op, rows=_log(rng, 1, min(1140150, 67000000 // width)), width=width, type=t, weight=rng.choice([t, "float32"]),
                    grad=rng.random() < 0.75)
    kind = rng.choice(["model", "table", "tensors"])
    return dict(op=op, layers=rng.choice([1, 2] if op == "adamw" else [1]) if kind == "model" else 0,
                table=_log(rng, 1500, 1140150) if kind != "tensors" else 0,
                tensors=_log(rng, 1, 401 if op == "adamw" else 20) if kind == "tensors" else 0,
                largest=_log(rng, 30, 400001 if op == "adamw" else 4000001) if kind == "tensors" else 0, type=t, clip=rng.random() < 0.5)


def _sizes(case):
    """Elements of each tensor: the model's parameters with so many attention layers, a table, tensors with lengths over all magnitudes."""
    sizes = []
    if case["layers"]:
        sizes += [3 * D * 4 * D, 3 * D * D, 3 * D, 3 * D, 2 * D * D, D, D, 1]
        sizes += case["layers"] * [4 * D * D, 6 * D * D, 6 * D * D, 6 * D, 4 * D * D, 2 * D, 3 * D * D, D, D * D, D, D, D]
    if case["table"]:
        sizes.append(case["table"] * D)
    n = case["tensors"]
    return sizes + [max(1, int(case["largest"] ** ((i + 0.5) / n))) for i in range(n)]


def work(case):
    size = SIZE[case["type"]]
    if case["op"] == "norm":
        n = case["rows"] * case["width"]
        both = 2 * case["width"] * SIZE[case["weight"]]
        if case["grad"]:
            return {"bytes": 4 * n * size + 2 * both, "flops": 20 * n}
        return {"bytes": 2 * n * size + both, "flops": 8 * n}
    n = sum(_sizes(case))
    if case["op"] == "adamw":
        return {"bytes": n * (3 * size + 16), "flops": n * (17 if case["clip"] else 15)}
    # codes in and out, exponents of the blocks; the moments' values in 16 bits
    return {"bytes": n * (3 * size + 4 + 4) + n / BLOCK * 4, "flops": n * (27 if case["clip"] else 25)}


# ---------------------------------------------------------------------------------------------- inputs
def prepare(case, seed):
    gen = torch.Generator(device="cuda").manual_seed(int(seed))
    randn = lambda *s: torch.randn(*s, device="cuda", generator=gen)
    rand = lambda *s: torch.rand(*s, device="cuda", generator=gen)
    t = TYPES[case["type"]]
    s = types.SimpleNamespace(op=case["op"])
    if s.op == "norm":
        rows, width, w = case["rows"], case["width"], TYPES[case["weight"]]
        # rows of their own sizes and offsets, columns of their own means
        s.x = (randn(rows, width) * torch.exp(0.5 * randn(rows, 1)) + 0.3 * randn(1, width) + randn(rows, 1)).to(t)
        s.weight, s.bias = (1 + 0.1 * randn(width)).to(w), (0.1 * randn(width)).to(w)
        s.eps, s.grad = 1e-5, None
        if case["grad"]:
            s.grad = randn(rows, width).to(t)
            for a in (s.x, s.weight, s.bias):
                a.requires_grad_(True)
        return s
    # tensors lie in one buffer, each from a multiple of a block on, as an allocator places them; what lies between is zero and stays so
    sizes = _sizes(case)
    begins = [0]
    for n in sizes:
        begins.append(begins[-1] + -(-n // BLOCK) * BLOCK)
    s.spans, total = [(b, b + n) for b, n in zip(begins, sizes)], begins[-1]
    s.begins, s.lengths = torch.tensor(begins[:-1], device="cuda"), torch.tensor(sizes, device="cuda")
    blocks = torch.tensor([-(-n // BLOCK) for n in sizes], device="cuda")
    s.begin_of_block = torch.repeat_interleave(s.begins, blocks)
    inside = torch.arange(total, device="cuda").view(-1, BLOCK) - s.begin_of_block[:, None] < torch.repeat_interleave(s.lengths, blocks)[:, None]
    inside = inside.view(-1).float()
    size = 1e-3 * torch.exp(randn(len(sizes)))                       # gradients of each tensor
    scale = torch.repeat_interleave(size, blocks * BLOCK) * inside
    del inside
    s.p = (0.05 * randn(total) * (scale > 0)).to(t)
    s.g = (scale * randn(total)).to(t)
    s.m, s.v = 0.3 * scale * randn(total), scale ** 2 * (0.5 + rand(total))
    del scale
    if case["table"]:
        # most rows of a table are not named by a step, some never were
        a, b = s.spans[-1]
        never = rand(case["table"], 1)
        for x, share in ((s.g, 0.7), (s.m, 0.1), (s.v, 0.1)):
            x[a:b].view(-1, D).mul_((never >= share).to(x.dtype))
    s.t, s.max_norm = STEPS, 1.0 if case["clip"] else None
    if s.op == "adamw8":
        zero = torch.zeros((), dtype=torch.int64, device="cuda")
        codes_m, exp_m = _encode(s.m, zero, 14, False)
        codes_v, exp_v = _encode(s.v, zero, 30, True)
        s.m, s.v, s.exponents = codes_m, codes_v, torch.stack([exp_m, exp_v], 1).contiguous()
    if own:
        from orca_b200.optim import AdamW
        s.params = [torch.nn.Parameter(s.p[a:b]) for a, b in s.spans]
        s.opt = AdamW(s.params, lr=LR, betas=BETAS, eps=EPS, weight_decay=DECAY, max_norm=s.max_norm, bits=8 if s.op == "adamw8" else 32)
        for p, (a, b) in zip(s.params, s.spans):
            p.grad = s.g[a:b]
            state = s.opt.state[p]
            state["step"].fill_(s.t)
            state["exp_avg"], state["exp_avg_sq"] = s.m[a:b], s.v[a:b]
            if s.op == "adamw8":
                state["exponents"] = s.exponents[a // BLOCK:-(-b // BLOCK)]
    return s


# ---------------------------------------------------------------------------------------------- the plain forms
def _norm(s):
    x, w = s.x.detach().float(), s.weight.detach().float()
    c = x - x.mean(1, keepdim=True)
    r = 1 / torch.sqrt((c * c).mean(1, keepdim=True) + s.eps)
    h = c * r
    out = (h * w + s.bias.detach().float()).to(s.x.dtype)
    if s.grad is None:
        return out
    g = s.grad.float()
    d = g * w
    dx = r * (d - d.mean(1, keepdim=True) - h * (d * h).mean(1, keepdim=True))
    # (sums over up to a million rows: in 64 bits)
    dw, db = (g * h).sum(0, dtype=torch.float64), g.sum(0, dtype=torch.float64)
    return out, dx.to(s.x.dtype), dw.to(s.weight.dtype), db.to(s.weight.dtype)


def _dither(place, step, second):
    """20 bits for each place in a tensor (int64) at a step, others for the second moment: the place's group of eight and the step through two rounds
    of multiplications (odd fractions of the golden ratio, of the roots of 2 and 3), then two steps an element of a linear congruence."""
    low = 0xffffffff
    x = ((place >> 3) * 0x9e3779b1 + (place >> 35) * 0x6a09e667 + step * 0xbb67ae85) & low
    x = ((x ^ (x >> 16)) * 0x6a09e667) & low
    x = ((x ^ (x >> 15)) * 0xbb67ae85) & low
    x = x ^ (x >> 16)
    a, c, mul, add = 1, 0, [], []
    for _ in range(16):
        a, c = (a * 1664525) & low, (c * 1664525 + 1013904223) & low
        mul.append(a)
        add.append(c)
    k = 2 * (place & 7) + int(second)
    mul, add = (torch.tensor(v, device=place.device) for v in (mul, add))
    return ((x * mul[k] + add[k]) & low) >> 12


def _power(e):
    """2^e in 32 bits, from its bits; e from -127 to 127."""
    return torch.where(e > -127, (e + 127) << 23, 1 << 22).to(torch.int32).view(torch.float32)


def _encode(x, u, top, square):
    """Codes and exponents of fp32 moments, whole blocks of them: positions on the scale of codes are the bits of fp32 numbers, subnormal
    ones too, once the block's binade is that of exponent `top`."""
    a = x.abs().view(-1, BLOCK)
    e = (a.amax(1).view(torch.int32) >> 23).clamp(min=33)
    fine = a * _power(128 - e)[:, None] * 2.0 ** (top - 128)
    codes = (fine.view(-1).view(torch.int32).long() + u) >> 20
    if square:
        codes = torch.where(x > 0, codes.clamp(min=1), codes)
    else:
        codes = codes + 128 * (x < 0)
    return codes.to(torch.uint8), e.to(torch.uint8)


def _decode(codes, e, top, square):
    size = (codes if square else codes & 127).int() << 20
    x = (size.view(torch.float32) * 2.0 ** (127 - top)).view(-1, BLOCK) * _power(e.int() - 127)[:, None]
    x = x.view(-1)
    return x if square else torch.where(codes > 127, -x, x)


def _adamw(s):
    s.t += 1
    (b1, b2), eight = BETAS, s.op == "adamw8"
    g, norm = s.g.float(), None
    if s.max_norm is not None:
        norm = torch.sqrt(s.g.double().square().sum())
        g = g * (s.max_norm / norm).clamp(max=1).float()
    if eight:
        # (rounded as the definition says, by which codes are decided: products in 32 bits, the last one and the sum together)
        f32 = lambda v: float(torch.tensor(v, dtype=torch.float32))
        m, v = _decode(s.m, s.exponents[:, 0], 14, False), _decode(s.v, s.exponents[:, 1], 30, True)
        m = (f32(b1) * m.double() + (f32(1 - b1) * g).double()).float()
        v = (f32(b2) * v.double() + (f32(1 - b2) * (g * g)).double()).float()
    else:
        m, v = b1 * s.m + (1 - b1) * g, b2 * s.v + (1 - b2) * g * g
    size = LR / (1 - b1 ** s.t)
    p = s.p.float() * (1 - LR * DECAY) - size * m / (torch.sqrt(v) / math.sqrt(1 - b2 ** s.t) + EPS)
    s.p.copy_(p)
    if not eight:
        s.m, s.v = m, v
        return s.p, m, v, norm if norm is None else norm.float()
    place = (torch.arange(len(p), device=p.device).view(-1, BLOCK) - s.begin_of_block[:, None]).view(-1)
    s.m, e_m = _encode(m, _dither(place, s.t, False), 14, False)
    s.v, e_v = _encode(v, _dither(place, s.t, True), 30, True)
    s.exponents = torch.stack([e_m, e_v], 1)
    m, v = _decode(s.m, e_m, 14, False).bfloat16(), _decode(s.v, e_v, 30, True).bfloat16()
    return s.p, [m[a:b] for a, b in s.spans], [v[a:b] for a, b in s.spans], norm if norm is None else norm.float()


def run(state):
    s = state
    if not own:
        return _norm(s) if s.op == "norm" else _adamw(s)
    if s.op == "norm":
        from orca_b200.norm import layer_norm
        out = layer_norm(s.x, s.weight, s.bias, s.eps)
        return out if s.grad is None else (out.detach(), *torch.autograd.grad(out, (s.x, s.weight, s.bias), s.grad))
    s.opt.step()
    if s.op == "adamw":
        return s.p, s.m, s.v, s.opt.grad_norm
    m, v = s.opt.moments()
    return s.p, m, v, s.opt.grad_norm


# ---------------------------------------------------------------------------------------------- the definition, in 64 bits
def _exact_norm(s):
    leaves = [a.detach().double().requires_grad_(s.grad is not None) for a in (s.x, s.weight, s.bias)]
    x, w, b = leaves
    var, mean = torch.var_mean(x, 1, correction=0, keepdim=True)
    out = (x - mean) * torch.rsqrt(var + s.eps) * w + b
    if s.grad is None:
        return out
    return (out.detach(), *torch.autograd.grad(out, leaves, s.grad.double()))


def _held(x, top, u, unsigned):
    """The values that one tensor's moments are held as: x in fp32, one tensor; u as `_dither` gives it."""
    n = len(x)
    x = torch.nn.functional.pad(x.double(), (0, -n % BLOCK)).view(-1, BLOCK)
    u = torch.nn.functional.pad(u.double(), (0, -n % BLOCK)).view(-1, BLOCK)
    size = x.abs()
    binade = lambda a: torch.frexp(a)[1].long() - 1                 # floor of the logarithm
    highest = binade(size.amax(1, keepdim=True)).clamp(min=33 - 127)
    exponent = torch.where(size > 0, binade(size) - highest + top, 0).clamp(min=1)
    unit = torch.ldexp(torch.ones_like(x), highest - top + exponent - 3)
    at = torch.round((size / unit + 8 * (exponent - 1)) * 2.0 ** 20)
    code = torch.floor((at + u) / 2.0 ** 20)
    if unsigned:
        code = torch.where(size > 0, code.clamp(min=1), code)
    exponent, mantissa = torch.div(code, 8, rounding_mode="floor"), code % 8
    value = torch.where(exponent > 0, 8 + mantissa, mantissa) * torch.ldexp(torch.ones_like(x), (highest - top - 3 + exponent.clamp(min=1).long()))
    return (value * torch.sign(x)).view(-1)[:n]


def _start64(codes, exponents, bits):
    """Values of one tensor's codes, `bits` of them below the sign."""
    c, top = codes.long(), 14 if bits == 7 else 30
    sign, c = (torch.where(c >= 128, -1.0, 1.0), c % 128) if bits == 7 else (1.0, c)
    e = exponents.long().repeat_interleave(BLOCK)[:len(c)] - 127 - top - 3
    value = torch.where(c < 8, c, 8 + c % 8).double()
    return sign * torch.ldexp(value, e + torch.div(c, 8, rounding_mode="floor").clamp(min=1))


def _exact_adamw(s):
    b1, b2 = BETAS
    t = s.t + 1
    total = sum(s.g[a:b].double().pow(2).sum() for a, b in s.spans) ** 0.5
    factor = 1.0 if s.max_norm is None else torch.clamp(s.max_norm / total, max=1.0).float().double()
    p64, means, squares = torch.zeros(len(s.p), dtype=torch.float64, device="cuda"), [], []
    near = lambda x: x.float().double()                             # to 32 bits
    for a, b in s.spans:
        g, p = s.g[a:b].double() * factor, s.p[a:b].double()
        if s.op == "adamw":
            m, v = s.m[a:b].double() * b1 + g * (1 - b1), s.v[a:b].double() * b2 + g * g * (1 - b2)
            means.append(m)
            squares.append(v)
        else:
            blocks = s.exponents[a // BLOCK:-(-b // BLOCK)]
            c = [float(torch.tensor(x).float()) for x in (b1, 1 - b1, b2, 1 - b2)]
            g = near(g)
            m = near(c[0] * _start64(s.m[a:b], blocks[:, 0], 7) + near(c[1] * g))
            v = near(c[2] * _start64(s.v[a:b], blocks[:, 1], 8) + near(c[3] * near(g * g)))
            place = torch.arange(b - a, device="cuda")
            means.append(_held(m, 14, _dither(place, t, False), False))
            squares.append(_held(v, 30, _dither(place, t, True), True))
        p64[a:b] = p - LR * DECAY * p - LR * (m / (1 - b1 ** t)) / ((v / (1 - b2 ** t)).sqrt() + EPS)
    if s.op == "adamw":
        flat = lambda parts: torch.cat([torch.nn.functional.pad(x, (0, -len(x) % BLOCK)) for x in parts])
        means, squares = flat(means), flat(squares)
    return p64, means, squares, None if s.max_norm is None else total


def exact(case, seed):
    s = prepare(case, seed)
    return _exact_norm(s) if s.op == "norm" else _exact_adamw(s)
