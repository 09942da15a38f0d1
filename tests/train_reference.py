"""Layer norm, AdamW and moments in 8 bits in 64 bits (NumPy), and how far arithmetic in 32 bits may be off them.

U is half a step of fp32 relative to a value.  Bounds are of first order, times 1 + 2^-7 for the terms behind."""
import numpy as np

U = 2.0 ** -24
MORE = 1 + 2.0 ** -7


# ---------------------------------------------------------------------------------------------- layer norm
def _depth(width):
    """Additions that a value goes through on its way into a row's sum: eight threads a row at least, whose sums are added in steps."""
    return -(-width // 8) + 40


def norm(x, w, b, eps):
    """y, h, r and the bounds of h and y before the last rounding, for x [rows, width]."""
    mean = x.mean(1, keepdims=True)
    c = x - mean
    var = (c * c).mean(1, keepdims=True)
    with np.errstate(divide="ignore", invalid="ignore"):
        r = 1 / np.sqrt(var + eps)
        h = c * r
    depth = _depth(x.shape[1])
    # sums are of differences from some number near the mean, the mean of some of the values or of all: off by `first` at most.  Differences are rounded,
    # and their mean is taken off them
    first = np.abs(c).max(1, keepdims=True) + (depth + 1) * U * np.abs(x).mean(1, keepdims=True)
    size = np.abs(c) + first
    off_c = U * size + depth * U * size.mean(1, keepdims=True) + 2 * U * (size + first)
    # the variance is that of the differences less the square of their mean; r has half its error and two roundings
    off_var = 2 * (off_c * size).mean(1, keepdims=True) + (depth + 4) * U * (size * size).mean(1, keepdims=True) + 3 * U * first * first
    with np.errstate(divide="ignore", invalid="ignore"):
        off_r = np.where(var + eps > 0, off_var / (2 * (var + eps)), 0) + 4 * U
    off_h = MORE * (off_c * r + np.abs(h) * (off_r + 2 * U))
    y = h * w + b
    return y, h, r, off_h, off_r, off_h * np.abs(w) + 3 * U * (np.abs(h * w) + np.abs(b))


def norm_grad(g, x, w, eps):
    """dx, dw, db and the bounds of each before the last rounding."""
    _, h, r, off_h, off_r, _ = norm(x, w, 0.0, eps)
    rows, width = x.shape
    d = g * w
    c1, c2 = d.mean(1, keepdims=True), (d * h).mean(1, keepdims=True)
    dx = r * (d - c1 - h * c2)
    depth = _depth(width)
    off_c1 = (depth + 2) * U * np.abs(d).mean(1, keepdims=True)
    off_c2 = (depth + 3) * U * np.abs(d * h).mean(1, keepdims=True) + (np.abs(d) * off_h).mean(1, keepdims=True)
    inner = np.abs(d) + np.abs(c1) + np.abs(h * c2)
    off = r * (4 * U * inner + off_c1 + np.abs(h) * off_c2 + off_h * np.abs(c2)) + (off_r + 2 * U) * r * inner
    # rows are added up in parts of 64, or of a 592nd of them; parts by sixteen threads a column, whose sums are added in order
    deep = min(rows, max(64, -(-rows // 592))) + 37 + 16 + 10
    off_w = deep * U * np.abs(g * h).sum(0) + (np.abs(g) * off_h).sum(0)
    return dx, (g * h).sum(0), g.sum(0), MORE * off, MORE * off_w, MORE * deep * U * np.abs(g).sum(0)


# ---------------------------------------------------------------------------------------------- AdamW
f32 = lambda v: np.float64(np.float32(v))


def factor(grads, max_norm):
    """The norm over all gradients, and the factor in 32 bits."""
    norm = np.sqrt(sum((g.astype(np.float64) ** 2).sum() for g in grads))
    return norm, (f32(max_norm / norm) if norm > max_norm else 1.0)


def squares(x):
    """The sum of squares of each row of x [threads, 16] (fp32) as a thread takes it: two sums in 32 bits from a power of two on that no square is above,
    with what each rounding leaves; products and sums that go together are rounded once."""
    f, wide = np.float32, np.longdouble
    fma = lambda a, b, c: (a.astype(wide) * b.astype(wide) + c.astype(wide)).astype(f)
    begin = (f(4) * ((np.abs(x).max(1).view(np.uint32) & np.uint32(0x7f800000)).view(f)) ** 2)[:, None]
    pairs = x.reshape(len(x), 8, 2)
    total, rest = np.repeat(begin, 2, 1), np.zeros((len(x), 2), f)
    for k in range(8):
        after = fma(pairs[:, k], pairs[:, k], total)
        by = after - total
        rest = rest + fma(pairs[:, k], pairs[:, k], -by)
        total = after
    total = (total - begin).astype(np.float64)
    return total[:, 0] + total[:, 1] + (rest[:, 0] + rest[:, 1]).astype(np.float64)


def adamw(p, g, m, v, t, lr, betas, eps, decay, f=1.0, eight=False):
    """p', m', v' and the bounds of each before the last rounding; with `eight` m' and v' as fp32 values, rounded as the format says."""
    b1, b2 = betas
    if eight:
        near = lambda x: x.astype(np.float32).astype(np.float64)
        g = near(g * f)
        m2 = near(f32(b1) * m + near(f32(1 - b1) * g))
        v2 = near(f32(b2) * v + near(f32(1 - b2) * near(g * g)))
        off_m, off_v = np.zeros_like(p), np.zeros_like(p)
    else:
        g = g * f
        m2, v2 = b1 * m + (1 - b1) * g, b2 * v + (1 - b2) * g * g
        # each coefficient, the factor's product, each product and the sum are rounded
        off_m = 4 * U * (np.abs(b1 * m) + np.abs((1 - b1) * g))
        off_v = 6 * U * v2 + 2.0 ** -149
    size, root = lr / (1 - b1 ** t), 1 / np.sqrt(1 - b2 ** t)
    low = np.sqrt(v2) * root + eps
    with np.errstate(divide="ignore", invalid="ignore"):
        new = p * (1 - lr * decay) - size * m2 / low
        # root of v': half its error, its own (two steps), none of a v' below 2^-126; its product, eps, their sum; the quotient (two steps), two products, size
        off_low = np.sqrt(v2 + off_v) * root - np.sqrt(v2) * root + 8 * U * low + np.where(v2 < 2.0 ** -125, np.sqrt(v2) * root, 0)
        off = 3 * U * np.abs(p) + size * off_m / low + np.abs(size * m2 / low) * (off_low / low + 8 * U)
    return new, m2, v2, MORE * off, MORE * off_m, MORE * off_v


def dither(n, t, second, first=0):
    """20 bits for each of n places from `first` on at step t."""
    i = np.arange(first, first + n, dtype=np.uint64)
    low = np.uint64(0xffffffff)
    u = lambda v: np.uint64(v)
    with np.errstate(over="ignore"):
        x = (((i >> u(3)) & low) * u(0x9e3779b1) + (i >> u(35)) * u(0x6a09e667) + u(t) * u(0xbb67ae85)) & low
        x = ((x ^ (x >> u(16))) * u(0x6a09e667)) & low
        x = ((x ^ (x >> u(15))) * u(0xbb67ae85)) & low
        x = x ^ (x >> u(16))
        for k in range(16):
            x = np.where(u(2) * (i & u(7)) + u(int(second)) >= u(k), (x * u(1664525) + u(1013904223)) & low, x)
    return (x >> u(12)).astype(np.float64)


def held(x, t, top, square, first=0):
    """The values that fp32 moments x (float64 array) are held as at step t, and their blocks' exponents; the first of them at a multiple of 256."""
    n = len(x)
    out, exponents = np.empty(n), []
    u = dither(n, t, square, first)
    for a in range(0, n, 256):
        v, d = x[a:a + 256], u[a:a + 256]
        if not np.isfinite(v).all():
            out[a:a + 256] = np.nan
            exponents.append(255)
            continue
        e = max(int(np.float32(np.abs(v).max()).view(np.int32) >> 23), 33)
        exponents.append(e)
        size = np.abs(v)
        with np.errstate(divide="ignore"):
            binade = np.where(size > 0, np.frexp(size)[1] - 1 + 127, 0)
        field = np.maximum(binade - e + top, 1)
        unit = np.ldexp(1.0, field + e - top - 127 - 3)
        at = np.rint((size / unit + 8 * (field - 1)) * 2.0 ** 20)
        code = np.floor((at + d) / 2.0 ** 20)
        if square:
            code = np.where(size > 0, np.maximum(code, 1), code)
        field, mantissa = code // 8, code % 8
        value = np.where(field > 0, 8 + mantissa, mantissa) * np.ldexp(1.0, (np.maximum(field, 1) + e - top - 127 - 3).astype(int))
        out[a:a + 256] = np.copysign(value, v)
    return out, np.array(exponents, dtype=np.uint8)


def one_apart(n, a, eps):
    """Layer norm of a row of n values that are zero but for one, a, with the gradient that is zero but for one, 1, at the same place (weights one): h there and
    elsewhere, dx there and elsewhere."""
    mean, var = a / n, a * a * (n - 1) / n / n
    r = 1 / np.sqrt(var + eps)
    here, else_ = (a - mean) * r, -mean * r
    return here, else_, r * (1 - 1 / n - here * here / n), r * (-1 / n - else_ * here / n)
