"""Plain forms, in 64 bits and on the CPU, of what the tests of packed rows and of lookups compare with."""
import numpy as np

D, GROUP, WORDS, KEY, HEAD = 172, 128, 24, 516, 528
EPS = 2.0 ** -24        # half a step of fp32
# the time encoding's cosine against 64 bits, over every float of every binade (csrc/common.cuh): the larger of its two forms
COS = 7.2e-7


def bf16_floor(x):
    """The largest bfloat16 that is not above x (float64 array of finite fp32 values)."""
    b = np.asarray(x, np.float32).view(np.uint32).astype(np.int64)
    down = np.where((b >> 31 == 1) & (b & 0xffff != 0), (b & 0xffff0000) + 0x10000, b & 0xffff0000)
    return down.astype(np.uint32)


def bf16_ceil_positive(x):
    """The smallest bfloat16 that is not below x >= 0 (float64)."""
    f = x.astype(np.float32)
    f = np.where(f.astype(np.float64) < x, np.nextafter(f, np.float32(np.inf)), f)
    b = f.view(np.uint32).astype(np.int64)
    return ((b + 0xffff) & 0xffff0000).astype(np.uint32)


def pack(x):
    """[m, 172] values (exact in fp32) -> words uint32 [m, 24]."""
    x = np.asarray(x, np.float64)
    words = np.zeros((len(x), WORDS), np.uint32)
    for g, c in enumerate((slice(0, GROUP), slice(GROUP, D))):
        v = x[:, c]
        with np.errstate(invalid="ignore"):
            fine = (np.abs(v) < 2.0 ** 126).all(1)
        v = np.where(fine[:, None], v, 0.0)
        off = bf16_floor(v.min(1))
        low = off.view(np.float32).astype(np.float64)
        step = bf16_ceil_positive((v.max(1) - low) / 15)
        s = step.view(np.float32).astype(np.float64)
        q = np.divide(v - low[:, None], s[:, None], out=np.zeros_like(v), where=s[:, None] > 0)
        code = np.rint(q).astype(np.uint32)
        words[:, g] = np.where(fine, off | (step >> 16), 0x7fc07fc0)
        code = np.where(fine[:, None], code, 0)
        at = np.arange(D)[c]
        for j, col in enumerate(at):
            words[:, 2 + col // 8] |= code[:, j].astype(np.uint32) << np.uint32(4 * (col % 8))
    return words


def unpack(words, exact=False):
    """words [.., 24] -> values, as they are held in fp32 (exact: offset + step * code in 64 bits)."""
    w = np.ascontiguousarray(words).view(np.uint32)
    col = np.arange(D)
    code = (w[..., 2 + col // 8] >> (4 * (col % 8)).astype(np.uint32)) & 15
    how = w[..., (col >= GROUP).astype(int)]
    step, off = (how << 16).view(np.float32).astype(np.float64), (how & 0xffff0000).view(np.float32).astype(np.float64)
    v = off + step * code
    return v if exact else v.astype(np.float32).astype(np.float64)


def attend(qt, rows, edges, w, nbr, eid, delta):
    """One row: the slots' values (float64 tables), the queries of two heads.  Returns ctx [1032] and a bound of the error
    of a computation in fp32 over the same values."""
    if len(nbr) == 0:
        return np.zeros(2 * KEY), 0.0
    angle = (delta.astype(np.float32)[:, None] * w.astype(np.float32)[None]).astype(np.float64)
    x = np.concatenate([rows[nbr], edges[eid], np.cos(angle)], 1)
    out, bound = np.zeros(2 * KEY), 0.0
    for h in range(2):
        q = qt[h * HEAD:h * HEAD + KEY].astype(np.float64)
        logit = x @ q
        p = np.exp(logit - logit.max())
        p /= p.sum()
        out[h * KEY:(h + 1) * KEY] = p @ x
        # A logit: at most 9 products of a pair in a row, both of the pair, five steps over the lanes and the value's own rounding:
        # 17 half steps of the sum of magnitudes; the cosine's error times the time part of the query.  A weight is off by twice a
        # logit's error, 4 half steps of the exponential and half a step of each of the logits' magnitudes (their difference).
        # A packed value is one fused multiplication and addition from its code: offset - 16 step is rounded (the offset is at most
        # the row's largest magnitude and 2^-7 of it, a step at most (2 + 2^-6) / 15 of it), and so is the value: 5 half steps of
        # the row's largest magnitude, also where the lowest and the highest code are missing.
        big = np.abs(x[:, :2 * D]).max(1) * np.abs(q[:2 * D]).sum()
        d = EPS * (17 * (np.abs(x) @ np.abs(q)) + 5 * big).max() + COS * np.abs(q[2 * D:]).sum()
        weight = 2 * d + EPS * (4 + 2 * np.abs(logit).max())
        # The weighted sum: a weight's error on numerator and total; a rounding a slot in both, two a rescaling step of the
        # running maximum; the value's rounding and the division.
        bound = max(bound, np.abs(x).max() * (2 * weight + EPS * (4 * len(nbr) + 16)) + COS)
    return out, bound


def lookup_grad(g, ids, n, scale, padding=None):
    """Gradient of a table in 64 bits, and the sum of magnitudes and the number of contributions of every row."""
    out, mag, cnt = np.zeros((n, g.shape[1])), np.zeros((n, g.shape[1])), np.zeros(n, np.int64)
    ok = (ids >= 0) & (ids < n)
    if padding is not None:
        ok &= ids != padding
    np.add.at(out, ids[ok], g[ok].astype(np.float64))
    np.add.at(mag, ids[ok], np.abs(g[ok].astype(np.float64)))
    np.add.at(cnt, ids[ok], 1)
    return out * scale, mag * abs(scale), cnt
