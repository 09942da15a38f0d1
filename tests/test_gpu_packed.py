"""Rows held in 4 bits on the GPU against plain forms in 64 bits (rows_reference.py).  What is held is equal bit for bit; attention is
within the bound that rows_reference.attend derives from the values at hand."""
import numpy as np
import pytest
import torch

import rows_reference as ref
from helpers import graph, state_dict

pytestmark = pytest.mark.gpu

D = 172
TYPES = {"float32": torch.float32, "bfloat16": torch.bfloat16, "float16": torch.float16}


@pytest.fixture(scope="module")
def dev():
    return torch.device("cuda:0")


def _u32(t):
    return t.cpu().numpy().view(np.uint32)


def _words(rs, n):
    """Random packed rows of moderate size; row 0 is zero."""
    w = rs.randint(0, 1 << 32, (n, ref.WORDS), dtype=np.uint64).astype(np.uint32)
    w[:, -1] &= 0xffff
    for g in range(2):
        step = ref.bf16_ceil_positive(rs.uniform(0.05, 0.4, n))
        off = ref.bf16_floor(rs.uniform(-3, 0.5, n).astype(np.float32))
        w[:, g] = off | (step >> 16)
    w[0] = 0
    return w


def _packed(dev, words):
    from orca_b200.packed import PackedRows
    return PackedRows.from_words(torch.from_numpy(words.view(np.int32)).to(dev))


def _time_w():
    return (1 / 10 ** np.linspace(0, 9, D)).astype(np.float32)


def _qt(rs, n, size=0.1):
    q = np.zeros((n, 2 * ref.HEAD), np.float32)
    for h in range(2):
        q[:, h * ref.HEAD:h * ref.HEAD + ref.KEY] = rs.randn(n, ref.KEY) * size
    q[:, ref.KEY:ref.HEAD] = np.nan            # (the columns between the heads are nobody's)
    q[:, ref.HEAD + ref.KEY:] = np.nan
    return q


# ------------------------------------------------------------------------------- push and pull
def _rows(rs, m, kind):
    x = rs.randn(m, D).astype(np.float32)
    if kind == "wide":
        x *= np.exp(rs.uniform(-60, 60, (m, 1))).astype(np.float32)
    elif kind == "shifted":
        x += (1000 * rs.randn(m, 1)).astype(np.float32)
    elif kind == "constant":
        x[:] = rs.randn(m, 1)
        x[::3] = 0
        x[1::3] = np.float32(1.5)
    elif kind == "grid":            # quotients that are borders between two codes
        x = rs.randint(0, 31, (m, D)).astype(np.float32) * 0.5
        x[:, 0], x[:, 1], x[:, 130], x[:, 131] = 0, 15, 0, 15
    elif kind == "tiny":
        x *= np.float32(1e-42)
    elif kind == "broken":
        x[0, 5], x[1, 140], x[2, 0], x[3, 171], x[4, 127], x[5, 128] = np.nan, np.nan, np.inf, -np.inf, 2.0 ** 126, -3e38
    return x


@pytest.mark.parametrize("kind", ["plain", "wide", "shifted", "constant", "grid", "tiny", "broken"])
@pytest.mark.parametrize("m", [1, 7, 1000])
def test_packing_is_the_format(dev, kind, m):
    from orca_b200.packed import PackedRows
    rs = np.random.RandomState(m)
    m = max(m, 6) if kind == "broken" else m
    x = _rows(rs, m, kind)
    p = PackedRows.of(torch.from_numpy(x).to(dev))
    want = ref.pack(x)
    assert np.array_equal(_u32(p.words), want)
    got = p.pull(torch.arange(m, device=dev)).cpu().numpy()
    assert np.array_equal(got, ref.unpack(want).astype(np.float32), equal_nan=True)
    # half a step at most, and half a step of fp32 of the value
    step = (want[:, :2] << 16).view(np.float32)
    off = np.abs(got.astype(np.float64) - x)
    half = np.where(np.arange(D) < ref.GROUP, step[:, :1], step[:, 1:]) / 2.0
    fine = np.isfinite(half)
    assert (off[fine] <= half[fine] + ref.EPS * np.abs(got[fine]) + 2.0 ** -149).all()
    p.check_status()


@pytest.mark.parametrize("kind", list(TYPES))
@pytest.mark.parametrize("m,n", [(1, 1), (33, 5), (600, 9228), (1024, 300), (1025, 300), (20001, 3000)])
def test_push_keeps_the_last_of_equal_ids(dev, kind, m, n):
    rs = np.random.RandomState(m)
    words = _words(rs, n)
    p = _packed(dev, words.copy())
    for turn in range(2):
        x = torch.from_numpy(rs.randn(m, D).astype(np.float32)).to(TYPES[kind])
        ids = rs.randint(0, n, m)
        p.push(x.to(dev), torch.from_numpy(ids).to(dev) if turn else ids)
        for i, row in zip(ids, ref.pack(x.float().numpy())):
            words[i] = row
        assert np.array_equal(_u32(p.words), words)
        assert int(p._record.abs().sum()) == 0
    p.check_status()


def test_push_takes_strides_and_other_types(dev):
    rs = np.random.RandomState(4)
    p = _packed(dev, _words(rs, 50))
    wide = torch.from_numpy(rs.randn(20, 2 * D + 3).astype(np.float32)).to(dev)
    ids = torch.from_numpy(rs.permutation(50)[:20]).to(dev)
    for x in (wide[:, 3:3 + D], wide[:, ::2][:, :D], wide[:, :D].double(), wide[:, :D].t().contiguous().t()):
        p.push(x, ids)
        assert np.array_equal(_u32(p.words)[ids.cpu().numpy()], ref.pack(x.float().cpu().numpy()))
    p.push(wide[:0, :D], ids[:0])
    assert p.pull([]).shape == (0, D)


def test_ids_outside_the_table(dev):
    from orca_b200._lib import OrcaError
    rs = np.random.RandomState(5)
    words = _words(rs, 40)
    p = _packed(dev, words.copy())
    x = rs.randn(4, D).astype(np.float32)
    p.push(torch.from_numpy(x).to(dev), torch.tensor([3, 40, -1, 1 << 40], device=dev))
    words[3] = ref.pack(x)[0]
    assert np.array_equal(_u32(p.words), words) and int(p._record.abs().sum()) == 0
    with pytest.raises(OrcaError):
        p.check_status()
    p.check_status()
    got = p.pull(torch.tensor([39, 40, -(1 << 40) + 3, 0], device=dev)).cpu().numpy()
    assert np.array_equal(got[0], ref.unpack(words[39]).astype(np.float32)) and not got[1:].any()
    with pytest.raises(OrcaError):
        p.check_status()
    for bad in ([40], [-1], np.array([0, 1 << 33])):
        with pytest.raises(OrcaError):
            p.pull(bad)


def test_push_replayed_from_a_graph(dev):
    """Other ids at every replay: nothing of one pass decides in the next."""
    rs = np.random.RandomState(6)
    words = _words(rs, 30)
    p = _packed(dev, words.copy())
    x = torch.zeros(64, D, device=dev)
    ids, pulled = torch.zeros(64, dtype=torch.int32, device=dev), torch.arange(30, dtype=torch.int32, device=dev)
    p.push(x[:1], ids[:1])                      # (makes the record)
    words[0] = 0
    side = torch.cuda.Stream()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g, stream=side):
        out = p.push_and_pull(x, ids, pulled)
    for _ in range(3):
        a, b = rs.randn(64, D).astype(np.float32), rs.randint(0, 30, 64).astype(np.int32)
        x.copy_(torch.from_numpy(a)), ids.copy_(torch.from_numpy(b))
        g.replay()
        for i, row in zip(b, ref.pack(a)):
            words[i] = row
        assert np.array_equal(_u32(p.words), words)
        assert np.array_equal(out.cpu().numpy(), ref.unpack(words).astype(np.float32))


def test_history_interface(dev):
    from orca_b200.packed import PackedHistory
    rs = np.random.RandomState(7)
    h = PackedHistory(60, D, dev, 10)
    assert not h.emb.any() and h.cache_flag.sum() == 0
    x = torch.from_numpy(rs.randn(12, D).astype(np.float32)).to(dev)
    ids = np.array([5, 6, 7, 5, 9, 59, 1, 2, 3, 4, 8, 5])
    got = h.push_and_pull(x, ids, [5, 59, 30])
    want = ref.unpack(ref.pack(x.cpu().numpy())).astype(np.float32)
    assert np.array_equal(got.cpu().numpy(), np.stack([want[11], want[5], np.zeros(D, np.float32)]))
    h.update_flag(np.array([3, 4]), None)
    assert h.cache_flag.nonzero()[0].tolist() == [3, 4]
    kept = h.emb.clone()
    h.reset_parameters()
    assert not h.emb.any()
    h.emb = kept                       # what is held already is held without a further error where its range is still spanned
    step = (_u32(h.rows.words)[:, :2] << 16).view(np.float32)
    assert float((h.emb - kept).abs().max()) <= step.max() / 2 * (1 + 2.0 ** -20)
    at = h.rows.words.data_ptr()
    h.emb = torch.ones(60, D, dtype=torch.float64)
    assert h.rows.words.data_ptr() == at and (h.emb == 1).all()       # (packed in place: graphs keep reading it)
    h.detach_history()
    h.check_status()


def test_first_push_in_a_capture_is_refused(dev):
    """What it makes would belong to the graph."""
    p = _packed(dev, _words(np.random.RandomState(30), 20))
    x, ids = torch.zeros(3, D, device=dev), torch.zeros(3, dtype=torch.int32, device=dev)
    keep = p.words.clone()
    with pytest.raises(RuntimeError, match="before capturing"):
        with torch.cuda.graph(torch.cuda.CUDAGraph()):
            out = p.pull(ids)
            p.push(x, ids)
    del out
    torch.cuda.synchronize()
    assert torch.equal(p.words, keep)
    p.push(x, ids)
    assert not p.pull(ids).any()


def test_offsets_past_32_bits(dev):
    """Rows, edges and slots that lie further than 2^32 bytes into their tables."""
    rs = np.random.RandomState(31)
    n, e = 46_000_000, 6_300_000
    from orca_b200.packed import PackedRows
    p, edges = PackedRows(n, dev), torch.empty(e, D, device=dev)
    ids = np.concatenate([n - 1 - np.arange(40), np.arange(1, 11)])
    x, ex = rs.randn(50, D).astype(np.float32), rs.randn(50, D).astype(np.float32)
    up = lambda a: torch.from_numpy(a).to(dev)
    p.push(up(x), ids)
    edges[e - 50:] = up(ex)
    held = ref.pack(x)
    assert np.array_equal(p.pull(ids).cpu().numpy(), ref.unpack(held).astype(np.float32))
    at, eat = rs.randint(0, 50, (30, 33)), rs.randint(0, 50, (30, 33))
    delta = rs.uniform(0, 1e6, (30, 33)).astype(np.float32)
    w, qt = _time_w(), _qt(rs, 30)
    ctx, valid = p.attend(up(qt), up(ids[at].astype(np.int32)), up((eat + e - 50).astype(np.int32)), up(delta), edges, up(w))
    rows64 = np.concatenate([np.zeros((1, D)), ref.unpack(held, True)])
    _check_tables(ctx, valid, qt, rows64, ex.astype(np.float64), w, at + 1, eat, delta)
    p.check_status()


# ------------------------------------------------------------------------------- attention over tables
def _tables(rs, rows, k, n, e, empty):
    nbr = np.where(rs.rand(rows, k) < empty, 0, rs.randint(1, n, (rows, k))).astype(np.int32)
    eid = np.where(nbr == 0, 0, rs.randint(0, e, (rows, k))).astype(np.int32)
    delta = np.exp(rs.uniform(0, 22, (rows, k))).astype(np.float32)       # up to 3.6e9: beyond the fixed-point cosine
    delta[rs.rand(rows, k) < 0.1] = 0
    return nbr, eid, delta


def _check_tables(got, valid, qt, rows64, edges64, w, nbr, eid, delta):
    got, valid = got.cpu().numpy().astype(np.float64), valid.cpu().numpy()
    for r in range(len(qt)):
        used = nbr[r] != 0
        want, bound = ref.attend(qt[r], rows64, edges64, w, nbr[r][used], eid[r][used], delta[r][used])
        assert valid[r] == used.any()
        assert np.abs(got[r] - want).max() <= bound, (r, np.abs(got[r] - want).max(), bound)


@pytest.mark.parametrize("edge", ["packed", "float32"])
@pytest.mark.parametrize("rows,k,empty", [(1, 1, 0.0), (1, 10, 0.0), (3, 10, 0.9), (5, 0, 0.0), (50, 10, 0.3), (301, 20, 0.1), (64, 32, 0.5),
                                          (40, 33, 0.0), (9, 64, 0.2), (2, 65, 0.0), (7, 129, 0.97), (3, 1000, 0.1), (1, 5003, 0.0),
                                          (4001, 4, 0.4), (20, 200, 1.0)])
def test_attend(dev, edge, rows, k, empty):
    rs = np.random.RandomState(rows * 7 + k)
    n, e = 90, 130
    words, w, qt = _words(rs, n), _time_w(), _qt(rs, rows)
    p = _packed(dev, words)
    if edge == "packed":
        ew = _words(rs, e)
        edges, edges64 = _packed(dev, ew), ref.unpack(ew, True)
    else:
        t = rs.randn(e, D).astype(np.float32)
        edges, edges64 = torch.from_numpy(t).to(dev), t.astype(np.float64)
    nbr, eid, delta = _tables(rs, rows, k, n, e, empty)
    up = lambda a: torch.from_numpy(a).to(dev)
    ctx, valid = p.attend(up(qt), up(nbr), up(eid), up(delta), edges, up(w))
    _check_tables(ctx, valid, qt, ref.unpack(words, True), edges64, w, nbr, eid, delta)
    again, _ = p.attend(up(qt), up(nbr), up(eid), up(delta), edges, up(w))
    assert torch.equal(ctx, again)
    p.check_status()


@pytest.mark.parametrize("size", [0.0, 1.0, 4.0])
def test_attend_logits_of_any_size(dev, size):
    rs = np.random.RandomState(11)
    words, ew, w, qt = _words(rs, 50), _words(rs, 60), _time_w(), _qt(rs, 30, size)
    nbr, eid, delta = _tables(rs, 30, 40, 50, 60, 0.2)
    up = lambda a: torch.from_numpy(a).to(dev)
    ctx, valid = _packed(dev, words).attend(up(qt), up(nbr), up(eid), up(delta), _packed(dev, ew), up(w))
    _check_tables(ctx, valid, qt, ref.unpack(words, True), ref.unpack(ew, True), w, nbr, eid, delta)


@pytest.mark.parametrize("k", [10, 300])
def test_values_that_are_not_numbers(dev, k):
    """In a row that no used slot names they change nothing; in one that is used, or in a query, they reach the result."""
    rs = np.random.RandomState(12)
    words, ew, w, qt = _words(rs, 50), _words(rs, 60), _time_w(), _qt(rs, 4)
    words[0], words[49], ew[0], ew[59] = 0x7fc07fc0, 0x7fc07fc0, 0x7fc07fc0, 0x7fc07fc0
    nbr, eid, delta = _tables(rs, 4, k, 49, 59, 0.2)
    eid[nbr != 0] = np.maximum(eid[nbr != 0], 1)
    nbr[0, -1], eid[1, 3], nbr[1, 3] = 49, 59, 4
    qt[2, 17] = np.nan
    delta[nbr == 0] = np.nan
    up = lambda a: torch.from_numpy(a).to(dev)
    ctx, valid = _packed(dev, words).attend(up(qt), up(nbr), up(eid), up(delta), _packed(dev, ew), up(w))
    got = ctx.cpu().numpy()
    assert np.isnan(got[0]).all() and np.isnan(got[1]).all()
    assert np.isnan(got[2][:ref.KEY]).all() and np.isfinite(got[2][ref.KEY:]).all()
    used = nbr[3] != 0
    want, bound = ref.attend(qt[3], np.nan_to_num(ref.unpack(words, True)), np.nan_to_num(ref.unpack(ew, True)), w, nbr[3][used], eid[3][used],
                             delta[3][used])
    assert np.abs(got[3] - want).max() <= bound and valid.all()


@pytest.mark.parametrize("k", [7, 200])
def test_logits_of_minus_infinity(dev, k):
    """Weights of zero, as the softmax has them; only where a row has no other slot is the result not a number."""
    rs = np.random.RandomState(13)
    words, ew, w = _words(rs, 50), np.zeros((3, ref.WORDS), np.uint32), np.zeros(D, np.float32)
    qt = _qt(rs, 2, 0.1)
    # column 0 of a row is 0 (times a query of minus infinity: not a number), so it is made 1 everywhere, -1 where a slot is to vanish
    rows = rs.randn(50, D).astype(np.float32)
    rows[:, 0], rows[25:, 0] = -1, 1
    words = ref.pack(rows)
    qt[:, [0, ref.HEAD]] = 0
    nbr = rs.randint(1, 25, (2, k)).astype(np.int32)
    nbr[0, ::2] = rs.randint(25, 50, len(nbr[0, ::2]))
    nbr[0, 0] = 25
    held = ref.unpack(words, True)
    up = lambda a: torch.from_numpy(a).to(dev)
    z = np.zeros((2, k), np.int32)
    p = _packed(dev, words)
    for q in (3e38, 1e37):         # the products of column 0 are +-q about, and the others vanish beside them
        big = qt.copy()
        big[:, [0, ref.HEAD]] = q
        ctx, _ = p.attend(up(big), up(nbr), up(z), up(z.astype(np.float32)), _packed(dev, ew), up(w))
        got = ctx.cpu().numpy().astype(np.float64)
        top = held[nbr[0], 0]
        want = held[nbr[0][top == top.max()]].mean(0)
        if q * top.max() > np.finfo(np.float32).max:      # (a logit of plus infinity: its softmax is not a number)
            assert np.isnan(got[0]).all()
        else:
            assert np.abs(got[0, :D] - want).max() <= 1e-5
    big[:, [0, ref.HEAD]] = -np.inf
    ctx, valid = p.attend(up(big[:1]), up(np.where(nbr[:1] >= 25, nbr[:1], 1)), up(z[:1]), up(z[:1].astype(np.float32)), _packed(dev, ew), up(w))
    assert np.isnan(ctx.cpu().numpy()).any() and valid.all()     # (plus infinity among them)
    only = np.where(nbr[:1] < 25, 25, nbr[:1]).astype(np.int32)   # column 0 positive everywhere: minus infinity in every slot
    ctx, valid = p.attend(up(big[:1]), up(only), up(z[:1]), up(z[:1].astype(np.float32)), _packed(dev, ew), up(w))
    assert np.isnan(ctx.cpu().numpy()).all() and valid.all()


@pytest.mark.parametrize("k", [3, 70])
def test_the_largest_values(dev, k):
    """Groups that span up to 2^127, beside ordinary ones: neighbours, edges and both.  Sums are formed before they are divided: three
    slots of one step have weights of 1 at most, so that they fit; seventy need not, and are infinite or NaN then."""
    rs = np.random.RandomState(29)
    words = _words(rs, 40)
    for g in range(2):
        step = ref.bf16_ceil_positive(rs.uniform(2.0 ** 118, 2.0 ** 123, 40))
        off = ref.bf16_floor((-rs.uniform(2.0 ** 120, 2.0 ** 126, 40)).astype(np.float32))
        words[20 + 10 * g:, g] = (off | (step >> 16))[20 + 10 * g:]
    p = _packed(dev, words)
    w, qt = _time_w(), _qt(rs, 12)
    for h in range(2):
        qt[:, h * ref.HEAD:h * ref.HEAD + 2 * D] *= np.float32(2.0 ** -122)
    nbr, eid = rs.randint(1, 40, (12, k)).astype(np.int32), rs.randint(1, 40, (12, k)).astype(np.int32)
    nbr[:4], eid[4:8] = nbr[:4] % 19 + 1, eid[4:8] % 19 + 1
    delta = rs.uniform(0, 100, (12, k)).astype(np.float32)
    up = lambda a: torch.from_numpy(a).to(dev)
    ctx, valid = p.attend(up(qt), up(nbr), up(eid), up(delta), p, up(w))
    assert valid.all()
    if k == 3:
        assert torch.isfinite(ctx).all()
        v = ref.unpack(words, True)
        _check_tables(ctx, valid, qt, v, v, w, nbr, eid, delta)
    p.check_status()


def test_slots_outside_the_tables(dev):
    from orca_b200._lib import OrcaError
    rs = np.random.RandomState(14)
    words, ew, w, qt = _words(rs, 50), _words(rs, 60), _time_w(), _qt(rs, 3)
    nbr, eid, delta = _tables(rs, 3, 12, 50, 60, 0.1)
    nbr[:, 0] = 5
    bad_nbr, bad_eid = nbr.copy(), eid.copy()
    bad_nbr[0, 4], bad_nbr[1, 5], bad_eid[2, 6] = 50, -7, 60
    bad_nbr[2, 6] = 3
    up = lambda a: torch.from_numpy(a).to(dev)
    p, e = _packed(dev, words), _packed(dev, ew)
    ctx, valid = p.attend(up(qt), up(bad_nbr), up(bad_eid), up(delta), e, up(w))
    with pytest.raises(OrcaError):
        p.check_status()
    nbr[0, 4] = nbr[1, 5] = nbr[2, 6] = 0
    _check_tables(ctx, valid, qt, ref.unpack(words, True), ref.unpack(ew, True), w, nbr, eid, delta)


@pytest.mark.parametrize("w", ["rising", "zero", "mixed"])
def test_other_time_weights(dev, w):
    """Not only the falling ones of the reference: any weights, arguments of any size."""
    rs = np.random.RandomState(15)
    tw = {"rising": _time_w()[::-1].copy(), "zero": np.zeros(D, np.float32),
          "mixed": (rs.randn(D) * 10.0 ** rs.uniform(-12, 3, D)).astype(np.float32)}[w]
    words, ew, qt = _words(rs, 50), _words(rs, 60), _qt(rs, 20)
    nbr, eid, delta = _tables(rs, 20, 12, 50, 60, 0.1)
    up = lambda a: torch.from_numpy(a).to(dev)
    ctx, valid = _packed(dev, words).attend(up(qt), up(nbr), up(eid), up(delta), _packed(dev, ew), up(tw))
    _check_tables(ctx, valid, qt, ref.unpack(words, True), ref.unpack(ew, True), tw, nbr, eid, delta)


def test_attend_is_the_gather_over_what_is_held(dev):
    """Against orca_attn_gather on the rows that the table stands for."""
    from orca_b200 import _lib
    rs = np.random.RandomState(16)
    words, w, qt = _words(rs, 200), _time_w(), np.nan_to_num(_qt(rs, 500))
    edges = rs.randn(300, D).astype(np.float32)
    nbr, eid, delta = _tables(rs, 500, 10, 200, 300, 0.2)
    nbr[:, 9] = np.maximum(nbr[:, 9], 1)
    up = lambda a: torch.from_numpy(a).to(dev)
    p = _packed(dev, words)
    d = [up(a) for a in (qt, nbr, eid, delta, edges, w)]
    ctx, valid = p.attend(*d)
    table = p.pull(torch.arange(200, device=dev))
    want, ok = torch.empty_like(ctx), torch.empty_like(valid)
    _lib.check(_lib.lib().orca_attn_gather(d[0].data_ptr(), table.data_ptr(), d[4].data_ptr(), d[5].data_ptr(), d[1].data_ptr(),
                                           d[2].data_ptr(), d[3].data_ptr(), 10, 500, None, want.data_ptr(), ok.data_ptr(), None,
                                           _lib.stream_ptr(dev)))
    assert torch.equal(valid, ok)
    assert float((ctx - want).abs().max()) < 1e-4      # (the tolerance of the gather kernel's own tests)


# ------------------------------------------------------------------------------- attention over lists
class Lists:
    """An adjacency made of given lengths; times with ties."""

    def __init__(self, rs, dev, lengths, n, e, span=2e8):
        self.n_nodes = len(lengths)
        self.ptr = np.concatenate([[0], np.cumsum(lengths)]).astype(np.int64)
        total = int(self.ptr[-1])
        self.ts = np.concatenate([np.sort(rs.randint(0, max(2, int(span) // 1000 if m > 50 else 6), m) * 1000.0) for m in lengths] + [np.zeros(0)])
        self.nbr = rs.randint(1, n, max(total, 1)).astype(np.int32)
        self.eid = rs.randint(0, e, max(total, 1)).astype(np.int32)
        up = lambda a: torch.from_numpy(a).to(dev)
        self.indptr, self.adj_nbr, self.adj_eid = up(self.ptr), up(self.nbr), up(self.eid)
        self.adj_ts = up(self.ts if total else np.zeros(1))

    def of(self, v, t, last):
        b = self.ptr[v]
        m = int(np.searchsorted(self.ts[b:self.ptr[v + 1]], t, side="left"))
        a = max(0, m - last) if last else 0
        delta = (t - self.ts[b + a:b + m].astype(np.float32).astype(np.float64)).astype(np.float32)
        return self.nbr[b + a:b + m], self.eid[b + a:b + m], delta


@pytest.mark.parametrize("edge", ["packed", "float32"])
@pytest.mark.parametrize("name,lengths,queries,last", [
    ("few", [0, 1, 5, 40], 9, None), ("one", [0, 17], 1, None), ("last", [0, 3, 64, 700, 12], 60, 10), ("parts", [0, 6400, 63, 64, 65, 1], 12, None),
    ("hub", [0, 60000, 10], 2, None), ("looked up together", [0, 40, 3, 130, 0, 2], 100, None),
    ("looked up alone", [0, 40, 3, 700, 0, 2], 129, 600), ("many", [0] + [int(v) for v in np.random.RandomState(1).lognormal(3, 1.3, 800)], 1500, None)])
def test_attend_lists(dev, edge, name, lengths, queries, last):
    rs = np.random.RandomState(len(lengths))
    n, e = 70, 110
    a = Lists(rs, dev, lengths, n, e)
    words, w, qt = _words(rs, n), _time_w(), _qt(rs, queries)
    nodes = rs.randint(0, len(lengths), queries).astype(np.int32)
    nodes[0] = 1
    times = rs.choice([2e8, 1e9, -1.0, 2000.0, 3000.0, 1e8], queries)
    times[0] = 3e8
    if edge == "packed":
        ew = _words(rs, e)
        edges, edges64 = _packed(dev, ew), ref.unpack(ew, True)
    else:
        t = rs.randn(e, D).astype(np.float32)
        edges, edges64 = torch.from_numpy(t).to(dev), t.astype(np.float64)
    p = _packed(dev, words)
    up = lambda x: torch.from_numpy(x).to(dev)
    ctx, valid = p.attend_lists(up(qt), a, up(nodes), up(times), edges, up(w), last=last)
    got, rows64 = ctx.cpu().numpy().astype(np.float64), ref.unpack(words, True)
    for r in range(queries):
        slots = a.of(nodes[r], times[r], last)
        want, bound = ref.attend(qt[r], rows64, edges64, w, *slots)
        assert valid[r].item() == (len(slots[0]) > 0)
        assert np.abs(got[r] - want).max() <= bound, (r, len(slots[0]), np.abs(got[r] - want).max(), bound)
        if len(slots[0]) > 1000:       # (long sums: the bound above counts a rounding a slot; what is reached is far below)
            assert np.linalg.norm(got[r] - want) <= 1e-5 * np.linalg.norm(want)
    again, _ = p.attend_lists(up(qt), a, nodes, times, edges, up(w), last=last)       # (from host arrays)
    assert torch.equal(ctx, again)
    p.check_status()


def test_lists_of_nodes_that_the_graph_does_not_have(dev):
    from orca_b200._lib import OrcaError
    rs = np.random.RandomState(21)
    a = Lists(rs, dev, [0, 9], 30, 30)
    p, e, w, qt = _packed(dev, _words(rs, 30)), _packed(dev, _words(rs, 30)), torch.from_numpy(_time_w()).to(dev), _qt(rs, 3)
    ctx, valid = p.attend_lists(torch.from_numpy(qt).to(dev), a, torch.tensor([2, 1, -5], device=dev), torch.full((3,), 1e9, device=dev), e, w)
    assert valid.tolist() == [0, 1, 0] and not ctx[0].any() and not ctx[2].any() and ctx[1].any()
    with pytest.raises(OrcaError):
        p.check_status()
    with pytest.raises(OrcaError):
        p.attend_lists(torch.from_numpy(qt).to(dev), a, [2, 1, 0], [0.0] * 3, e, w)


def test_what_attention_refuses(dev):
    from orca_b200 import _lib
    rs = np.random.RandomState(20)
    a = Lists(rs, dev, [0, 9], 30, 30)
    p, e, w = _packed(dev, _words(rs, 30)), _packed(dev, _words(rs, 30)), torch.from_numpy(_time_w()).to(dev)
    qt, nodes, times = torch.from_numpy(_qt(rs, 3)).to(dev), torch.ones(3, dtype=torch.int32, device=dev), torch.full((3,), 1e9, device=dev)
    nbr = torch.ones(3, 4, dtype=torch.int32, device=dev)
    delta, edges = torch.ones(3, 4, device=dev), torch.zeros(30, D, device=dev)
    good = dict(qt=qt, nbr=nbr, eid=nbr, delta=delta, edges=e, time_w=w)
    p.attend(**good)
    p.attend(**{**good, "edges": edges, "nbr": nbr.t().contiguous().t(), "delta": delta[:, :1].expand(3, 4)})
    for bad in [dict(qt=qt.double()), dict(qt=qt[:, :1032]), dict(qt=qt.cpu()), dict(qt=qt[:, 1:]), dict(nbr=nbr[:2]), dict(nbr=nbr.long()),
                dict(eid=nbr[:, :3]), dict(delta=delta.double()), dict(delta=delta.cpu()), dict(edges=edges[:0]), dict(edges=edges.half()),
                dict(edges=edges[:, :171]), dict(edges=edges.t()), dict(edges=e.words), dict(edges=None), dict(time_w=w[:171]), dict(time_w=w.double())]:
        with pytest.raises(ValueError):
            p.attend(**{**good, **bad})
    with pytest.raises(NotImplementedError):
        p.attend(**{**good, "qt": qt.clone().requires_grad_(True)})
    good = dict(qt=qt, finder=a, nodes=nodes, timestamps=times, edges=e, time_w=w)
    p.attend_lists(**good, last=2)
    for bad in [dict(nodes=nodes[:2]), dict(timestamps=times[:2]), dict(last=0), dict(last=-3), dict(edges=edges.bfloat16()), dict(time_w=w[:, None])]:
        with pytest.raises(ValueError):
            p.attend_lists(**{**good, **bad})
    for bad in (nodes.short(), nodes.float()):
        with pytest.raises(TypeError):
            p.attend_lists(**{**good, "nodes": bad})
    with pytest.raises(_lib.OrcaError):               # (what the library itself refuses)
        _lib.rows().attend_lists(p.words, p.status, qt, e.words, w, a.indptr, a.adj_nbr, a.adj_eid, a.adj_ts, 2, nodes, times.double(), -1)
    with pytest.raises(ValueError):
        p.push(torch.zeros(3, D, device=dev), [1, 2])
    for bad in (torch.zeros(3, 171, device=dev), torch.zeros(D, device=dev), [[0.0] * D]):
        with pytest.raises(ValueError):
            p.push(bad, [1, 2, 3])
    p.push(torch.zeros(0, D, device=dev), [])
    assert p.pull([]).shape == (0, D)
    p.check_status()


def test_no_queries(dev):
    rs = np.random.RandomState(22)
    a = Lists(rs, dev, [0, 9], 30, 30)
    p, e, w = _packed(dev, _words(rs, 30)), _packed(dev, _words(rs, 30)), torch.from_numpy(_time_w()).to(dev)
    qt = torch.zeros(0, 2 * ref.HEAD, device=dev)
    none = torch.zeros(0, 10, dtype=torch.int32, device=dev)
    assert p.attend(qt, none, none, none.float(), e, w)[0].shape == (0, 1032)
    assert p.attend_lists(qt, a, [], [], e, w)[1].shape == (0,)


# ------------------------------------------------------------------------------- streams and graphs
def test_two_streams_and_a_graph(dev):
    """Two calls at once on streams of their own, and a captured pair of calls replayed with other inputs."""
    rs = np.random.RandomState(23)
    a = Lists(rs, dev, [0, 5000, 30, 700], 70, 110)
    words, ew, w = _words(rs, 70), _words(rs, 110), _time_w()
    p, e, tw = _packed(dev, words), _packed(dev, ew), torch.from_numpy(w).to(dev)
    up = lambda x: torch.from_numpy(x).to(dev)
    nodes, times = up(rs.randint(1, 4, 40).astype(np.int32)), up(np.full(40, 1e9))
    qs = [up(_qt(rs, 40)) for _ in range(4)]
    nbr, eid, delta = (up(x) for x in _tables(rs, 40, 300, 70, 110, 0.1))
    want = [(p.attend_lists(q, a, nodes, times, e, tw), p.attend(q, nbr, eid, delta, e, tw)) for q in qs]
    torch.cuda.synchronize()
    streams = [torch.cuda.Stream() for _ in range(2)]
    got = [None, None]
    for turn in range(10):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                got[i] = (p.attend_lists(qs[i], a, nodes, times, e, tw), p.attend(qs[i], nbr, eid, delta, e, tw))
    torch.cuda.synchronize()
    for g, v in zip(got, want):
        assert all(torch.equal(x, y) for x, y in zip((*g[0], *g[1]), (*v[0], *v[1])))
    q = qs[0].clone()
    g = torch.cuda.CUDAGraph()
    with torch.cuda.graph(g):
        out = (p.attend_lists(q, a, nodes, times, e, tw), p.attend(q, nbr, eid, delta, e, tw))
    for i in (2, 3, 0):
        q.copy_(qs[i])
        g.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(x, y) for x, y in zip((*out[0], *out[1]), (*want[i][0], *want[i][1])))


def test_calls_from_threads(dev):
    """Calls from two threads at once, each on a stream of its own."""
    import threading
    rs = np.random.RandomState(32)
    a = Lists(rs, dev, [0, 900, 30, 70], 70, 110)
    p, e, tw = _packed(dev, _words(rs, 70)), _packed(dev, _words(rs, 110)), torch.from_numpy(_time_w()).to(dev)
    nodes, times = rs.randint(1, 4, 20), np.full(20, 1e9)
    qs = [torch.from_numpy(_qt(rs, 20)).to(dev) for _ in range(2)]
    want = [p.attend_lists(q, a, nodes, times, e, tw)[0] for q in qs]
    torch.cuda.synchronize()
    wrong = []

    def work(i):
        with torch.cuda.stream(torch.cuda.Stream()):
            for _ in range(50):
                if not torch.equal(p.attend_lists(qs[i], a, nodes, times, e, tw)[0], want[i]):
                    wrong.append(i)

    threads = [threading.Thread(target=work, args=(i,)) for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not wrong


# ------------------------------------------------------------------------------- together, in the model
def test_the_models_batches_refuse_a_history_in_4_bits(dev):
    """They would read and write the copy that its `emb` is."""
    from orca_b200.packed import PackedHistory
    from test_gpu_model import make_model
    g = graph("t_nb2")
    tgn = make_model(g)
    call = lambda: tgn.compute_edge_probabilities(g.sources[:20], g.destinations[:20], g.destinations[:20], g.timestamps[:20],
                                                  g.edge_idxs[:20], g.spec.n_degree, False, False, None)
    fp32 = tgn.embedding_module.histories[0]
    for before in (False, True):               # (whether the model has described itself to the library already)
        tgn.embedding_module.histories[0] = PackedHistory(g.n_nodes, D, dev)
        with pytest.raises(TypeError):
            call()
        tgn.embedding_module.histories[0] = fp32
        call()


def test_embeddings_of_the_model_over_a_packed_history(dev):
    """TGN.packed_embeddings against the oracle's attention layer on the rows that the history stands for."""
    from oracle import tgn_oracle
    from orca_b200.packed import PackedHistory, PackedRows
    from test_gpu_model import make_model
    g = graph("t_nb2")
    tgn = make_model(g)
    rs = np.random.RandomState(24)
    h = PackedHistory(g.n_nodes, D, dev)
    table = rs.randn(g.n_nodes, D).astype(np.float32)
    table[0] = 0
    h.push(torch.from_numpy(table).to(dev), np.arange(g.n_nodes))
    held = ref.unpack(ref.pack(table))
    nodes, times = g.sources[-300:], g.timestamps[-300:]
    nodes = np.concatenate([nodes, [g.n_nodes - 1]])
    times = np.concatenate([times, [0.0]])                       # (before everything: no slots)
    p = {k: torch.from_numpy(v) for k, v in state_dict(2).items()}
    adj = tgn_oracle.Adjacency(g.sources, g.destinations, g.edge_idxs, g.timestamps, g.n_nodes)
    edge_rows = PackedRows.of(tgn.edge_raw_features)
    for k, edges in ((10, None), (None, edge_rows)):
        got = tgn.packed_embeddings(h, nodes, times, k, edges).cpu().numpy()
        width = k or int(max(len(adj.nbr[adj.indptr[v]:adj.indptr[v + 1]]) for v in set(nodes.tolist())))
        nbr, eid, et = tgn_oracle.sample_neighbors(adj, nodes, times, width)
        ef = g.edge_features if edges is None else ref.unpack(_u32(edge_rows.words))
        dt = torch.from_numpy((times[:, None] - et).astype(np.float32))
        want = tgn_oracle.attention_layer(p, 1, torch.from_numpy(held[nodes]).float(), torch.from_numpy(held[nbr]).float(),
                                          torch.from_numpy(np.asarray(ef)[eid]).float(), dt, torch.from_numpy(nbr)).numpy()
        rel = np.abs(got - want) / np.maximum(np.abs(want), 0.05)
        assert rel.max() < 1e-3           # (the tolerance of the projections' own tests)
    h.check_status()


def test_train_pack_attend(dev):
    """A run as it would be used: rows of a table are trained by lookups, packed, pulled and attended over."""
    from orca_b200.lookup import lookup_rows
    from orca_b200.packed import PackedRows
    rs = np.random.RandomState(25)
    table = torch.from_numpy((0.1 * rs.randn(80, D)).astype(np.float32)).to(dev).requires_grad_(True)
    ids = torch.from_numpy(rs.randint(0, 80, 500)).to(dev)
    goal = torch.from_numpy(rs.randn(500, D).astype(np.float32)).to(dev)
    start = table.detach().cpu().numpy().astype(np.float64)
    rows = lookup_rows(table, ids, scale=2.0, padding=0)
    ((rows - goal) ** 2).sum().backward()
    want, mag, cnt = ref.lookup_grad((2 * (2 * start[ids.cpu().numpy()] - goal.cpu().numpy())), ids.cpu().numpy(), 80, 2.0, 0)
    # each contribution is off by 3 roundings, each of cnt additions and the scale by one
    assert (np.abs(table.grad.cpu().numpy() - want) <= ref.EPS * (cnt[:, None] + 6) * mag + 1e-30).all()
    with torch.no_grad():
        table -= 0.01 * table.grad
    p = PackedRows.of(table)
    held = ref.pack(table.detach().cpu().numpy())
    assert np.array_equal(_u32(p.words), held)
    w, qt, ew = _time_w(), _qt(rs, 30), _words(rs, 60)
    nbr, eid, delta = _tables(rs, 30, 10, 80, 60, 0.2)
    up = lambda a: torch.from_numpy(a).to(dev)
    ctx, valid = p.attend(up(qt), up(nbr), up(eid), up(delta), _packed(dev, ew), up(w))
    _check_tables(ctx, valid, qt, ref.unpack(held, True), ref.unpack(ew, True), w, nbr, eid, delta)
