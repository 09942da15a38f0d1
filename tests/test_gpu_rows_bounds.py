"""Long sums against bounds that follow the order in which they are formed, so that a part that is left out shows."""
import numpy as np
import pytest
import torch

import rows_reference as ref
from test_gpu_packed import _check_tables, _packed, _qt, _time_w, _words

pytestmark = pytest.mark.gpu

CHUNK, WARPS, FEW, FEW_WAYS = 32, 8, 2048, 4


def _depth(n, cnt):
    """Additions that a contribution goes through on its way into its row's sum, of cnt of n ids.  Few ids: four sums of every fourth
    contribution, then three additions.  Else 32 of a chunk one after the other; the chunks' sums one after the other, up to 16 of them, or
    by eight warps in turn, whose sums are then added one after the other."""
    if n <= FEW:
        return -(-cnt // FEW_WAYS) + FEW_WAYS - 1
    parts = cnt // CHUNK + 2
    return CHUNK + np.where(parts <= 16, 16, -(-parts // WARPS) + WARPS - 1)


@pytest.mark.parametrize("dtype", [torch.float32, torch.bfloat16], ids=str)
@pytest.mark.parametrize("m,n,width,skew", [(66001, 3, 5, 0), (20011, 50, 172, 4), (9000, 12, 172, 0), (2048, 7, 172, 0), (600, 2, 33, 0),
                                            (2049, 5, 172, 0), (40000, 400, 60, 9)])
def test_gradients_of_hubs(m, n, width, skew, dtype):
    """An error of depth * 2^-24 of the sum of magnitudes, the scale's rounding and the type's.  Of 66 001 contributions to one row: 0.7 (fp32) for a
    sum of about 260; a chunk's sum is about 6."""
    from orca_b200.lookup import lookup_grad
    rs = np.random.RandomState(m)
    ids = np.full(m, n - 1) if skew == 0 else (rs.rand(m) ** skew * n).astype(np.int64)
    g = torch.from_numpy(rs.randn(m, width).astype(np.float32)).to(dtype)
    want, mag, cnt = ref.lookup_grad(g.double().numpy(), ids, n, 0.75)
    got = lookup_grad(g.cuda(), torch.from_numpy(ids).cuda(), n, 0.75).double().cpu().numpy()
    half = torch.finfo(dtype).eps / 2
    bound = ref.EPS * (_depth(m, cnt)[:, None] + 1) * (1 + 2.0 ** -7) * mag + half * np.abs(want)
    assert (np.abs(got - want) <= bound).all()


@pytest.mark.parametrize("rows,k", [(12, 70), (3, 300), (100, 300), (1, 2000)])
def test_large_values_over_many_steps_and_parts(rows, k):
    """Groups that span 2^107 / (k / 300) beside ordinary ones: 2^12 of them times k is below 2^128, so that every sum fits, over
    several stages of a row and over parts that are joined."""
    dev = torch.device("cuda:0")
    rs = np.random.RandomState(rows + k)
    low = 2.0 ** (20 + max(0, np.ceil(np.log2(k / 300))))
    words = _words(rs, 40)
    for g in range(2):
        step = ref.bf16_ceil_positive(rs.uniform(2.0 ** 118, 2.0 ** 123, 40) / low)
        off = ref.bf16_floor((-rs.uniform(2.0 ** 120, 2.0 ** 126, 40) / low).astype(np.float32))
        words[20 + 10 * g:, g] = (off | (step >> 16))[20 + 10 * g:]
    p, w, qt = _packed(dev, words), _time_w(), _qt(rs, rows)
    for h in range(2):
        qt[:, h * ref.HEAD:h * ref.HEAD + 2 * 172] *= np.float32(2.0 ** -127 * low)
    nbr, eid = rs.randint(1, 40, (rows, k)).astype(np.int32), rs.randint(1, 40, (rows, k)).astype(np.int32)
    delta = rs.uniform(0, 100, (rows, k)).astype(np.float32)
    up = lambda a: torch.from_numpy(a).to(dev)
    ctx, valid = p.attend(up(qt), up(nbr), up(eid), up(delta), p, up(w))
    assert bool(valid.all()) and bool(torch.isfinite(ctx).all())
    v = ref.unpack(words, True)
    _check_tables(ctx, valid, qt, v, v, w, nbr, eid, delta)
    # columns of the time encoding stand beside values 2^100 as large: by themselves, as weighted sums of cosines
    got = ctx.cpu().numpy().astype(np.float64)
    for r in range(rows):
        x = np.concatenate([v[nbr[r]], v[eid[r]], np.cos((delta[r][:, None] * w[None]).astype(np.float64))], 1)
        for h in range(2):
            q = qt[r, h * ref.HEAD:h * ref.HEAD + ref.KEY].astype(np.float64)
            logit = x @ q
            weights = np.exp(logit - logit.max())
            want = weights / weights.sum() @ x[:, 344:]
            # (rows_reference.attend's bound of a weight, times columns of at most 1)
            big = np.abs(x[:, :344]).max(1) * np.abs(q[:344]).sum()
            d = ref.EPS * (17 * (np.abs(x) @ np.abs(q)) + 5 * big).max() + ref.COS * np.abs(q[344:]).sum()
            bound = 2 * (2 * d + ref.EPS * (4 + 2 * np.abs(logit).max())) + ref.EPS * (4 * k + 16) + ref.COS
            assert np.abs(got[r, h * ref.KEY + 344:(h + 1) * ref.KEY] - want).max() <= bound
