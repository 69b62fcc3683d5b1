"""GPU: the 16-bit window of the paged cache: what a query does not see, what is not finite, and its precision."""
import numpy as np
import pytest
import torch

import paged_plain as plain
from test_gpu_paged import DT, f32, ints, make, tokens

pytestmark = pytest.mark.gpu


def put(cache, k, v, row=0):
    o = ints(0, k.shape[0])
    cache.extend(rows=ints(row), offsets=o)
    cache.append(0, k.cuda(), v.cuda(), rows=ints(row), offsets=o)


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("group", [1, 2, 4, 5, 8, 16])
@pytest.mark.parametrize("lq, bad_from", [(2, 1), (3, 1), (3, 2), (5, 3)])
@pytest.mark.parametrize("bad", [float("nan"), float("-inf")])
def test_later_tokens_do_not_reach_earlier_queries(d, group, lq, bad_from, bad):
    """Of the lq newest tokens those from `bad_from` on have keys and values that are not finite: the queries before them are unaffected, however query
    tokens and heads are shared out in passes.  (Tolerance: that of the finite case.)"""
    n = 150
    cache = make(1, 1, d, "bf16", 128)
    k, v = tokens(n, 1, d, torch.bfloat16, 8)
    first = n - lq + bad_from
    good = (k[:first].clone(), v[:first].clone())
    k[first:], v[first:] = bad, bad
    put(cache, k, v)
    q = torch.randn(1, lq, group, d, generator=torch.Generator().manual_seed(group)).bfloat16().cuda()
    got = cache.attend(0, q, out_dtype=torch.float32)[0].double().cpu().numpy()
    want = plain.attention(f32(q[0, :bad_from].cpu()), *plain.held(f32(good[0]), f32(good[1]), 128), d ** -0.5)
    for j in range(bad_from):
        for h in range(group):
            assert np.linalg.norm(got[j, h] - want[j, h]) <= 3e-5 * np.linalg.norm(want[j, h]), (j, h)
    assert not np.isfinite(got[bad_from:]).any()


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n, lq, group", [(20, 1, 4), (150, 1, 8), (150, 3, 2), (40, 2, 8), (330, 1, 5)])
def test_infinite_values(dt, d, n, lq, group):
    """Values that are infinite in the window: a sum of positive multiples of them is that infinity, of both signs NaN, and a NaN is NaN; channels without any are
    what they are without them."""
    cache = make(1, 1, d, dt, 128)
    k, v = tokens(n, 1, d, DT[dt], 5)
    spoilt = v.clone()
    at = n - lq - 3                                               # every query sees it
    spoilt[at, 0, 3], spoilt[at - 1, 0, 7] = float("inf"), float("-inf")
    spoilt[at, 0, 9], spoilt[at - 2, 0, 9] = float("inf"), float("-inf")
    spoilt[at, 0, 11], spoilt[at, 0, d - 1] = float("nan"), float("inf")
    spoilt[at - 1, 0, d - 1] = float("inf")
    spoilt[n - 1, 0, 20] = float("inf")                           # the last query only sees this one
    put(cache, k, spoilt)
    q = torch.randn(1, lq, group, d, generator=torch.Generator().manual_seed(group)).to(DT[dt]).cuda()
    got = cache.attend(0, q, out_dtype=torch.float32)[0].cpu().numpy()
    kk, vv = plain.held(f32(k), f32(v), 128)
    want = plain.attention(f32(q[0].cpu()), kk, vv, d ** -0.5)
    inf = np.inf
    assert (got[..., 3] == inf).all() and (got[..., 7] == -inf).all() and (got[..., d - 1] == inf).all()
    assert np.isnan(got[..., 9]).all() and np.isnan(got[..., 11]).all() and (got[-1, :, 20] == inf).all()
    plain_channels = [c for c in range(d) if c not in (3, 7, 9, 11, d - 1, 20)]
    for j in range(lq):
        for h in range(group):
            x, y = got[j, h, plain_channels], want[j, h, plain_channels]
            assert np.linalg.norm(x - y) <= 3e-5 * np.linalg.norm(y), (j, h)
    if lq > 1:
        assert np.abs(got[:-1, :, 20] - want[:-1, :, 20]).max() <= 3e-5 * np.linalg.norm(want, axis=-1).max()


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("d", [64, 128])
def test_probabilities_have_the_precision_of_fp32(dt, d):
    """One token has the largest logit and no value, 90 others have the same smaller logit and the value 1: the output is 90 p / (1 + 90 p), so an error of p is not averaged
    away.  128 queries give 128 different p from 1/2 to 2^-16.  The logit is one exact product times the scale: at most 2^-24 of 11.1 in the product and in the factor to
    base 2, together 1.4e-6 (natural log units; the largest logit's own error is as large only where its size is, and it is chosen as zero here); the exponential 2^-22, sums
    and the quotient 2^-22: 1.9e-6 of the output in the worst case, 3e-6 is asked for."""
    n = 91
    cache = make(1, 1, d, dt, 128)
    k, v = torch.zeros(n, 1, d), torch.ones(n, 1, d)
    k[1:, 0, 0] = -1.0
    v[0] = 0.0
    put(cache, k.to(DT[dt]), v.to(DT[dt]))
    size = torch.linspace(0.6, 11.0, 128)
    errors = []
    for i in range(0, 128, 8):
        q = torch.zeros(1, 1, 8, d)
        q[0, 0, :, 0] = size[i:i + 8]
        q = q.to(DT[dt])
        got = cache.attend(0, q.cuda(), out_dtype=torch.float32, scaling=1.0)[0, 0].double().cpu().numpy()
        p = np.exp(-q[0, 0, :, 0].double().numpy())
        want = 90 * p / (1 + 90 * p)
        errors.append(got / want[:, None] - 1)
        assert np.abs(errors[-1]).max() <= 3e-6, (i, np.abs(errors[-1]).max())
    # in the mean square: a logit of up to 15.9 (base 2) rounds by up to 2^-21, 1.9e-7 of the exponential; the factor to base 2 adds 1.5e-7 and the exponential 1e-7
    assert np.square(errors).mean() ** 0.5 <= 5e-7, np.square(errors).mean() ** 0.5
