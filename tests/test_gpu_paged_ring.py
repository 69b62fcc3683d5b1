"""GPU: the 16-bit window of the paged cache: what a query does not see."""
import numpy as np
import pytest
import torch

import paged_plain as plain
from test_gpu_paged import f32, ints, make, tokens

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
