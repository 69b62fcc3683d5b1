"""GPU: shared prefixes of the paged cache, where batches are wide and prefixes short, rows stay out of their group, values need more than 16 bits, and runs of pages are long.

Helpers and the tolerance for sharing are those of test_gpu_paged_views.py.
"""
import numpy as np
import pytest
import torch

import paged_plain as plain
from test_gpu_paged import DT, f32, ints, make, tokens
from test_gpu_paged_views import SHARED_TOL, close, grouped, query, shares

pytestmark = pytest.mark.gpu


def spoil_workspaces(cache):
    """What earlier calls left in the workspaces is NaN."""
    for held in cache._workspaces.values():
        for _, _, t in held:
            t.fill_(255)


WIDE = [
    # rows, query rows per kv head, kv heads, pages of the prefix: tiles of more than 128 query rows, whose pages are two steps each, and fewer than 296 steps
    (256, 1, 8, 6), (256, 1, 8, 10), (256, 1, 8, 15), (128, 2, 8, 12), (128, 2, 8, 14), (128, 2, 8, 16), (85, 3, 8, 17), (200, 1, 8, 8), (160, 1, 32, 4),
]


@pytest.mark.parametrize("rows, group, kvh, pages", WIDE)
@pytest.mark.parametrize("d, dt", [(128, "bf16"), (128, "fp16"), (64, "bf16"), (64, "fp16")])
def test_wide_batches_behind_short_prefixes(rows, group, kvh, pages, d, dt):
    """The merge reads what this call wrote, whatever stood in the workspace before."""
    residual = 64
    prompt = pages * 64 + residual
    cache, members, _ = grouped([(prompt, [0] * rows)], kvh, d, dt, residual, pages=64, max_length=2048)
    kids = members[0]
    q = query(rows, 1, group * kvh, d, dt, 11)
    o = ints(0, rows)
    want = cache.attend(0, q, rows=ints(*kids), out_dtype=torch.float32)
    cache.attend(0, q, rows=ints(*kids), groups=o, out_dtype=torch.float32)
    spoil_workspaces(cache)
    got = cache.attend(0, q, rows=ints(*kids), groups=o, out_dtype=torch.float32)
    cache.check()
    if d == 128:                                                   # at head_dim 64 the shortest of them do not pay
        assert shares(cache, q, kids, o) == [pages] * rows and not torch.equal(got, want)
    close(got, want.double().cpu().numpy(), SHARED_TOL)
    assert torch.equal(cache.attend(0, q, rows=ints(*kids), groups=o, out_dtype=torch.float32), got)


@pytest.mark.parametrize("live, pays", [(8, False), (16, False), (40, True)])
def test_whether_sharing_pays_is_a_matter_of_the_rows_that_share(live, pays):
    """A padded batch of 64 entries behind 101 pages: 8 or 16 live rows are attended as without groups, bit for bit; 40 share."""
    cache, members, _ = grouped([(101 * 64 + 64, [1 + i % 50 for i in range(64)])], 8, 128, "bf16", 64)
    kids = members[0]
    cache.lengths[torch.tensor(kids[live:], device="cuda")] = 0
    q = query(64, 1, 32, 128, "bf16", 12)
    want = cache.attend(0, q, rows=ints(*kids), out_dtype=torch.float32)
    got = cache.attend(0, q, rows=ints(*kids), groups=ints(0, 64), out_dtype=torch.float32)
    cache.check()
    assert torch.equal(got, want) != pays
    assert not got[live:].any()
    close(got, want.double().cpu().numpy(), SHARED_TOL)
