"""GPU: attention of the paged cache over windows with sinks and over prefixes that rows share, against 64-bit attention.

Tolerances, before any run.  A window goes through the kernels of ordinary attention: 3e-5 of the output's norm (as in test_gpu_paged.py).  Shared prefixes, fp32 output: P is a f16
number of at least 2^-14 of the row's largest wherever it matters, rounded by 2^-12 of itself, and so is every value; both roundings are independent from token to token, so their sum is at most
2^-12 of sqrt(sum p^2 v^2) each in the root mean square.  That is what the output's norm itself is made of where tokens' values are independent, and the output is no smaller; twice
2^-12 * sqrt(2) allows for the spread of 128 channels: 7e-4.  Keys have 22 bits, logits of up to 30 then 30 * 2^-22 = 7e-6, and sums in the tensor cores (truncated) 2^-23 times 4 per page: below
5e-4 of what is allowed.  16-bit output is the fp32 output rounded once.
"""
import numpy as np
import pytest
import torch

import paged_plain as plain
from test_gpu_paged import DT, f32, fill, ints, make, tokens

pytestmark = pytest.mark.gpu
TOL, SHARED_TOL = 3e-5, 7e-4


def windowed(q, k, v, scaling, window, sinks):
    """q [l, H, D]: the newest l of k's, v's n tokens -> [l, H, D] in 64 bits"""
    lq, hq, d = q.shape
    n, kvh = k.shape[:2]
    out = np.zeros((lq, hq, d))
    for j in range(lq):
        pos = n - lq + j
        if pos < 0:
            continue
        seen = [t for t in range(pos + 1) if t > pos - window or t < sinks]
        for h in range(hq):
            s = k[seen, h // (hq // kvh)] @ q[j, h].astype(np.float64) * scaling
            w = np.exp(s - s.max())
            out[j, h] = (w / w.sum()) @ v[seen, h // (hq // kvh)]
    return out


def query(b, lq, hq, d, dt, seed):
    return torch.randn(b, lq, hq, d, generator=torch.Generator().manual_seed(seed)).to(DT[dt]).cuda()


def close(got, want, tol):
    g = got.double().cpu().numpy()
    assert g.shape == want.shape
    for at in np.ndindex(*want.shape[:-1]):
        size = np.linalg.norm(want[at])
        if size == 0:
            assert not g[at].any(), at
        else:
            err = np.linalg.norm(g[at] - want[at])
            assert err <= tol * size, (at, err / size)


# ---- windows

WINDOWS = [
    # head_dim, type, kv heads, query heads, residual, query tokens, lengths, window, sinks
    (128, "bf16", 2, 8, 128, 1, [0, 1, 63, 64, 128, 192, 193, 700], 1, 0),
    (128, "bf16", 2, 8, 128, 1, [0, 1, 63, 64, 128, 192, 193, 700], 100, 4),
    (128, "fp16", 1, 8, 64, 1, [64, 127, 128, 129, 1000], 64, 64),
    (128, "bf16", 2, 2, 0, 1, [1, 63, 64, 65, 128, 192, 640], 65, 1),
    (64, "bf16", 2, 8, 128, 1, [1, 192, 320, 777], 300, 130),
    (64, "fp16", 3, 3, 0, 2, [0, 1, 2, 64, 65, 130, 400], 63, 3),
    (128, "bf16", 1, 5, 128, 3, [1, 2, 3, 195, 400, 900], 130, 200),
    (64, "bf16", 1, 4, 0, 5, [3, 64, 66, 68, 130, 333], 2, 0),
    (128, "bf16", 1, 3, 192, 9, [5, 256, 600], 4, 5),
    (128, "fp16", 2, 32, 64, 1, [130, 515], 1 << 30, 0),
    (128, "bf16", 1, 4, 64, 70, [30, 71, 500], 50, 9),
]


@pytest.mark.parametrize("d, dt, kvh, hq, residual, lq, lengths, window, sinks", WINDOWS)
def test_window(d, dt, kvh, hq, residual, lq, lengths, window, sinks):
    cache = make(len(lengths), kvh, d, dt, residual)
    kv = fill(cache, lengths, 2, seed=d + hq)
    q = query(len(lengths), lq, hq, d, dt, 5)
    order = list(range(len(lengths)))[::-1]
    got = cache.attend(0, q, rows=ints(*order), window=window, sinks=sinks, out_dtype=torch.float32)
    cache.check()
    assert torch.equal(cache.attend(0, q, rows=ints(*order), window=window, sinks=sinks), got.to(DT[dt]))
    for i, r in enumerate(order):
        k, v = plain.held(f32(kv[r][0]), f32(kv[r][1]), residual)
        close(got[i], windowed(f32(q[i].cpu()), k, v, d ** -0.5, window, sinks), TOL)


def test_a_window_that_reaches_everything_is_ordinary_attention():
    cache = make(3, 2, 128, "bf16", 128)
    fill(cache, [10, 500, 900], 1)
    q = query(3, 2, 8, 128, "bf16", 1)
    whole = cache.attend(0, q, out_dtype=torch.float32)
    for window, sinks in ((900, 0), (2 ** 31 - 1, 0), (2 ** 40, 2 ** 40), (1, 900), (300, 700)):
        assert torch.equal(cache.attend(0, q, window=window, sinks=sinks, out_dtype=torch.float32), whole), (window, sinks)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
@pytest.mark.parametrize("lq", [1, 3])
def test_tokens_behind_the_window_do_not_reach_it(bad, lq):
    """In the ring, a token that is not finite and that no query, or not every query, sees: who does not see it is unaffected."""
    n, d, window, sinks = 150, 128, 40, 2
    cache = make(1, 1, d, "bf16", 128)
    k, v = tokens(n, 1, d, torch.bfloat16, 8)
    good = plain.held(f32(k), f32(v), 128)
    at = [n - lq - window, 5, sinks] + ([n - lq + 1 - window] if lq > 1 else [])      # out of everyone's sight; and out of the later queries'
    k[at], v[at] = bad, bad
    o = ints(0, n)
    cache.extend(offsets=o)
    cache.append(0, k.cuda(), v.cuda(), offsets=o)
    q = query(1, lq, 4, d, "bf16", 1)
    got = cache.attend(0, q, window=window, sinks=sinks, out_dtype=torch.float32)[0]
    want = windowed(f32(q[0].cpu()), *good, d ** -0.5, window, sinks)
    if lq == 1:
        close(got, want, TOL)
    else:
        assert not torch.isfinite(got[0]).any()
        close(got[1:], want[1:], TOL)


def test_pages_behind_the_window_are_not_read():
    """Their table entries may be gone (a program that frees them): no error, the same output."""
    cache = make(1, 2, 128, "bf16", 64)
    fill(cache, [1000], 1)
    q = query(1, 1, 8, 128, "bf16", 1)
    want = cache.attend(0, q, window=200, sinks=70, out_dtype=torch.float32)
    cache.block_table[0, 2:12] = -1               # tokens 128 .. 767; the window begins at 800
    assert torch.equal(cache.attend(0, q, window=200, sinks=70, out_dtype=torch.float32), want)
    cache.check()
    cache.attend(0, q, window=400, sinks=70)
    with pytest.raises(Exception, match="outside the cache"):
        cache.check()


# ---- shared prefixes

def grouped(groups, kvh, d, dt, residual, pages=1024, max_length=8192):
    """A cache whose rows were forked from prompts: groups [(prompt tokens, [own tokens, ...]), ...].  Returns it, the rows of each group, and every row's keys and values."""
    rows = sum(1 + len(own) for _, own in groups)
    cache = make(rows, kvh, d, dt, residual, max_length=max_length, pages=pages)
    members, kv, at = [], {}, 0
    for g, (prompt, own) in enumerate(groups):
        home, kids = at, list(range(at + 1, at + 1 + len(own)))
        at += 1 + len(own)
        pk, pv = tokens(prompt, kvh, d, DT[dt], 100 + g)
        o = ints(0, prompt)
        cache.extend(rows=ints(home), offsets=o)
        cache.append(0, pk.cuda(), pv.cuda(), rows=ints(home), offsets=o)
        cache.fork(ints(*[home] * len(kids)), ints(*kids))
        new = [tokens(n, kvh, d, DT[dt], 1000 * g + i) for i, n in enumerate(own)]
        o = ints(0, *np.cumsum(own).tolist())
        cache.extend(rows=ints(*kids), offsets=o)
        if sum(own):
            cache.append(0, torch.cat([x[0] for x in new]).cuda(), torch.cat([x[1] for x in new]).cuda(), rows=ints(*kids), offsets=o)
        for r, (k, v) in zip(kids, new):
            kv[r] = torch.cat([pk, k]), torch.cat([pv, v])
        members.append(kids)
    cache.check()
    return cache, members, kv


def shares(cache, q, order, groups):
    """Whether a call of this shape shares anything, as the kernels left it in the workspace: pages taken care of, by list entry."""
    import ctypes
    from muzero_b200.kernels._cabi import PagedView, stream_ptr
    view = PagedView(0, 0, groups.data_ptr(), groups.shape[0] - 1)
    lib = cache._lib
    head = lib.mz_paged_attention_workspace_bytes(cache._ref, q.shape[0], q.shape[1], q.shape[2])
    whole = lib.mz_paged_attention_view_workspace_bytes(cache._ref, ctypes.byref(view), q.shape[0], q.shape[1], q.shape[2])
    if whole == head:
        return None
    at = -(-head // 128) * 128
    ws = cache._workspaces[stream_ptr(cache.device)][-1][2]
    torch.cuda.synchronize()
    return ws[at:at + 4 * q.shape[0]].view(torch.int32).tolist()


GROUPS = [
    # head_dim, type, kv heads, query heads, residual, query tokens, groups of (prompt, own tokens), pages that are shared (None: too little for the host)
    (128, "bf16", 8, 32, 128, 1, [(3500, [0, 1, 5, 64, 65, 100, 130, 300] * 8)], True),          # two tiles of 128 rows
    (128, "fp16", 8, 64, 64, 1, [(2000, [3, 70, 9, 200] * 4), (700, [0, 0, 0, 0] * 3), (1500, [17] * 10)], True),
    (64, "bf16", 8, 32, 128, 4, [(4000, [4, 5, 100, 33] * 4)], True),                             # query tokens of their own
    (64, "fp16", 4, 20, 0, 3, [(3100, [3, 4, 64, 65, 61] * 6), (900, [10, 90] * 5)], True),       # no ring to speak of: the last pages are not whole for every query
    (128, "bf16", 2, 16, 0, 1, [(6000, [0] * 40)], True),
    (128, "bf16", 4, 4, 192, 1, [(7000, [1, 2, 3] * 25)], True),
    (128, "bf16", 8, 32, 128, 5, [(1700, [9, 8, 7] * 10)], True),                                 # 600 rows per kv head: three tiles
    (128, "bf16", 8, 32, 128, 1, [(300, [1, 2, 3, 4])], False),
]


@pytest.mark.parametrize("d, dt, kvh, hq, residual, lq, groups, pays", GROUPS)
def test_shared_prefixes(d, dt, kvh, hq, residual, lq, groups, pays):
    cache, members, kv = grouped(groups, kvh, d, dt, residual)
    order = [r for kids in members for r in kids]
    o = ints(*np.cumsum([0] + [len(kids) for kids in members]).tolist())
    q = query(len(order), lq, hq, d, dt, 7)
    want = cache.attend(0, q, rows=ints(*order), out_dtype=torch.float32).double().cpu().numpy()      # 3e-5 from the definition, and tested to be
    got = cache.attend(0, q, rows=ints(*order), groups=o, out_dtype=torch.float32)
    cache.check()
    skip = shares(cache, q, order, o)
    if pays:
        expect = []
        for kids in members:
            n = min(min(plain.packed(len(kv[r][0]), residual), len(kv[r][0]) - lq + 1) // 64 for r in kids)
            first = cache.block_table[kids[0]].tolist()
            same = [i for i in range(n) if all(cache.block_table[r, i].item() == first[i] for r in kids)]
            expect += [len(same)] * len(kids)
        assert max(skip) > 0 and all(a in (b, 0) for a, b in zip(skip, expect)), (skip, expect)
    close(got, want, SHARED_TOL)
    assert torch.equal(cache.attend(0, q, rows=ints(*order), groups=o), got.to(DT[dt]))
    assert torch.equal(cache.attend(0, q, rows=ints(*order), groups=o, out_dtype=torch.float32), got)
    for i in range(0, len(order), 11):                            # a few against the definition
        k, v = plain.held(f32(kv[order[i]][0]), f32(kv[order[i]][1]), residual)
        close(got[i], plain.attention(f32(q[i].cpu()), k, v, d ** -0.5), SHARED_TOL)


@pytest.fixture(scope="module")
def common():
    """64 rows behind a prompt of 3000 tokens, head_dim 64"""
    cache, members, kv = grouped([(3000, [1 + i % 70 for i in range(64)])], 8, 64, "bf16", 128)
    return cache, members[0], kv


def test_entries_outside_groups_and_groups_of_one(common):
    cache, kids, _ = common
    q = query(len(kids), 1, 32, 64, "bf16", 3)
    rows = ints(*kids)
    want = cache.attend(0, q, rows=rows, out_dtype=torch.float32).double().cpu().numpy()
    for o in ([3, 60], [0, 1, 1, 50, 64], [0, 0, 64, 64], [0, 64]):
        got = cache.attend(0, q, rows=rows, groups=ints(*o), out_dtype=torch.float32)
        close(got, want, SHARED_TOL)
        skip = shares(cache, q, kids, ints(*o))
        lone = [i for i in range(64) if not any(a <= i < b and b - a > 1 for a, b in zip(o, o[1:]))]
        assert max(skip) == 44 and all(skip[i] == 0 for i in lone), (o, skip)
    assert torch.equal(cache.attend(0, q, rows=rows, groups=ints(5), out_dtype=torch.float32), cache.attend(0, q, rows=rows, out_dtype=torch.float32))      # no group at all
    cache.check()


@pytest.mark.parametrize("o", [[0, 30, 20, 64], [-1, 64], [0, 65], [64, 0]])
def test_group_offsets_that_do_not_ascend(common, o):
    cache, kids, _ = common
    q = query(len(kids), 1, 32, 64, "bf16", 3)
    got = cache.attend(0, q, rows=ints(*kids), groups=ints(*o), out_dtype=torch.float32)
    with pytest.raises(Exception, match="outside the cache"):
        cache.check()
    assert torch.equal(got, cache.attend(0, q, rows=ints(*kids), out_dtype=torch.float32))
    cache.check()


def test_the_same_row_twice_and_rows_that_are_not_there(common):
    cache, kids, _ = common
    rows = list(kids)
    rows[5], rows[40] = rows[6], rows[6]
    q = query(len(rows), 1, 32, 64, "bf16", 4)
    got = cache.attend(0, q, rows=ints(*rows), groups=ints(0, 64), out_dtype=torch.float32)
    close(got, cache.attend(0, q, rows=ints(*rows), out_dtype=torch.float32).double().cpu().numpy(), SHARED_TOL)
    cache.check()
    rows[0], rows[9], rows[30] = -1, -1, cache.rows                # the others share all the same
    got = cache.attend(0, q, rows=ints(*rows), groups=ints(0, 64), out_dtype=torch.float32)
    assert [i for i, n in enumerate(shares(cache, q, rows, ints(0, 64))) if n != 44] == [0, 9, 30]
    with pytest.raises(Exception, match="outside the cache"):
        cache.check()
    assert not got[[0, 9, 30]].any()
    close(got, cache.attend(0, q, rows=ints(*rows), out_dtype=torch.float32).double().cpu().numpy(), SHARED_TOL)
    with pytest.raises(Exception, match="outside the cache"):
        cache.check()


def test_a_padded_batch(common):
    """Rows of the batch that are empty, or so short that they have no page: they stay out, the others share."""
    cache, kids, _ = common
    before = cache.lengths.clone()
    short = {kids[0]: 0, kids[7]: 0, kids[20]: 1, kids[21]: 130, kids[63]: 0}
    for r, n in short.items():
        cache.lengths[r] = n
    q = query(len(kids), 1, 32, 64, "bf16", 6)
    want = cache.attend(0, q, rows=ints(*kids), out_dtype=torch.float32)
    got = cache.attend(0, q, rows=ints(*kids), groups=ints(0, 64), out_dtype=torch.float32)
    skip = shares(cache, q, kids, ints(0, 64))
    cache.lengths.copy_(before)
    cache.check()
    assert [i for i, n in enumerate(skip) if n != 44] == [0, 7, 20, 21, 63]
    assert not got[[0, 7, 63]].any()
    close(got, want.double().cpu().numpy(), SHARED_TOL)


@pytest.mark.parametrize("scaling", [None, 0.5, -0.3, 0.0])
def test_scalings(common, scaling):
    cache, kids, _ = common
    q = query(len(kids), 1, 32, 64, "bf16", 3)
    want = cache.attend(0, q, rows=ints(*kids), scaling=scaling, out_dtype=torch.float32).double().cpu().numpy()
    close(cache.attend(0, q, rows=ints(*kids), groups=ints(0, 64), scaling=scaling, out_dtype=torch.float32), want, SHARED_TOL)


@pytest.mark.parametrize("bad", [float("nan"), float("inf"), float("-inf")])
def test_a_query_that_is_not_finite_spoils_its_own_row_only(common, bad):
    cache, kids, _ = common
    q = query(len(kids), 1, 32, 64, "bf16", 3)
    clean = cache.attend(0, q, rows=ints(*kids), groups=ints(0, 64), out_dtype=torch.float32)
    q[17, 0, 2, 33] = bad
    got = cache.attend(0, q, rows=ints(*kids), groups=ints(0, 64), out_dtype=torch.float32)
    same = torch.ones(len(kids), 32, dtype=torch.bool)
    same[17, 2] = False
    assert torch.equal(got[:, 0].cpu()[same], clean[:, 0].cpu()[same]) and torch.isnan(got[17, 0, 2]).all()


@pytest.mark.parametrize("dt", ["bf16", "fp16"])
@pytest.mark.parametrize("scale", [1e-5, 1.0, 1e4])
def test_pages_and_queries_of_very_unlike_ranges(dt, scale):
    """Values of some pages 1e3 times those of others, keys with outlier channels and a constant part (rows that do not straddle zero), a token that takes nearly all, queries of every size."""
    kvh, d, prompt, n = 4, 128, 3000, 64
    cache = make(n + 1, kvh, d, dt, 64, max_length=4096, pages=512)
    k, v = tokens(prompt, kvh, d, torch.float32, 5)
    k[:, 1] += 7.0
    k[:, 2, :5] *= 20.0
    k[:, 3, 64:] -= 3.0
    v[::3] = v[::3].abs() + 0.5
    v[640:1280] *= 1e-3
    v[1280:1344] *= 30.0
    v[1344:1408] = 0.0
    k[77, 0] *= 8.0
    k, v = ((x * s).clamp(-6e4, 6e4).to(DT[dt]) for x, s in ((k, scale), (v, scale)))
    o = ints(0, prompt)
    cache.extend(rows=ints(n), offsets=o)
    cache.append(0, k.cuda(), v.cuda(), rows=ints(n), offsets=o)
    kids = list(range(n))
    cache.fork(ints(*[n] * n), ints(*kids))
    q = torch.randn(n, 1, 16, d, generator=torch.Generator().manual_seed(2)) / scale
    q *= torch.logspace(-3, 0, n).view(n, 1, 1, 1)
    q = q.clamp(-6e4, 6e4).to(DT[dt]).cuda()
    want = cache.attend(0, q, rows=ints(*kids), out_dtype=torch.float32)
    got = cache.attend(0, q, rows=ints(*kids), groups=ints(0, n), out_dtype=torch.float32)
    assert max(shares(cache, q, kids, ints(0, n))) == 45
    close(got, want.double().cpu().numpy(), SHARED_TOL)


def test_many_small_groups():
    """More units than a CTA lists at a time: 300 groups of three rows with tables of their own."""
    kvh, d, rows = 32, 64, 900
    cache = make(rows, kvh, d, "bf16", 0, max_length=256 * 64, pages=2100)
    gen = torch.Generator(device="cuda").manual_seed(1)
    cache.store.random_(0, 256, generator=gen)
    words = cache.store.view(1, 2100, kvh, 4608)
    for at in (2048, 4352):                                        # codes as they come; words with moderate scales that straddle zero
        w = words[..., at:at + 256].view(torch.int32)
        w.copy_((torch.randint(64, 128, w.shape, device="cuda", generator=gen, dtype=torch.int32) << 16) | 0x3400)
    table = torch.full((rows, cache.block_table.shape[1]), -1, dtype=torch.int32)
    for g in range(300):
        table[3 * g:3 * g + 3, :7] = torch.arange(7 * g, 7 * g + 7, dtype=torch.int32)
    cache.block_table.copy_(table)
    cache.lengths.fill_(7 * 64)
    q = query(rows, 1, 8 * kvh, d, "bf16", 9)
    o = torch.arange(0, rows + 1, 3, dtype=torch.int32, device="cuda")
    got = cache.attend(0, q, groups=o, out_dtype=torch.float32)
    cache.check()
    skip = shares(cache, q, list(range(rows)), o)
    assert set(skip) == {7}
    close(got[::7].reshape(-1, d), cache.attend(0, q, out_dtype=torch.float32)[::7].reshape(-1, d).double().cpu().numpy(), SHARED_TOL)


def test_captured_replayed_and_on_another_stream(common):
    """A captured call follows lengths and tables as they are at its replay; two graphs on one stream share a workspace and run one after the other."""
    cache, kids, _ = common
    rows, o = ints(*kids), ints(0, 64)
    q = query(len(kids), 1, 32, 64, "bf16", 3)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        cache.attend(0, q, rows=rows, groups=o)
    torch.cuda.synchronize()
    graphs = []
    for kw in (dict(groups=o), dict(window=500, sinks=4)):
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=side):
            out = cache.attend(0, q, rows=rows, **kw)
        graphs.append((graph, out, kw))
    before = cache.lengths.clone()
    for shift in (0, 1):
        cache.lengths.copy_(before - 64 * shift * (torch.arange(cache.rows, device="cuda", dtype=torch.int32) % 2))
        cache.lengths.clamp_(min=0)
        torch.cuda.synchronize()
        with torch.cuda.stream(side):
            for graph, _, _ in graphs:
                graph.replay()
        torch.cuda.synchronize()
        for _, out, kw in graphs:
            assert torch.equal(out, cache.attend(0, q, rows=rows, **kw))
    cache.lengths.copy_(before)
    cache.check()


def test_outputs_strides_and_types(common):
    cache, kids, _ = common
    q = query(len(kids), 1, 32, 64, "bf16", 3)
    strided = torch.zeros(len(kids), 32, 3 * 64, dtype=torch.bfloat16, device="cuda")
    strided[..., 64:128] = q[:, 0]
    for kw in (dict(groups=ints(0, 64)), dict(window=300, sinks=2)):
        want = cache.attend(0, q, rows=ints(*kids), **kw)
        out = torch.empty(len(kids), 32, 64, dtype=torch.bfloat16, device="cuda")
        assert cache.attend(0, strided[..., 64:128], rows=ints(*kids), out=out, **kw) is out
        assert torch.equal(out, want[:, 0])


def test_a_step_of_serving_with_all_of_them():
    """A prompt, its forks, decode steps with shared attention in one layer and a window in the other, and what the rows hold read back: all from the same tokens."""
    kvh, hq, d, n = 8, 32, 64, 48
    cache = make(n + 1, kvh, d, "bf16", 128, layers=2, max_length=8192, pages=1024)
    prompt = tokens(4000, kvh, d, torch.bfloat16, 1)
    o = ints(0, 4000)
    cache.extend(rows=ints(n), offsets=o)
    for layer in range(2):
        cache.append(layer, prompt[0].cuda(), prompt[1].cuda(), rows=ints(n), offsets=o)
    kids = list(range(n))
    cache.fork(ints(*[n] * n), ints(*kids))
    steps = [tokens(n, kvh, d, torch.bfloat16, 50 + i) for i in range(70)]
    rows = ints(*kids)
    for k, v in steps:
        cache.extend(rows=rows)
        for layer in range(2):
            cache.append(layer, k.cuda(), v.cuda(), rows=rows)
        q = query(n, 1, hq, d, "bf16", 3)
        shared = cache.attend(0, q, rows=rows, groups=ints(0, n), out_dtype=torch.float32)
        near = cache.attend(1, q, rows=rows, window=256, sinks=4, out_dtype=torch.float32)
    cache.check()
    for r in (0, 17, 47):
        k = torch.cat([prompt[0]] + [s[0][r:r + 1] for s in steps])
        v = torch.cat([prompt[1]] + [s[1][r:r + 1] for s in steps])
        kk, vv = plain.held(f32(k), f32(v), 128)
        close(shared[r], plain.attention(f32(q[r].cpu()), kk, vv, d ** -0.5), SHARED_TOL)
        close(near[r], windowed(f32(q[r].cpu()), kk, vv, d ** -0.5, 256, 4), TOL)
        for layer in range(2):
            rk, rv = cache.read(layer, rows=ints(r), offsets=ints(0, len(k)), tokens=len(k), out_dtype=torch.float32)
            assert np.array_equal(rk.cpu().numpy(), kk.astype(np.float32)) and np.array_equal(rv.cpu().numpy(), vv.astype(np.float32))


def test_misaligned_operands_and_small_workspaces_are_refused(common):
    """At the C entry: before anything is launched."""
    import ctypes
    from muzero_b200.kernels import _cabi
    cache, kids, _ = common
    o = ints(0, 64)
    lib, v = cache._lib, _cabi.PagedView(0, 0, o.data_ptr(), 1)
    need = lib.mz_paged_attention_view_workspace_bytes(cache._ref, ctypes.byref(v), 64, 1, 32)
    ws, q, rows = torch.zeros(need + 64, dtype=torch.uint8, device="cuda"), query(64, 1, 32, 64, "bf16", 1), ints(*kids)
    out = torch.zeros_like(q)

    def call(query=0, at=0, size=need, groups=o.data_ptr()):
        a = _cabi.PagedAttentionArgs(q.data_ptr() + query, 2048, 2048, 64, 64, 1, 32, rows.data_ptr(), 0.125, out.data_ptr(), 2, ws.data_ptr() + at, size)
        w = _cabi.PagedView(0, 0, groups, 1)
        return lib.mz_paged_attention_view(cache._ref, 0, ctypes.byref(a), ctypes.byref(w), _cabi.stream_ptr(cache.device))

    for kw, text in ((dict(query=8), "16-byte aligned"), (dict(at=16), "32-byte"), (dict(size=need - 1), "needed"), (dict(groups=None), "groups is NULL")):
        assert call(**kw) != 0 and text in _cabi.last_error(), kw
    assert call(at=32) == 0
    assert torch.equal(out, cache.attend(0, q, rows=rows, groups=o))


CHILD = r"""
import sys, torch
sys.path[:0] = [{root!r}, {root!r} + "/tests"]
import muzero_b200 as mz
from muzero_b200.kernels._cabi import load_library
lib = load_library()
assert lib.mz_bounds_violations(None, None, None, 0) == 0
for d, dt, rows in ((128, torch.bfloat16, 70), (64, torch.float16, 24)):
    n = rows + 1
    cache = mz.MuZeroPagedCache.allocate(layers=1, kv_heads=8, head_dim=d, pages=256, rows=n, max_length=8192, dtype=dt)
    o = torch.tensor([0, 6000], dtype=torch.int32, device="cuda")
    home = torch.tensor([rows], dtype=torch.int32, device="cuda")
    cache.extend(rows=home, offsets=o)
    k, v = (torch.randn(6000, 8, d, device="cuda", dtype=dt) for _ in range(2))
    cache.append(0, k, v, rows=home, offsets=o)
    kids = torch.arange(rows, dtype=torch.int32, device="cuda")
    cache.fork(home.expand(rows).contiguous(), kids)
    q = torch.randn(rows, 1, 64 if d == 64 else 32, d, device="cuda", dtype=dt)
    for kw in (dict(groups=torch.tensor([0, rows - 1], dtype=torch.int32, device="cuda")), dict(window=700, sinks=70)):
        good = cache.attend(0, q, rows=kids, **kw)
        assert torch.isfinite(good).all()
        lib.mz_debug_fail_waits(1)
        bad = cache.attend(0, q, rows=kids, **kw)
        torch.cuda.synchronize()
        lib.mz_debug_fail_waits(0)
        assert torch.isnan(bad).all(), kw
        assert torch.equal(cache.attend(0, q, rows=kids, **kw), good)
    cache.read(0, offsets=torch.tensor([0, 100], dtype=torch.int32, device="cuda"), rows=home, tokens=100)
    cache.check()
assert lib.mz_bounds_violations(None, None, None, 0) == 0
print("views checked build ok")
"""


def test_checked_build_and_waits_that_run_out():
    """In the checked build: no guarded store out of bounds; where every wait runs out the outputs are NaN, the call ends, the next one is right."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    lib = os.path.join(root, "muzero_b200", "lib", "libmuzero_b200_bounds.so")
    if not os.path.exists(lib):
        pytest.skip("the checked library has not been built")
    env = dict(os.environ, MUZERO_B200_LIB=lib)
    res = subprocess.run([sys.executable, "-c", CHILD.format(root=root)], env=env, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and "views checked build ok" in res.stdout, res.stdout + res.stderr
