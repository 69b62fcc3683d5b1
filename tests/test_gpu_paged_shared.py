"""GPU: shared prefixes of the paged cache, where batches are wide and prefixes short, rows stay out of their group, values need more than 16 bits, and runs of pages are long.

Helpers and SHARED_TOL are those of test_gpu_paged_views.py.  FINE_TOL, before any run: keys, values and probabilities are two f16 numbers each, 2^-22 of themselves; logits of up to 30 (base 2: 43)
carry that of their terms and 2^-23 of a running sum for each of 16 products, of which all but the last few are small: 1e-5; the output's sums lose at most 2^-23 in each of 12 products per page, and a
CTA has at most three pages of these prefixes, a stream two: 3e-6; the exponential 2^-22.  Together below 2e-5, and with the 16-bit window's 1e-5 what ordinary attention is held to: 3e-5.
"""
import numpy as np
import pytest
import torch

import paged_plain as plain
from test_gpu_paged import DT, f32, ints, make, tokens
from test_gpu_paged_views import SHARED_TOL, close, grouped, query, shares

pytestmark = pytest.mark.gpu
FINE_TOL = 3e-5


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


@pytest.mark.parametrize("d, dt, hq, lq", [(128, "bf16", 32, 1), (128, "fp16", 32, 1), (64, "bf16", 32, 1), (64, "fp16", 16, 2), (128, "bf16", 8, 3)])
def test_shared_attention_is_as_exact_as_ordinary_attention(d, dt, hq, lq):
    cache, members, kv = grouped([(3000, [3 + i % 70 for i in range(64)])], 8, d, dt, 128)
    kids = members[0]
    q = query(64, lq, hq, d, dt, 13)
    got = cache.attend(0, q, rows=ints(*kids), groups=ints(0, 64), out_dtype=torch.float32)
    cache.check()
    assert min(shares(cache, q, kids, ints(0, 64))) >= 44
    want = cache.attend(0, q, rows=ints(*kids), out_dtype=torch.float32)
    assert not torch.equal(got, want)
    close(got, want.double().cpu().numpy(), 2 * FINE_TOL)
    for i in (0, 31, 63):
        k, v = plain.held(f32(kv[kids[i]][0]), f32(kv[kids[i]][1]), 128)
        close(got[i], plain.attention(f32(q[i].cpu()), k, v, d ** -0.5), FINE_TOL)


@pytest.mark.parametrize("d, dt, group", [(128, "bf16", 4), (128, "fp16", 2), (64, "bf16", 4)])
def test_long_runs_of_pages_lose_nothing(d, dt, group):
    """A CTA takes hundreds of pages one after the other, of values that are all of one sign (the tensor cores' sums are cut off towards zero).  A long table needs few pages: it
    names each of 50 many times, and attention over it is that over 50 with their weights multiplied."""
    rows, kvh, distinct, times, residual = 64, 8, 50, 160, 64
    n = distinct * times * 64 + residual
    cache = make(rows, kvh, d, dt, residual, max_length=n, pages=distinct + 6)
    g = torch.Generator().manual_seed(3)
    k = torch.randn(distinct * 64 + residual, kvh, d, generator=g).to(DT[dt])
    v = (1 + 0.2 * torch.randn(k.shape, generator=g)).to(DT[dt])
    o = ints(0, k.shape[0])
    cache.extend(rows=ints(0), offsets=o)
    cache.append(0, k.cuda(), v.cuda(), rows=ints(0), offsets=o)
    cache.check()
    ids = cache.block_table[0, :distinct].clone()
    cache.block_table[:, :distinct * times] = ids[torch.randperm(distinct * times, generator=g).cuda() % distinct]
    cache.lengths.fill_(n)
    cache.tail.copy_(1 + torch.randn(cache.tail.shape, generator=g).to(cache.dtype).cuda() / 8)
    q = query(rows, 1, group * kvh, d, dt, 14)
    got = cache.attend(0, q, groups=ints(0, rows), out_dtype=torch.float32)
    cache.check()
    assert shares(cache, q, None, ints(0, rows)) == [distinct * times] * rows
    held_k, held_v = plain.held(f32(k), f32(v), residual)
    place = [(n - residual + i) % cache.tail.shape[4] for i in range(residual)]
    ring = cache.tail[0].double().cpu().numpy()[:, :, :, place]
    for r in (0, 37):
        for h in range(kvh):
            kk, vv = (np.concatenate([x[:distinct * 64, h], y]) for x, y in ((held_k, ring[r, 0, h]), (held_v, ring[r, 1, h])))
            s = q[r, 0, h * group:(h + 1) * group].double().cpu().numpy() @ kk.T * d ** -0.5
            w = np.exp(s - s.max(-1, keepdims=True))
            w[:, :distinct * 64] *= times
            close(got[r, 0, h * group:(h + 1) * group], w @ vv / w.sum(-1, keepdims=True), FINE_TOL)


@pytest.mark.parametrize("d, group, rows, pages, pays", [(128, 4, 8, 64, False), (128, 4, 32, 64, True), (128, 4, 4, 600, False), (128, 8, 4, 1000, True), (64, 4, 8, 64, False), (64, 4, 64, 64, True)])
def test_the_rule_on_both_sides(d, group, rows, pages, pays):
    """Where sharing was measured to cost more, a call with groups gives what one without does, bit for bit."""
    cache = make(rows, 8, d, "bf16", 64, max_length=pages * 64 + 64, pages=pages)
    random_pages(cache, 1)
    cache.block_table.copy_(torch.arange(pages, dtype=torch.int32).expand(rows, -1))
    cache.lengths.fill_(pages * 64 + 64)
    q = query(rows, 1, group * 8, d, "bf16", 15)
    want = cache.attend(0, q, out_dtype=torch.float32)
    got = cache.attend(0, q, groups=ints(0, rows), out_dtype=torch.float32)
    cache.check()
    assert torch.equal(got, want) != pays
    close(got, want.double().cpu().numpy(), 2 * FINE_TOL)


def random_pages(cache, seed):
    """Codes as they come, words with moderate scales that straddle zero."""
    gen = torch.Generator(device="cuda").manual_seed(seed)
    d = cache.head_dim
    cache.store.random_(0, 256, generator=gen)
    for at in (32 * d, 68 * d):
        w = cache.store[..., at:at + 4 * d].view(torch.int32)
        w.copy_((torch.randint(64, 128, w.shape, device="cuda", generator=gen, dtype=torch.int32) << 16) | 0x3400)
    cache.tail.copy_(torch.randn(cache.tail.shape, device="cuda", generator=gen))


def test_more_units_than_a_cta_lists_at_a_time():
    """200 groups of five rows with tables of their own and 64 kv heads: 86 units to a CTA, that share."""
    kvh, d, rows = 64, 64, 1000
    cache = make(rows, kvh, d, "bf16", 0, max_length=16 * 64, pages=1400)
    random_pages(cache, 2)
    table = torch.full((rows, cache.block_table.shape[1]), -1, dtype=torch.int32)
    for g in range(200):
        table[5 * g:5 * g + 5, :7] = torch.arange(7 * g, 7 * g + 7, dtype=torch.int32)
    cache.block_table.copy_(table)
    cache.lengths.fill_(7 * 64)
    q = query(rows, 1, 8 * kvh, d, "bf16", 9)
    o = torch.arange(0, rows + 1, 5, dtype=torch.int32, device="cuda")
    got = cache.attend(0, q, groups=o, out_dtype=torch.float32)
    cache.check()
    want = cache.attend(0, q, out_dtype=torch.float32)
    assert set(shares(cache, q, None, o)) == {7} and not torch.equal(got, want)
    close(got[::7].reshape(-1, d), want[::7].reshape(-1, d).double().cpu().numpy(), 2 * FINE_TOL)


@pytest.mark.parametrize("dt, span", [("bf16", 20), ("fp16", 10)])
def test_scales_that_are_very_unlike_within_a_page(dt, span):
    """Channels of the keys, and tokens of the values, whose sizes go down to 2^-20 of the largest, and queries that make up for it: every channel weighs the same.  A scale of
    2^-20 is still a normal f16 number once the page's largest is 2^14, and its remainder has an error of 2^-19."""
    kvh, d, rows, pages = 8, 128, 64, 46
    cache = make(rows + 1, kvh, d, dt, 64, max_length=4096, pages=64)
    g = torch.Generator().manual_seed(6)
    n = pages * 64 + 64
    down = torch.exp2(-span * torch.rand(d, generator=g))
    k = (torch.randn(n, kvh, d, generator=g) * down).to(DT[dt])
    v = (torch.randn(n, kvh, d, generator=g) * torch.exp2(-span * torch.rand(n, 1, 1, generator=g))).to(DT[dt])
    o = ints(0, n)
    cache.extend(rows=ints(rows), offsets=o)
    cache.append(0, k.cuda(), v.cuda(), rows=ints(rows), offsets=o)
    kids = list(range(rows))
    cache.fork(ints(*[rows] * rows), ints(*kids))
    q = (torch.randn(rows, 1, 4 * kvh, d, generator=g) / down).to(DT[dt]).cuda()
    got = cache.attend(0, q, rows=ints(*kids), groups=ints(0, rows), out_dtype=torch.float32)
    cache.check()
    assert not torch.equal(got, cache.attend(0, q, rows=ints(*kids), out_dtype=torch.float32))
    kk, vv = plain.held(f32(k), f32(v), 64)
    for i in (0, 40):
        close(got[i], plain.attention(f32(q[i].cpu()), kk, vv, d ** -0.5), FINE_TOL)


@pytest.mark.parametrize("args, shared", [(["--rows", "32", "--requests", "33", "--new-tokens", "6"], True), (["--rows", "8", "--prefix", "500", "--requests", "9", "--new-tokens", "20"], False)])
def test_the_example_shares_its_prefix(args, shared):
    """With its default prefix the serving example's batch takes the prefix once; its attention is checked against pages that are decoded in torch (bf16 output), and so is `read`."""
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_serving.py")
    spec = importlib.util.spec_from_file_location("paged_serving", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    out = m.main(["--layers", "2", *args])
    assert out["batch"]["shared"] == shared and out["batch"]["read"]
    assert max(out["batch"]["error"], out["error"]) <= 2.0 ** -8


@pytest.mark.parametrize("d, batch, lq, hq", [(128, 64, 1, 32), (64, 9, 40, 20), (128, 64, 512, 32)])
def test_the_size_of_a_workspace_for_groups(d, batch, lq, hq):
    """What a call with groups needs beyond one without: records, sums of long runs, and a few numbers per entry and group."""
    import ctypes
    from muzero_b200.kernels._cabi import PagedView
    cache = make(batch, 4, d, "bf16", 64, max_length=1 << 17, pages=8)
    o = ints(0, batch)
    view = PagedView(0, 0, o.data_ptr(), 1)
    lib = cache._lib
    more = lib.mz_paged_attention_view_workspace_bytes(cache._ref, ctypes.byref(view), batch, lq, hq) - lib.mz_paged_attention_workspace_bytes(cache._ref, batch, lq, hq)
    sms = torch.cuda.get_device_properties(0).multi_processor_count
    assert 0 <= more - ((batch * lq * hq + 256 * sms) * (4 * d + 8) + 1024 * sms * d) <= 1024 + 16 * batch


def test_graphs_of_one_stream_replayed_on_two():
    """Two steps of layers, captured on the same stream, are replayed at the same time on two others: each has its own workspace, and so has what runs outside of them meanwhile."""
    layers, rows, d, pages = 4, 64, 64, 60
    cache = make(rows, 8, d, "bf16", 64, max_length=pages * 64 + 128, pages=pages, layers=layers)
    for layer in range(layers):
        random_pages(cache, 20 + layer)
    cache.block_table.copy_(torch.arange(cache.block_table.shape[1], dtype=torch.int32) % pages)
    cache.lengths.copy_(torch.arange(rows, dtype=torch.int32) * 3 + pages * 64 - 200)
    q = [query(rows, 1, 32, d, "bf16", 16 + i) for i in range(2)]
    calls = [lambda i=i, kw=kw: [cache.attend(layer, q[i], **kw) for layer in range(layers)] for i, kw in enumerate((dict(groups=ints(0, rows)), dict(window=1500, sinks=70)))]
    want = [call() for call in calls]
    capture, streams = torch.cuda.Stream(), [torch.cuda.Stream() for _ in range(2)]
    graphs, outs = [], []
    torch.cuda.synchronize()
    for call in calls + calls:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1], stream=capture):
            outs.append(call())
    for _ in range(20):
        for out in outs:
            for x in out:
                x.zero_()
        torch.cuda.synchronize()
        for i, (graph, out) in enumerate(zip(graphs, outs)):
            with torch.cuda.stream(streams[i % 2]):
                graph.replay()
        here = [call() for call in calls]
        torch.cuda.synchronize()
        for got in (outs[:2], outs[2:], here):
            assert all(torch.equal(x, y) for a, b in zip(got, want) for x, y in zip(a, b))
    cache.check()


@pytest.mark.parametrize("prompts, pages, pays", [((2000, 1900, 1500), (30, 22), False), ((6000, 5900, 4500), (92, 69), True)])
def test_which_groups_share(prompts, pages, pays):
    """Groups of one batch are weighed each for itself: the pair stays out, the others take their pages once, if what that saves is worth a call that shares (kv heads x pages x
    (13 x 16 rows - 34 and 13 x 10 - 34) tenths of a row's visit: 59 thousand of 104, and 181)."""
    groups = [(prompts[0], [3, 70, 9, 200] * 4), (prompts[1], [5, 6]), (prompts[2], [17] * 10)]
    cache, members, _ = grouped(groups, 8, 128, "fp16", 64)
    order = [r for kids in members for r in kids]
    o = ints(0, 16, 18, 28)
    q = query(len(order), 1, 64, 128, "fp16", 7)
    want = cache.attend(0, q, rows=ints(*order), out_dtype=torch.float32)
    got = cache.attend(0, q, rows=ints(*order), groups=o, out_dtype=torch.float32)
    cache.check()
    assert shares(cache, q, order, o) == [pages[0]] * 16 + [0] * 2 + [pages[1]] * 10
    # (where the others share, the pair's steps are cut otherwise, and rounded otherwise)
    assert all(torch.equal(got[i], want[i]) != pays for i in (*range(16), *range(18, 28))) and (pays or torch.equal(got, want))
    close(got, want.double().cpu().numpy(), 2 * FINE_TOL)


@pytest.mark.parametrize("d, dt, hq, lq, rows, own", [(128, "bf16", 32, 70, 6, [70, 100, 200]), (64, "fp16", 16, 130, 3, [5, 140, 131]), (128, "bf16", 8, 300, 2, [300, 40]),
                                                      (64, "bf16", 20, 33, 5, [0, 33, 64])])
def test_blocks_of_query_tokens(d, dt, hq, lq, rows, own):
    """Tens to hundreds of query tokens of each row, some of them in the prefix, whose last pages then are not whole for every query."""
    kvh, residual = 4, 64
    cache, members, kv = grouped([(3300, (own * rows)[:rows])], kvh, d, dt, residual)
    kids = members[0]
    q = query(rows, lq, hq, d, dt, 17)
    o = ints(0, rows)
    want = cache.attend(0, q, rows=ints(*kids), out_dtype=torch.float32)
    got = cache.attend(0, q, rows=ints(*kids), groups=o, out_dtype=torch.float32)
    cache.check()
    pages = min(min(plain.packed(len(kv[r][0]), residual), len(kv[r][0]) - lq + 1) // 64 for r in kids)
    table = cache.block_table[kids].cpu()
    pages = next((i for i in range(pages) if len(set(table[:, i].tolist())) > 1), pages)
    assert shares(cache, q, kids, o) == [pages] * rows and not torch.equal(got, want)
    close(got, want.double().cpu().numpy(), 2 * FINE_TOL)
    r = 1
    k, v = plain.held(f32(kv[kids[r]][0]), f32(kv[kids[r]][1]), residual)
    at = [0, lq // 2, lq - 1]
    n = len(k)
    for j in at:
        close(got[r, j:j + 1], plain.attention(f32(q[r, j:j + 1].cpu()), k[:n - lq + j + 1], v[:n - lq + j + 1], d ** -0.5), FINE_TOL)
