"""GPU: the paged cache against its definition (bytes of pages, 64-bit attention) and a host model of its tables.

Tolerances, before any run.  Pages, rings, tables, lengths and counts are equal.  Attention with fp32 output: logits of up to about 30 carry 2^-23 of
themselves (4e-6), the exponential 2^-22, sums of a few thousand terms less than 1e-6 of their norm, and a ring's probabilities are two 16-bit
parts, 2^-16 (bf16): 3e-5 of the output's norm.  16-bit output is the fp32 output rounded once, bit for bit.
"""
import numpy as np
import pytest
import torch

import paged_plain as plain

pytestmark = pytest.mark.gpu
DT = {"bf16": torch.bfloat16, "fp16": torch.float16}
TOL = 3e-5


def ints(*v):
    return torch.tensor(v, dtype=torch.int32, device="cuda")


def tokens(n, kvh, d, dt, seed):
    g = torch.Generator().manual_seed(seed)
    scale = torch.exp(torch.randn(d, generator=g))
    return (torch.randn(n, kvh, d, generator=g) * scale).to(dt), torch.randn(n, kvh, d, generator=g).to(dt)


def make(rows, kvh, d, dt, residual, max_length=4096, pages=256, layers=1):
    import muzero_b200 as mz
    return mz.MuZeroPagedCache.allocate(layers=layers, kv_heads=kvh, head_dim=d, pages=pages, rows=rows, max_length=max_length, residual_length=residual, dtype=DT[dt])


def fill(cache, lengths, chunks, seed=0, layer=0):
    """appends rows of these lengths, in `chunks` rounds; returns the rows' keys and values"""
    kv = [tokens(n, cache.kv_heads, cache.head_dim, cache.dtype, seed + 97 * i) for i, n in enumerate(lengths)]
    for c in range(chunks):
        part = [(n * c // chunks, n * (c + 1) // chunks) for n in lengths]
        offs = np.concatenate([[0], np.cumsum([b - a for a, b in part])])
        o = ints(*offs.tolist())
        cache.extend(offsets=o)
        k = torch.cat([kv[i][0][a:b] for i, (a, b) in enumerate(part)]).cuda()
        v = torch.cat([kv[i][1][a:b] for i, (a, b) in enumerate(part)]).cuda()
        if offs[-1]:
            cache.append(layer, k, v, offsets=o, max_new=max(b - a for a, b in part))
    cache.check()
    return kv


def f32(t):
    return t.float().numpy()


def assert_row(cache, row, k, v, layer=0):
    """a row's pages and ring hold exactly these tokens"""
    n, d = k.shape[0], cache.head_dim
    assert int(cache.lengths[row]) == n
    np_ = plain.packed(n, cache.residual_length) // 64
    ids = cache.block_table[row].tolist()
    assert all(i >= 0 for i in ids[:np_]) and all(i == -1 for i in ids[np_:])
    for p in range(np_):
        raw = cache.store[layer, ids[p]].cpu().numpy()
        for h in range(cache.kv_heads):
            s = slice(64 * p, 64 * p + 64)
            assert np.array_equal(raw[h], plain.pack_page(f32(k[s, h]), f32(v[s, h]))), (row, p, h)
    ring = cache.tail.shape[4]
    at = [t % ring for t in range(64 * np_, n)]
    for side, x in ((0, k), (1, v)):
        assert torch.equal(cache.tail[layer, row, side].cpu()[:, at].view(torch.int16), x[64 * np_:].transpose(0, 1).view(torch.int16))


def check_attention(cache, kv, q, rows, layer=0, scaling=None):
    got = cache.attend(layer, q, rows=ints(*rows), out_dtype=torch.float32, scaling=scaling)
    cache.check()
    assert got.shape == q.shape and got.dtype == torch.float32
    assert torch.equal(cache.attend(layer, q, rows=ints(*rows), scaling=scaling), got.to(cache.dtype))
    for i, r in enumerate(rows):
        k, v = plain.held(f32(kv[r][0]), f32(kv[r][1]), cache.residual_length)
        want = plain.attention(f32(q[i].cpu()), k, v, cache.head_dim ** -0.5 if scaling is None else scaling)
        g = got[i].double().cpu().numpy()
        for j in range(q.shape[1]):
            for h in range(q.shape[2]):
                err, size = np.linalg.norm(g[j, h] - want[j, h]), np.linalg.norm(want[j, h])
                assert err <= TOL * size, (r, j, h, err / max(size, 1e-30))
    return got


CASES = [
    # head_dim, type, kv heads, query heads, residual, query tokens, lengths
    (128, "bf16", 2, 8, 128, 1, [0, 1, 63, 64, 128, 191, 192, 193, 255, 256, 700]),
    (128, "fp16", 1, 8, 64, 1, [64, 127, 128, 129, 1000]),
    (128, "bf16", 2, 2, 0, 1, [1, 63, 64, 65, 128, 129, 192, 640]),
    (64, "bf16", 2, 8, 128, 1, [1, 192, 320, 333, 777]),
    (64, "fp16", 3, 3, 0, 2, [0, 1, 2, 64, 65, 130]),
    (128, "bf16", 1, 5, 128, 3, [1, 2, 3, 192, 195, 400]),
    (64, "bf16", 1, 4, 0, 5, [3, 64, 66, 68, 130, 200]),
    (128, "fp16", 2, 32, 64, 1, [130, 515]),
    (128, "bf16", 1, 3, 192, 9, [5, 256, 300]),
]


@pytest.mark.parametrize("d, dt, kvh, hq, residual, lq, lengths", CASES)
@pytest.mark.parametrize("chunks", [1, 4])
def test_append_and_attend(d, dt, kvh, hq, residual, lq, lengths, chunks):
    cache = make(len(lengths), kvh, d, dt, residual)
    kv = fill(cache, lengths, chunks, seed=d + hq)
    for r in range(len(lengths)):
        assert_row(cache, r, *kv[r])
    q = torch.randn(len(lengths), lq, hq, d, generator=torch.Generator().manual_seed(hq)).to(DT[dt]).cuda()
    order = list(range(len(lengths)))[::-1]
    check_attention(cache, kv, q, order)
    check_attention(cache, kv, q, order, scaling=0.5)


def test_token_by_token_equals_at_once():
    """One token at a time past two flushes, other rows joining and resting: the same bytes, and attention after every step."""
    kvh, hq, d = 2, 8, 128
    cache = make(3, kvh, d, "bf16", 64)
    kv = [tokens(300, kvh, d, torch.bfloat16, 5 + i) for i in range(3)]
    length = [0, 0, 0]
    for step in range(300):
        rows = [r for r in range(3) if (step + r) % (r + 1) == 0]
        cache.extend(rows=ints(*rows))
        k = torch.stack([kv[r][0][length[r]] for r in rows]).cuda()
        v = torch.stack([kv[r][1][length[r]] for r in rows]).cuda()
        cache.append(0, k, v, rows=ints(*rows))
        for r in rows:
            length[r] += 1
        if step in (0, 1, 64, 127, 128, 191, 192, 255, 299):
            have = {r: (kv[r][0][:length[r]], kv[r][1][:length[r]]) for r in range(3)}
            for r in range(3):
                assert_row(cache, r, *have[r])
            q = torch.randn(3, 1, hq, d, generator=torch.Generator().manual_seed(step)).bfloat16().cuda()
            check_attention(cache, have, q, [0, 1, 2])


@pytest.mark.parametrize("scale", [1e-6, 1e-3, 1e4])
@pytest.mark.parametrize("dt", ["bf16", "fp16"])
def test_scales(scale, dt):
    """Values of any size: the fixed point scales with them.  (At 1e-6 the scale words are f16's smallest numbers and rows become coarse; what is tested is the
    attention over what the pages then hold.)"""
    cache = make(1, 1, 128, dt, 0)
    k, v = tokens(500, 1, 128, torch.float32, 3)
    kv = [((k * scale).clamp(-6e4, 6e4).to(DT[dt]), (v * scale).clamp(-6e4, 6e4).to(DT[dt]))]
    o = ints(0, 500)
    cache.extend(offsets=o)
    cache.append(0, kv[0][0].cuda(), kv[0][1].cuda(), offsets=o)
    assert_row(cache, 0, *kv[0])
    q = (torch.randn(1, 1, 4, 128, generator=torch.Generator().manual_seed(1)) / min(scale, 1.0)).clamp(-6e4, 6e4).to(DT[dt]).cuda()
    check_attention(cache, kv, q, [0], scaling=0.05 / max(scale, 1.0))


def test_rows_that_are_not_ordinary():
    """Constant, zero, NaN, infinite, huge, tiny and one-sided rows, as keys and as values: bytes as defined."""
    d = 128
    x = torch.randn(128, 1, d, generator=torch.Generator().manual_seed(2))
    y = torch.randn(128, 1, d, generator=torch.Generator().manual_seed(4))
    for t in (x, y):
        for a, s in ((0, slice(None)), (1, slice(0, 64))):          # channels (keys' rows) and tokens (values' rows)
            pick = (lambda i: t[:64, 0, i]) if a == 0 else (lambda i: t[i, 0, s])
            pick(0).fill_(0.0)
            pick(1).fill_(3.5)
            pick(2).fill_(-7.0)
            pick(3)[5] = float("nan")
            pick(4)[7] = float("inf")
            pick(5)[9] = float("-inf")
            pick(6).fill_(float("nan"))
            pick(7).mul_(1e38)
            pick(8).mul_(1e-30)
            pick(9).mul_(1e-7)
            pick(10).abs_().add_(2.0)
            pick(11).abs_().neg_().sub_(0.5)
            pick(12).copy_(torch.linspace(-1e-6, 1e-6, 64))
            pick(13).abs_().mul_(1e-6)
            pick(14).fill_(-0.0)
    for dt in (torch.bfloat16, torch.float16):
        cache = make(1, 1, d, "bf16" if dt == torch.bfloat16 else "fp16", 0)
        k, v = x.to(dt), y.to(dt)
        o = ints(0, 128)
        cache.extend(offsets=o)
        cache.append(0, k.cuda(), v.cuda(), offsets=o)
        assert_row(cache, 0, k, v)


@pytest.mark.parametrize("residual", [0, 128])
@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_what_a_query_does_not_see_does_not_reach_it(residual, bad):
    """The newest of three query tokens' key and value are not finite: the two before it are unaffected, its own outputs are NaN."""
    n, d = 210, 128
    cache = make(1, 1, d, "bf16", residual)
    k, v = tokens(n, 1, d, torch.bfloat16, 8)
    good = [(k[:-1].clone(), v[:-1].clone())]
    k[-1], v[-1] = bad, bad
    o = ints(0, n)
    cache.extend(offsets=o)
    cache.append(0, k.cuda(), v.cuda(), offsets=o)
    q = torch.randn(1, 3, 4, d, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    got = cache.attend(0, q, out_dtype=torch.float32).double().cpu().numpy()
    kk, vv = plain.held(f32(good[0][0]), f32(good[0][1]), residual)
    assert plain.packed(n, residual) == plain.packed(n - 1, residual)
    want = plain.attention(f32(q[0, :2].cpu()), kk, vv, d ** -0.5)
    assert np.linalg.norm(got[0, :2] - want) <= 3e-5 * np.linalg.norm(want)
    assert not np.isfinite(got[0, 2]).any()


@pytest.mark.parametrize("bad", [float("nan"), float("inf")])
def test_a_query_that_is_not_finite_spoils_its_own_row_only(bad):
    cache = make(1, 2, 128, "bf16", 0)
    kv = fill(cache, [320], 1)
    q = torch.randn(1, 1, 8, 128, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
    clean = cache.attend(0, q, out_dtype=torch.float32)
    q[0, 0, 2, 77] = bad
    got = cache.attend(0, q, out_dtype=torch.float32)
    others = [h for h in range(8) if h != 2]
    assert torch.equal(got[0, 0, others], clean[0, 0, others]) and torch.isnan(got[0, 0, 2]).all()
    del kv


def test_strides_and_alignment():
    """Keys and values as slices of a fused projection, as transposed views and off any 16-byte boundary; queries likewise."""
    kvh, hq, d, n = 2, 8, 64, 150
    k, v = tokens(n, kvh, d, torch.bfloat16, 1)
    fused = torch.zeros(n, kvh, 3 * d, dtype=torch.bfloat16)
    fused[..., d:2 * d], fused[..., 2 * d:] = k, v
    fused = fused.cuda()
    odd = torch.zeros(n * kvh * d + 1, dtype=torch.bfloat16, device="cuda")
    odd[1:] = v.flatten().cuda()
    forms = [(fused[..., d:2 * d], fused[..., 2 * d:]), (k.transpose(0, 1).contiguous().cuda().transpose(0, 1), odd[1:].view(n, kvh, d)),
             (k.transpose(1, 2).contiguous().cuda().transpose(1, 2), v.cuda())]
    q = torch.randn(1, 2, hq, d, generator=torch.Generator().manual_seed(1)).bfloat16()
    qodd = torch.zeros(q.numel() + 3, dtype=torch.bfloat16, device="cuda")
    qodd[3:] = q.flatten().cuda()
    outs = []
    for (kf, vf), qf in zip(forms, (q.cuda(), q.transpose(1, 2).contiguous().cuda().transpose(1, 2), qodd[3:].view(q.shape))):
        cache = make(1, kvh, d, "bf16", 64)
        o = ints(0, n)
        cache.extend(offsets=o)
        cache.append(0, kf, vf, offsets=o)
        assert_row(cache, 0, k, v)
        outs.append(cache.attend(0, qf))
    assert torch.equal(outs[0], outs[1]) and torch.equal(outs[0], outs[2])
    three = cache.attend(0, q[:, 1].cuda())                        # [batch, heads, dim]: one token
    assert three.shape == (1, hq, d) and torch.equal(three, outs[0][:, 1])


def test_rows_pages_and_counts_against_a_model():
    """A few hundred random extensions, forks, releases and compactions: tables, lengths and counts as the model says, contents of all rows kept."""
    rng = np.random.default_rng(11)
    rows, pages, kvh, d, residual = 6, 20, 1, 64, 64
    cache = make(rows, kvh, d, "fp16", residual, max_length=900, pages=pages, layers=2)
    model = plain.Model(rows, pages, cache.block_table.shape[1], residual)
    have = [[(torch.zeros(0, kvh, d, dtype=torch.float16),) * 2 for _ in range(rows)] for _ in range(2)]
    refused = 0
    for step in range(250):
        what = rng.choice(["extend", "extend", "extend", "fork", "free", "compact"])
        if what == "extend":
            some = rng.permutation(rows)[:rng.integers(1, rows + 1)].tolist()
            counts = [int(rng.choice([0, 1, 5, 64, 130])) for _ in some]
            o = ints(*np.concatenate([[0], np.cumsum(counts)]).tolist())
            expect = model.extend(some, counts)
            cache.extend(rows=ints(*some), offsets=o)
            new = [[tokens(c, kvh, d, torch.float16, 1000 * step + 10 * i + layer) for i, c in enumerate(counts)] for layer in range(2)]
            for layer in range(2):
                if sum(counts):
                    cache.append(layer, torch.cat([x[0] for x in new[layer]]).cuda(), torch.cat([x[1] for x in new[layer]]).cuda(), rows=ints(*some), offsets=o)
            if expect:
                refused += 1
                with pytest.raises(Exception, match="free pages" if expect == 1 else "outgrew"):
                    cache.check()
            else:
                for layer in range(2):
                    for r, x in zip(some, new[layer]):
                        have[layer][r] = tuple(torch.cat([a, b]) for a, b in zip(have[layer][r], x))
        elif what == "fork":
            p = rng.permutation(rows).tolist()
            m = int(rng.integers(1, rows // 2 + 1))
            target, source = p[:m], [int(rng.choice(p[m:])) for _ in range(m)]
            model.fork(source, target)
            cache.fork(ints(*source), ints(*target))
            for layer in range(2):
                for s, t in zip(source, target):
                    have[layer][t] = have[layer][s]
        elif what == "free":
            some = rng.permutation(rows)[:2].tolist()
            model.free(some)
            cache.free(ints(*some, some[0]))                       # a row listed twice is released once
            for layer in range(2):
                for r in some:
                    have[layer][r] = (torch.zeros(0, kvh, d, dtype=torch.float16),) * 2
        else:
            model.compact()
            cache.compact()
        cache.check()
        assert cache.block_table.tolist() == model.table and cache.lengths.tolist() == model.length and cache.page_refs.tolist() == model.refs, (step, what)
        if step % 25 == 24:
            for layer in range(2):
                for r in range(rows):
                    assert_row(cache, r, *have[layer][r], layer=layer)
    assert refused > 0 and cache.free_pages() == sum(c == 0 for c in model.refs)


def test_copy_pages():
    cache = make(2, 2, 64, "bf16", 0, pages=9, layers=3)
    fill(cache, [200, 130], 1)
    cache.store.random_(0, 256)
    before = cache.store.clone()
    cache.copy_pages(ints(1, 3, 1), ints(7, 5, 8))
    before[:, [7, 5, 8]] = before[:, [1, 3, 1]]
    assert torch.equal(cache.store, before)
    cache.copy_pages(ints(1, 100), ints(6, 2))                     # the second pair is not one: skipped, reported
    before[:, 6] = before[:, 1]
    assert torch.equal(cache.store, before)
    with pytest.raises(Exception, match="outside"):
        cache.check()


def test_what_the_device_finds_wrong():
    """Bad indexes are reported and touch nothing; a failed extension keeps the append that follows from writing."""
    from muzero_b200.kernels import MuZeroKernelError
    cache = make(2, 1, 64, "bf16", 0, pages=2, max_length=640)
    kv = fill(cache, [100, 40], 1)
    state = [t.clone() for t in (cache.store, cache.tail, cache.block_table, cache.lengths, cache.page_refs)]

    def unchanged():
        return all(torch.equal(a, b) for a, b in zip(state, (cache.store, cache.tail, cache.block_table, cache.lengths, cache.page_refs)))

    k, v = tokens(200, 1, 64, torch.bfloat16, 1)
    o = ints(0, 0, 200)
    cache.extend(offsets=o)
    cache.append(0, k.cuda(), v.cuda(), offsets=o)
    assert unchanged()
    with pytest.raises(MuZeroKernelError, match="free pages"):
        cache.check()
    cache.check()                                                  # forgotten
    for call in (lambda: cache.extend(rows=ints(5)), lambda: cache.free(ints(-1)), lambda: cache.fork(ints(0), ints(7)), lambda: cache.fork(ints(0), ints(0)),
                 lambda: cache.append(0, k[:1].cuda(), v[:1].cuda(), rows=ints(9)), lambda: cache.extend(offsets=ints(0, 5, 3))):
        call()
        assert unchanged()
        with pytest.raises(MuZeroKernelError, match="outside"):
            cache.check()
    q = torch.randn(2, 1, 4, 64, device="cuda", dtype=torch.bfloat16)
    got = cache.attend(0, q, rows=ints(0, 6))
    assert (got[1] == 0).all() and torch.equal(got[0], cache.attend(0, q[:1], rows=ints(0))[0])
    with pytest.raises(MuZeroKernelError, match="outside"):
        cache.check()
    cache.block_table[0, 0] = 1 << 20                              # a table that somebody has spoilt
    assert torch.isfinite(cache.attend(0, q)).all()
    with pytest.raises(MuZeroKernelError, match="outside"):
        cache.check()
    del kv


def test_lengths_that_the_table_has_no_room_for():
    """Spoilt lengths, whose steps added up would pass 32 bits, are reported; the rows beside them keep their results."""
    from muzero_b200.kernels import MuZeroKernelError
    n, d = 160, 64
    cache = make(n, 1, d, "bf16", 0, max_length=640, pages=16)
    fill(cache, [200, 70] + [0] * (n - 2), 1)
    q = torch.randn(n, 1, 2, d, device="cuda", dtype=torch.bfloat16)
    want = cache.attend(0, q, out_dtype=torch.float32)
    cache.lengths[2:] = 0x7fffffff
    got = cache.attend(0, q, out_dtype=torch.float32)
    assert torch.allclose(got[:2], want[:2], rtol=0, atol=1e-5) and torch.isfinite(got).all()
    with pytest.raises(MuZeroKernelError, match="outside"):
        cache.check()
    cache.lengths[2:] = -5
    assert (cache.attend(0, q)[2:] == 0).all()
    cache.check()


def test_refusals():
    import muzero_b200 as mz
    cache = make(2, 2, 64, "bf16", 0)
    k = torch.zeros(2, 2, 64, dtype=torch.bfloat16, device="cuda")
    for call in (lambda: cache.append(0, k.half(), k), lambda: cache.append(0, k, k[:1]), lambda: cache.append(0, k[:1], k[:1]), lambda: cache.append(0, k.cpu(), k),
                 lambda: cache.extend(rows=torch.tensor([0], device="cuda")), lambda: cache.extend(rows=ints(0, 1), offsets=ints(0, 1)),
                 lambda: cache.attend(0, torch.zeros(2, 1, 4, 32, dtype=torch.bfloat16, device="cuda")), lambda: cache.attend(0, torch.zeros(2, 1, 4, 64, device="cuda")),
                 lambda: cache.attend(0, k.view(2, 1, 2, 64), out=torch.zeros(3, device="cuda")), lambda: cache.fork(ints(0, 1), ints(1)),
                 lambda: cache.attend(0, k.view(2, 1, 2, 64), rows=ints(0)),
                 lambda: mz.MuZeroPagedCache.allocate(layers=1, kv_heads=1, head_dim=96, pages=1, rows=1, max_length=64),
                 lambda: mz.MuZeroPagedCache.allocate(layers=1, kv_heads=1, head_dim=64, pages=1, rows=1, max_length=64, residual_length=100),
                 lambda: mz.MuZeroPagedCache.allocate(layers=1, kv_heads=1, head_dim=64, pages=1, rows=1, max_length=64, dtype=torch.float32)):
        with pytest.raises(ValueError):
            call()
    for call in (lambda: cache.append(5, k, k), lambda: cache.attend(0, torch.zeros(2, 1, 3, 64, dtype=torch.bfloat16, device="cuda")),
                 lambda: cache.attend(0, k.view(2, 1, 2, 64), out_dtype=torch.float16)):
        with pytest.raises(mz.kernels.MuZeroKernelError):
            call()


def test_streams_and_graphs():
    """A decode step captured in a graph, replayed on tensors that change, equals eager calls; two streams have workspaces of their own."""
    kvh, hq, d = 2, 8, 128
    a, b = make(2, kvh, d, "bf16", 64), make(2, kvh, d, "bf16", 64)
    fill(a, [150, 300], 1)
    fill(b, [150, 300], 1)
    k, v = (x.cuda() for x in tokens(2, kvh, d, torch.bfloat16, 50))
    q = torch.randn(2, 1, hq, d, device="cuda", dtype=torch.bfloat16)
    a.attend(0, q)                                                 # tables are in place before the capture
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        a.extend()
        a.append(0, k, v)
        out = a.attend(0, q)
    for step in range(140):
        nk, nv = (x.cuda() for x in tokens(2, kvh, d, torch.bfloat16, 60 + step))
        k.copy_(nk)
        v.copy_(nv)
        q.normal_()
        graph.replay()
        b.extend()
        b.append(0, k, v)
        assert torch.equal(out, b.attend(0, q)), step
    for x in ("store", "tail", "block_table", "lengths", "page_refs"):
        assert torch.equal(getattr(a, x), getattr(b, x)), x
    with torch.cuda.stream(side):
        side.wait_stream(torch.cuda.default_stream())
        other = b.attend(0, q)
    torch.cuda.synchronize()
    assert torch.equal(other, out)
    a.check()


def test_runs_are_equal_bit_for_bit():
    cache = make(5, 4, 128, "bf16", 128, pages=400, max_length=6000)
    fill(cache, [5000, 1, 900, 128, 3000], 1)
    q = torch.randn(5, 1, 16, 128, device="cuda", dtype=torch.bfloat16)
    first = cache.attend(0, q, out_dtype=torch.float32)
    for _ in range(20):
        assert torch.equal(cache.attend(0, q, out_dtype=torch.float32), first)


def test_a_machine_full_of_steps():
    """More steps than twice the CTAs (parts of unlike size), many short rows between, and rows that share pages."""
    kvh, hq, d = 8, 32, 128
    lengths = [9000, 0, 3, 4500, 64, 200] + [130, 0, 700, 1] * 6
    cache = make(len(lengths) + 1, kvh, d, "bf16", 0, max_length=9200, pages=1200)
    kv = fill(cache, lengths + [0], 1)
    cache.fork(ints(3), ints(len(lengths)))
    kv[len(lengths)] = kv[3]
    q = torch.randn(len(lengths) + 1, 1, hq, d, device="cuda", dtype=torch.bfloat16)
    out = cache.attend(0, q, out_dtype=torch.float32)
    for r in (0, 1, 2, 3, 5, 8, len(lengths)):
        k, v = plain.held(f32(kv[r][0]), f32(kv[r][1]), 0)
        want = plain.attention(f32(q[r].cpu()), k, v, d ** -0.5)
        assert np.linalg.norm(out[r].double().cpu().numpy() - want) <= 3e-5 * max(np.linalg.norm(want), 1e-30), r
    same = cache.attend(0, q[:1].expand(2, 1, hq, d), rows=ints(3, len(lengths)), out_dtype=torch.float32)
    assert torch.allclose(same[0], same[1], rtol=0, atol=1e-5)      # the same tokens, cut elsewhere


def test_many_rows():
    """The most rows that a call takes, each in a place of its own."""
    n, d = 1024, 64
    cache = make(n, 1, d, "fp16", 0, max_length=256, pages=4 * n)
    lengths = [(i * 37) % 200 for i in range(n)]
    kv = fill(cache, lengths, 1)
    q = torch.randn(n, 1, 1, d, device="cuda", dtype=torch.float16)
    order = torch.randperm(n, generator=torch.Generator().manual_seed(0))
    out = cache.attend(0, q, rows=order.int().cuda(), out_dtype=torch.float32)
    for i in (0, 1, 500, 1022, 1023):
        r = int(order[i])
        k, v = plain.held(f32(kv[r][0]), f32(kv[r][1]), 0)
        want = plain.attention(f32(q[i].cpu()), k, v, d ** -0.5)
        assert np.linalg.norm(out[i].double().cpu().numpy() - want) <= 3e-5 * np.linalg.norm(want) + 1e-30, i
    with pytest.raises(Exception, match="1024"):
        cache.attend(0, torch.zeros(1025, 1, 1, d, device="cuda", dtype=torch.float16), rows=torch.zeros(1025, dtype=torch.int32, device="cuda"))


def test_offsets_past_32_bits():
    """A pool of more than 2^32 bytes, pages in its last part, and compaction from there."""
    kvh, d = 8, 128
    pages = (1 << 32) // (kvh * 72 * d) + 40
    cache = make(1, kvh, d, "bf16", 0, max_length=640, pages=pages)
    cache.page_refs[:pages - 30] = 1                               # taken, as if by others
    kv = fill(cache, [500], 1)
    assert int(cache.block_table[0, 0]) == pages - 30
    assert_row(cache, 0, *kv[0])
    q = torch.randn(1, 1, 32, d, device="cuda", dtype=torch.bfloat16)
    before = cache.attend(0, q)
    cache.page_refs[5:12] = 0
    cache.compact()
    assert cache.block_table[0, :7].tolist() == list(range(5, 12))
    assert torch.equal(cache.attend(0, q), before)
    assert_row(cache, 0, *kv[0])


CHILD = r"""
import ctypes, sys, torch
sys.path.insert(0, {root!r})
import muzero_b200 as mz
from muzero_b200.kernels._cabi import load_library
lib = load_library()
assert lib.mz_bounds_violations(None, None, None, 0) == 0
cache = mz.MuZeroPagedCache.allocate(layers=1, kv_heads=2, head_dim=128, pages=64, rows=3, max_length=2048)
o = torch.tensor([0, 900, 901, 1300], dtype=torch.int32, device="cuda")
cache.extend(offsets=o)
k, v = (torch.randn(1300, 2, 128, device="cuda", dtype=torch.bfloat16) for _ in range(2))
cache.append(0, k, v, offsets=o)
q = torch.randn(3, 1, 8, 128, device="cuda", dtype=torch.bfloat16)
good = cache.attend(0, q)
assert torch.isfinite(good).all()
lib.mz_debug_fail_waits(1)
bad = cache.attend(0, q)
torch.cuda.synchronize()
lib.mz_debug_fail_waits(0)
assert torch.isnan(bad[0]).all() and torch.isnan(bad[2]).all() and torch.equal(bad[1], good[1])     # row 1 has no pages: no products to wait for
assert torch.equal(cache.attend(0, q), good)
cache.check()
assert lib.mz_bounds_violations(None, None, None, 0) == 0
print("paged checked build ok")
"""


def test_checked_build_and_waits_that_run_out():
    """In the checked build: no guarded store out of bounds; products that never come make the rows that needed them NaN, the call ends, the next one is right."""
    import os
    import subprocess
    import sys
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    lib = os.path.join(root, "muzero_b200", "lib", "libmuzero_b200_bounds.so")
    if not os.path.exists(lib):
        pytest.skip("the checked library has not been built")
    env = dict(os.environ, MUZERO_B200_LIB=lib)
    res = subprocess.run([sys.executable, "-c", CHILD.format(root=root)], env=env, capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and "paged checked build ok" in res.stdout, res.stdout + res.stderr


def test_the_example_runs(capsys):
    import importlib.util
    import os
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_serving.py")
    spec = importlib.util.spec_from_file_location("paged_serving", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    out = m.main(["--layers", "2", "--rows", "6", "--prefix", "300", "--requests", "15", "--new-tokens", "40"])
    assert out["requests"] >= 15 and out["error"] <= 2.0 ** -8          # bf16 output
