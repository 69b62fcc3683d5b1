"""GPU: tokens of the paged cache read back, against the codec's definition.

A value is A + T w / 32 with a f16 anchor A, a f16 scale T and a whole number w of at most 127: an f32 number unless A's and T w / 32's bits lie more than 24 apart, and the kernel rounds once to f32.  So
f32 output is the definition's value rounded to f32, and 16-bit output that rounded once more: equal, bit for bit, to the same two roundings here.
"""
import numpy as np
import pytest
import torch

import paged_plain as plain
from test_gpu_paged import DT, f32, fill, ints, make, tokens

pytestmark = pytest.mark.gpu


def expected(k, v, residual, dt):
    top = float(torch.finfo(dt).max)
    return tuple(torch.from_numpy(x.astype(np.float32)).clamp(-top, top).to(dt) for x in plain.held(f32(k), f32(v), residual))


CASES = [
    (128, "bf16", 2, 128, [0, 1, 63, 64, 191, 192, 193, 700]),
    (128, "fp16", 1, 64, [64, 127, 128, 129, 1000]),
    (64, "bf16", 3, 0, [1, 63, 64, 65, 128, 640]),
    (64, "fp16", 2, 192, [5, 255, 256, 333]),
]


@pytest.mark.parametrize("d, dt, kvh, residual, lengths", CASES)
@pytest.mark.parametrize("wide", [False, True])
def test_rows_back(d, dt, kvh, residual, lengths, wide):
    cache = make(len(lengths), kvh, d, dt, residual)
    kv = fill(cache, lengths, 2, seed=d)
    out = torch.float32 if wide else DT[dt]
    order = list(range(len(lengths)))[::-1]
    for firsts in ([0] * len(order), [min(n, 70) for n in (lengths[r] for r in order)], [n // 2 for n in (lengths[r] for r in order)]):
        counts = [lengths[r] - f for r, f in zip(order, firsts)]
        offsets = [0] + np.cumsum(counts).tolist()
        first = ints(*firsts) if any(firsts) else None
        k, v = cache.read(0, rows=ints(*order), offsets=ints(*offsets), first=first, tokens=offsets[-1], out_dtype=torch.float32 if wide else None)
        cache.check()
        assert k.dtype == out and k.shape == (offsets[-1], kvh, d)
        for i, r in enumerate(order):
            wk, wv = expected(*kv[r], residual, out)
            assert torch.equal(k[offsets[i]:offsets[i + 1]].cpu(), wk[firsts[i]:]) and torch.equal(v[offsets[i]:offsets[i + 1]].cpu(), wv[firsts[i]:]), r


def test_padded_batches_and_places_of_nobody():
    """Equal steps of offsets: what a row does not have reads as zero.  Places before the first entry, behind the last and of empty entries stay; rows may be repeated."""
    cache = make(3, 2, 128, "bf16", 64)
    kv = fill(cache, [30, 200, 0], 1)
    k, v = (torch.full((5 + 4 * 256 + 9, 2, 128), 7.0, dtype=torch.bfloat16, device="cuda") for _ in range(2))
    offsets = [5 + 256 * i for i in range(5)]
    assert cache.read(0, rows=ints(1, 0, 2, 1), offsets=ints(*offsets), out=(k, v))[0] is k
    for x, side in ((k.cpu(), 0), (v.cpu(), 1)):
        assert (x[:5] == 7).all() and (x[5 + 1024:] == 7).all()
        for i, r in enumerate((1, 0, 2, 1)):
            want = expected(*kv[r], 64, torch.bfloat16)[side]
            assert torch.equal(x[offsets[i]:offsets[i] + len(want)], want) and not x[offsets[i] + len(want):offsets[i + 1]].any()
    # from far behind a row's end, and nothing at all
    k, v = cache.read(0, rows=ints(1, 1), offsets=ints(0, 100, 100), first=ints(2 ** 31 - 1, 0), tokens=100)
    assert not k.any() and not v.any()
    k, v = cache.read(0, offsets=ints(0, 0, 0, 0), tokens=0)
    assert k.shape == (0, 2, 128)
    cache.check()


def test_strided_outputs_and_a_layer_of_several():
    cache = make(2, 4, 64, "fp16", 0, layers=3)
    kv = fill(cache, [150, 77], 1, layer=2)
    by_head = [torch.zeros(4, 230, 64, dtype=torch.float16, device="cuda") for _ in range(2)]
    fused = torch.zeros(230, 4, 3, 64, dtype=torch.float16, device="cuda")
    for k, v in ((by_head[0].transpose(0, 1), by_head[1].transpose(0, 1)), (fused[:, :, 1], fused[:, :, 2])):
        cache.read(2, offsets=ints(0, 150, 227), out=(k, v))
        for at, r in ((0, 0), (150, 1)):
            for x, want in zip((k, v), expected(*kv[r], 0, torch.float16)):
                assert torch.equal(x[at:at + len(want)].cpu(), want)
        assert not k[227:].any()
    assert not fused[:, :, 0].any()


def test_values_at_the_ends_of_the_types():
    """A scale is a f16 number and may be a little too large, so that the level of f16's largest number lies beyond it: held to the type's range."""
    cache = make(1, 1, 128, "fp16", 0)
    k = torch.zeros(64, 1, 128)
    k[::2] = 65504.0
    k[1::4] = -65504.0
    k = k.half()
    cache.extend(offsets=ints(0, 64))
    cache.append(0, k.cuda(), k.cuda(), offsets=ints(0, 64))
    got = cache.read(0, offsets=ints(0, 64), tokens=64)
    for x, want in zip(got, expected(k, k, 0, torch.float16)):
        assert torch.isfinite(x).all() and torch.equal(x.cpu(), want)
    wide = cache.read(0, offsets=ints(0, 64), tokens=64, out_dtype=torch.float32)[0]
    assert wide.abs().max() >= 65504


def test_what_is_wrong_on_the_device_is_reported():
    """Rows that are not there and offsets that are taken back are skipped; a page that is not there reads as zero."""
    cache = make(2, 1, 64, "bf16", 0)
    kv = fill(cache, [200, 200], 1)
    out = [torch.full((300, 1, 64), 3.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    cache.read(0, rows=ints(0, 7, -1), offsets=ints(0, 100, 200, 300), out=tuple(out))
    with pytest.raises(Exception, match="outside the cache"):
        cache.check()
    assert torch.equal(out[0][:100].cpu(), expected(*kv[0], 0, torch.bfloat16)[0][:100]) and (out[0][100:] == 3).all()
    cache.block_table[1, 1] = -1
    k, v = cache.read(0, rows=ints(1), offsets=ints(0, 200), tokens=200)
    with pytest.raises(Exception, match="outside the cache"):
        cache.check()
    assert not k[64:128].any() and not v[64:128].any() and torch.equal(k[:64].cpu(), expected(*kv[1], 0, torch.bfloat16)[0][:64])
    out = [torch.full((50, 1, 64), 3.0, dtype=torch.bfloat16, device="cuda") for _ in range(2)]
    cache.read(0, rows=ints(0, 0), offsets=ints(0, 80, 20), out=tuple(out))       # more places than there are, then none
    assert torch.equal(out[0].cpu(), expected(*kv[0], 0, torch.bfloat16)[0][:50])
    cache.check()


def test_many_entries_and_a_graph():
    cache = make(4, 2, 64, "bf16", 64)
    kv = fill(cache, [100, 65, 400, 1], 1)
    rng = np.random.default_rng(3)
    rows = rng.integers(0, 4, 3000)
    counts = rng.integers(0, 5, 3000)
    first = rng.integers(0, 120, 3000)
    offsets = np.concatenate([[0], np.cumsum(counts)])
    args = dict(rows=ints(*rows.tolist()), offsets=ints(*offsets.tolist()), first=ints(*first.tolist()))
    out = tuple(torch.empty((int(offsets[-1]), 2, 64), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        cache.read(0, out=out, **args)
    graph.replay()
    torch.cuda.synchronize()
    want = [expected(*x, 64, torch.bfloat16) for x in kv]
    for x, side_ in zip(out, range(2)):
        whole = [torch.cat([w[side_], torch.zeros(200, 2, 64, dtype=torch.bfloat16)]) for w in want]
        assert torch.equal(x.cpu(), torch.cat([whole[r][f:f + n] for r, f, n in zip(rows, first, counts)]))
