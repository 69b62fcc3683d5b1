"""GPU: an extension that is refused, for whatever reason, leaves the cache as it was, and so do the appends that follow it; the next one that succeeds
counts, whether or not anybody has asked for the error meanwhile."""
import pytest
import torch

from test_gpu_paged import assert_row, check_attention, fill, ints, make, tokens

pytestmark = pytest.mark.gpu
NAMES = ("store", "tail", "block_table", "lengths", "page_refs")


def state_of(cache):
    return [getattr(cache, n).clone() for n in NAMES]


def assert_unchanged(cache, state):
    for name, was in zip(NAMES, state):
        assert torch.equal(getattr(cache, name), was), name


@pytest.mark.parametrize("residual", [0, 64])
@pytest.mark.parametrize("rows, offsets, count", [([0, 9], None, 2), ([1, -1], [0, 70, 71], 71), ([0, 2], [0, 5, 3], 5), ([2, 0, 1], [0, 66, 130, 129], 130)])
def test_a_bad_index_among_good_ones_changes_nothing(rows, offsets, count, residual):
    """Rows that end just behind a page's end, one of them sharing its pages: an append that took the refused tokens for announced ones would write over the
    newest live tokens and quantize a shared page anew."""
    from muzero_b200.kernels import MuZeroKernelError
    cache = make(3, 2, 64, "bf16", residual)
    kv = fill(cache, [residual + 130, residual + 65], 1)
    cache.fork(ints(0), ints(2))
    state = state_of(cache)
    k, v = (x.cuda() for x in tokens(count, 2, 64, torch.bfloat16, 7))
    o = None if offsets is None else ints(*offsets)
    for asked in (False, True):                                    # the error is asked for before the append, or after it
        cache.extend(rows=ints(*rows), offsets=o)
        if asked:
            with pytest.raises(MuZeroKernelError, match="outside"):
                cache.check()
        cache.append(0, k, v, rows=ints(*rows), offsets=o)
        assert_unchanged(cache, state)
        with pytest.raises(MuZeroKernelError, match="outside"):    # (the append reports the bad index as well)
            cache.check()
    cache.append(0, k[:1], v[:1], rows=ints(0))                    # good lists, but nothing has been announced
    assert_unchanged(cache, state)
    cache.check()
    q = torch.randn(3, 1, 4, 64, device="cuda", dtype=torch.bfloat16)
    check_attention(cache, {0: kv[0], 1: kv[1], 2: kv[0]}, q, [0, 1, 2])


@pytest.mark.parametrize("asked", [False, True])
def test_the_next_extension_counts(asked):
    """Too few pages, then room, then an extension that succeeds: its tokens are written although nobody has asked for the error in between."""
    from muzero_b200.kernels import MuZeroKernelError
    kvh, d = 2, 128
    cache = make(3, kvh, d, "bf16", 0, pages=4, max_length=512, layers=2)
    kv = [fill(cache, [100, 64, 70], 1)]
    k1, v1 = tokens(100, kvh, d, torch.bfloat16, 33)
    offs = ints(0, 100)
    cache.append(1, torch.cat([x[0] for x in kv[0]]).cuda(), torch.cat([x[1] for x in kv[0]]).cuda(), offsets=ints(0, 100, 164, 234))
    state = state_of(cache)
    lost, lost_v = tokens(200, kvh, d, torch.bfloat16, 34)
    cache.extend(rows=ints(0), offsets=ints(0, 200))               # needs three pages, one is free
    for layer in range(2):
        cache.append(layer, lost.cuda(), lost_v.cuda(), rows=ints(0), offsets=ints(0, 200))
    assert_unchanged(cache, state)
    if asked:
        with pytest.raises(MuZeroKernelError, match="free pages"):
            cache.check()
    cache.free(ints(1))
    cache.extend(rows=ints(0), offsets=offs)
    for layer in range(2):
        cache.append(layer, k1.cuda(), v1.cuda(), rows=ints(0), offsets=offs)
    row = tuple(torch.cat([a, b]) for a, b in zip(kv[0][0], (k1, v1)))
    for layer in range(2):
        assert_row(cache, 0, *row, layer=layer)
        assert_row(cache, 2, *kv[0][2], layer=layer)
    got = cache.attend(1, torch.ones(1, 4, d, device="cuda", dtype=torch.bfloat16), rows=ints(0))
    assert torch.isfinite(got).all()
    if not asked:
        with pytest.raises(MuZeroKernelError, match="free pages"):
            cache.check()
    cache.check()
    q = torch.randn(2, 1, 4, d, device="cuda", dtype=torch.bfloat16)
    check_attention(cache, {0: row, 2: kv[0][2]}, q, [0, 2], layer=1)


def test_a_captured_step_goes_on_after_a_refusal():
    """A captured step runs out of pages, room is made between two replays, and the replays that follow write what they announce."""
    from muzero_b200.kernels import MuZeroKernelError
    kvh, d = 1, 64
    cache = make(2, kvh, d, "fp16", 0, pages=2, max_length=512)
    kv = fill(cache, [64, 127], 1)                                 # both pages are taken, row 1 needs another one with its next token
    k, v = (torch.zeros(1, kvh, d, dtype=torch.float16, device="cuda") for _ in range(2))
    rows = ints(1)
    cache.attend(0, torch.zeros(1, 1, 2, d, dtype=torch.float16, device="cuda"), rows=rows)
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        cache.extend(rows=rows)
        cache.append(0, k, v, rows=rows)
    new = tokens(5, kvh, d, torch.float16, 9)
    state = state_of(cache)
    for step in range(5):
        k.copy_(new[0][step:step + 1])
        v.copy_(new[1][step:step + 1])
        graph.replay()
        if step == 0:
            assert_unchanged(cache, state)                         # refused: token 0 is lost, and that is reported
            cache.free(ints(0))
    assert_row(cache, 1, torch.cat([kv[1][0], new[0][1:]]), torch.cat([kv[1][1], new[1][1:]]))
    with pytest.raises(MuZeroKernelError, match="free pages"):
        cache.check()
