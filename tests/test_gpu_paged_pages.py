"""GPU: attention over what pages hold: bytes that no append has written, rows of very unlike scales."""
import numpy as np
import pytest
import torch

import paged_plain as plain
from test_gpu_paged import DT, check_attention, f32, fill, ints, make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("group", [2, 8])
def test_pages_of_any_bytes(d, group):
    """Pages that nobody has written (a store taken over as it was): the call ends, whatever the words say, rows beside them keep their results, and so does the next
    call.  Every upper half of a word that is no anchor stands for a zero level between 0 and 127, its sign bit set or not."""
    cache = make(3, 2, d, "bf16", 0, pages=40)
    fill(cache, [640, 300, 200], 1)
    q = torch.randn(3, 1, 2 * group, d, device="cuda", dtype=torch.bfloat16)
    want, store = cache.attend(0, q, out_dtype=torch.float32), cache.store.clone()
    mine = cache.block_table[0, :10].long()
    words = torch.cat([torch.arange(32 * d, 36 * d), torch.arange(68 * d, 72 * d)]).view(-1, 4).cuda()
    halves = torch.arange(words.shape[0], device="cuda") % 256
    halves = halves % 128 | (halves // 128) << 15                 # 0 .. 127 and 0x8000 .. 0x807f
    for form in range(3):
        if form == 0:
            cache.store[:, mine] = torch.randint(0, 256, cache.store[:, mine].shape, device="cuda", dtype=torch.uint8)
        elif form == 1:
            cache.store[:, mine] = 255
        else:
            cache.store[:, mine] = 0
            page = cache.store[0, mine]
            page[:, :, words[:, 1]] = 0x3c                         # T = 1
            page[:, :, words[:, 2]] = (halves & 255).byte()
            page[:, :, words[:, 3]] = (halves >> 8).byte()
            cache.store[0, mine] = page
        got = cache.attend(0, q, out_dtype=torch.float32)
        torch.cuda.synchronize()
        assert torch.allclose(got[1:], want[1:], rtol=0, atol=1e-5 * float(want.abs().max()))
    assert torch.isfinite(got).all()                               # (the last form's words are all in order but for their sign)
    cache.store.copy_(store)
    assert torch.equal(cache.attend(0, q, out_dtype=torch.float32), want)
    cache.check()


def scales_case(d, k, v, q):
    """one row of k, v [n, 1, d], queries q [1, 1, heads, d] -> output and the same in 64 bits, [heads, d], and the pages' largest T on either side"""
    k, v, q = k.bfloat16(), v.bfloat16(), q.bfloat16()
    cache = make(1, 1, d, "bf16", 0)
    o = ints(0, k.shape[0])
    cache.extend(offsets=o)
    cache.append(0, k.cuda(), v.cuda(), offsets=o)
    got = cache.attend(0, q.cuda(), out_dtype=torch.float32)[0, 0].double().cpu().numpy()
    want = plain.attention(f32(q[0]), *plain.held(f32(k), f32(v), 0), d ** -0.5)[0]
    top = []
    for words in (plain.quantize(f32(k[:, 0]).reshape(-1, 64, d).swapaxes(1, 2))[1], plain.quantize(f32(v[:, 0]).reshape(-1, 64))[1]):
        top.append(float((words & 0xFFFF).astype(np.uint16).view(np.float16).max()))
    return got, want, top


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("ratio", [0, 4, 7, 10, 12, 14])
def test_channels_of_unlike_scales(d, ratio):
    """Key channels 2^ratio times as large as the others, whose queries are as much smaller, or zero.  q T is rounded to 2^-31 of a power of two above the product of the
    largest |q| and T (both up to twice those), levels are 64 / 32 in the mean: an error of a logit of sqrt(d) * 2^-29 * |q| T * 2 / sqrt(3) * scaling in the mean square, and
    of the output as large in parts of it; twice that, beside the tolerance of ordinary rows."""
    gen = torch.Generator().manual_seed(ratio)
    k, v, q = (torch.randn(*s, generator=gen) for s in ((1024, 1, d), (1024, 1, d), (1, 1, 4, d)))
    for c, factor in ((5, 2.0 ** -ratio), (17, 0.0)):
        k[..., c] *= 2.0 ** ratio
        q[..., c] *= factor
    got, want, (top, _) = scales_case(d, k, v, q)
    for h in range(4):
        logit = d ** 0.5 * 2.0 ** -29 * float(q[0, 0, h].abs().max()) * top * 2 / 3 ** 0.5 * d ** -0.5
        assert np.linalg.norm(got[h] - want[h]) <= (3e-5 + 2 * logit) * np.linalg.norm(want[h]), h


@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("ratio, bits", [(0, 0), (4, 0), (10, 0), (4, 6), (7, 9), (10, 12), (13, 15)])
def test_tokens_of_unlike_scales(d, ratio, bits):
    """Every 64th token's value is 2^ratio times as large as the others', and its probability 2^-bits times as large.  p T is rounded to 2^-31 of a power of two above the
    largest T (up to twice that): an error of each channel of sqrt(tokens) * 2^-30 * T * 2 / sqrt(3) in the mean square, before the division by a sum of at least 1; twice
    that, beside the tolerance of ordinary rows."""
    n = 1024
    gen = torch.Generator().manual_seed(ratio + bits)
    k, v, q = (torch.randn(*s, generator=gen) for s in ((n, 1, d), (n, 1, d), (1, 1, 4, d)))
    v[::64] *= 2.0 ** ratio
    q[..., 3], k[..., 3] = 4.0, 0.0
    k[::64, :, 3] = -bits * 0.6931 * d ** 0.5 / 4
    got, want, (_, top) = scales_case(d, k, v, q)
    for h in range(4):
        assert np.linalg.norm(got[h] - want[h]) <= 3e-5 * np.linalg.norm(want[h]) + 2 * (n * d) ** 0.5 * 2.0 ** -30 * top * 2 / 3 ** 0.5, h


@pytest.mark.parametrize("bits", [4, 8, 12, 16])
def test_a_token_that_takes_nearly_all(bits):
    """The first token has 2^bits times the probability of the others and hardly a value: what the others carry keeps the precision that p T of 31 bits leaves it, of
    n tokens whose p is 2^-bits (bound as above, T as for ordinary rows)."""
    n, d = 1024, 128
    gen = torch.Generator().manual_seed(bits)
    k, v, q = (torch.randn(*s, generator=gen) for s in ((n, 1, d), (n, 1, d), (1, 1, 4, d)))
    v[0] *= 1e-3
    q[..., 3], k[..., 3] = 4.0, 0.0
    k[0, :, 3] = bits * 0.6931 * d ** 0.5 / 4
    got, want, (_, top) = scales_case(d, k, v, q)
    for h in range(4):
        assert np.linalg.norm(got[h] - want[h]) <= 3e-5 * np.linalg.norm(want[h]) + 2 * (n * d) ** 0.5 * 2.0 ** -30 * top * 2 / 3 ** 0.5, h


@pytest.mark.parametrize("d, dt, kvh, hq, residual, lq", [(128, "bf16", 1, 3, 0, 130), (64, "fp16", 2, 4, 64, 77), (128, "bf16", 2, 8, 128, 33), (64, "bf16", 1, 8, 0, 64)])
def test_a_block_of_new_tokens(d, dt, kvh, hq, residual, lq):
    """As many query tokens as a short prompt has: their own tokens stand in pages and in the window, some rows are shorter than the block."""
    lengths = [lq + 200, lq, lq - 20, 1, 0, 300]
    cache = make(len(lengths), kvh, d, dt, residual)
    kv = fill(cache, lengths, 1, seed=lq)
    q = torch.randn(len(lengths), lq, hq, d, generator=torch.Generator().manual_seed(hq)).to(DT[dt]).cuda()
    check_attention(cache, kv, q, list(range(len(lengths))))
