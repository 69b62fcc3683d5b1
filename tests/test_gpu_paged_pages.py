"""GPU: attention over what pages hold: bytes that no append has written, rows of very unlike scales."""
import pytest
import torch

from test_gpu_paged import fill, make

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
