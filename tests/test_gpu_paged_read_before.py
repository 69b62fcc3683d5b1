"""GPU: reading from before a row's first token: zeros, as for every token that a row does not have, and nothing is left unwritten."""
import pytest
import torch

from test_gpu_paged import fill, ints, make
from test_gpu_paged_read import expected

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dt, out", [(torch.bfloat16, torch.bfloat16), (torch.bfloat16, torch.float32)])
def test_a_batch_padded_on_the_left(dt, out):
    lengths, most = [0, 1, 63, 64, 65, 200, 321], 330
    cache = make(len(lengths), 2, 128, "bf16", 64)
    kv = fill(cache, lengths, 1, seed=4)
    k, v = (torch.full((most * len(lengths), 2, 128), float("nan"), dtype=out, device="cuda") for _ in range(2))
    cache.read(0, offsets=ints(*[most * i for i in range(len(lengths) + 1)]), first=ints(*[n - most for n in lengths]), out=(k, v))
    cache.check()
    for x, side in ((k.cpu(), 0), (v.cpu(), 1)):
        for i, n in enumerate(lengths):
            part = x[most * i:most * (i + 1)]
            assert not part[:most - n].any() and torch.equal(part[most - n:], expected(*kv[i], 64, out)[side]), n


def test_from_far_before_and_past_the_end():
    cache = make(2, 1, 64, "bf16", 0)
    kv = fill(cache, [70, 70], 1)
    firsts, counts = [-2 ** 31, -2 ** 31 + 1, -1, -64, -65, -200, -70], [100, 1, 1, 64, 66, 400, 70]
    offsets = [0]
    for n in counts:
        offsets.append(offsets[-1] + n)
    k, v = (torch.full((offsets[-1], 1, 64), float("nan"), dtype=torch.bfloat16, device="cuda") for _ in range(2))
    cache.read(0, rows=ints(*[i % 2 for i in range(len(counts))]), offsets=ints(*offsets), first=ints(*firsts), out=(k, v))
    cache.check()
    for x, side in ((k.cpu(), 0), (v.cpu(), 1)):
        for i, (first, n) in enumerate(zip(firsts, counts)):
            want = torch.zeros(n, 1, 64, dtype=torch.bfloat16)
            held = expected(*kv[i % 2], 0, torch.bfloat16)[side]
            for t in range(max(first, 0), min(first + n, 70)):
                want[t - first] = held[t]
            assert torch.equal(x[offsets[i]:offsets[i] + n], want), (first, n)
