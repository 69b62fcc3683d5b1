"""GPU: the paged cache's calls: what the host refuses, first calls, arguments at their limits."""
import pytest
import torch

from test_gpu_paged import make

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("off, gap", [(16, 0), (0, 16), (8, 0)])
def test_tensors_that_the_kernels_cannot_read_are_refused(off, gap):
    """A store that begins, or whose pages begin, between 32-byte boundaries; a ring between 16-byte ones: refused before anything reads them."""
    import muzero_b200 as mz
    c = make(2, 2, 64, "bf16", 64, pages=3)
    rest = dict(block_table=c.block_table, lengths=c.lengths, page_refs=c.page_refs, status=c.status, residual_length=64)
    size = 2 * 4608 + gap
    raw = torch.zeros(off + 3 * size, dtype=torch.uint8, device="cuda")
    store = raw[off:].as_strided((1, 3, 2, 4608), (3 * size, size, 4608, 1))
    with pytest.raises(ValueError, match="boundaries"):
        mz.MuZeroPagedCache(store=store, tail=c.tail, **rest)
    tail = torch.zeros(c.tail.numel() + 4, dtype=c.dtype, device="cuda")[4:].view(c.tail.shape)
    with pytest.raises(ValueError, match="boundaries"):
        mz.MuZeroPagedCache(store=c.store, tail=tail, **rest)
