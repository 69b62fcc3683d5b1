"""GPU: the paged cache's calls: what the host refuses, first calls, arguments at their limits."""
import os
import subprocess
import sys

import pytest
import torch

from test_gpu_paged import assert_row, ints, make, tokens

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


FIRST = r"""
import sys, torch
sys.path[:0] = [{root!r}, {root!r} + "/tests"]
import paged_plain as plain
from test_gpu_paged import assert_row, check_attention, ints, make, tokens
cache = make(2, 2, 128, "bf16", 0, pages=16, max_length=640)
k, v = tokens(330, 2, 128, torch.bfloat16, 3)
kd, vd, q = k.cuda(), v.cuda(), torch.randn(2, 1, 8, 128, device="cuda", dtype=torch.bfloat16)
o, rows = ints(0, 200, 330), ints(0, 1)
torch.cuda.synchronize()
side = torch.cuda.Stream()
if {captured}:
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph, stream=side):
        cache.extend(offsets=o)
        cache.append(0, kd, vd, offsets=o)
        out = cache.attend(0, q)
    graph.replay()
else:
    with torch.cuda.stream(side):
        cache.extend(offsets=o)
        cache.append(0, kd, vd, offsets=o)
        out = cache.attend(0, q)
torch.cuda.synchronize()
cache.check()
kv = [(k[:200], v[:200]), (k[200:], v[200:])]
for r in range(2):
    assert_row(cache, r, *kv[r])
check_attention(cache, kv, q, [0, 1])
assert torch.equal(out, cache.attend(0, q))
print("first call ok")
"""


@pytest.mark.parametrize("captured", [True, False])
def test_the_first_calls_of_a_process(captured):
    """The first calls of all stand in a captured graph, or on a stream that does not wait for the legacy one: the codec's tables are in place."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    res = subprocess.run([sys.executable, "-c", FIRST.format(root=root, captured=captured)], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and "first call ok" in res.stdout, res.stdout + res.stderr


@pytest.mark.parametrize("most", [300, 301, 1 << 20, (1 << 31) - 64, (1 << 31) - 63, (1 << 31) - 1])
def test_a_bound_on_new_tokens_may_be_any(most):
    """`max_new` is a bound: the largest there is does no more than the tokens' number."""
    cache = make(2, 1, 64, "bf16", 64)
    k, v = tokens(310, 1, 64, torch.bfloat16, 4)
    o = ints(0, 300, 310)
    cache.extend(offsets=o)
    cache.append(0, k.cuda(), v.cuda(), offsets=o, max_new=most)
    cache.check()
    assert_row(cache, 0, k[:300], v[:300])
    assert_row(cache, 1, k[300:], v[300:])


def test_the_example_checks_rows_that_were_decoded():
    """The serving example checks a decoded row, a branch and the prefix in every layer (bf16 output), and a row's keys against those that were written (error of
    the 4-bit codec on normal rows: 0.085)."""
    import importlib.util
    path = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "examples", "paged_serving.py")
    spec = importlib.util.spec_from_file_location("paged_serving", path)
    m = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(m)
    out = m.main(["--layers", "3", "--rows", "8", "--prefix", "500", "--requests", "40", "--new-tokens", "96", "--seed", "1"])
    assert out["branches"] > 0 and set(out["errors"]) == {"first", "branch", "prefix"}
    assert max(out["errors"].values()) <= 2.0 ** -8 and 0.0 < out["held"] <= 0.1
