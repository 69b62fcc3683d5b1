"""GPU: the tables of the compander are in place for the first call, whatever its stream."""
import os
import subprocess
import sys

import pytest

pytestmark = pytest.mark.gpu

FIRST = r"""
import sys, torch
sys.path.insert(0, {root!r})
import muzero_b200 as mz
x = torch.randn(4096, 64, generator=torch.Generator().manual_seed(1)).bfloat16().cuda()
torch.cuda.synchronize()
side = torch.cuda.Stream()
with torch.cuda.stream(side):
    first = [mz.quantize_rows(x, {bits}, 2.0, 1e-8, torch.bfloat16)]
    first.append(mz.dequantize_rows(*first[0], {bits}, 2.0, 64, torch.float32))
torch.cuda.synchronize()
again = [mz.quantize_rows(x, {bits}, 2.0, 1e-8, torch.bfloat16)]
again.append(mz.dequantize_rows(*again[0], {bits}, 2.0, 64, torch.float32))
torch.cuda.synchronize()
assert all(torch.equal(a, b) for a, b in zip(first[0], again[0])) and torch.equal(first[1], again[1])
print("first call ok")
"""


@pytest.mark.parametrize("bits", [4, 8])
def test_first_call_on_a_stream_of_its_own(bits):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    res = subprocess.run([sys.executable, "-c", FIRST.format(root=root, bits=bits)], capture_output=True, text=True, timeout=300)
    assert res.returncode == 0 and "first call ok" in res.stdout, res.stdout + res.stderr
