"""Paged cache, what needs no GPU: the codec's tables and quality, the ABI's structs, refusals."""
import ctypes
import os
import subprocess
import tempfile

import numpy as np
import pytest
import torch

from paged_plain import BOOK, NEAREST, dequantize, quantize

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))


def test_books_of_the_library():
    from muzero_b200.kernels._cabi import load_library
    book, nearest = np.zeros((128, 16), np.uint8), np.zeros((128, 128), np.uint8)
    assert load_library().mz_paged_books(book.ctypes.data, nearest.ctypes.data) == 0
    assert np.array_equal(book, BOOK) and np.array_equal(nearest, NEAREST)
    # what the kernels rely on: seven bits, ascending, the zero level exact, both ends reached (but for the few books whose last code is the zero level)
    assert BOOK.max() <= 127 and BOOK.min() >= 0 and (np.diff(BOOK, axis=1) > 0).all()
    z = np.arange(128)
    assert all(z[i] in BOOK[i] for i in z)
    assert load_library().mz_paged_books(None, None) == 1


@pytest.mark.parametrize("shift", [0.0, 0.7, 3.0])
def test_codec_error_is_that_of_the_contiguous_codec(oracle, shift):
    """Levels in 127ths instead of exact ones: at most 2 % more error than the contiguous store's codec on the same rows.  (A level is off by at most half
    a 127th of the range where neighbouring levels are 5 to 14 apart: 0.5 / sqrt(3) against gaps / sqrt(12) of 2.7 on average adds about 1 %.)"""
    x = (torch.randn(4000, 64, generator=torch.Generator().manual_seed(3)) + shift)
    back = torch.from_numpy(dequantize(*quantize(x.numpy())))
    packed, mn, scale = oracle.quantize_rows_oracle(x, 4, 2.0, 1e-8, torch.float16)
    ref = oracle.dequantize_rows_oracle(packed, mn, scale, 4, 2.0, 64, torch.float32)
    mine, theirs = (back - x).pow(2).mean().sqrt(), (ref.double() - x).pow(2).mean().sqrt()
    assert mine <= 1.02 * theirs, (mine, theirs)


def test_codec_error_is_within_half_a_gap():
    """|x - value| is at most half the gap between the levels beside x, plus what two roundings may add: half a level where x is rounded to one, and another 0.57
    where the zero level is rounded and the scale is (f16, 2^-11 of 127 levels)."""
    rng = np.random.default_rng(5)
    x = np.concatenate([rng.standard_normal((200, 64)) * s + c for s, c in ((1, 0), (1e-2, 0), (50, 0), (1, 4), (1, -9))]).astype(np.float32)
    codes, words = quantize(x)
    t = (words & 0xFFFF).astype(np.uint16).view(np.float16).astype(np.float64) / 32
    err = np.abs(dequantize(codes, words) - x) / t[:, None]
    gap = np.diff(BOOK, axis=1).max()
    assert err.max() <= gap / 2 + 0.5 + 0.57


def test_structs_match_the_header():
    from muzero_b200.kernels import _cabi
    src = '#include <stdio.h>\n#include "muzero_b200.h"\nint main(){printf("%zu %zu\\n", sizeof(mz_paged_cache), sizeof(mz_paged_attention_args));return 0;}\n'
    with tempfile.TemporaryDirectory() as td:
        c, exe = os.path.join(td, "s.c"), os.path.join(td, "s")
        open(c, "w").write(src)
        subprocess.check_call(["gcc", "-I", os.path.join(ROOT, "include"), c, "-o", exe])
        a, b = map(int, subprocess.check_output([exe]).split())
    assert ctypes.sizeof(_cabi.PagedCache) == a and ctypes.sizeof(_cabi.PagedAttentionArgs) == b


def _cache(**kw):
    from muzero_b200.kernels._cabi import MZ_BF16, PagedCache
    at = 1 << 20                                  # never dereferenced: the calls are refused before a launch
    f = dict(layers=2, rows=4, pages=8, width=3, kv_heads=2, head_dim=128, residual=128, ring=256, kv_dtype=MZ_BF16, store=at, store_stride_layer=8 * 18432,
             store_stride_page=18432, tail=at, tail_stride_layer=4 * 131072, tail_stride_row=131072, block_table=at, lengths=at, page_refs=at, status=at)
    f.update(kw)
    return PagedCache(**f)


@pytest.mark.parametrize("field, value", [("head_dim", 96), ("kv_dtype", 0), ("residual", 100), ("residual", -64), ("ring", 128), ("pages", 0), ("store", None),
                                          ("store", (1 << 20) + 8), ("store_stride_page", 1000), ("tail_stride_row", 4), ("lengths", None), ("width", 1 << 25)])
def test_a_cache_that_cannot_be_is_refused(field, value):
    from muzero_b200.kernels import _cabi
    lib = _cabi.load_library()
    c = _cache(**{field: value})
    assert lib.mz_paged_extend(c, None, None, 1, None) == 1
    assert lib.mz_paged_free(c, 1 << 20, 1, None) == 1
    assert lib.mz_paged_fork(c, 1 << 20, 1 << 20, 1, None) == 1
    assert lib.mz_paged_copy_pages(c, 1 << 20, 1 << 20, 1, None) == 1
    assert lib.mz_paged_append(c, 0, 1 << 20, 256, 128, 1 << 20, 256, 128, None, None, 1, 1, 1, None) == 1
    assert lib.mz_paged_compact(c, 1 << 20, 1 << 20, None) == 1
    assert lib.mz_paged_compact_workspace_bytes(c) == 0
    assert lib.mz_paged_attention(c, 0, _cabi.PagedAttentionArgs(), None) == 1
    assert _cabi.last_error()


def test_calls_that_cannot_be_are_refused():
    from muzero_b200.kernels import _cabi
    lib, c, at = _cabi.load_library(), _cache(), 1 << 20
    assert lib.mz_paged_extend(c, None, None, 5, None) == 1                               # more entries than rows
    assert lib.mz_paged_extend(c, at, None, 5000, None) == 1
    assert lib.mz_paged_extend(c, None, None, 0, None) == 0                               # nothing to do
    assert lib.mz_paged_append(c, 2, at, 256, 128, at, 256, 128, None, None, 1, 1, 1, None) == 1       # no such layer
    assert lib.mz_paged_append(c, 0, at, 256, 128, at, 256, 128, None, None, 2, 3, 1, None) == 1       # three tokens for two rows
    assert lib.mz_paged_append(c, 0, at + 2, 256, 128, at, 256, 128, None, None, 1, 1, 1, None) == 1   # not aligned
    assert lib.mz_paged_append(c, 0, at, 257, 128, at, 256, 128, None, None, 1, 1, 1, None) == 1
    assert "aligned" in _cabi.last_error()
    assert lib.mz_paged_append(c, 0, None, 256, 128, None, 256, 128, None, None, 0, 0, 0, None) == 0
    assert lib.mz_paged_compact(c, at, 4, None) == 4 and "workspace" in _cabi.last_error()
    assert lib.mz_paged_fork(c, at, at, 5, None) == 1
    assert lib.mz_paged_fork(c, None, None, 1, None) == 1
    assert lib.mz_paged_copy_pages(c, at, at, 9, None) == 1


def test_cpu_tensors_are_rejected():
    import muzero_b200 as mz
    from muzero_b200.kernels import MuZeroKernelError
    with pytest.raises(MuZeroKernelError):
        mz.MuZeroPagedCache.allocate(layers=1, kv_heads=2, head_dim=64, pages=4, rows=2, max_length=256, device="cpu")


def test_sizes():
    from muzero_b200.cache.paged import packed_tokens, page_bytes
    assert page_bytes(128) == 9216 and page_bytes(64) == 4608
    assert [packed_tokens(n, 128) for n in (0, 1, 128, 191, 192, 255, 256, 4224)] == [0, 0, 0, 0, 64, 64, 128, 4096]
    assert [packed_tokens(n, 0) for n in (0, 63, 64, 65)] == [0, 0, 64, 64]
