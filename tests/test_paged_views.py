"""Paged cache: what windows, groups and reading refuse, without a GPU."""
import ctypes

import pytest

from test_paged_host import _cache


def _args(**change):
    from muzero_b200.kernels import _cabi
    at = 1 << 20
    a = _cabi.PagedAttentionArgs(query=at, q_stride_b=1024, q_stride_l=1024, q_stride_h=128, batch=1, q_len=1, q_heads=8, scaling=1.0, out=at, out_dtype=2,
                                 workspace=at, workspace_bytes=1 << 40)
    for k, v in change.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("view, text", [((-1, 0, None, 0), "window -1"), ((5, -1, None, 0), "sinks -1"), ((0, 4, None, 0), "sinks without a window"),
                                        ((5, 0, 1 << 20, 2), "a window bounds"), ((0, 0, 1 << 20, -1), "-1 groups"), ((0, 0, 1 << 20, 1025), "1025 groups")])
def test_views_that_are_refused(view, text):
    from muzero_b200.kernels import _cabi
    lib, v = _cabi.load_library(), _cabi.PagedView(*view)
    assert lib.mz_paged_attention_view(_cache(), 0, _args(), v, None) != 0 and text in _cabi.last_error()
    assert lib.mz_paged_attention_view_workspace_bytes(_cache(), v, 1, 1, 8) == 0


def test_views_share_the_checks_of_attention():
    from muzero_b200.kernels import _cabi
    lib, v = _cabi.load_library(), _cabi.PagedView(100, 0, None, 0)
    for change, text in ((dict(q_heads=7), "q_heads 7"), (dict(batch=1025), "batch 1025"), (dict(out_dtype=1), "out_dtype")):
        assert lib.mz_paged_attention_view(_cache(), 0, _args(rows=1 << 20, **change), v, None) != 0 and text in _cabi.last_error()
    assert lib.mz_paged_attention_view(_cache(), 99, _args(), v, None) != 0 and "layer 99" in _cabi.last_error()
    assert lib.mz_paged_attention_view(_cache(), 0, _args(), None, None) != 0 and "view is NULL" in _cabi.last_error()


def test_structs_match_the_header():
    import os
    import subprocess
    import tempfile
    from muzero_b200.kernels import _cabi
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    src = '#include <stdio.h>\n#include "muzero_b200.h"\nint main(){printf("%zu %zu\\n", sizeof(mz_paged_view), sizeof(mz_paged_read_args));return 0;}\n'
    with tempfile.TemporaryDirectory() as td:
        c, exe = os.path.join(td, "s.c"), os.path.join(td, "s")
        open(c, "w").write(src)
        subprocess.check_call(["gcc", "-I", os.path.join(root, "include"), c, "-o", exe])
        a, b = map(int, subprocess.check_output([exe]).split())
    assert ctypes.sizeof(_cabi.PagedView) == a and ctypes.sizeof(_cabi.PagedReadArgs) == b


@pytest.mark.parametrize("change, text", [(dict(batch=4097), "batch 4097"), (dict(tokens=-1), "-1 tokens"), (dict(dtype=1), "dtype"), (dict(key=None), "NULL"), (dict(offsets=None), "NULL"),
                                          (dict(key=(1 << 20) + 8), "16-byte"), (dict(v_stride_head=132), "16 bytes"), (dict(rows=None, batch=4000), "batch 4000 of")])
def test_reads_that_are_refused(change, text):
    from muzero_b200.kernels import _cabi
    at = 1 << 20
    a = _cabi.PagedReadArgs(key=at, value=at, dtype=2, k_stride_token=1024, k_stride_head=128, v_stride_token=1024, v_stride_head=128, rows=at, offsets=at, first=None, batch=1, tokens=64)
    for k, v in change.items():
        setattr(a, k, v)
    lib = _cabi.load_library()
    assert lib.mz_paged_read(_cache(), 0, a, None) != 0 and text in _cabi.last_error()
    assert lib.mz_paged_read(_cache(), 99, a, None) != 0 and "layer 99" in _cabi.last_error()


@pytest.mark.parametrize("kw, text", [(dict(window=0), "at least 1"), (dict(window=-3), "at least 1"), (dict(sinks=4), "beside a `window`"), (dict(window=5, sinks=-1), "beside a `window`"),
                                      (dict(window=5, groups=[0, 1]), "without a `window`"), (dict(groups=[]), "one more"), (dict(groups=[0.0, 1.0]), "int32")])
def test_arguments_of_attend(kw, text):
    import torch
    from test_paged_calls import _host_cache
    if "groups" in kw:
        kw = dict(kw, groups=torch.tensor(kw["groups"], dtype=torch.float32 if kw["groups"][:1] == [0.0] and isinstance(kw["groups"][0], float) else torch.int32))
    c = _host_cache()
    c.head_dim, c.dtype, c.kv_heads = 64, torch.bfloat16, 2
    with pytest.raises(ValueError, match=text):
        c.attend(0, torch.zeros(1, 8, 64, dtype=torch.bfloat16), **kw)


def test_arguments_of_read():
    import torch
    from test_paged_calls import _host_cache
    c = _host_cache()
    c.head_dim, c.dtype, c.kv_heads, c.rows = 64, torch.bfloat16, 2, 4
    o = torch.tensor([0, 5], dtype=torch.int32)
    good = torch.zeros(8, 2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="how many places"):
        c.read(0, offsets=o)
    for out, kw in (((good, good[:7]), {}), ((good, good.float()), {}), ((good.float(), good.float()), dict(out_dtype=torch.bfloat16)), ((good, good), dict(tokens=9)), ((good[:, :1], good[:, :1]), {})):
        with pytest.raises(ValueError, match="two tensors"):
            c.read(0, offsets=o, out=out, **kw)
    with pytest.raises(ValueError, match="16-byte pieces"):
        c.read(0, offsets=o, out=(good.transpose(1, 2).contiguous().transpose(1, 2), good))
    with pytest.raises(ValueError, match="`first`"):
        c.read(0, offsets=o, out=(good, good), first=torch.zeros(3, dtype=torch.int32))
