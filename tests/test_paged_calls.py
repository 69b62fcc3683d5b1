"""Paged cache, the host side of its calls, without a GPU."""
import pytest

from test_paged_host import _cache


@pytest.mark.parametrize("change", [dict(store=(1 << 20) + 16), dict(store_stride_page=18432 + 16), dict(store_stride_layer=8 * 18432 + 16)])
def test_a_store_that_32_byte_loads_cannot_read_is_refused(change):
    """Attention reads the 32 bytes of a row of codes with one load: pages begin on 32-byte boundaries.  Refused by every call, before a launch."""
    from muzero_b200.kernels import _cabi
    lib, at = _cabi.load_library(), 1 << 20
    c = _cache(**change)
    args = _cabi.PagedAttentionArgs(query=at, q_stride_b=1024, q_stride_l=1024, q_stride_h=128, batch=1, q_len=1, q_heads=8, scaling=1.0, out=at, out_dtype=2,
                                    workspace=at, workspace_bytes=1 << 30)
    for call in (lambda: lib.mz_paged_attention(c, 0, args, None), lambda: lib.mz_paged_extend(c, None, None, 1, None),
                 lambda: lib.mz_paged_append(c, 0, at, 256, 128, at, 256, 128, None, None, 1, 1, 1, None), lambda: lib.mz_paged_compact(c, at, 1 << 20, None)):
        assert call() == 1
        assert "32" in _cabi.last_error()


@pytest.mark.parametrize("change", [dict(store=(1 << 20) + 32), dict(store_stride_page=18432 + 32), dict(store_stride_layer=8 * 18432 + 32)])
def test_a_store_on_32_byte_boundaries_is_taken(change):
    from muzero_b200.kernels import _cabi
    assert _cabi.load_library().mz_paged_extend(_cache(**change), None, None, 0, None) == 0          # checked, and nothing to do


def _host_cache():
    """A cache's host side without a device."""
    import torch
    from muzero_b200.cache.paged import MuZeroPagedCache
    c = object.__new__(MuZeroPagedCache)
    c.device, c._workspaces = torch.device("cpu"), {}
    return c


@pytest.mark.parametrize("sizes", [range(1 << 20, 9 << 20, 1 << 16), range(9 << 20, 1 << 20, -(1 << 16)), [5, 1 << 22, 7, 1 << 23, (1 << 23) + 1]])
def test_workspaces_of_growing_calls(sizes):
    """What a stream's calls of many sizes hold together is less than four times what the largest needs: a workspace that has to grow doubles at least, and its
    predecessors are smaller than it all together."""
    c = _host_cache()
    for n in sizes:
        at, size, t = c._workspace(n, 1)
        assert size >= n and t.numel() == size and t.data_ptr() == at
    held = [w[1] for w in c._workspaces[1]]
    assert sum(held) < 4 * max(max(sizes), 1 << 20) and sum(held[:-1]) < held[-1]
    small = c._workspace(3, 2)                                     # another stream's own
    assert small[1] == 1 << 20 and len(c._workspaces) == 2


def test_calls_of_two_threads_have_their_own_arguments(monkeypatch):
    """Two threads attend at the same time, on streams of their own: what the library finds in its argument block is the caller's query, output and workspace, also when
    the other thread has come as far as the library meanwhile."""
    import ctypes
    import threading

    import torch
    from muzero_b200.cache import paged
    from muzero_b200.kernels._cabi import PagedAttentionArgs
    c = _host_cache()
    c.head_dim, c.dtype, c._needs, c._ref = 64, torch.bfloat16, {}, None
    both = threading.Barrier(2, timeout=20)
    seen = {}

    class Library:
        @staticmethod
        def mz_paged_attention_workspace_bytes(*_):
            return 1 << 20

        @staticmethod
        def mz_paged_attention(_, layer, ref, stream):
            both.wait()                                            # both have filled their blocks
            a = ctypes.cast(ref, ctypes.POINTER(PagedAttentionArgs)).contents
            seen[layer] = a.query, a.out, a.workspace, a.batch, a.q_heads, a.scaling, stream
            both.wait()
            return 0

    c._lib = Library
    monkeypatch.setattr(paged, "stream_ptr", lambda device: threading.current_thread().name)
    monkeypatch.setattr(paged, "on_device", lambda device, fn, *args: fn(*args))
    queries = [torch.zeros(1 + i, 1, 2 + 2 * i, 64, dtype=torch.bfloat16) for i in range(2)]
    outs = [torch.empty_like(q) for q in queries]
    threads = [threading.Thread(target=lambda i=i: c.attend(i, queries[i], out=outs[i], scaling=float(i)), name=f"stream {i}") for i in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    for i in range(2):
        ws = c._workspaces[f"stream {i}"][-1][0]
        assert seen[i] == (queries[i].data_ptr(), outs[i].data_ptr(), ws, 1 + i, 2 + 2 * i, float(i), f"stream {i}")


def test_index_vectors():
    """A vector of one entry is contiguous whatever its stride; longer ones that are not, other types and other shapes are refused."""
    import torch
    from muzero_b200.cache.paged import _index
    cpu = torch.device("cpu")
    whole = torch.arange(6, dtype=torch.int32)
    for one in (whole[::2][:1], whole[:1].expand(1), torch.arange(4, dtype=torch.int32).view(2, 2)[:1, 1]):
        assert _index(one, "rows", cpu, 1) == one.data_ptr()
    assert _index(whole[2:], "rows", cpu, 4) == whole.data_ptr() + 8
    for bad in (whole[::2], whole[:1].expand(3), whole.long(), whole.view(2, 3)):
        with pytest.raises(ValueError):
            _index(bad, "rows", cpu)
