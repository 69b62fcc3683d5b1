"""Paged cache: what its handle keeps between calls, without a GPU."""
import pytest
import torch

from test_paged_calls import _host_cache


@pytest.fixture
def cache(monkeypatch):
    """The host side of a cache on a library that notes the workspaces it is given."""
    import ctypes

    from muzero_b200.cache import paged
    from muzero_b200.kernels._cabi import PagedAttentionArgs
    c = _host_cache()
    c.head_dim, c.dtype, c._needs, c._ref, c.given = 64, torch.bfloat16, {}, None, []

    class Library:
        mz_paged_attention_workspace_bytes = staticmethod(lambda *_: 100)
        mz_paged_attention_view_workspace_bytes = staticmethod(lambda *_: 100)

        @staticmethod
        def mz_paged_attention(_, layer, ref, stream):
            a = ctypes.cast(ref, ctypes.POINTER(PagedAttentionArgs)).contents
            c.given.append((a.workspace, a.workspace_bytes))
            return 0

        @staticmethod
        def mz_paged_attention_view(_, layer, ref, view, stream):
            return Library.mz_paged_attention(_, layer, ref, stream)

    c._lib = Library
    monkeypatch.setattr(paged, "stream_ptr", lambda device: 7)
    monkeypatch.setattr(paged, "on_device", lambda device, fn, *args: fn(*args))
    return c


def test_a_window_that_changes_in_every_step_does_not_fill_the_handle(cache):
    q = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    for window in range(1, 5000):
        cache.attend(0, q, window=window, sinks=window % 3)
    assert len(cache._needs) <= 1024 and len(set(cache.given)) == 1


def test_captured_calls_have_workspaces_of_their_graph(cache, monkeypatch):
    """While a stream is captured the handle keeps nothing: the memory is the graph's, and neither another graph's nor that of calls outside."""
    q = torch.zeros(1, 2, 64, dtype=torch.bfloat16)
    cache.attend(0, q)
    outside = cache.given[-1]
    held = []
    empty = torch.empty
    monkeypatch.setattr(torch, "empty", lambda *a, **kw: held.append(empty(*a, **kw)) or held[-1])
    from muzero_b200.cache import paged
    monkeypatch.setattr(paged, "_capturing", lambda device: True)
    for kw in ({}, dict(window=5), {}):
        cache.attend(0, q, **kw)
        assert cache.given[-1] == (held[-1].data_ptr(), 100)
    assert [w[:2] for w in cache._workspaces[7]] == [outside] and len({x for x in cache.given}) == 4
    monkeypatch.setattr(paged, "_capturing", lambda device: False)
    cache.attend(0, q)
    assert cache.given[-1] == outside
