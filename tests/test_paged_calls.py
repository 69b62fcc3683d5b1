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
