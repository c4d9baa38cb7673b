"""The largest calls of the 4-bit paged key/value cache, without a GPU: what one launch cannot take is refused by its sizes, before any
device work. No counterpart in the reference."""
import ctypes as C

import pytest

from jepa_amd import _lib

P = 0x10000      # a non-null, 16-byte aligned address that no refused call reads


def attention(heads, kvh, n_seq, n_rows, width=1, kind=0):
    L = _lib.lib()
    L.jepa_error_reset()
    s = _lib.CacheShape(heads, kvh, 32, 16, 10)
    rc = L.jepa_amd_cache_attention(0, C.byref(s), P, kind, P, heads * 32, n_seq, n_rows, P, P, P, width, 1.0, 1, P, heads * 32, P, 1 << 50, None)
    return rc, _lib.error_text()


@pytest.mark.parametrize("kind", [0, 1, 30])
def test_workgroups_of_one_launch(kind):
    """4096 sequences over 4096 K/V heads are more workgroups than a launch has, however few their rows."""
    rc, text = attention(4096, 4096, 4096, 4096, kind=kind)
    assert rc == -1 and "jepa_amd_cache_attention" in text and "workgroups" in text


def test_heads_of_rows_of_one_launch():
    rc, text = attention(4096, 1, 1, 1 << 15)
    assert rc == -1 and "heads of rows" in text
    L = _lib.lib()
    s = _lib.CacheShape(4096, 4096, 32, 16, 10)
    for call in (L.jepa_amd_cache_store, L.jepa_amd_cache_read):
        L.jepa_error_reset()
        args = (0, P, 131072, P, 131072, 1 << 15, P) if call is L.jepa_amd_cache_store else (P, 1 << 15, 0, P, 131072, P, 131072)
        assert call(0, C.byref(s), P, *args, None) == -1 and "heads of rows" in _lib.error_text()


def test_no_rows_are_never_too_many():
    """A call without rows has nothing to launch: it gets as far as the device."""
    rc, text = attention(4096, 4096, 4096, 0)
    assert rc == 0 or "workgroups" not in text
