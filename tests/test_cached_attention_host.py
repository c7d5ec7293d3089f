"""How cached_attention's rows and keys are shared out, on the CPU."""
import ctypes

import pytest

from test_kv_cache_host import c_arg


@pytest.mark.parametrize("window", [(1 << 30) + 1, (1 << 31) - 1, 1 << 31, 1 << 32, (1 << 63) - 8, (1 << 63) - 1])
def test_no_window(lib, window):
    """A window that is wider than any text is none, whatever its number."""
    n = ctypes.c_size_t(0)

    def size(w, **kw):
        arg = c_arg(**{"max_pages": 4096, "table_stride": 4096, **kw})
        assert lib.tmac_cached_attn_workspace(arg, 2, 1, 6, w, 2, ctypes.byref(n)) == 0
        return n.value

    for kw in ({}, {"format": 0}, {"max_pages": 1 << 20, "table_stride": 1 << 20}):
        assert size(window, **kw) == size(1 << 30, **kw) > 0
