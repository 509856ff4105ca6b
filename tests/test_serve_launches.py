"""Sizes of paged attention whose threads no launch holds are refused, on the host."""
import ctypes

import pytest

from aps2026_amd import capi


@pytest.mark.parametrize("kv_heads,max_kv,code,word", [
    (16, 64, capi.APS_ERR_SHAPE, "workgroups"),      # 2^24 workgroups of 256 threads and more
    (4, 64, capi.APS_ERR_ARG, "overlap"),            # 2^22: taken, and then refused for out over q
])
def test_threads_of_a_launch(kv_heads, max_kv, code, word):
    p, L = 1 << 20, capi.lib()
    cache = capi.KvCacheDesc(p, p, None, None, 8, 16, kv_heads, 64, capi.DTYPE_BF16)
    rc = L.aps_attention_paged(ctypes.byref(cache), p, kv_heads * 64, capi.DTYPE_BF16, 1 << 20, kv_heads, p, p, p, 4,
                               1 << 20, 1, max_kv, 64, 0, 0.1, p, None, 0, None)
    assert rc == code and word in capi.last_error()
