"""fa_kv_attention_work without a GPU: scratch sizes from the sizes alone."""
import ctypes as C

import numpy as np
import pytest

from ai_amd import _native as N

L = N.lib()


def work(cache, batch, heads):
    n = C.c_size_t(7)
    return L.fa_kv_attention_work(C.byref(cache), C.byref(batch), heads, C.byref(n)), n.value


@pytest.mark.parametrize("codes,scales", [(None, None), (None, 256), (256, None), (264, 256), (256, 260)])
def test_scratch_is_sized_before_the_pool_is_allocated(codes, scales):
    """Neither the cache's buffers nor the batch's arrays are looked at."""
    mem = np.zeros(64, np.uint8)
    full = N.KvCache(256, 256, 1000, 8, 128)
    arrays = N.KvBatch(mem.ctypes.data, 500, mem.ctypes.data, mem.ctypes.data, 3, 3)
    rc, want = work(full, arrays, 32)
    assert rc == N.FA_OK and want > 0
    assert work(N.KvCache(codes, scales, 1000, 8, 128), N.KvBatch(None, 500, None, None, 3, 3), 32) == (N.FA_OK, want)


def test_sizes_are_still_refused():
    batch = N.KvBatch(None, 500, None, None, 3, 3)
    for bad in ((-1, 8, 128), (10, 0, 128), (10, 65536, 128), (10, 8, 0), (10, 8, 513)):
        assert work(N.KvCache(None, None, *bad), batch, 32) == (N.FA_ERR_ARG, 0)
