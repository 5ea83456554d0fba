"""KVCache.AppendRoPE's own checks at their edges, without a GPU."""
import numpy as np
import pytest

import test_step_refusals as R
from ai_amd import _native as N
from ai_amd import kvcache
from ai_amd.tensor import TensorError


@pytest.fixture
def cache():
    c = kvcache.KVCache.__new__(kvcache.KVCache)
    c.kv_heads, c.head_dim, c.blocks, c.ctx = 1, 8, 4, R.NoGpu()
    c._codes, c._scales = N.vp(R.P), N.vp(R.P)
    c.cache = N.KvCache(R.P, R.P, 4, 1, 8)
    c._free, c._tables, c._lengths, c._next = [3, 2, 1, 0], {}, {}, 0
    yield c
    c._codes = c._scales = N.vp()


@pytest.mark.parametrize("k", [5.0, [1.0, 2.0], np.zeros((2, 1, 7))])
def test_keys_of_another_shape(cache, k):
    """An error of the cache's kind, whatever is given for rows."""
    with pytest.raises(TensorError, match="want"):
        cache.AppendRoPE([cache.Add()], None, k, k, base=1e4)


def test_positions_of_all_32_bits(cache):
    """Both ends reach the library (which has no context here); one past either is refused."""
    s = cache.Add()
    k = np.zeros((2, 1, 8), np.float32)
    with pytest.raises(TensorError, match="ctx is NULL"):
        cache.AppendRoPE([s], None, k, k, [2], base=1e4, positions=[2 ** 31 - 1, -2 ** 31])
    for p in (2 ** 31, -2 ** 31 - 1):
        with pytest.raises(TensorError, match="positions"):
            cache.AppendRoPE([s], None, k, k, [2], base=1e4, positions=[0, p])
