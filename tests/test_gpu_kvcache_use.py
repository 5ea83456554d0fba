"""The 8-bit key/value cache on the GPU: uses of its calls that go wrong silently where they go wrong."""
import ctypes as C

import numpy as np
import pytest

import kv_lib as K
import kv_oracle as O
import test_gpu_kvcache as G
from ai_amd import _native as N

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("dtype,D,H,length,n,blocks", [
    ("f32", 256, 3, 8000, 800, 10),  # 19 tiles of 128 rows on 125 blocks, for 256 workgroups
    ("bf16", 64, 3, 8000, 800, 5)])  # for 512
def test_parts_are_joined_as_they_were_written(ctx, dtype, D, H, length, n, blocks):
    """Split tiles of many rows: the kernel that writes the parts leaves their length, in blocks, in the last word of the
    scratch's counters, where the launch that joins them takes it from; the other words end as they began, at zero."""
    r = G.rng(3)
    cache, ref, tables = G.fill(ctx, r, [length], 1, D, dtype)
    q = G.make(r, (n, H, D), dtype)
    b = K.Batch(ctx, tables, [length], [0, n])
    need = C.c_size_t(0)
    N.check(ctx.h, N.lib().fa_kv_attention_work(C.byref(cache.c), C.byref(b.b), H, C.byref(need)))
    bq, bo, w = K.Buf(ctx, q), K.Buf(ctx, nbytes=q.nbytes, fill=0x5A), K.Buf(ctx, nbytes=need.value, fill=0xFF)
    N.check(ctx.h, N.lib().fa_kv_attention_dev(ctx.h, C.byref(cache.c), C.byref(b.b), K.dt(q), bq.p, *K.st(q), H, 1, 0,
                                               0.1, bo.p, w.p, need.value))
    ctx.sync()
    head = w.get((4096,), np.uint32)
    assert head[-1] == blocks and not head[:-1].any()
    rows = [0, 1, n // 2, n - 1]
    k, v = ref.tokens(tables[0], length)
    want, tol = O.attention(K.wide(q[rows]), k, v, O.sees(length, n, True, 0)[rows], float(np.float32(0.1)))
    if dtype == "bf16":
        tol = tol + G.BF * O.attention(K.wide(q[rows]), k, np.abs(v), O.sees(length, n, True, 0)[rows],
                                       float(np.float32(0.1)))[0]
    G.close(bo.get(q.shape, q.dtype)[rows], want, tol, f"{dtype} {D} dims in parts of {blocks} blocks")
    for x in (bq, bo, w, b, cache):
        x.free()
