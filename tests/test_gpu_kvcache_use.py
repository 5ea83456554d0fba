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


# ---- row starts that are not in order ----------------------------------------------------------

GUARD = 4096


class Guarded:
    """A device buffer between two guards of its own bytes."""

    def __init__(self, ctx, a):
        self.a = np.ascontiguousarray(a)
        side = np.full(GUARD, 0xC3, np.uint8)
        self.buf = K.Buf(ctx, np.concatenate([side, self.a.view(np.uint8).ravel(), side]))
        self.p = self.buf.p.value + GUARD

    def get(self):
        """What it holds; its guards have to be as they were."""
        x = self.buf.get((self.buf.nbytes,), np.uint8)
        assert (x[:GUARD] == 0xC3).all() and (x[-GUARD:] == 0xC3).all()
        return x[GUARD:-GUARD].view(self.a.dtype).reshape(self.a.shape)

    def free(self):
        self.buf.free()


@pytest.mark.parametrize("width", [5, 20000])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("cu", [[0, 500, 20, 10 ** 9], [-7, -9, -2 ** 31, 4], [100, 50, 2, 1], [2 ** 31 - 1] * 4,
                                [0, 0, 700, 3]])
def test_row_starts_out_of_order_write_nothing_else(ctx, cu, dtype, width):
    """Whatever row starts the device holds: attention and reading back write rows of their outputs, writing blocks of the
    tables, and nothing else; the same pool then serves a call in order as if nothing had been."""
    r = G.rng(6)
    H, Hkv, D, lengths = 2, 1, 64, [300, 300, 300]
    blocks, tables = K.tables_for(r, lengths, extra=3, width=width)
    mine = np.zeros(blocks, bool)
    mine[tables[tables < blocks]] = True
    code_bytes = N.lib().fa_kv_codes_bytes(blocks, Hkv, D)
    codes = Guarded(ctx, np.full((blocks, code_bytes // blocks), 0x7F, np.uint8))
    scales = Guarded(ctx, np.full((blocks, Hkv * 2), 1.0, np.float32))
    cache = K.Cache.__new__(K.Cache)
    cache.ctx, cache.blocks, cache.Hkv, cache.D, cache.Dp = ctx, blocks, Hkv, D, D
    cache.c = N.KvCache(codes.p, scales.p, blocks, Hkv, D)
    k, v = G.make(r, (900, Hkv, D), dtype), G.make(r, (900, Hkv, D), dtype)
    full = K.Batch(ctx, tables, lengths, K.cu_of(lengths))
    K.write(cache, full, k, v)
    q = G.make(r, (900, H, D), dtype)
    before = K.attend(cache, full, q, scale=0.125)
    held = codes.get().copy(), scales.get().copy()
    L = N.lib()
    for rows in (40, 500):
        for lens in ([300, -5, 300], lengths):
            b = K.Batch(ctx, tables, lens, cu, rows=rows)
            size = (rows, H, D)
            bq, bo = Guarded(ctx, q[:rows]), Guarded(ctx, np.zeros(size, q.dtype))
            bk, bv = (Guarded(ctx, np.zeros((rows, Hkv, D), k.dtype)) for _ in range(2))
            N.check(ctx.h, L.fa_kv_attention_dev(ctx.h, C.byref(cache.c), C.byref(b.b), K.dt(q), bq.p, *K.st(q), H, 1, 0,
                                                 0.125, bo.p, None, 0))
            N.check(ctx.h, L.fa_kv_read_dev(ctx.h, C.byref(cache.c), C.byref(b.b), K.dt(k), bk.p, bv.p))
            ctx.sync()
            for x in (bq, bo, bk, bv):
                x.get()
            for x, y in zip(held, (codes.get(), scales.get())):
                np.testing.assert_array_equal(x, y)
            ik, iv = Guarded(ctx, k[:rows]), Guarded(ctx, v[:rows])
            N.check(ctx.h, L.fa_kv_write_dev(ctx.h, C.byref(cache.c), C.byref(b.b), K.dt(k), ik.p, *K.st(k), iv.p,
                                             *K.st(v)))
            ctx.sync()
            for x, y in zip(held, (codes.get(), scales.get())):
                np.testing.assert_array_equal(x[~mine], y[~mine])
            for x in (ik, iv):
                np.testing.assert_array_equal(x.get().view(np.uint8), x.a.view(np.uint8))
            for x in (b, bq, bo, bk, bv, ik, iv):
                x.free()
            codes.buf.put(np.concatenate([np.full(GUARD, 0xC3, np.uint8), held[0].ravel()]))
            scales.buf.put(np.concatenate([np.full(GUARD, 0xC3, np.uint8), held[1].view(np.uint8).ravel()]))
            np.testing.assert_array_equal(K.attend(cache, full, q, scale=0.125), before)
    for x in (full, codes, scales):
        x.free()
