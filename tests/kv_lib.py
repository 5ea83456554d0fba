"""The device entry points of the key/value cache on numpy arrays, for the tests."""
import ctypes as C

import numpy as np

from ai_amd import _native as N
from ai_amd import synth as S


class Buf:
    """A device buffer with the bytes of an array."""

    def __init__(self, ctx, a=None, nbytes=None, fill=None):
        self.ctx = ctx
        self.nbytes = int(nbytes if nbytes is not None else a.nbytes)
        self.p = C.c_void_p()
        N.check(ctx.h, N.lib().fa_device_alloc(ctx.h, max(self.nbytes, 16), C.byref(self.p)))
        if fill is not None:
            a = np.full(self.nbytes, fill, np.uint8)
        if a is not None:
            self.put(a)

    def put(self, a):
        a = np.ascontiguousarray(a)
        N.check(self.ctx.h, N.lib().fa_memcpy_h2d(self.ctx.h, self.p, a.ctypes.data, a.nbytes))

    def get(self, shape, dtype):
        out = np.empty(shape, dtype)
        N.check(self.ctx.h, N.lib().fa_memcpy_d2h(self.ctx.h, out.ctypes.data, self.p, out.nbytes))
        return out

    def free(self):
        N.lib().fa_device_free(self.ctx.h, self.p)
        self.p = None


class Cache:
    """A pool whose bytes are NaN codes and NaN scales to begin with."""

    def __init__(self, ctx, blocks, kv_heads, D, fill=0x7F):
        self.ctx, self.blocks, self.Hkv, self.D = ctx, blocks, kv_heads, D
        self.Dp = -(-D // 64) * 64
        n = N.lib().fa_kv_codes_bytes(blocks, kv_heads, D)
        assert n == blocks * kv_heads * 2 * 64 * self.Dp
        self.codes = Buf(ctx, nbytes=n, fill=fill)
        self.scales = Buf(ctx, nbytes=blocks * kv_heads * 8, fill=0xFF)
        self.c = N.KvCache(self.codes.p, self.scales.p, blocks, kv_heads, D)

    def state(self):
        return (self.codes.get((self.blocks, self.Hkv, 2, 64 * self.Dp), np.uint8),
                self.scales.get((self.blocks, self.Hkv, 2), np.uint32))

    def free(self):
        self.codes.free()
        self.scales.free()


def split_codes(codes, D):
    """codes [.., 2, 64 * Dp] as [.., 2, 64 tokens, D], by the layout that the header states."""
    t, d = np.arange(64)[:, None], np.arange(D)[None, :]
    k = (d // 64) * 4096 + t * 64 + d % 64
    v = d * 64 + 16 * (t // 4 % 4) + 4 * (t // 16) + t % 4
    return np.stack([codes[..., 0, :][..., k], codes[..., 1, :][..., v]], -3)


class Batch:
    def __init__(self, ctx, tables, lengths, cu, rows=None, nseq=None):
        self.tables = np.ascontiguousarray(tables, np.int32)
        self.lengths = np.asarray(lengths, np.int32)
        self.cu = np.asarray(cu, np.int32)
        self.bufs = [Buf(ctx, x) for x in (self.tables, self.lengths, self.cu)]
        self.rows = int(self.cu[-1] if rows is None else rows)
        self.nseq = len(self.lengths)
        self.b = N.KvBatch(self.bufs[0].p, self.tables.shape[1], self.bufs[1].p, self.bufs[2].p, self.nseq, self.rows)

    def host(self):
        return N.KvBatch(self.tables.ctypes.data, self.tables.shape[1], self.lengths.ctypes.data, self.cu.ctypes.data,
                         self.nseq, self.rows)

    def free(self):
        for b in self.bufs:
            b.free()


def dt(a):
    return N.FA_DT_BF16 if a.dtype == np.uint16 else N.FA_DT_F32


def wide(a):
    return S.bf16_to_f32(a) if a.dtype == np.uint16 else a


def st(a):
    return a.strides[0] // a.itemsize, a.strides[1] // a.itemsize


def span_of(a):
    """The memory under a strided view, from its first element on."""
    n = sum((s - 1) * t for s, t in zip(a.shape, a.strides)) // a.itemsize + 1
    return np.lib.stride_tricks.as_strided(a, (n,), (a.itemsize,))


def write(cache, batch, k, v):
    ctx = cache.ctx
    bk, bv = Buf(ctx, span_of(k)), Buf(ctx, span_of(v))
    N.check(ctx.h, N.lib().fa_kv_write_dev(ctx.h, C.byref(cache.c), C.byref(batch.b), dt(k), bk.p, *st(k), bv.p,
                                           *st(v)))
    ctx.sync()
    bk.free()
    bv.free()


def read(cache, batch, dtype=np.float32):
    ctx = cache.ctx
    shape = (batch.rows, cache.Hkv, cache.D)
    size = int(np.prod(shape)) * np.dtype(dtype).itemsize
    bk, bv = Buf(ctx, nbytes=size, fill=0x5A), Buf(ctx, nbytes=size, fill=0x5A)
    N.check(ctx.h, N.lib().fa_kv_read_dev(ctx.h, C.byref(cache.c), C.byref(batch.b),
                                          N.FA_DT_F32 if dtype == np.float32 else N.FA_DT_BF16, bk.p, bv.p))
    ctx.sync()
    got = bk.get(shape, dtype), bv.get(shape, dtype)
    bk.free()
    bv.free()
    return got


def attend(cache, batch, q, causal=True, window=0, scale=1.0, work=False):
    """Output [rows, H, D]; rows that are not written keep bytes of 0x5A."""
    ctx = cache.ctx
    H = q.shape[1]
    bq, bo = Buf(ctx, span_of(q)), Buf(ctx, nbytes=q.shape[0] * H * cache.D * q.itemsize, fill=0x5A)
    w, need = None, C.c_size_t(0)
    if work:
        N.check(ctx.h, N.lib().fa_kv_attention_work(C.byref(cache.c), C.byref(batch.b), H, C.byref(need)))
        w = Buf(ctx, nbytes=need.value, fill=0xFF)
    N.check(ctx.h, N.lib().fa_kv_attention_dev(ctx.h, C.byref(cache.c), C.byref(batch.b), dt(q), bq.p, *st(q), H,
                                               int(causal), window, scale, bo.p, w.p if w else None, need.value))
    ctx.sync()
    out = bo.get((q.shape[0], H, cache.D), q.dtype)
    for b in (bq, bo, w):
        if b:
            b.free()
    return out


SPARE = 0  # table entries of a sequence more than it uses, as in a program with longest lengths in mind


def tables_for(r, lengths, extra=2, width=None):
    """A pool size and block tables that hand its blocks out in random order; unused entries are out of range."""
    used = [-(-l // 64) for l in lengths]
    blocks = sum(used) + extra
    perm = r.permutation(blocks)
    width = max(max(used, default=0), 1) + SPARE if width is None else width
    t = np.full((len(lengths), width), 2 ** 31 - 1, np.int32)
    at = 0
    for i, u in enumerate(used):
        t[i, :u] = perm[at:at + u]
        at += u
    return blocks, t


def cu_of(ns):
    return np.concatenate([[0], np.cumsum(ns)]).astype(np.int32)
