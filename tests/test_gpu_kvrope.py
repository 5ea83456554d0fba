"""Rotary positions on the way into the 8-bit key/value cache, on the GPU
against the definition (decode_oracle.py, kv_oracle.py): codes and scales to
the bit, queries to the rounding of their type."""
import ctypes as C

import numpy as np
import pytest

import decode_oracle as O
import kv_lib as K
import kv_oracle as KO
import test_gpu_kvcache as G
import test_gpu_kvcache_use as use
from ai_amd import _native as N
from ai_amd import synth as S
from ai_amd.kvcache import KVCache

pytestmark = pytest.mark.gpu


class Step:
    """Device copies of a step's tensors; q_out (0x5A bytes to begin with) may be q itself."""

    def __init__(self, ctx, q, k, v, positions=None, in_place=False):
        self.ctx, self.q, self.k, self.v = ctx, q, k, v
        self.bufs = [None if x is None else K.Buf(ctx, K.span_of(x)) for x in (q, k, v)]
        self.pos = None if positions is None else K.Buf(ctx, np.asarray(positions, np.int32))
        self.in_place = in_place
        self.out = None
        if q is not None:
            self.out = self.bufs[0] if in_place else K.Buf(ctx, nbytes=q.size * q.itemsize, fill=0x5A)

    def call(self, cache, batch, base, dims):
        rope = N.KvRope(base, dims, self.pos.p if self.pos else None)
        bq, bk, bv = self.bufs
        q = self.q
        return N.lib().fa_kv_write_rope_dev(
            self.ctx.h, C.byref(cache.c), C.byref(batch.b), C.byref(rope), K.dt(self.k), bq.p if bq else None,
            *(K.st(q) if bq else (0, 0)), q.shape[1] if bq else 0, self.out.p if bq else None, bk.p, *K.st(self.k),
            bv.p, *K.st(self.v))

    def run(self, cache, batch, base, dims):
        N.check(self.ctx.h, self.call(cache, batch, base, dims))
        self.ctx.sync()
        return None if self.q is None else self.out.get(self.q.shape, self.q.dtype)

    def free(self):
        for b in {id(x): x for x in (*self.bufs, self.pos, self.out) if x}.values():
            b.free()


def check_queries(got, q, positions, base, dims, rows=None):
    """Within a rounding of the type of the definition (float32: of both products, should a cosine's last bit differ)."""
    rows = slice(None) if rows is None else rows
    want = O.rotate(K.wide(q), positions, base, dims).astype(np.float64)[rows]
    g = K.wide(got).astype(np.float64)[rows]
    mag = np.abs(K.wide(q)).max(-1, keepdims=True)[rows] * 2
    tol = (2.0 ** -8 * np.abs(want) if got.dtype == np.uint16 else 0) + 2.0 ** -22 * mag + 1e-40
    assert (np.isnan(g) == np.isnan(want)).all()
    fin = np.isfinite(want)
    assert (np.abs(g - want) <= tol)[fin].all(), np.abs(g - want)[fin].max()
    np.testing.assert_array_equal(got[rows][..., dims:], q[rows][..., dims:])


def check_cache(cache, ref, D):
    codes, scales = cache.state()
    got = KO.DECODE[K.split_codes(codes, D)]
    known = ~np.isnan(ref.exp)
    with np.errstate(invalid="ignore"):
        want_scales = np.where(known, 2.0 ** np.nan_to_num(ref.exp), 0).astype(np.float32)
    np.testing.assert_array_equal(scales.view(np.float32)[known], want_scales[known])
    written = ~np.isnan(ref.val)
    np.testing.assert_array_equal(got[written], ref.val[written])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,dims", [(2, 2), (8, 6), (40, 40), (64, 64), (66, 66), (66, 10), (80, 80), (96, 64), (128, 128),
                                    (128, 34), (192, 192), (256, 256), (256, 2), (320, 320), (512, 512), (511, 256),
                                    (63, 62)])
def test_head_dims_and_rotary_dims(ctx, D, dims, dtype):
    """Prompts, tokens that continue blocks, and single ones; queries of one, three and eight heads for a key's."""
    r = G.rng(D * 1000 + dims)
    Hkv, base = 2, 10000.0
    steps = [(5, 64, 1, 130, 0), (1, 1, 63, 2, 1), (60, 70, 0, 1, 90), (1, 1, 1, 1, 1)]
    final = [sum(s[i] for s in steps) for i in range(5)]
    blocks, tables = K.tables_for(r, final)
    cache, ref = K.Cache(ctx, blocks, Hkv, D), KO.RefCache(blocks, Hkv, D)
    lengths = [0] * 5
    for ns, group in zip(steps, (3, 1, 8, 3)):
        lengths = [a + n for a, n in zip(lengths, ns)]
        cu = K.cu_of(ns)
        rows = int(cu[-1])
        q, k, v = (G.make(r, (rows, h, D), dtype) for h in (Hkv * group, Hkv, Hkv))
        pos = np.concatenate([np.arange(l - n, l) for l, n in zip(lengths, ns)])
        b = K.Batch(ctx, tables, lengths, cu)
        s = Step(ctx, q, k, v)
        check_queries(s.run(cache, b, base, dims), q, pos, base, dims)
        ref.write(tables, lengths, cu, O.rotate(K.wide(k), pos, base, dims), K.wide(v))
        check_cache(cache, ref, D)
        s.free()
        b.free()
    cache.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("lengths,ns", [([700, 3], [700, 2]), ([40, 90, 64], [1, 1, 1]), ([3000], [257])])
def test_given_positions_near_and_far(ctx, lengths, ns, dtype):
    """Positions that are not places: repeated, negative, of both ends of 32 bits."""
    r = G.rng(7)
    H, Hkv, D = 6, 2, 64
    cache, ref, tables = G.fill(ctx, r, [l - n for l, n in zip(lengths, ns)], Hkv, D, dtype,
                                extra=sum(-(-l // 64) for l in lengths) + 4, width=60)
    free = [i for i in range(cache.blocks) if i not in set(tables.ravel().tolist())]
    for i, l in enumerate(lengths):
        for j in range(-(-l // 64)):
            if not 0 <= tables[i, j] < cache.blocks:
                tables[i, j] = free.pop()
    cu = K.cu_of(ns)
    rows = int(cu[-1])
    q, k, v = (G.make(r, (rows, h, D), dtype) for h in (H, Hkv, Hkv))
    pos = r.integers(-2 ** 31, 2 ** 31, rows).astype(np.int32)
    pos[0], pos[-1] = 2 ** 31 - 1, -2 ** 31
    pos[::3] = r.integers(0, 10 ** 6, len(pos[::3]))
    pos[1:3] = 5
    b = K.Batch(ctx, tables, lengths, cu)
    for base in (1e6, 500.0):
        s = Step(ctx, q, k, v, pos)
        check_queries(s.run(cache, b, base, D), q, pos, base, D)
        ref.write(tables, lengths, cu, O.rotate(K.wide(k), pos, base, D), K.wide(v))
        check_cache(cache, ref, D)
        s.free()
    b.free()
    cache.free()


@pytest.mark.parametrize("base", [0.25, 1.0, 1e-3])
def test_bases_up_to_one(ctx, base):
    """Angles that grow with the pair instead of falling, past 2^31."""
    r = G.rng(8)
    D, n = 32, 70
    blocks, tables = K.tables_for(r, [n])
    cache, ref = K.Cache(ctx, blocks, 1, D), KO.RefCache(blocks, 1, D)
    q, k, v = (G.make(r, (n, 1, D), "f32") for _ in range(3))
    pos = np.concatenate([np.arange(n - 6), [2 ** 31 - 1, -2 ** 31, 2 ** 30, 12345678, -1, 2 ** 24]])
    b = K.Batch(ctx, tables, [n], [0, n])
    s = Step(ctx, q, k, v, pos)
    check_queries(s.run(cache, b, base, D), q, pos, base, D)
    ref.write(tables, [n], [0, n], O.rotate(k, pos, base, D), v)
    check_cache(cache, ref, D)
    for x in (s, b, cache):
        x.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("pad", [4, 1])
def test_strides_and_one_buffer(ctx, dtype, pad):
    """q, k and v as parts of one row, with a row stride that keeps or loses alignment."""
    r = G.rng(9)
    H, Hkv, D, lengths, ns = 4, 2, 64, [100, 30], [70, 30]
    whole = G.make(r, (100, (H + 2 * Hkv) * D + pad), dtype)
    q, k, v = (np.lib.stride_tricks.as_strided(whole[:, a * D:], (100, h, D),
                                               (whole.strides[0], D * whole.itemsize, whole.itemsize))
               for a, h in ((0, H), (H, Hkv), (H + Hkv, Hkv)))
    cache, ref, tables = G.fill(ctx, r, [30, 0], Hkv, D, dtype, extra=4, width=2)
    free = [i for i in range(cache.blocks) if i not in set(tables.ravel().tolist())]
    tables[0, 1], tables[1, 0] = free[:2]
    pos = np.concatenate([np.arange(30, 100), np.arange(30)])
    b = K.Batch(ctx, tables, lengths, K.cu_of(ns))
    s = Step(ctx, q, k, v)
    check_queries(s.run(cache, b, 1e4, D), q, pos, 1e4, D)
    ref.write(tables, lengths, K.cu_of(ns), O.rotate(K.wide(k), pos, 1e4, D), K.wide(v))
    check_cache(cache, ref, D)
    for x in (s, b, cache):
        x.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,dims,n", [(64, 64, 300), (128, 128, 1), (66, 34, 70), (256, 256, 65)])
def test_queries_in_place(ctx, D, dims, n, dtype):
    r = G.rng(10)
    blocks, tables = K.tables_for(r, [n])
    cache = K.Cache(ctx, blocks, 1, D)
    q, k, v = (G.make(r, (n, h, D), dtype) for h in (5, 1, 1))
    b = K.Batch(ctx, tables, [n], [0, n])
    s, t = Step(ctx, q, k, v), Step(ctx, q, k, v, in_place=True)
    np.testing.assert_array_equal(s.run(cache, b, 1e4, dims), t.run(cache, b, 1e4, dims))
    for x in (s, t, b, cache):
        x.free()


def test_no_queries_and_empty_batches(ctx):
    r = G.rng(11)
    D = 64
    blocks, tables = K.tables_for(r, [50])
    cache, ref = K.Cache(ctx, blocks, 1, D), KO.RefCache(blocks, 1, D)
    k, v = (G.make(r, (50, 1, D), "f32") for _ in range(2))
    b = K.Batch(ctx, tables, [50], [0, 50])
    s = Step(ctx, None, k, v)
    s.run(cache, b, 1e4, D)
    ref.write(tables, [50], [0, 50], O.rotate(k, np.arange(50), 1e4, D), v)
    check_cache(cache, ref, D)
    before = cache.state()
    for batch in (K.Batch(ctx, tables, [50], [0, 0], rows=0), K.Batch(ctx, tables, [50], [0, 0], rows=50)):
        s.run(cache, batch, 1e4, D)
        batch.free()
    for x, y in zip(before, cache.state()):
        np.testing.assert_array_equal(x, y)
    for x in (s, b, cache):
        x.free()


def test_special_values(ctx):
    """NaN and infinities spoil their own pair and nothing else; magnitudes up to float32's largest."""
    r = G.rng(12)
    D, n = 64, 64
    blocks, tables = K.tables_for(r, [n])
    cache, ref = K.Cache(ctx, blocks, 1, D), KO.RefCache(blocks, 1, D)
    q, k, v = (G.make(r, (n, 1, D), "f32") for _ in range(3))
    for x in (q, k):
        x[3, 0, 5], x[4, 0, 40], x[5, 0, 0] = np.nan, np.inf, -np.inf
        x[6], x[7] = 3e38, 1e-42
    b = K.Batch(ctx, tables, [n], [0, n])
    s = Step(ctx, q, k, v)
    got = s.run(cache, b, 1e4, D)
    want = O.rotate(q, np.arange(n), 1e4, D)
    assert (np.isnan(got) == np.isnan(want)).all() and np.isnan(want).sum() == 2  # the pair of the NaN
    np.testing.assert_array_equal(np.isinf(got), np.isinf(want))  # an infinity times cosines and sines that are not 0
    assert np.isinf(want[[4, 5]]).sum() == 4
    assert np.isfinite(got[np.r_[0:3, 8:n]]).all()
    kr = O.rotate(k, np.arange(n), 1e4, D)
    ref.write(tables, [n], [0, n], kr, v)
    codes, scales = cache.state()
    block = tables[0, 0]
    np.testing.assert_array_equal(np.isnan(KO.DECODE[K.split_codes(codes, D)][block, 0, 0]), np.isnan(ref.val[block, 0, 0]))
    check_cache(cache, ref, D)
    for x in (s, b, cache):
        x.free()


def test_queries_of_tokens_without_a_block(ctx):
    """Table entries outside the pool, or a table too short: nothing is written, queries are rotated all the same."""
    r = G.rng(13)
    D, Hkv, H = 64, 1, 2
    tables = np.array([[0, 99], [-1, 1]], np.int32)
    lengths, ns = [200, 70], [190, 70]
    cache = K.Cache(ctx, 3, Hkv, D)
    rows = sum(ns)
    q, k, v = (G.make(r, (rows, h, D), "f32") for h in (H, Hkv, Hkv))
    b = K.Batch(ctx, tables, lengths, K.cu_of(ns))
    s = Step(ctx, q, k, v)
    pos = np.concatenate([np.arange(10, 200), np.arange(70)])
    check_queries(s.run(cache, b, 1e4, D), q, pos, 1e4, D)
    codes, scales = cache.state()
    assert (codes[2] == 0x7F).all() and (scales[2] == 0xFFFFFFFF).all()
    for x in (s, b, cache):
        x.free()


def test_rows_behind_the_last_sequence_stay(ctx):
    r = G.rng(14)
    D = 128
    blocks, tables = K.tables_for(r, [30])
    cache = K.Cache(ctx, blocks, 1, D)
    q, k, v = (G.make(r, (80, h, D), "bf16") for h in (3, 1, 1))
    b = K.Batch(ctx, tables, [30], [0, 30], rows=80)
    s = Step(ctx, q, k, v)
    got = s.run(cache, b, 1e4, D)
    check_queries(got, q, np.r_[0:30, np.zeros(50)], 1e4, D, slice(0, 30))
    assert (got[30:].view(np.uint8) == 0x5A).all()
    for x in (s, b, cache):
        x.free()


@pytest.mark.parametrize("cu", [[0, 500, 20, 10 ** 9], [-7, -9, -2 ** 31, 4], [100, 50, 2, 1], [2 ** 31 - 1] * 4])
def test_row_starts_out_of_order_write_nothing_else(ctx, cu):
    """Whatever the device's arrays hold: queries within their rows, blocks of the tables, nothing else."""
    r = G.rng(15)
    H, Hkv, D, rows = 2, 1, 64, 500
    blocks, tables = K.tables_for(r, [300] * 3, extra=3)
    mine = np.zeros(blocks, bool)
    mine[tables[tables < blocks]] = True
    codes = use.Guarded(ctx, np.full((blocks, 2 * 64 * D), 0x7F, np.uint8))
    scales = use.Guarded(ctx, np.full((blocks, 2), 1.0, np.float32))
    cache = N.KvCache(codes.p, scales.p, blocks, Hkv, D)
    q, k, v = (use.Guarded(ctx, G.make(r, (rows, h, D), "f32")) for h in (H, Hkv, Hkv))
    pos = use.Guarded(ctx, np.arange(rows, dtype=np.int32))
    for lens in ([300, -5, 300], [300, 300, 300]):
        b = K.Batch(ctx, tables, lens, cu, rows=rows)
        out = use.Guarded(ctx, np.zeros((rows, H, D), np.float32))
        for p in (pos.p, None):
            rope = N.KvRope(1e4, D, p)
            N.check(ctx.h, N.lib().fa_kv_write_rope_dev(ctx.h, C.byref(cache), C.byref(b.b), C.byref(rope), 0, q.p, H * D, D,
                                                        H, out.p, k.p, D, D, v.p, D, D))
        ctx.sync()
        out.get()
        assert (codes.get()[~mine] == 0x7F).all() and (scales.get()[~mine] == 1.0).all()
        for x in (q, k, v, pos):
            np.testing.assert_array_equal(x.get(), x.a)
        b.free()
        out.free()
    for x in (codes, scales, q, k, v, pos):
        x.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_equals_rotating_first_and_the_host_call(ctx, dtype):
    """The same bytes as fa_kv_write of keys rotated before (in float32), and from the host entry point and KVCache."""
    r = G.rng(16)
    H, Hkv, D, ns = 6, 2, 64, [90, 1, 200]
    rows = sum(ns)
    q, k, v = (G.make(r, (rows, h, D), dtype) for h in (H, Hkv, Hkv))
    pos = np.concatenate([np.arange(n) for n in ns])
    blocks, tables = K.tables_for(r, ns)
    a, b, c = (K.Cache(ctx, blocks, Hkv, D) for _ in range(3))
    batch = K.Batch(ctx, tables, ns, K.cu_of(ns))
    s = Step(ctx, q, k, v)
    got = s.run(a, batch, 1e6, D)
    K.write(b, batch, O.rotate(K.wide(k), pos, 1e6, D), K.wide(v))
    out = np.empty_like(q)
    rope, host = N.KvRope(1e6, D, None), batch.host()
    N.check(ctx.h, N.lib().fa_kv_write_rope(ctx.h, C.byref(c.c), C.byref(host), C.byref(rope), K.dt(k), q.ctypes.data,
                                            *K.st(q), H, out.ctypes.data, k.ctypes.data, *K.st(k), v.ctypes.data, *K.st(v)))
    np.testing.assert_array_equal(out, got)
    for x, y, z in zip(a.state(), b.state(), c.state()):
        np.testing.assert_array_equal(x, y)
        np.testing.assert_array_equal(x, z)
    with KVCache(Hkv, D, 1000, ctx=ctx) as cache:
        seqs = [cache.Add() for _ in ns]
        np.testing.assert_array_equal(cache.AppendRoPE(seqs, q, k, v, ns, base=1e6), got)
        assert cache.AppendRoPE([seqs[0]], None, k[:1], v[:1], base=1e6, positions=[7]) is None
        assert cache.Len(seqs[0]) == 91
        kk, _ = cache.Read(seqs[2])
        ref = KO.RefCache(blocks, Hkv, D)
        ref.write(tables, ns, K.cu_of(ns), O.rotate(K.wide(k), pos, 1e6, D), K.wide(v))
        np.testing.assert_array_equal(kk, ref.tokens(tables[2], 200)[0].astype(np.float32))
    for x in (s, batch, a, b, c):
        x.free()


@pytest.mark.parametrize("nseq", [1, 65, 700])
def test_many_sequences(ctx, nseq):
    r = G.rng(17)
    D, Hkv, H = 32, 1, 2
    ns = r.integers(0, 4, nseq)
    ns[0] = 3
    lengths = ns + r.integers(0, 100, nseq)
    blocks, tables = K.tables_for(r, lengths)
    cache, ref = K.Cache(ctx, blocks, Hkv, D, fill=0), KO.RefCache(blocks, Hkv, D)
    old = lengths - ns
    k, v = (G.make(r, (int(old.sum()), Hkv, D), "f32") for _ in range(2))
    if len(k):
        b = K.Batch(ctx, tables, old, K.cu_of(old))
        K.write(cache, b, k, v)
        ref.write(tables, old, K.cu_of(old), k, v)
        b.free()
    rows = int(ns.sum())
    q, k, v = (G.make(r, (rows, h, D), "f32") for h in (H, Hkv, Hkv))
    pos = np.concatenate([np.arange(l - n, l) for l, n in zip(lengths, ns)])
    b = K.Batch(ctx, tables, lengths, K.cu_of(ns))
    s = Step(ctx, q, k, v)
    check_queries(s.run(cache, b, 1e4, D), q, pos, 1e4, D)
    ref.write(tables, lengths, K.cu_of(ns), O.rotate(k, pos, 1e4, D), v)
    check_cache(cache, ref, D)
    for x in (s, b, cache):
        x.free()


def test_offsets_past_32_bits(ctx):
    """Rows whose stride takes their offsets past 2^32 bytes, and 2^31 elements."""
    r = G.rng(18)
    D, H, n = 64, 1, 3
    stride = (1 << 30) + 64
    blocks, tables = K.tables_for(r, [n])
    cache, ref = K.Cache(ctx, blocks, 1, D), KO.RefCache(blocks, 1, D)
    big = K.Buf(ctx, nbytes=4 * (2 * stride + D))
    rows = [G.make(r, (1, D), "f32") for _ in range(n)]
    L = N.lib()
    for i, x in enumerate(rows):
        N.check(ctx.h, L.fa_memcpy_h2d(ctx.h, big.p.value + 4 * i * stride, x.ctypes.data, x.nbytes))
    out = K.Buf(ctx, nbytes=n * D * 4, fill=0x5A)
    b = K.Batch(ctx, tables, [n], [0, n])
    rope = N.KvRope(1e4, D, None)
    N.check(ctx.h, L.fa_kv_write_rope_dev(ctx.h, C.byref(cache.c), C.byref(b.b), C.byref(rope), 0, big.p, stride, D, H,
                                          out.p, big.p, stride, D, big.p, stride, D))
    ctx.sync()
    x = np.stack(rows)
    check_queries(out.get((n, 1, D), np.float32), x, np.arange(n), 1e4, D)
    ref.write(tables, [n], [0, n], O.rotate(x, np.arange(n), 1e4, D), x)
    check_cache(cache, ref, D)
    for y in (big, out, b, cache):
        y.free()
