"""The 8-bit key/value cache on the GPU: uses of its calls that go wrong silently where they go wrong."""
import ctypes as C
import os
import subprocess
import sys

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

# ---- many rows under capture -------------------------------------------------------------------

HIP = {"hipStreamBeginCapture": [C.c_void_p, C.c_int], "hipStreamEndCapture": [C.c_void_p, C.POINTER(C.c_void_p)],
       "hipGraphInstantiate": [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t],
       "hipGraphLaunch": [C.c_void_p, C.c_void_p], "hipGraphDestroy": [C.c_void_p], "hipGraphExecDestroy": [C.c_void_p]}


def captured_chunks(ctx, dtype, D, H, Hkv, width, split):
    """A step of chunks (written, attended to) captured before any call of its kernels ran, replayed four times with other
    tokens, lengths, row starts and tables, with eager calls and synchronisation between, against the eager calls."""
    hip = C.CDLL("libamdhip64.so")
    for name, types in HIP.items():
        getattr(hip, name).argtypes = types
    L, r, rows = N.lib(), G.rng(41), 600
    plans = [([700, 400], [0, 350, 600]), ([1200, 290], [0, 310, 600]), ([300, 640], [0, 300, 590]),
             ([64, 1270], [0, 3, 600])]
    blocks = 2 * width if width < 100 else 60
    cache = K.Cache(ctx, blocks, Hkv, D, fill=0)
    b = K.Batch(ctx, np.full((2, width), -1, np.int32), plans[0][0], plans[0][1], rows=rows)
    like = G.make(r, (1,), dtype)
    bufs = {n: K.Buf(ctx, nbytes=rows * h * D * like.itemsize, fill=0) for n, h in
            (("k", Hkv), ("v", Hkv), ("q", H), ("out", H))}
    need = C.c_size_t(0)
    N.check(ctx.h, L.fa_kv_attention_work(C.byref(cache.c), C.byref(b.b), H, C.byref(need)))
    work = K.Buf(ctx, nbytes=need.value, fill=0)

    def step(w, nbytes):
        N.check(ctx.h, L.fa_kv_write_dev(ctx.h, C.byref(cache.c), C.byref(b.b), K.dt(like), bufs["k"].p, Hkv * D, D,
                                         bufs["v"].p, Hkv * D, D))
        N.check(ctx.h, L.fa_kv_attention_dev(ctx.h, C.byref(cache.c), C.byref(b.b), K.dt(like), bufs["q"].p, H * D, D, H,
                                             1, 0, 0.09, bufs["out"].p, w, nbytes))

    graph, ex = C.c_void_p(), C.c_void_p()
    ctx.sync()
    assert hip.hipStreamBeginCapture(ctx.stream, 2) == 0
    step(work.p, need.value)
    assert hip.hipStreamEndCapture(ctx.stream, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(ex), graph, None, None, 0) == 0
    for turn, (lengths, cu) in enumerate(plans):
        perm, t, at = r.permutation(blocks), np.full((2, width), -1, np.int32), 0
        for i, length in enumerate(lengths):
            u = -(-length // 64)
            t[i, :u] = perm[at:at + u]
            at += u
        for x, y in zip(b.bufs, (t, np.array(lengths, np.int32), np.array(cu, np.int32))):
            x.put(y)
        for n, h in (("k", Hkv), ("v", Hkv), ("q", H)):
            bufs[n].put(G.make(r, (rows, h, D), dtype))
        if turn == 0:  # what the sequences hold before the step
            for x in (cache.codes, cache.scales):
                x.put(np.zeros(x.nbytes, np.uint8) if x is cache.codes else np.ones(x.nbytes // 4, np.float32))
        state = cache.state()
        bufs["out"].put(np.full(bufs["out"].nbytes, 0x5A, np.uint8))
        assert hip.hipGraphLaunch(ex, ctx.stream) == 0
        ctx.sync()
        got, after = bufs["out"].get((rows, H, D), like.dtype), cache.state()
        head = work.get((need.value // 4,), np.uint32)[:4096] if need.value else np.zeros(1, np.uint32)
        assert (head[-1] > 0) == split  # the launch was cut in parts
        cache.codes.put(state[0])
        cache.scales.put(state[1])
        bufs["out"].put(np.full(bufs["out"].nbytes, 0x5A, np.uint8))
        step(None, 0)
        ctx.sync()
        np.testing.assert_array_equal(got.view(np.uint8), bufs["out"].get((rows, H, D), like.dtype).view(np.uint8))
        for x0, x1 in zip(after, cache.state()):
            np.testing.assert_array_equal(x0, x1)
        assert np.isfinite(K.wide(got[:cu[-1]])).all() and (got[cu[-1]:].view(np.uint8) == 0x5A).all()
    hip.hipGraphExecDestroy(ex)
    hip.hipGraphDestroy(graph)
    for x in (*bufs.values(), work, b, cache):
        x.free()


CHUNKS = [("bf16", 128, 8, 2, 200, True), ("f32", 128, 8, 2, 200, True), ("bf16", 64, 32, 32, 20, False),
          ("f32", 192, 32, 32, 20, False)]


@pytest.mark.parametrize("case", CHUNKS)
def test_captured_chunks_replay_with_new_contents(ctx, case):
    captured_chunks(ctx, *case)


@pytest.mark.parametrize("case", [CHUNKS[0], CHUNKS[3]])
def test_first_call_of_a_process_is_captured(case):
    """The kernel's own setting is made where its first call is under capture."""
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = ("import sys; sys.path[:0] = ['tests', '.']; import test_gpu_kvcache_use as t; from ai_amd import _native as N; "
            f"t.captured_chunks(N.Context(0), *{case!r}); print('done', flush=True)")
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.strip() == "done", r.stderr[-2000:]
