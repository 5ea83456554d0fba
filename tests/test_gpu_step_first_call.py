"""A decoding step's operators whose first call of a process is under capture: what their kernels need set is set there,
and replays with other contents equal eager calls."""
import ctypes as C
import os
import subprocess
import sys

import numpy as np
import pytest

import kv_lib as K
import test_gpu_f8 as F
import test_gpu_kvcache as G
import test_gpu_kvrope as R
from ai_amd import _native as N

pytestmark = pytest.mark.gpu


def captured(ctx, dtype, D, rows, n, k, vocab, filters):
    import test_gpu_decode_step as T  # (its hip(): the functions of graphs)
    hip, L, r = T.hip(), N.lib(), G.rng(D + n)
    Hkv, H = 2, 4
    blocks, tables = K.tables_for(r, [rows + 70])
    cache = K.Cache(ctx, blocks, Hkv, D, fill=0)
    cache.scales.put(np.ones(blocks * Hkv * 2, np.float32))
    batch = K.Batch(ctx, tables, [rows + 70], [0, rows])
    q, kk, v = (G.make(r, (rows, h, D), dtype) for h in (H, Hkv, Hkv))
    s = R.Step(ctx, q, kk, v)
    w = (r.standard_normal((n, k)) / np.sqrt(k)).astype(np.float32)
    codes, scales = (K.Buf(ctx, nbytes=f(n, k), fill=0xFF) for f in (L.fa_f8_codes_bytes, L.fa_f8_scales_bytes))
    held, m = N.F8Matrix(codes.p, scales.p, n, k), 24
    bw, ba, bc = K.Buf(ctx, w), K.Buf(ctx, nbytes=m * k * 4, fill=0), K.Buf(ctx, nbytes=m * n * 4, fill=0)
    bl, bu = K.Buf(ctx, nbytes=m * vocab * 4, fill=0), K.Buf(ctx, nbytes=m * 4, fill=0)
    ids, logp = K.Buf(ctx, nbytes=m * 4, fill=0), K.Buf(ctx, nbytes=m * 4, fill=0)
    settings = [K.Buf(ctx, x) for x in (np.full(m, 0.8, np.float32), np.full(m, 40, np.int32), np.full(m, 0.9, np.float32))]
    need = [C.c_size_t(0), C.c_size_t(0)]
    N.check(ctx.h, L.fa_matmul_f8_work(m, C.byref(held), C.byref(need[0])))
    N.check(ctx.h, L.fa_sample_work(m, vocab, C.byref(need[1])))
    work = [K.Buf(ctx, nbytes=max(x.value, 16), fill=0xFF) for x in need]
    st = N.Sampling(settings[0].p, settings[1].p if filters else None, settings[2].p if filters else None, None)

    def step(own):
        p = [(None, 0)] * 2 if own else [(x.p, y.value) for x, y in zip(work, need)]
        N.check(ctx.h, s.call(cache, batch, 1e4, D))
        N.check(ctx.h, L.fa_f8_write_dev(ctx.h, C.byref(held), 0, bw.p, k))
        N.check(ctx.h, L.fa_matmul_f8_dev(ctx.h, m, 0, ba.p, k, C.byref(held), None, F.DT[dtype], bc.p, n, *p[0]))
        N.check(ctx.h, L.fa_sample_dev(ctx.h, m, vocab, 0, bl.p, vocab, C.byref(st), bu.p, ids.p, logp.p, *p[1]))

    def state():
        return [s.out.get(q.shape, q.dtype), bc.get(m * n * (4 if dtype == "f32" else 2), np.uint8), ids.get(m, np.uint32),
                logp.get(m, np.uint32), codes.get(codes.nbytes, np.uint8), scales.get(scales.nbytes, np.uint8),
                *cache.state()]

    graph, ex = C.c_void_p(), C.c_void_p()
    ctx.sync()
    assert hip.hipStreamBeginCapture(ctx.stream, 2) == 0
    step(False)
    assert hip.hipStreamEndCapture(ctx.stream, C.byref(graph)) == 0
    assert hip.hipGraphInstantiate(C.byref(ex), graph, None, None, 0) == 0
    for turn in range(3):
        for b, x in zip(s.bufs, (q, kk, v)):
            b.put(G.make(r, x.shape, dtype))
        bw.put((r.standard_normal((n, k)) / np.sqrt(k)).astype(np.float32))
        ba.put(r.standard_normal((m, k)).astype(np.float32))
        bl.put((r.standard_normal((m, vocab)) * 3).astype(np.float32))
        bu.put(r.random(m).astype(np.float32))
        before = cache.state()
        assert hip.hipGraphLaunch(ex, ctx.stream) == 0
        ctx.sync()
        got = state()
        cache.codes.put(before[0])
        cache.scales.put(before[1])
        step(turn % 2 == 0)
        ctx.sync()
        for x, y in zip(got, state()):
            np.testing.assert_array_equal(x, y)
        assert (got[2].view(np.int32) >= 0).all()
    hip.hipGraphExecDestroy(ex)
    hip.hipGraphDestroy(graph)
    for x in (*settings, *work, ids, logp, bl, bu, bw, ba, bc, codes, scales, s, batch, cache):
        x.free()


CASES = [("f32", 512, 200, 300, 4000, 70000, True), ("bf16", 256, 65, 8000, 300, 5000, True),
         ("bf16", 66, 1, 40, 9000, 70000, False)]


@pytest.mark.parametrize("case", CASES)
def test_captured_and_replayed(ctx, case):
    captured(ctx, *case)


@pytest.mark.parametrize("case", CASES)
def test_first_call_of_a_process(case):
    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    code = ("import sys; sys.path[:0] = ['tests', '.']; import test_gpu_step_first_call as t; from ai_amd import _native as "
            f"N; t.captured(N.Context(0), *{case!r}); print('done', flush=True)")
    r = subprocess.run([sys.executable, "-c", code], cwd=root, capture_output=True, text=True, timeout=100)
    assert r.returncode == 0 and r.stdout.strip() == "done", r.stderr[-2000:]
