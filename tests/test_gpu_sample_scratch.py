"""The scratch that sampling asks for, and the calls that need less."""
import ctypes as C

import numpy as np
import pytest

import kv_lib as K
import test_gpu_kvcache as G
import test_gpu_kvcache_use as use
import test_gpu_sample as T
from ai_amd import _native as N

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("settings", [False, True])
@pytest.mark.parametrize("rows,vocab", [(1, 1), (700, 3), (1, 70001), (37, 49999), (300, 4097), (3, 262144)])
def test_draws_without_filters_need_the_heads_of_slices(ctx, rows, vocab, settings):
    """The header's bound for them suffices, guards around it, and gives what the context's own scratch gives; with a
    filter it is too little."""
    r = G.rng(rows + vocab)
    L = N.lib()
    l, u = T.logits(r, rows, vocab, "f32"), T.numbers(r, rows)
    t = r.choice([0.0, 0.7, 1.3], rows).astype(np.float32)
    want = T.draw(ctx, l, u, **(dict(temperature=t) if settings else {}))
    size = 24 * rows * -(-vocab // 4096) + 256
    bufs = [K.Buf(ctx, x) for x in (l, u, t)]
    ids, logp = K.Buf(ctx, nbytes=4 * rows, fill=0x5A), K.Buf(ctx, nbytes=4 * rows, fill=0x5A)
    work = use.Guarded(ctx, np.full(size, 0xFF, np.uint8))
    s = N.Sampling(bufs[2].p, None, None, None)

    def call(s):
        return L.fa_sample_dev(ctx.h, rows, vocab, N.FA_DT_F32, bufs[0].p, vocab, s, bufs[1].p, ids.p, logp.p, work.p, size)

    N.check(ctx.h, call(C.byref(s) if settings else None))
    ctx.sync()
    work.get()
    np.testing.assert_array_equal(ids.get(rows, np.int32), want[0])
    np.testing.assert_array_equal(logp.get(rows, np.uint32), want[1].view(np.uint32))
    for name in ("top_k", "top_p", "min_p"):
        f = N.Sampling(bufs[2].p, None, None, None)
        setattr(f, name, bufs[1].p)  # (refused before anything reads it)
        assert call(C.byref(f)) == N.FA_ERR_ARG and b"work" in L.fa_last_error(ctx.h)
    for b in (*bufs, ids, logp, work):
        b.free()


def test_short_rows_list_no_more_than_they_have(ctx):
    """2 bytes for each token of a row shorter than a slice, beside its sums; filters of all kinds within it."""
    r = G.rng(9)
    need = C.c_size_t(0)
    for vocab in (1, 2, 300, 4095):
        N.check(ctx.h, N.lib().fa_sample_work(1000, vocab, C.byref(need)))
        assert need.value <= 1000 * (12 * 1024 + 2 * vocab + 24 + 128 + 4) + 6 * 256
        l, u, s = T.logits(r, 40, vocab, "f32", "ties"), T.numbers(r, 40), T.settings(r, 40)
        T.check(T.draw(ctx, l, u, work=True, **s), l, u, **s)
