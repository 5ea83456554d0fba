"""What a KVCache holds of the device, without one: its pool is freed once, however the program lets go of it, and a
call that fails leaves its sequences as they were."""
import ctypes as C
import gc

import numpy as np
import pytest

from ai_amd import _native as N
from ai_amd import kvcache as M
from ai_amd.tensor import TensorError

REAL = N.lib()


class FakeLib:
    """Allocations and contexts as numbers; every operator succeeds."""

    def __init__(self):
        self.fa_kv_codes_bytes = REAL.fa_kv_codes_bytes
        self.held, self.log = {}, []

    def fa_device_alloc(self, ctx, n, out):
        p = 256 * (len(self.log) + 1)
        self.held[p] = ctx
        self.log.append(("alloc", p))
        C.cast(out, C.POINTER(C.c_void_p))[0] = p
        return N.FA_OK

    def fa_device_free(self, ctx, p):
        assert self.held.pop(p.value) == ctx
        self.log.append(("free", p.value))
        return N.FA_OK

    def fa_destroy(self, ctx):
        self.log.append(("destroy", ctx))

    def fa_last_error(self, ctx):
        return b"no"

    def fa_kv_write(self, *a):
        return N.FA_OK

    fa_kv_attention = fa_kv_read = fa_kv_write


@pytest.fixture
def fake(monkeypatch):
    lib = FakeLib()
    monkeypatch.setattr(N, "lib", lambda: lib)
    return lib


def context(h):
    c = N.Context.__new__(N.Context)  # as after fa_create
    c.h = h
    N.own(c)
    return c


def test_a_dropped_cache_frees_its_pool(fake):
    ctx = context(7)
    c = M.KVCache(2, 64, 640, ctx=ctx)
    assert len(fake.held) == 2
    del c
    gc.collect()
    assert not fake.held
    ctx.close()


def test_a_context_closes_its_caches_first(fake):
    ctx, other = context(7), context(8)
    a, b, c = M.KVCache(2, 64, 640, ctx=ctx), M.KVCache(1, 64, 64, ctx=other), M.KVCache(1, 64, 64, ctx=ctx)
    ctx.close()
    assert set(fake.held.values()) == {8} and fake.log[-1] == ("destroy", 7)
    with pytest.raises(TensorError, match="closed"):
        a.Append([a.Add()], np.zeros((1, 2, 64), np.float32), np.zeros((1, 2, 64), np.float32))
    for x in (a, c, b):
        x.close()
        x.close()
    ctx.close()
    assert not fake.held and [e for e, _ in fake.log].count("free") == 6
    other.close()
    assert [e for e in fake.log if e[0] == "destroy"] == [("destroy", 7), ("destroy", 8)]


def test_a_call_that_fails_early_leaves_the_sequences(fake, monkeypatch):
    """Whatever goes wrong after blocks were handed out, before the library is called or while it runs."""
    c = M.KVCache(2, 64, 640, ctx=context(7))
    a, b = c.Add(), c.Add()
    x = np.zeros((100, 2, 64), np.float32)
    c.Append([a], x[:70], x[:70], [70])

    def fails(*args):
        raise error

    for error, name in ((MemoryError(), "_batch"), (KeyboardInterrupt(), "_batch"), (KeyboardInterrupt(), None)):
        with monkeypatch.context() as m:
            if name:
                m.setattr(M.KVCache, name, fails)
            else:
                m.setattr(FakeLib, "fa_kv_write", fails)
            with pytest.raises(type(error)):
                c.Append([a, b], x, x, [60, 40])
        assert (c.Len(a), c.Len(b), c.Room()) == (70, 0, 640 - 128)
    c.Append([a, b], x, x, [60, 40])
    assert (c.Len(a), c.Len(b), c.Room()) == (130, 40, 640 - 256)
    c.close()
    c.ctx.close()


def test_sizes_past_their_integers_are_refused(fake):
    """The library takes 32-bit sizes: larger ones are refused, not cut to their low bits."""
    ctx = context(7)
    for args in ((2 ** 32 + 2, 64, 640), (2, 2 ** 32 + 64, 640), (2, 64, 2 ** 38 + 64)):
        with pytest.raises(TensorError):
            M.KVCache(*args, ctx=ctx)
    c = M.KVCache(2, 64, 640, ctx=ctx)
    a = c.Add()
    k = np.zeros((1, 2, 64), np.float32)
    c.Append([a], k, k)
    for window in (2 ** 31, 2 ** 32, -1, -2 ** 32 + 5):
        with pytest.raises(TensorError, match="window"):
            c.Attention([a], k, window=window)
    c.Attention([a], k, window=2 ** 31 - 1)
    c.close()
    ctx.close()
    assert not fake.held
