"""The key/value cache without a GPU: its reference against arithmetic, the
exported sizes, and every refusal (arguments are checked before the context
is used)."""
import ctypes as C

import numpy as np
import pytest

import kv_oracle as O
from ai_amd import _native as N
from ai_amd import kvcache as M
from ai_amd.tensor import TensorError

L = N.lib()


def test_reference_rounding():
    """Every code is its own nearest value; between two neighbours the nearer wins, the even one on ties."""
    v = np.sort(O.DECODE[np.isfinite(O.DECODE)])
    v = np.unique(v)
    assert v.max() == 448 and (O.round_e4m3(v) == v).all() and len(v) == 253
    mid = (v[1:] + v[:-1]) / 2
    up = O.round_e4m3(mid * (1 + 1e-9) + 1e-13)
    assert (O.round_e4m3(mid + (v[1:] - v[:-1]) * 1e-6) == v[1:]).all() and np.isfinite(up).all()
    assert (O.round_e4m3(mid - (v[1:] - v[:-1]) * 1e-6) == v[:-1]).all()
    codes = {float(O.DECODE[b]): b for b in range(256) if np.isfinite(O.DECODE[b])}
    assert all(codes[float(t)] % 2 == 0 or t == 0 for t in O.round_e4m3(mid))


def test_reference_scale():
    assert O.scale_exp(np.array([448.0])) == 0 and O.scale_exp(np.array([448.0001])) == 1
    assert O.scale_exp(np.array([224.0])) == -1 and O.scale_exp(np.array([0.0, np.nan, np.inf])) == -80
    assert O.scale_exp(np.array([3.4028235e38])) == 120
    r = np.random.default_rng(0)
    x = r.standard_normal(1000) * 100
    e = O.scale_exp(x)
    assert np.abs(x).max() <= 448 * 2.0 ** e and np.abs(x).max() > 448 * 2.0 ** (e - 1)
    # what one write loses: half a step of four bits, or of the smallest code
    y = O.round_e4m3(x * 2.0 ** -e) * 2.0 ** e
    assert (np.abs(x - y) <= np.maximum(np.abs(x) * 2.0 ** -4, 2.0 ** (e - 10))).all()


def test_codes_bytes():
    f = L.fa_kv_codes_bytes
    assert f(10, 3, 64) == 10 * 3 * 2 * 4096 and f(1, 1, 1) == 8192 and f(2, 1, 65) == 2 * 2 * 8192
    assert f(1 << 20, 8, 512) == (1 << 20) * 8 * 2 * 64 * 512
    assert f(0, 1, 64) == 0
    for bad in ((-1, 1, 64), (1, 0, 64), (1, 70000, 64), (1, 1, 0), (1, 1, 513)):
        assert f(*bad) == 0


class Call:
    """Arguments of a call that would be right but for the context, on the host."""

    def __init__(self, lengths=(70, 5), ns=(3, 5), table=((2, 0), (1, -1)), blocks=4, Hkv=2, D=64):
        self.mem = np.zeros(1 << 16, np.uint8)
        at = (self.mem.ctypes.data + 255) & ~255
        self.cache = N.KvCache(at, at, blocks, Hkv, D)
        self.tables = np.array(table, np.int32)
        self.lengths = np.array(lengths, np.int32)
        self.cu = np.concatenate([[0], np.cumsum(ns)]).astype(np.int32)
        self.batch = N.KvBatch(self.tables.ctypes.data, self.tables.shape[1], self.lengths.ctypes.data,
                               self.cu.ctypes.data, len(self.lengths), int(self.cu[-1]))
        self.x = np.zeros((int(max(self.cu[-1], 1)), 8, D), np.float32)
        self.p, self.H, self.dtype, self.st = self.x.ctypes.data, 4, 0, (8 * D, D)
        self.window, self.scale = 0, 0.125

    def write(self, host=True):
        f = L.fa_kv_write if host else L.fa_kv_write_dev
        return f(None, C.byref(self.cache), C.byref(self.batch), self.dtype, self.p, *self.st, self.p, *self.st)

    def read(self, host=True):
        f = L.fa_kv_read if host else L.fa_kv_read_dev
        return f(None, C.byref(self.cache), C.byref(self.batch), self.dtype, self.p, self.p)

    def attend(self, host=True):
        a = (None, C.byref(self.cache), C.byref(self.batch), self.dtype, self.p, *self.st, self.H, 1, self.window,
             self.scale, self.p)
        return L.fa_kv_attention(*a) if host else L.fa_kv_attention_dev(*a, None, 0)

    def refused(self, words, which=("write", "read", "attend"), host=(True, False)):
        for w in which:
            for h in host:
                rc = getattr(self, w)(h)
                msg = L.fa_last_error(None).decode()
                assert rc == N.FA_ERR_ARG and words in msg, (w, h, rc, msg)


def test_right_arguments_get_as_far_as_the_context():
    Call().refused("ctx is NULL")
    Call(lengths=(), ns=(), table=np.zeros((0, 1))).refused("ctx is NULL")


@pytest.mark.parametrize("change,words", [
    (lambda c: setattr(c.cache, "blocks", -1), "blocks"), (lambda c: setattr(c.cache, "kv_heads", 0), "heads"),
    (lambda c: setattr(c.cache, "kv_heads", 70000), "heads"), (lambda c: setattr(c.cache, "head_dim", 0), "dimension"),
    (lambda c: setattr(c.cache, "head_dim", 513), "dimension"), (lambda c: setattr(c.cache, "codes", None), "NULL"),
    (lambda c: setattr(c.cache, "scales", None), "NULL"),
    (lambda c: setattr(c.cache, "codes", c.cache.codes + 8), "aligned"),
    (lambda c: setattr(c.batch, "nseq", -1), "negative"), (lambda c: setattr(c.batch, "rows", -1), "negative"),
    (lambda c: setattr(c.batch, "table_stride", -1), "negative"), (lambda c: setattr(c, "dtype", 7), "dtype"),
    (lambda c: setattr(c.batch, "lengths", None), "NULL"), (lambda c: setattr(c.batch, "cu_rows", None), "NULL"),
    (lambda c: setattr(c.batch, "tables", None), "NULL"), (lambda c: setattr(c, "p", None), "NULL"),
    (lambda c: setattr(c.batch, "rows", 2 ** 31), "more than one call")])
def test_refusals(change, words):
    c = Call()
    change(c)
    c.refused(words)


def test_refusals_of_strides_and_attention():
    c = Call()
    c.st = (-1, 64)
    c.refused("stride", ("write", "attend"))
    c.st = (64, -1)
    c.refused("stride", ("write", "attend"))
    for H in (0, 3, -2, 65536):
        c = Call()
        c.H = H
        c.refused("query heads", ("attend",))
    c = Call()
    c.window = -1
    c.refused("window", ("attend",))
    for s in (np.nan, np.inf):
        c = Call()
        c.scale = s
        c.refused("scale", ("attend",))


def test_refusals_of_host_batches():
    host = (True,)
    c = Call()
    c.cu[0] = 1
    c.refused("starts at", host=host)
    c = Call()
    c.cu[1] = 9
    c.refused("falls", host=host)
    c = Call()
    c.cu[2] = 40
    c.lengths[1] = 200
    c.refused("ends at", host=host)
    Call(lengths=(2, 5)).refused("tokens but", host=host)
    Call(lengths=(129, 5), ns=(1, 5), table=((2, 0), (1, -1))).refused("table entries", host=host)
    Call(table=((2, 4), (1, -1))).refused("outside", host=host)
    Call(table=((2, -1), (1, -1))).refused("outside", host=host)
    Call(table=((9, 0), (1, -1))).refused("outside", ("attend",), host)  # a block below the first row: only attention sees it
    Call(table=((9, 0), (1, -1))).refused("ctx is NULL", ("write", "read"), host)
    Call(table=((2, 1), (1, -1))).refused("written twice", ("write",), host)
    Call(table=((2, 1), (1, -1))).refused("ctx is NULL", ("read", "attend"), host)
    Call(lengths=(130, 5), ns=(70, 5), table=((3, 0, 0), (1, 1, 1))).refused("written twice", ("write",), host)
    c = Call(lengths=(70, -3), ns=(3, 0))
    c.refused("tokens but", host=host)


def test_refusals_of_sizes_past_a_launch():
    """More workgroups than a launch counts, positions and offsets past their integers."""
    c = Call()
    c.batch.table_stride = 1 << 25
    c.refused("table rows")
    n = C.c_size_t(7)
    assert L.fa_kv_attention_work(C.byref(c.cache), C.byref(c.batch), 4, C.byref(n)) == N.FA_ERR_ARG and n.value == 0
    c = Call()
    c.batch.nseq, c.batch.rows, c.H = 1 << 24, 1 << 24, 2
    c.refused("workgroups", host=(False,))
    c.batch.nseq = c.batch.rows = (1 << 24) - 1
    c.refused("ctx is NULL", ("write", "read"), host=(False,))
    c = Call()
    c.cache.head_dim, c.batch.rows = 512, (1 << 28) - 64  # 16 rows a workgroup
    c.refused("workgroups", ("attend",), host=(False,))
    for st in ((1 << 58, 64), (64, 1 << 58), ((1 << 63) - 1, 0)):
        c = Call()
        c.st = st
        c.refused("too large", ("write", "attend"))
    for s in (3e38, -3e38):
        c = Call()
        c.scale = s
        c.refused("scale", ("attend",))


def test_blocks_behind_the_window_need_no_table_entry():
    c = Call(lengths=(130, 5), ns=(2, 5), table=((-1, 2, 0), (1, -1, -1)))
    c.refused("outside", ("attend",), (True,))
    c.window = 65  # the first row, 128, sees 64 .. 129
    c.refused("ctx is NULL", ("attend",), (True,))
    c.window = 66
    c.refused("outside", ("attend",), (True,))


def test_work_size():
    n = C.c_size_t(7)
    c = Call()
    f = L.fa_kv_attention_work
    assert f(C.byref(c.cache), C.byref(c.batch), 4, None) == N.FA_ERR_ARG
    assert f(C.byref(c.cache), None, 4, C.byref(n)) == N.FA_ERR_ARG
    assert f(C.byref(c.cache), C.byref(c.batch), 3, C.byref(n)) == N.FA_ERR_ARG and n.value == 0
    assert f(C.byref(c.cache), C.byref(c.batch), 4, C.byref(n)) == N.FA_OK and n.value == 0  # two blocks: not split
    c.batch.table_stride = 1000
    assert f(C.byref(c.cache), C.byref(c.batch), 4, C.byref(n)) == N.FA_OK and 0 < n.value < 1 << 28
    c.batch.rows = 0
    assert f(C.byref(c.cache), C.byref(c.batch), 4, C.byref(n)) == N.FA_OK and n.value == 0


# ---- the Python class's own bookkeeping -----------------------------------------------------

class FakeLib:
    """Counts blocks in place of the device: allocation and the three operators always succeed."""

    def __init__(self, real):
        self.fa_kv_codes_bytes = real.fa_kv_codes_bytes
        self.rc = 0

    def fa_device_alloc(self, ctx, n, out):
        C.cast(out, C.POINTER(C.c_void_p))[0] = 256
        return 0

    def fa_device_free(self, ctx, p):
        return 0

    def fa_kv_write(self, *a):
        return self.rc

    def fa_last_error(self, ctx):
        return b"no"

    fa_kv_attention = fa_kv_read = fa_kv_write


class FakeCtx:
    h = 1


@pytest.fixture
def fake(monkeypatch):
    lib = FakeLib(L)
    monkeypatch.setattr(N, "lib", lambda: lib)
    return lib


def test_cache_blocks_are_handed_out_and_back(fake):
    c = M.KVCache(2, 64, 640, ctx=FakeCtx())
    assert c.blocks == 10 and c.Room() == 640
    a, b = c.Add(), c.Add()
    x = np.zeros((200, 2, 64), np.float32)
    c.Append([a, b], x, x, [130, 70])
    assert c.Len(a) == 130 and c.Len(b) == 70 and c.Room() == 640 - 5 * 64
    assert len(set(c._tables[a] + c._tables[b])) == 5
    c.Append([b], x[:58], x[:58], [58])  # fits into its last block
    assert c.Room() == 640 - 5 * 64
    with pytest.raises(TensorError, match="free"):
        c.Append([a], np.zeros((400, 2, 64), np.float32), np.zeros((400, 2, 64), np.float32), [400])
    fake.rc = N.FA_ERR_HIP  # a call that fails leaves the sequences as they were
    with pytest.raises(N.FaError):
        c.Append([a, b], x, x, [100, 100])
    fake.rc = 0
    assert c.Len(a) == 130 and c.Len(b) == 128 and c.Room() == 640 - 5 * 64
    c.Truncate(a, 64)
    assert c.Room() == 640 - 3 * 64 and len(c._tables[a]) == 1
    c.Free(b)
    assert c.Room() == 640 - 64
    with pytest.raises(TensorError, match="no sequence"):
        c.Len(b)
    batch, keep = c._batch([a], [3])
    assert batch.nseq == 1 and batch.rows == 3 and keep[1].tolist() == [64]
    c.close()
    with pytest.raises(TensorError, match="closed"):
        c.Append([a], x[:1], x[:1])


def test_cache_refusals(fake):
    for args in ((0, 64, 64), (1, 0, 64), (1, 513, 64), (1, 64, 0), (1, 64, -5)):
        with pytest.raises(TensorError):
            M.KVCache(*args, ctx=FakeCtx())
    c = M.KVCache(2, 64, 640, ctx=FakeCtx())
    a = c.Add()
    k = np.zeros((3, 2, 64), np.float32)
    for bad in (lambda: c.Append([a], k, k), lambda: c.Append([a], k, k[:2], [3]), lambda: c.Append([a], k, k, [-3]),
                lambda: c.Append([a], k, k.astype(np.uint16), [3]), lambda: c.Append([a], k[:, :1], k[:, :1], [3]),
                lambda: c.Append([a], k[0], k[0], [3]), lambda: c.Append([a, a], k, k, [1, 2]),
                lambda: c.Append([a + 1], k, k, [3]), lambda: c.Read(a, 1), lambda: c.Truncate(a, 1),
                lambda: c.Truncate(a, -1), lambda: c.Attention([a], np.zeros((1, 2, 63), np.float32)),
                lambda: c.Read(a, 0, dtype=np.float64)):
        with pytest.raises(TensorError):
            bad()
    c.close()
