"""A decoding step's operators without a GPU: their references against
arithmetic, the exported sizes, and every refusal (arguments are checked before
the context is used)."""
import ctypes as C

import numpy as np
import pytest

import decode_oracle as O
import test_kvcache as K
from ai_amd import _native as N
from ai_amd import f8, kvcache
from ai_amd import sample as smp
from ai_amd.tensor import TensorError

L = N.lib()
P = 0x1000  # a pointer that no refused call follows
NAN, INF = float("nan"), float("inf")


def refused(rc, text):
    msg = L.fa_last_error(None).decode()
    assert rc == N.FA_ERR_ARG and text in msg, (rc, msg)


# ---- references -----------------------------------------------------------------------------


def test_reference_rotation():
    r = np.random.default_rng(0)
    x = r.standard_normal((5, 2, 10)).astype(np.float32)
    pos = np.array([0, 1, 7, 100000, -3])
    y = O.rotate(x, pos, 1e4, 6)
    np.testing.assert_array_equal(y[0], x[0])           # position 0 turns nothing
    np.testing.assert_array_equal(y[..., 6:], x[..., 6:])
    z = (x[..., :3] + 1j * x[..., 3:6]) * np.exp(1j * pos[:, None, None] * 1e4 ** (-2 * np.arange(3) / 6))
    np.testing.assert_allclose(y[..., :3] + 1j * y[..., 3:6], z, atol=1e-6)


def test_reference_quantize():
    r = np.random.default_rng(1)
    x = (r.standard_normal((3, 300)) * 10.0 ** r.uniform(-30, 30, (3, 1))).astype(np.float32)
    x[0, :128] = 0
    x[1, 5], x[2, 299] = np.nan, -np.inf
    x[2, 0] = 3.4e38
    q, e = O.quantize(x)
    assert q.shape == (3, 3, 128) and e[0, 0] == -80 and e[2, 0] == 120 and (q[:, 2, 44:] == 0).all()
    v = O.values(q, e, 300)
    fin = np.isfinite(x)
    assert (np.isnan(v) == ~fin).all()
    block = np.arange(300) // 128
    near = np.maximum(np.abs(x) * 2.0 ** -4, 2.0 ** (e[:, block] - 10))
    near[2, 0] = np.inf  # above 240 * 2^120
    assert (np.abs(v - x)[fin] <= near[fin]).all()
    assert v[2, 0] == 240 * 2.0 ** 120
    q, e = O.quantize(np.array([[448.0], [448.00003], [224.0]]))
    assert e[:, 0].tolist() == [0, 1, -1]


def test_reference_sampling():
    l = np.log(np.array([1.0, 4, 2, 2, 1]))
    ids = [O.sample(l, u)[0] for u in np.arange(10) / 10 + 1e-9]
    assert ids == [0, 1, 1, 1, 1, 2, 2, 3, 3, 4]
    assert [O.sample(l, u, top_k=2)[0] for u in (0.0, 0.6, 0.7, 0.99)] == [1, 1, 2, 2]   # ties: the lower id
    assert [O.sample(l, u, top_p=0.7)[0] for u in (0.0, 0.7, 0.9)] == [1, 2, 3]           # 4 + 2 < 7, + 2
    assert [O.sample(l, u, min_p=0.5)[0] for u in (0.0, 0.6, 0.9)] == [1, 2, 3]
    assert O.sample(l, 0.9, temperature=0) == (1, 0.0) and O.sample(l, 0.99, top_p=0.0)[0] == 1
    assert O.sample(np.array([-INF, NAN]), 0.5)[0] == -1
    assert O.sample(np.array([1.0, INF, INF]), 0.6) == (2, np.log(0.5))
    assert abs(O.sample(l, 0.0)[1] - np.log(0.1)) < 1e-12


# ---- rotary writing ---------------------------------------------------------------------------


class Rope(K.Call):
    def __init__(self, **kw):
        super().__init__(**kw)
        self.rope = N.KvRope(1e4, 64, None)
        self.q, self.out = self.p, self.p

    def call(self, host=True, rope=True):
        f = L.fa_kv_write_rope if host else L.fa_kv_write_rope_dev
        return f(None, C.byref(self.cache), C.byref(self.batch), C.byref(self.rope) if rope else None, self.dtype,
                 self.q, *self.st, self.H, self.out, self.p, *self.st, self.p, *self.st)


@pytest.mark.parametrize("host", [True, False])
def test_rope_refusals(host):
    c = Rope()
    refused(c.call(host), "ctx is NULL")
    refused(c.call(host, rope=False), "rope is NULL")
    for base in (0.0, -1.0, NAN, INF):
        c = Rope()
        c.rope.base = base
        refused(c.call(host), "base")
    for dims in (0, -2, 3, 66, 1):
        c = Rope()
        c.rope.dims = dims
        refused(c.call(host), "rotary dims")
    for heads in (-2, 3, 65534):
        c = Rope()
        c.H = heads
        refused(c.call(host), "heads")
    c = Rope()
    c.H = 0
    refused(c.call(host), "queries of no heads")
    c.q = c.out = None
    refused(c.call(host), "ctx is NULL")
    for what in ("q", "out"):
        c = Rope()
        setattr(c, what, None)
        refused(c.call(host), "NULL buffer")
    c = Rope()
    c.p = None
    refused(c.call(host), "NULL buffer")
    c = Rope()
    c.st = (-1, 64)
    refused(c.call(host), "negative stride")
    c = Rope()
    c.st = (1 << 60, 64)
    refused(c.call(host), "too large")
    c = Rope()
    c.dtype = 2
    refused(c.call(host), "unknown dtype")
    c = Rope()
    c.cache.head_dim = 513
    refused(c.call(host), "head dimension")


def test_rope_refuses_what_the_batch_cannot_do():
    refused(Rope(table=((2, 0), (7, -1))).call(), "outside 0..3")
    refused(Rope(table=((2, 1), (1, -1))).call(), "written twice")
    refused(Rope(lengths=(2, 5)).call(), "2 tokens but 3 rows")


# ---- products ------------------------------------------------------------------------------------


def test_f8_sizes():
    f, g = L.fa_f8_codes_bytes, L.fa_f8_scales_bytes
    assert f(3, 128) == 384 and f(3, 129) == 768 and f(5, 1) == 640 and f(0, 5) == 0 and f(5, 0) == 0
    assert g(3, 128) == 12 and g(3, 512) == 12 and g(3, 513) == 24 and g(1, 1) == 4
    for bad in ((-1, 1), (1, -1), (1 << 27, 1), (1, 1 << 24)):
        assert f(*bad) == 0 and g(*bad) == 0
    assert f((1 << 27) - 1, 200) == ((1 << 27) - 1) * 256


class F8:
    def __init__(self):
        self.w = N.F8Matrix(P, P, 10, 200)
        self.m, self.adt, self.a, self.lda, self.cdt, self.c, self.ldc = 3, 0, P, 200, 0, P, 10
        self.e = N.Epilogue(None, None, 0, None, 10, None, 10)

    def call(self, host=True, work=None, nbytes=0):
        a = (None, self.m, self.adt, self.a, self.lda, C.byref(self.w), C.byref(self.e), self.cdt, self.c, self.ldc)
        return L.fa_matmul_f8(*a) if host else L.fa_matmul_f8_dev(*a, work, nbytes)


@pytest.mark.parametrize("host", [True, False])
def test_product_refusals(host):
    def change(text, **kw):
        c = F8()
        for k, v in kw.items():
            setattr(c.w if k in ("codes", "scales", "n", "k") else c.e if k in ("act", "mul", "ldm", "residual", "ldr")
                    else c, k, v)
        refused(c.call(host), text)

    change("ctx is NULL")
    change("outside [0..2^27)", n=-1)
    change("outside [0..2^27)", n=1 << 27)
    change("outside [0..2^27)", k=1 << 24)
    change("outside [0..2^27)", m=-1)
    change("outside [0..2^27)", m=1 << 27)
    change("more than one call takes", m=(1 << 27) - 1, n=(1 << 27) - 1, ldc=1 << 27)
    change("NULL matrix buffer", codes=None)
    change("NULL matrix buffer", scales=None)
    change("aligned", codes=P + 8)
    change("aligned", scales=P + 2)
    change("unknown dtype 2", adt=2)
    change("unknown dtype 7", cdt=7)
    change("leading dimension 199", lda=199)
    change("leading dimension 9", ldc=9)
    change("leading dimension", lda=(1 << 30) + 1)
    change("unknown activation", act=4)
    change("Mul: leading dimension 9", mul=P, ldm=9)
    change("Residual: leading dimension 9", residual=P, ldr=9)
    change("NULL buffer", a=None)
    change("NULL buffer", c=None)
    f = L.fa_matmul_f8 if host else lambda *a: L.fa_matmul_f8_dev(*a, None, 0)
    refused(f(None, 1, 0, P, 1, None, None, 0, P, 1), "matrix is NULL")


@pytest.mark.parametrize("name", ["fa_f8_write", "fa_f8_write_dev", "fa_f8_read", "fa_f8_read_dev"])
def test_conversion_refusals(name):
    f = getattr(L, name)
    w = N.F8Matrix(P, P, 10, 200)
    refused(f(None, C.byref(w), 0, P, 200), "ctx is NULL")
    refused(f(None, None, 0, P, 200), "matrix is NULL")
    refused(f(None, C.byref(w), 3, P, 200), "unknown dtype")
    refused(f(None, C.byref(w), 0, P, 199), "leading dimension")
    refused(f(None, C.byref(w), 0, None, 200), "NULL buffer")
    refused(f(None, C.byref(N.F8Matrix(None, P, 10, 200)), 0, P, 200), "NULL matrix buffer")
    refused(f(None, C.byref(N.F8Matrix(P, P, 10, -1)), 0, P, 200), "outside")


def test_work_sizes():
    need = C.c_size_t(7)
    w = N.F8Matrix(None, None, 10, 200)  # sizes only: before anything is allocated
    assert L.fa_matmul_f8_work(5, C.byref(w), C.byref(need)) == N.FA_OK and need.value >= 0
    refused(L.fa_matmul_f8_work(-1, C.byref(w), C.byref(need)), "outside")
    refused(L.fa_matmul_f8_work(1, None, C.byref(need)), "matrix is NULL")
    refused(L.fa_matmul_f8_work(1, C.byref(w), None), "bytes is NULL")
    assert L.fa_matmul_f8_work(0, C.byref(w), C.byref(need)) == N.FA_OK and need.value == 0
    assert L.fa_sample_work(4, 1000, C.byref(need)) == N.FA_OK
    refused(L.fa_sample_work(4, 0, C.byref(need)), "vocabulary")
    refused(L.fa_sample_work(1 << 20, 5, C.byref(need)), "rows")
    refused(L.fa_sample_work(4, 5, None), "bytes is NULL")


# ---- sampling ----------------------------------------------------------------------------------------


@pytest.mark.parametrize("host", [True, False])
def test_sampling_refusals(host):
    def call(rows=2, vocab=5, dtype=0, logits=P, ld=5, u=P, ids=P):
        a = (None, rows, vocab, dtype, logits, ld, None, u, ids, None)
        return L.fa_sample(*a) if host else L.fa_sample_dev(*a, None, 0)

    refused(call(), "ctx is NULL")
    refused(call(rows=-1), "rows")
    refused(call(rows=1 << 20), "rows")
    refused(call(vocab=0), "vocabulary")
    refused(call(vocab=(1 << 24) + 1, ld=1 << 25), "vocabulary")
    refused(call(dtype=2), "unknown dtype")
    refused(call(ld=4), "leading dimension")
    refused(call(ld=1 << 41), "leading dimension")
    for name in ("logits", "u", "ids"):
        refused(call(**{name: None}), "NULL buffer")


# ---- the Python classes' own checks (before anything reaches the library) -----------------------------


class NoGpu:
    h = None


def test_python_refusals():
    x = np.zeros((2, 5), np.float32)
    with pytest.raises(TensorError, match="2-D"):
        f8.F8Matrix(np.zeros(5), ctx=NoGpu())
    with pytest.raises(TensorError, match="want logits"):
        smp.Sample(x[0], 0.5, ctx=NoGpu())
    with pytest.raises(TensorError, match="no numbers"):
        smp.Sample(x, None, ctx=NoGpu())
    with pytest.raises(TensorError, match="top_p has shape"):
        smp.Sample(x, [0.5, 0.5], top_p=[1.0], ctx=NoGpu())
    with pytest.raises(TensorError, match="not a whole number"):
        smp.Sample(x, [0.5, 0.5], top_k=2.5, ctx=NoGpu())
    with pytest.raises(TensorError, match="ctx is NULL"):
        smp.Sample(x, [0.5, 0.5], top_k=10 ** 12, ctx=NoGpu())
    m = f8.F8Matrix.__new__(f8.F8Matrix)
    m.ctx, m._codes, m._scales, m.n, m.k = NoGpu(), N.vp(), N.vp(), 3, 5
    for use in (m.Values, lambda: m.MatMul(x)):
        with pytest.raises(TensorError, match="closed"):
            use()
    m._codes = N.vp(P)
    with pytest.raises(TensorError, match="times the transpose"):
        m.MatMul(np.zeros((2, 4), np.float32))
    with pytest.raises(TensorError, match="dtype"):
        m.MatMul(x, dtype=np.float64)
    with pytest.raises(TensorError, match="Bias has shape"):
        m.MatMul(x, f8.Fused(Bias=np.zeros(4)))
    m._codes = N.vp()


def test_python_append_refusals(monkeypatch):
    c = kvcache.KVCache.__new__(kvcache.KVCache)
    c.kv_heads, c.head_dim, c.blocks, c.ctx = 1, 8, 4, NoGpu()
    c._codes, c._scales = N.vp(P), N.vp(P)
    c.cache = N.KvCache(P, P, 4, 1, 8)
    c._free, c._tables, c._lengths, c._next = [3, 2, 1, 0], {}, {}, 0
    s = c.Add()
    k, q = np.zeros((2, 1, 8), np.float32), np.zeros((2, 3, 8), np.float32)
    for kw, text in ((dict(base=0.0), "base"), (dict(base=1e4, dims=3), "rotary dims"), (dict(base=1e4, dims=16), "rotary"),
                     (dict(base=1e4, dims=2 ** 40), "rotary dims"), (dict(base=1e4, positions=[1]), "positions"),
                     (dict(base=1e4, positions=[1, 2 ** 31]), "positions"),
                     (dict(base=1e4, positions=[0.5, 1.0]), "positions"), (dict(base=1e4), "ctx is NULL")):
        with pytest.raises(TensorError, match=text):
            c.AppendRoPE([s], q, k, k, [2], **kw)
        assert c.Len(s) == 0 and c.Room() == 256  # nothing was added
    with pytest.raises(TensorError, match="2 queries|queries for"):
        c.AppendRoPE([s], q[:1], k, k, [2], base=1e4)
    with pytest.raises(TensorError, match="q is"):
        c.AppendRoPE([s], q.astype(np.uint16), k, k, [2], base=1e4)
    with pytest.raises(TensorError, match="given twice"):
        c.AppendRoPE([s, s], q, k, k, base=1e4)
    c._codes = c._scales = N.vp()
