"""Products with weights in 8 bits on the GPU against the definition
(decode_oracle.py): what is held, to the bit; products within bounds derived
there, and to the bit where every sum is exact."""
import ctypes as C

import numpy as np
import pytest

import decode_oracle as O
import kv_lib as K
import test_gpu_kvcache as G
import test_gpu_kvcache_use as use
from ai_amd import _native as N
from ai_amd import f8
from ai_amd import synth as S
from ai_amd import tensor as T

pytestmark = pytest.mark.gpu
DT = {"f32": N.FA_DT_F32, "bf16": N.FA_DT_BF16}
NP = {"f32": np.float32, "bf16": np.uint16}


class Held:
    """A matrix in 8 bits on the device, its bytes 0xFF before it is written."""

    def __init__(self, ctx, n, k):
        L = N.lib()
        self.ctx, self.n, self.k, self.kb = ctx, n, k, -(-k // 128)
        self.codes = use.Guarded(ctx, np.full(L.fa_f8_codes_bytes(n, k), 0xFF, np.uint8))
        self.scales = use.Guarded(ctx, np.full(L.fa_f8_scales_bytes(n, k), 0xFF, np.uint8))
        self.w = N.F8Matrix(self.codes.p, self.scales.p, n, k)

    def write(self, x):
        b = K.Buf(self.ctx, K.span_of(x))
        N.check(self.ctx.h, N.lib().fa_f8_write_dev(self.ctx.h, C.byref(self.w), K.dt(x), b.p,
                                                    max(x.strides[0] // x.itemsize, x.shape[1])))
        self.ctx.sync()
        b.free()
        return self

    def read(self, dtype="f32", pad=0):
        out = K.Buf(self.ctx, nbytes=self.n * (self.k + pad) * (4 if dtype == "f32" else 2), fill=0x5A)
        N.check(self.ctx.h, N.lib().fa_f8_read_dev(self.ctx.h, C.byref(self.w), DT[dtype], out.p, self.k + pad))
        self.ctx.sync()
        got = out.get((self.n, self.k + pad), NP[dtype])
        out.free()
        assert (got[:, self.k:].view(np.uint8) == 0x5A).all()
        return got[:, :self.k]

    def free(self):
        self.codes.free()
        self.scales.free()


def product(ctx, held, a, cdt, e=None, pad=0, work=False):
    """C and the guards of everything the call may touch, checked."""
    m, n = len(a), held.n
    L = N.lib()
    ba = use.Guarded(ctx, K.span_of(a))
    c = use.Guarded(ctx, np.full((m, n + pad), 0x5A5A5A5A if cdt == "f32" else 0x5A5A, np.uint32 if cdt == "f32" else np.uint16))
    bufs, ep = [], N.Epilogue(None, None, 0, None, n, None, n)
    for name, x in (e or {}).items():
        if name == "act":
            ep.act = x
            continue
        bufs.append(use.Guarded(ctx, K.span_of(x)))
        setattr(ep, name, bufs[-1].p)
        if x.ndim == 2:
            setattr(ep, {"mul": "ldm", "residual": "ldr"}[name], x.strides[0] // 4)
    w, need = None, C.c_size_t(0)
    if work:
        N.check(ctx.h, L.fa_matmul_f8_work(m, C.byref(held.w), C.byref(need)))
        w = use.Guarded(ctx, np.full(need.value, 0xFF, np.uint8))
    N.check(ctx.h, L.fa_matmul_f8_dev(ctx.h, m, K.dt(a), ba.p, max(a.strides[0] // a.itemsize, held.k, 1), C.byref(held.w),
                                      C.byref(ep) if e is not None else None, DT[cdt], c.p, n + pad, w.p if w else None,
                                      need.value))
    ctx.sync()
    got = c.get()
    if cdt == "f32":
        got = got.view(np.float32)
    for b in (ba, *bufs):
        np.testing.assert_array_equal(b.get().view(np.uint8), b.a.view(np.uint8))
    if w:
        w.get()
    assert (got[:, n:].view(np.uint8) == 0x5A).all()
    for b in (ba, c, w, *bufs):
        if b:
            b.free()
    return np.ascontiguousarray(got[:, :n])


def check(got, want, tol, what):
    g = K.wide(got).astype(np.float64)
    assert g.shape == want.shape
    nan = np.isnan(want)
    assert (np.isnan(g) == nan).all(), what
    d = np.abs(g - want)
    worst = float((d / tol)[~nan].max()) if (~nan).any() else 0.0
    print(f"{what}: {worst:.3g} of the bound", flush=True)
    assert (d <= tol)[~nan].all(), (what, worst)


def case(ctx, m, n, k, adt, cdt, seed=0, epi=(), pad=0, work=False, tails=False):
    r = G.rng(seed + m * 7 + n * 3 + k)
    a = r.standard_normal((m, k)) * np.exp((1.5 if tails else 0.5) * r.standard_normal((m, k if tails else 1)))
    a, w = a.astype(np.float32), (r.standard_normal((n, k)) / np.sqrt(max(k, 1))).astype(np.float32)
    a = S.f32_to_bf16(a) if adt == "bf16" else a
    held = Held(ctx, n, k).write(w)
    e = {}
    make = dict(bias=lambda: r.standard_normal(n), row_scale=lambda: r.standard_normal(m),
                mul=lambda: r.standard_normal((m, n)), residual=lambda: r.standard_normal((m, n)))
    for x in epi:
        if isinstance(x, int):
            e["act"] = x
        else:
            e[x] = make[x]().astype(np.float32)
    got = product(ctx, held, a, cdt, e if epi else None, pad, work)
    want, tol = O.product(K.wide(a).astype(np.float64), w.astype(np.float64), cdt == "bf16", **e)
    check(got, want, tol, f"{m}x{n}x{k} {adt}->{cdt} {epi}")
    held.free()


# ---- what is held ----------------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,k", [(1, 1), (3, 127), (5, 128), (2, 129), (17, 300), (1, 640), (300, 512), (4, 513), (1000, 4)])
def test_write_and_read_are_exact(ctx, n, k, dtype):
    r = G.rng(n * 1000 + k)
    x = (r.standard_normal((n, k)) * np.exp(3 * r.standard_normal((n, 1)))).astype(np.float32)
    x = S.f32_to_bf16(x) if dtype == "bf16" else x
    h = Held(ctx, n, k).write(x)
    q, e = O.quantize(K.wide(x))
    want = O.values(q, e, k).astype(np.float32)
    np.testing.assert_array_equal(h.read(), want)
    np.testing.assert_array_equal(S.bf16_to_f32(h.read("bf16", 3)), want)
    codes = h.codes.get().reshape(n, h.kb * 128)
    assert (codes[:, k:] == 0).all()
    scales = h.scales.get().reshape(n, -1)
    np.testing.assert_array_equal(scales[:, :h.kb], (e + 127).astype(np.uint8))
    assert (scales[:, h.kb:] == 127).all()
    h.free()


def test_special_values_are_held(ctx):
    x = np.zeros((6, 256), np.float32)
    x[0, :3] = np.nan, np.inf, -np.inf
    x[0, 5] = 1.0
    x[1, 200] = 3.4028235e38
    x[1, 201] = -3.3e38
    x[2] = 1e-30
    x[3] = 1e-45
    x[4, ::2] = -0.0
    x[5, :128] = np.inf
    h = Held(ctx, 6, 256).write(x)
    got = h.read()
    q, e = O.quantize(x)
    np.testing.assert_array_equal(got, O.values(q, e, 256).astype(np.float32))
    assert np.isnan(got[0, :3]).all() and got[0, 5] == 1.0 and got[1, 200] == np.float32(240 * 2.0 ** 120)
    h.free()


def test_rows_of_other_strides(ctx):
    r = G.rng(3)
    for ld, off in ((301, 0), (304, 1), (304, 4)):
        x = r.standard_normal((20, ld + 8)).astype(np.float32).ravel()[off:off + 20 * ld].reshape(20, ld)[:, :300]
        h = Held(ctx, 20, 300).write(x)
        q, e = O.quantize(x)
        np.testing.assert_array_equal(h.read(), O.values(q, e, 300).astype(np.float32))
        h.free()


# ---- products ----------------------------------------------------------------------------------


@pytest.mark.parametrize("cdt", ["f32", "bf16"])
@pytest.mark.parametrize("adt", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(1, 1, 1), (1, 17, 128), (2, 64, 127), (3, 100, 129), (16, 33, 640), (17, 256, 384),
                                   (31, 48, 2048), (33, 130, 65), (64, 64, 1024), (65, 300, 257), (130, 129, 512),
                                   (257, 513, 300), (300, 1, 700), (5, 1000, 33)])
def test_product_sizes(ctx, m, n, k, adt, cdt):
    case(ctx, m, n, k, adt, cdt)


@pytest.mark.parametrize("cdt", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(1, 5000, 768), (8, 4096, 1024), (40, 2000, 4096), (500, 1152, 768), (1024, 512, 256),
                                   (700, 900, 1300)])
def test_product_larger(ctx, m, n, k, cdt):
    case(ctx, m, n, k, "bf16", cdt, work=True)


@pytest.mark.parametrize("cdt", ["f32", "bf16"])
@pytest.mark.parametrize("m", [1, 6, 40, 300])
@pytest.mark.parametrize("epi", [("bias",), ("row_scale",), (1,), (2,), (3,), ("mul",), ("residual",),
                                 ("bias", "row_scale", 2, "mul", "residual"), ()])
def test_epilogues(ctx, m, epi, cdt):
    case(ctx, m, 150, 200, "f32", cdt, epi=epi, pad=3)


@pytest.mark.parametrize("cdt", ["f32", "bf16"])
@pytest.mark.parametrize("m", [1, 16, 50, 400])
def test_long_tails(ctx, m, cdt):
    """Activations over many binades: where the 8-bit units cut most."""
    case(ctx, m, 300, 1024, "f32", cdt, tails=True)


@pytest.mark.parametrize("cdt", ["f32", "bf16"])
@pytest.mark.parametrize("m", [1, 2, 15, 16, 17, 32, 33, 64, 100, 129, 256, 300])
@pytest.mark.parametrize("n,k", [(40, 128), (200, 700), (513, 1536)])
def test_exact_sums(ctx, m, n, k, cdt):
    """Operands of -1, 0 and 1 with a block's scale of its own: sums are whole numbers times it, to the bit; a term lost
    or read twice, or a scale of another block or row, shows."""
    r = G.rng(m + n + k)
    kb = -(-k // 128)
    mine = np.arange(k) // 128
    a = r.integers(-1, 2, (m, k)).astype(np.float32)
    w = r.integers(-1, 2, (n, k)).astype(np.float32)
    a[:, ::128], w[:, ::128] = 1, 1
    sa, sw = 2.0 ** r.integers(-3, 4, (m, kb)), 2.0 ** r.integers(-3, 4, (n, kb))
    a, w = (a * sa[:, mine]).astype(np.float32), (w * sw[:, mine]).astype(np.float32)
    want = a.astype(np.float64) @ w.astype(np.float64).T
    held = Held(ctx, n, k).write(w)
    got = K.wide(product(ctx, held, a, cdt))
    if cdt == "bf16":  # one rounding of an exact sum
        want = S.bf16_to_f32(S.f32_to_bf16(want.astype(np.float32)))
    np.testing.assert_array_equal(got, want.astype(np.float32))
    held.free()


@pytest.mark.parametrize("cdt", ["f32", "bf16"])
@pytest.mark.parametrize("m,n", [(1, 60), (20, 200), (200, 300)])
def test_nan_stays_in_its_row_and_column(ctx, m, n, cdt):
    r = G.rng(m)
    k = 390
    a, w = r.standard_normal((m, k)).astype(np.float32), r.standard_normal((n, k)).astype(np.float32)
    a[m // 2, 389], w[n // 3, 130] = np.inf, np.nan
    held = Held(ctx, n, k).write(w)
    got = np.isnan(K.wide(product(ctx, held, a, cdt)))
    want = np.zeros((m, n), bool)
    want[m // 2], want[:, n // 3] = True, True
    np.testing.assert_array_equal(got, want)
    held.free()


@pytest.mark.parametrize("cdt", ["f32", "bf16"])
def test_empty_sizes(ctx, cdt):
    """No columns of A: the epilogue of zero; no rows, no features: nothing."""
    L = N.lib()
    bias = np.arange(7, dtype=np.float32)
    held = N.F8Matrix(None, None, 7, 0)
    bb, c = K.Buf(ctx, bias), use.Guarded(ctx, np.zeros((3, 7), np.float32 if cdt == "f32" else np.uint16))
    e = N.Epilogue(bb.p, None, 0, None, 7, None, 7)
    N.check(ctx.h, L.fa_matmul_f8_dev(ctx.h, 3, 0, None, 0, C.byref(held), C.byref(e), DT[cdt], c.p, 7, None, 0))
    ctx.sync()
    np.testing.assert_array_equal(K.wide(c.get()), np.broadcast_to(bias, (3, 7)))
    for m, n in ((0, 7), (3, 0)):
        N.check(ctx.h, L.fa_matmul_f8_dev(ctx.h, m, 0, None, 5, C.byref(N.F8Matrix(None, None, n, 0)), None, DT[cdt], None, 7,
                                          None, 0))
    bb.free()
    c.free()


def test_strided_operands(ctx):
    """Rows of A and of the epilogue's matrices that are not aligned, or lie apart."""
    r = G.rng(4)
    for ld, off, adt in ((261, 0, "f32"), (264, 3, "f32"), (260, 2, "bf16"), (259, 1, "bf16"), (264, 8, "bf16")):
        for m in (2, 70):
            flat = r.standard_normal(m * ld + 16).astype(np.float32)
            flat = S.f32_to_bf16(flat) if adt == "bf16" else flat
            a = flat[off:off + m * ld].reshape(m, ld)[:, :257]
            w = r.standard_normal((90, 257)).astype(np.float32)
            mul = r.standard_normal((m, 95)).astype(np.float32)[:, :90]
            held = Held(ctx, 90, 257).write(w)
            got = product(ctx, held, a, "f32", dict(mul=mul), pad=1)
            want, tol = O.product(K.wide(np.ascontiguousarray(a)).astype(np.float64), w.astype(np.float64), False, mul=mul)
            check(got, want, tol, f"ld {ld} off {off} {adt} m {m}")
            held.free()


@pytest.mark.parametrize("cdt", ["f32", "bf16"])
def test_same_results_every_time(ctx, cdt):
    r = G.rng(5)
    for m, n, k in ((3, 2000, 4096), (48, 512, 4096), (300, 260, 1000)):
        a, w = r.standard_normal((m, k)).astype(np.float32), r.standard_normal((n, k)).astype(np.float32)
        held = Held(ctx, n, k).write(w)
        first = product(ctx, held, a, cdt)
        for i in range(3):
            np.testing.assert_array_equal(product(ctx, held, a, cdt, work=i > 0), first)
        held.free()


def test_host_entry_points_and_the_class(ctx):
    r = G.rng(6)
    m, n, k = 9, 70, 200
    x, w = r.standard_normal((m, k)).astype(np.float32), r.standard_normal((n, k)).astype(np.float32)
    bias, mul = r.standard_normal(n).astype(np.float32), r.standard_normal((m, n)).astype(np.float32)
    held = Held(ctx, n, k).write(w)
    with f8.F8Matrix(w, ctx=ctx) as M:
        np.testing.assert_array_equal(M.Values(), held.read())
        np.testing.assert_array_equal(M.Values(dtype=np.uint16), held.read("bf16"))
        for xs, adt in ((x, "f32"), (S.f32_to_bf16(x), "bf16"), (np.asfortranarray(x), "f32")):
            for cdt in ("f32", "bf16"):
                np.testing.assert_array_equal(M.MatMul(xs, dtype=NP[cdt]),
                                              product(ctx, held, np.ascontiguousarray(xs), cdt))
        f = T.Fused(Bias=bias, Act=T.GELUAct, Mul=mul)
        np.testing.assert_array_equal(M.MatMul(x, f), product(ctx, held, x, "f32", dict(bias=bias, act=2, mul=mul)))
        assert M.MatMul(x[:0]).shape == (0, n)
        # rows of C that lie apart on the host keep what is between them
        c = np.full((m, n + 5), 7.0, np.float32)
        N.check(ctx.h, N.lib().fa_matmul_f8(ctx.h, m, 0, x.ctypes.data, k, C.byref(M.matrix), None, 0, c.ctypes.data, n + 5))
        np.testing.assert_array_equal(c[:, :n], M.MatMul(x))
        assert (c[:, n:] == 7).all()
    held.free()


def test_work_is_checked(ctx):
    held = Held(ctx, 600, 300).write(np.ones((600, 300), np.float32))
    need = C.c_size_t(0)
    a, c = K.Buf(ctx, np.ones((500, 300), np.float32)), K.Buf(ctx, nbytes=500 * 600 * 4)
    L = N.lib()
    N.check(ctx.h, L.fa_matmul_f8_work(500, C.byref(held.w), C.byref(need)))
    assert need.value > 0
    w = K.Buf(ctx, nbytes=need.value + 16)
    for p, size in ((w.p.value, need.value - 1), (w.p.value + 8, need.value)):
        rc = L.fa_matmul_f8_dev(ctx.h, 500, 0, a.p, 300, C.byref(held.w), None, 0, c.p, 600, p, size)
        assert rc == N.FA_ERR_ARG and "work" in L.fa_last_error(ctx.h).decode()
    N.check(ctx.h, L.fa_matmul_f8_dev(ctx.h, 500, 0, a.p, 300, C.byref(held.w), None, 0, c.p, 600, w.p.value + 16, need.value))
    ctx.sync()
    np.testing.assert_array_equal(c.get((500, 600), np.float32), 300)
    for b in (a, c, w, held):
        b.free()


# ---- K in parts --------------------------------------------------------------------------------


@pytest.mark.parametrize("cdt", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(17, 1, 2048), (20, 200, 2088), (32, 129, 4096), (33, 70, 5000), (64, 65, 2176),
                                   (130, 300, 3333), (1, 3000, 8192), (16, 1100, 16000), (200, 64, 9000)])
def test_long_rows(ctx, m, n, k, cdt):
    """Few tiles and long rows: parts of K that several workgroups sum, an uneven last part among them."""
    case(ctx, m, n, k, "bf16", cdt, work=k % 2 == 0, epi=("bias", 2, "mul", "residual"), pad=3)


def test_long_rows_give_the_same_bits(ctx):
    """Whichever workgroup joins the parts; and on work that held another call's counts."""
    r = G.rng(91)
    held = [Held(ctx, n, k).write(r.standard_normal((n, k)).astype(np.float32)) for n, k in ((300, 8192), (100, 5000))]
    a = [r.standard_normal((m, h.k)).astype(np.float32) for m, h in zip((40, 20), held)]
    first = [product(ctx, h, x, "f32") for h, x in zip(held, a)]
    for i in range(12):
        for h, x, want in zip(held, a, first):
            np.testing.assert_array_equal(product(ctx, h, x, "f32", work=i % 3 == 0), want)
    for h in held:
        h.free()


@pytest.mark.parametrize("cdt", ["f32", "bf16"])
@pytest.mark.parametrize("m,n,k", [(1700, 2000, 700), (100, 26000, 130), (1000, 4100, 1153), (300, 32768, 260)])
def test_tiles_about_as_many_as_cus(ctx, m, n, k, cdt):
    case(ctx, m, n, k, "bf16", cdt, epi=("residual",))


@pytest.mark.parametrize("cdt", ["f32", "bf16"])
@pytest.mark.parametrize("m", [3, 20, 70])
def test_very_long_rows(ctx, m, cdt):
    case(ctx, m, 3, 200001, "f32", cdt, work=True)
