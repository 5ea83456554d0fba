"""The 8-bit key/value cache on the GPU against its 64-bit definition
(kv_oracle.py): codes and scales to the bit, attention within bounds derived
there, the cases that its documentation states, and a run of the operators
together. Every device buffer of a cache starts as NaN codes and scales, so a
byte that should not be read shows.

bf16 tolerances: weights are rounded once (2^-8 of their value) and so are the
outputs."""
import ctypes as C

import numpy as np
import pytest

import kv_lib as K
import kv_oracle as O
from ai_amd import _native as N
from ai_amd import synth as S
from ai_amd import tensor as T
from ai_amd.kvcache import KVCache

pytestmark = pytest.mark.gpu

BF = 2.0 ** -8  # half a step of bf16, relative


@pytest.fixture(params=[0, 20000], ids=["tables as long as needed", "longer tables"])
def spare(request, monkeypatch):
    """Attention is divided by what the tables have room for: with long ones many rows take the kernel for them."""
    monkeypatch.setattr(K, "SPARE", request.param)


def rng(seed):
    return np.random.default_rng(seed)


def make(r, shape, dtype, size=1.0):
    x = (size * r.standard_normal(shape)).astype(np.float32)
    return S.f32_to_bf16(x) if dtype == "bf16" else x


def close(got, want, tol, what=""):
    """Elementwise: got within tol of want; bf16 outputs rounded once, their weights too."""
    g = K.wide(got).astype(np.float64)
    assert g.shape == want.shape
    lim = tol + np.abs(want) * (BF if got.dtype == np.uint16 else O.U) + 1e-37
    d = np.abs(g - want)
    worst = float((d / lim).max()) if d.size else 0.0
    print(f"{what}: max |d| {d.max() if d.size else 0:.3g}, {worst:.3g} of the bound", flush=True)
    assert np.isfinite(g).all() and (d <= lim).all(), (what, np.argwhere(~(d <= lim))[:4], worst)


def fill(ctx, r, lengths, Hkv, D, dtype="f32", extra=2, width=None):
    """A cache that holds sequences of these lengths, and its reference."""
    blocks, tables = K.tables_for(r, lengths, extra, width)
    cache = K.Cache(ctx, blocks, Hkv, D)
    ref = O.RefCache(blocks, Hkv, D)
    rows = sum(lengths)
    k, v = make(r, (rows, Hkv, D), dtype), make(r, (rows, Hkv, D), dtype, 2.0)
    if rows:
        b = K.Batch(ctx, tables, lengths, K.cu_of(lengths))
        K.write(cache, b, k, v)
        ref.write(tables, lengths, K.cu_of(lengths), K.wide(k), K.wide(v))
        b.free()
    return cache, ref, tables


def attention_case(ctx, seed, dtype, D, H, Hkv, lengths, ns, causal=True, window=0, work=False, width=None, scale=None):
    r = rng(seed)
    cache, ref, tables = fill(ctx, r, lengths, Hkv, D, dtype, width=width)
    scale = 1 / np.sqrt(D) if scale is None else scale
    cu = K.cu_of(ns)
    q = make(r, (int(cu[-1]), H, D), dtype)
    b = K.Batch(ctx, tables, lengths, cu)
    got = K.attend(cache, b, q, causal, window, scale, work)
    scale32 = float(np.float32(scale))
    for i, (length, n) in enumerate(zip(lengths, ns)):
        k, v = ref.tokens(tables[i], length)
        rows = slice(cu[i], cu[i + 1])
        want, tol = O.attention(K.wide(q[rows]), k, v, O.sees(length, n, causal, window), scale32)
        if dtype == "bf16":
            absv = O.attention(K.wide(q[rows]), k, np.abs(v), O.sees(length, n, causal, window), scale32)[0]
            tol = tol + BF * absv
        close(got[rows], want, tol, f"{dtype} D={D} H={H}/{Hkv} len={length} n={n} causal={causal} window={window}")
    b.free()
    cache.free()


# ---- writing and reading back ------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [1, 40, 64, 66, 128, 200, 256, 320, 512])
def test_write_and_read_are_exact(ctx, D, dtype):
    """Whole prompts, then tokens that continue blocks with growing and shrinking magnitudes: codes, scales and what is
    read back equal the definition; blocks that are not written keep every byte."""
    r = rng(D * 7 + len(dtype))
    Hkv = 3
    steps = [(5, 64, 1, 130, 0), (1, 1, 63, 2, 1), (60, 70, 0, 1, 200), (1, 1, 1, 1, 1)]
    final = [sum(s[i] for s in steps) for i in range(5)]
    blocks, tables = K.tables_for(r, final)
    cache, ref = K.Cache(ctx, blocks, Hkv, D), O.RefCache(blocks, Hkv, D)
    lengths = [0] * 5
    for step, ns in enumerate(steps):
        lengths = [a + n for a, n in zip(lengths, ns)]
        cu = K.cu_of(ns)
        rows = int(cu[-1])
        size = np.exp(r.uniform(-3, 3) * r.standard_normal((rows, Hkv, 1)))
        k, v = (make(r, (rows, Hkv, D), "f32") * size.astype(np.float32) for _ in range(2))
        if dtype == "bf16":
            k, v = S.f32_to_bf16(k), S.f32_to_bf16(v)
        b = K.Batch(ctx, tables, lengths, cu)
        K.write(cache, b, k, v)
        ref.write(tables, lengths, cu, K.wide(k), K.wide(v))
        b.free()
        codes, scales = cache.state()
        got = O.DECODE[K.split_codes(codes, D)]
        used = {int(t) for i in range(5) for t in tables[i, :-(-lengths[i] // 64)]}
        for i in range(blocks):
            if i not in used:
                assert (codes[i] == 0x7F).all() and (scales[i] == 0xFFFFFFFF).all(), f"block {i} was written"
        for i in range(5):
            for p in range(-(-lengths[i] // 64)):
                blk, m = tables[i, p], min(64, lengths[i] - p * 64)
                np.testing.assert_array_equal(got[blk][:, :, :m], ref.val[blk][:, :, :m])
                np.testing.assert_array_equal(scales[blk].view(np.float32), 2.0 ** ref.exp[blk])
    b = K.Batch(ctx, tables, lengths, K.cu_of(lengths))
    for kind in (np.float32, np.uint16):
        k, v = K.read(cache, b, kind)
        for i in range(5):
            rows = slice(b.cu[i], b.cu[i + 1])
            for x, want in zip((k, v), ref.tokens(tables[i], lengths[i])):
                np.testing.assert_array_equal(K.wide(x[rows]).astype(np.float64), want)
    b.free()
    cache.free()


def test_write_many_rows_and_few_use_the_same_places(ctx):
    """One sequence with many rows (units by block) and many with one (units by row)."""
    r = rng(5)
    for lengths, ns in (([4000], [3900]), ([100 + i for i in range(90)], [1] * 90), ([700, 3, 0, 900], [650, 2, 0, 3])):
        cache, ref, tables = fill(ctx, r, [l - n for l, n in zip(lengths, ns)], 2, 64,
                                  width=-(-max(lengths) // 64))
        used = sorted(set(range(cache.blocks + sum(lengths) // 64 + 2 * len(lengths))))
        cache.free()
        blocks, tables = K.tables_for(r, lengths)
        cache, ref = K.Cache(ctx, blocks, 2, 64), O.RefCache(blocks, 2, 64)
        for stop in ([l - n for l, n in zip(lengths, ns)], lengths):
            n = stop if stop is not lengths else ns
            cu = K.cu_of(n)
            k, v = make(r, (int(cu[-1]), 2, 64), "f32"), make(r, (int(cu[-1]), 2, 64), "f32", 3.0)
            b = K.Batch(ctx, tables, stop, cu)
            if cu[-1]:
                K.write(cache, b, k, v)
                ref.write(tables, stop, cu, k, v)
            b.free()
        b = K.Batch(ctx, tables, lengths, K.cu_of(lengths))
        k, v = K.read(cache, b)
        for i in range(len(lengths)):
            for x, want in zip((k, v), ref.tokens(tables[i], lengths[i])):
                np.testing.assert_array_equal(x[b.cu[i]:b.cu[i + 1]], want)
        b.free()
        cache.free()
        assert used


def test_write_strides_and_rows_behind(ctx):
    """Keys and values as views of a q|k|v product and of a [heads, rows, dims] array; rows behind the last sequence are
    neither read (NaN there) nor written back."""
    r = rng(11)
    Hkv, D, rows = 2, 80, 50
    lengths, cu = [30, 17], [0, 30, 47]
    blocks, tables = K.tables_for(r, lengths)
    qkv = make(r, (rows, 5 * D + 3), "f32")
    qkv[47:] = np.nan
    k = np.lib.stride_tricks.as_strided(qkv[:, D:], (rows, Hkv, D), (qkv.strides[0], D * 4, 4))
    heads_first = make(r, (Hkv, rows, D), "f32")
    v = heads_first.transpose(1, 0, 2)
    cache, ref = K.Cache(ctx, blocks, Hkv, D), O.RefCache(blocks, Hkv, D)
    b = K.Batch(ctx, tables, lengths, cu, rows=rows)
    K.write(cache, b, k, v)
    ref.write(tables, lengths, cu, k, v)
    gk, gv = K.read(cache, b)
    for i in range(2):
        wk, wv = ref.tokens(tables[i], lengths[i])
        np.testing.assert_array_equal(gk[cu[i]:cu[i + 1]], wk)
        np.testing.assert_array_equal(gv[cu[i]:cu[i + 1]], wv)
    assert (gk[47:].view(np.uint32) == 0x5A5A5A5A).all() and (gv[47:].view(np.uint32) == 0x5A5A5A5A).all()
    q = np.lib.stride_tricks.as_strided(qkv, (rows, 2, D), (qkv.strides[0], D * 4, 4))
    out = K.attend(cache, b, q, scale=0.1)
    assert (out[47:].view(np.uint32) == 0x5A5A5A5A).all() and np.isfinite(out[:47]).all()
    b.free()
    cache.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_strides_of_many_rows(ctx, spare, dtype):
    """Queries as a view of a q|k|v product with rows of any alignment; rows behind the last sequence stay as they are."""
    r = rng(13)
    for D, pad in ((80, 3), (128, 8)):
        H, Hkv, rows = 4, 2, 330
        lengths, cu = [200, 128], [0, 200, 320]
        cache, ref, tables = fill(ctx, r, lengths, Hkv, D, dtype)
        qkv = make(r, (rows, 6 * D + pad), dtype)
        q = np.lib.stride_tricks.as_strided(qkv[:, D:], (rows, H, D), (qkv.strides[0], D * qkv.itemsize, qkv.itemsize))
        b = K.Batch(ctx, tables, lengths, cu, rows=rows)
        got = K.attend(cache, b, q, scale=0.1)
        assert (got[320:].view(np.uint8) == 0x5A).all()
        for i in range(2):
            at = slice(cu[i], cu[i + 1])
            qi, mask = K.wide(np.ascontiguousarray(q[at])), O.sees(lengths[i], cu[i + 1] - cu[i], True, 0)
            wk, wv = ref.tokens(tables[i], lengths[i])
            scale = float(np.float32(0.1))
            want, tol = O.attention(qi, wk, wv, mask, scale)
            if dtype == "bf16":
                tol = tol + BF * O.attention(qi, wk, np.abs(wv), mask, scale)[0]
            close(got[at], want, tol, f"strided, {D} dims, sequence {i}")
        b.free()
        cache.free()


def test_write_special_values(ctx):
    """Zeros, the smallest and largest magnitudes, ties between codes, and values that are not finite."""
    D, Hkv = 64, 1
    big = np.float32(3.4028235e38)
    rows = [np.zeros(D), np.full(D, 1e-45), np.full(D, 3e-25), np.full(D, big), np.linspace(-448, 448, D),
            np.full(D, 449.0), np.where(np.arange(D) % 7 == 0, np.inf, 1.0), np.where(np.arange(D) == 3, np.nan, -2.0),
            2.0 ** (np.arange(D) - 40.0), (17 + np.arange(D)) / 16.0, -np.zeros(D)]
    x = np.array(rows, np.float32)[:, None, :]
    n = len(rows)
    lengths = [64 * n]
    tables = np.arange(n, dtype=np.int32)[None]
    # one token to a block, so that each has a scale of its own
    cache, ref = K.Cache(ctx, n, Hkv, D), O.RefCache(n, Hkv, D)
    for i in range(n):
        b = K.Batch(ctx, tables, [64 * i + 1], [0, 1])
        K.write(cache, b, x[i:i + 1], x[i:i + 1])
        ref.write(tables, [64 * i + 1], [0, 1], x[i:i + 1], x[i:i + 1])
        k, v = K.read(cache, b)
        want = ref.tokens(tables[0], 64 * i + 1)[0][-1:]
        np.testing.assert_array_equal(k.astype(np.float64), want)
        np.testing.assert_array_equal(v.astype(np.float64), want)
        b.free()
    cache.free()
    assert lengths


def test_write_drops_what_followed_and_reuses_blocks(ctx):
    """Writing at an earlier position ends the sequence there; a block handed out again starts a new scale at its first
    place."""
    r = rng(3)
    cache, ref = K.Cache(ctx, 2, 1, 64), O.RefCache(2, 1, 64)
    tables = np.array([[1, 0]], np.int32)
    for length, n, size in ((100, 100, 1000.0), (71, 7, 1.0), (40, 40, 0.01), (64, 24, 5.0), (65, 1, 1e-3)):
        k, v = make(r, (n, 1, 64), "f32", size), make(r, (n, 1, 64), "f32", size)
        b = K.Batch(ctx, tables, [length], [0, n])
        K.write(cache, b, k, v)
        ref.write(tables, [length], [0, n], k, v)
        b.free()
        b = K.Batch(ctx, tables, [length], [0, length])
        got = K.read(cache, b)
        for x, want in zip(got, ref.tokens(tables[0], length)):
            np.testing.assert_array_equal(x, want)
        b.free()
    cache.free()


# ---- attention ------------------------------------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D", [1, 40, 64, 96, 128, 192, 200, 256, 320, 512])
def test_attention_head_dims(ctx, D, dtype):
    """Single tokens and a few, at each head dim, over one token to several blocks."""
    attention_case(ctx, D + 1, dtype, D, 6, 2, [1, 2, 63, 64, 65, 200, 321], [1, 2, 1, 3, 1, 5, 1])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("H,Hkv", [(1, 1), (3, 1), (8, 8), (16, 1), (40, 2), (32, 8)])
def test_attention_head_layouts(ctx, H, Hkv, dtype):
    attention_case(ctx, H * 100 + Hkv, dtype, 64, H, Hkv, [70, 1, 300], [1, 1, 20])


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("causal,window", [(True, 0), (False, 0), (True, 1), (True, 64), (True, 100), (False, 1),
                                           (False, 37), (False, 1000), (True, 2 ** 31 - 1), (False, 2 ** 31 - 1)])
def test_attention_masks(ctx, spare, causal, window, dtype):
    """Chunks and whole prompts under each mask, windows shorter and longer than a block and than the sequence."""
    attention_case(ctx, 17 + window % 97, dtype, 128, 4, 2, [150, 64, 400, 10], [150, 7, 90, 1], causal, window)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,H,Hkv,lengths,ns", [
    (128, 4, 1, [3000], [1]), (64, 2, 2, [5000, 1, 700], [1, 1, 1]), (256, 3, 1, [2100, 33], [4, 33]),
    (512, 2, 2, [900], [2]), (128, 8, 2, [1500, 1400], [40, 1]), (40, 5, 1, [9000], [3]),
    (128, 2, 1, [300 + 17 * i for i in range(20)], [1 + i % 3 for i in range(20)])])
def test_attention_split_token_axis(ctx, D, H, Hkv, lengths, ns, dtype):
    """Few rows on many blocks: the blocks are cut into parts and joined, with the caller's scratch or the context's."""
    attention_case(ctx, D + len(lengths), dtype, D, H, Hkv, lengths, ns, work=dtype == "f32")
    attention_case(ctx, D + len(lengths) + 1, dtype, D, H, Hkv, lengths, ns, causal=False, window=777,
                   work=dtype == "bf16", width=400)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,H,Hkv,lengths,ns", [
    (128, 8, 2, [640, 200, 333], [640, 200, 333]), (64, 4, 4, [300] * 3, [257, 300, 128]),
    (256, 3, 1, [500, 129], [400, 129]), (192, 2, 1, [260], [260]), (96, 6, 2, [700], [130]),
    (320, 2, 1, [200], [200])])
def test_attention_prompts(ctx, spare, D, H, Hkv, lengths, ns, dtype):
    attention_case(ctx, D + H, dtype, D, H, Hkv, lengths, ns)
    attention_case(ctx, D + H + 1, dtype, D, H, Hkv, lengths, ns, window=90)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,H,Hkv,lengths,ns", [(128, 8, 2, [5000], [40]), (64, 2, 1, [2000, 9000], [100, 130]),
                                                (256, 3, 1, [1500], [70]), (192, 1, 1, [3000], [129])])
def test_attention_few_tiles_of_many_rows_split(ctx, spare, D, H, Hkv, lengths, ns, dtype):
    """Chunks on long contexts: few tiles of 128 rows, whose blocks are cut into parts and joined."""
    attention_case(ctx, D + H, dtype, D, H, Hkv, lengths, ns, work=dtype == "f32")
    attention_case(ctx, D + H + 1, dtype, D, H, Hkv, lengths, ns, causal=False, window=1100, work=dtype == "bf16")


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_attention_many_sequences(ctx, dtype):
    """More sequences than a wave has lanes, some empty, some without rows; split and not."""
    r = rng(77)
    lengths = [int(x) for x in r.integers(0, 700, 130)]
    lengths[5] = lengths[64] = 0
    ns = [min(l, int(r.integers(0, 4))) for l in lengths]
    attention_case(ctx, 78, dtype, 64, 2, 1, lengths, ns, width=11)
    attention_case(ctx, 79, dtype, 64, 16, 16, lengths, [min(l, 1) for l in lengths])


def test_thousands_of_sequences(ctx):
    """Sequence starts found in two rounds and more, one row each: written, read back, attended to."""
    r = rng(80)
    B, D = 4500, 64
    lengths = [int(x) for x in r.integers(1, 4, B)]
    blocks = B
    tables = r.permutation(blocks).astype(np.int32)[:, None]
    cache, ref = K.Cache(ctx, blocks, 1, D), O.RefCache(blocks, 1, D)
    for step in range(1, 4):
        now = [min(l, step) for l in lengths]
        ns = [int(l >= step) for l in lengths]
        cu = K.cu_of(ns)
        k, v = make(r, (int(cu[-1]), 1, D), "f32"), make(r, (int(cu[-1]), 1, D), "f32")
        b = K.Batch(ctx, tables, now, cu)
        K.write(cache, b, k, v)
        ref.write(tables, now, cu, k, v)
        b.free()
    b = K.Batch(ctx, tables, lengths, K.cu_of(lengths))
    gk, gv = K.read(cache, b)
    q = make(r, (int(b.cu[-1]), 2, D), "f32")
    out = K.attend(cache, b, q, scale=0.125)
    for i in range(B):
        wk, wv = ref.tokens(tables[i], lengths[i])
        rows = slice(b.cu[i], b.cu[i + 1])
        np.testing.assert_array_equal(gk[rows], wk)
        np.testing.assert_array_equal(gv[rows], wv)
        if i % 50 == 0:
            want, tol = O.attention(q[rows], wk, wv, O.sees(lengths[i], lengths[i], True, 0), 0.125)
            close(out[rows], want, tol, f"sequence {i}")
    b.free()
    cache.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [2, 150])
def test_attention_scores_that_rise_and_fall(ctx, spare, dtype, n):
    """Scores that rise by thousands of times their weights' range from block to block, and fall again: the reference
    of the weights follows, in both kernels, split and not."""
    r = rng(90 + n)
    for length, H in ((700, 4), (300, 1)):
        D = 64
        blocks, tables = K.tables_for(r, [length])
        cache, ref = K.Cache(ctx, blocks, 1, D), O.RefCache(blocks, 1, D)
        k = make(r, (length, 1, D), "f32", 0.1)
        k[:, 0, 0] = np.concatenate([np.linspace(0, 60, length // 2), np.linspace(60, -20, length - length // 2)])
        v = make(r, (length, 1, D), "f32")
        q = make(r, (n, H, D), "f32", 0.1)
        q[:, :, 0] = 1.0
        if dtype == "bf16":
            k, v, q = (S.f32_to_bf16(x) for x in (k, v, q))
        b = K.Batch(ctx, tables, [length], [0, length])
        K.write(cache, b, k, v)
        b.free()
        ref.write(tables, [length], [0, length], K.wide(k), K.wide(v))
        b = K.Batch(ctx, tables, [length], [0, n])
        wk, wv = ref.tokens(tables[0], length)
        for scale in (1.0, -1.0):
            got = K.attend(cache, b, q, scale=scale)
            mask = O.sees(length, n, True, 0)
            want, tol = O.attention(K.wide(q), wk, wv, mask, scale)
            if dtype == "bf16":
                tol = tol + BF * O.attention(K.wide(q), wk, np.abs(wv), mask, scale)[0]
            close(got, want, tol, f"rising scores, {n} rows, scale {scale}")
        b.free()
        cache.free()


def test_attention_score_range(ctx, spare):
    """Scores of hundreds either way, scale 0, a negative scale."""
    for scale in (3.0, 0.0, -0.7):
        attention_case(ctx, 23, "f32", 64, 4, 2, [200, 90], [3, 90], scale=scale)


def test_attention_value_scales_far_apart(ctx, spare):
    """Blocks whose values are 2^60 apart, large and tiny ones: weights meet each block's own scale."""
    r = rng(31)
    lengths, D = [64 * 5], 64
    blocks, tables = K.tables_for(r, lengths)
    cache, ref = K.Cache(ctx, blocks, 1, D), O.RefCache(blocks, 1, D)
    k, v = make(r, (320, 1, D), "f32"), make(r, (320, 1, D), "f32")
    for i, e in enumerate((0, 30, -30, 110, -70)):
        v[i * 64:(i + 1) * 64] *= np.float32(2.0 ** e)
    b = K.Batch(ctx, tables, lengths, [0, 320])
    K.write(cache, b, k, v)
    ref.write(tables, lengths, [0, 320], k, v)
    q = make(r, (320, 2, D), "f32")
    got = K.attend(cache, b, q, True, 64, 0.125)
    wk, wv = ref.tokens(tables[0], 320)
    want, tol = O.attention(q, wk, wv, O.sees(320, 320, True, 64), 0.125)
    close(got, want, tol, "value scales")
    b.free()
    cache.free()


def test_attention_value_scales_far_apart_few_rows(ctx):
    """The same with three rows on a split axis."""
    r = rng(32)
    lengths, D = [64 * 20], 128
    blocks, tables = K.tables_for(r, lengths)
    cache, ref = K.Cache(ctx, blocks, 1, D), O.RefCache(blocks, 1, D)
    k, v = make(r, (1280, 1, D), "f32"), make(r, (1280, 1, D), "f32")
    for i in range(20):
        v[i * 64:(i + 1) * 64] *= np.float32(2.0 ** (-3 * i))
    b = K.Batch(ctx, tables, lengths, [0, 1280])
    K.write(cache, b, k, v)
    b.free()
    ref.write(tables, lengths, [0, 1280], k, v)
    q = make(r, (3, 1, D), "f32")
    wk, wv = ref.tokens(tables[0], 1280)
    b = K.Batch(ctx, tables, lengths, [0, 3])
    for window in (0, 70):
        got = K.attend(cache, b, q, True, window, 0.125)
        want, tol = O.attention(q, wk, wv, O.sees(1280, 3, True, window), 0.125)
        close(got, want, tol, f"value scales, window {window}")
    b.free()
    cache.free()


def test_attention_empty_rows_and_lengths(ctx, spare):
    """A sequence of no tokens, one without rows, more rows than tokens: rows that see nothing are zeros."""
    r = rng(2)
    for dtype in ("f32", "bf16"):
        cache, ref, tables = fill(ctx, r, [5, 0, 70], 1, 64, dtype)
        b = K.Batch(ctx, tables, [5, 0, 70], [0, 9, 12, 12])
        q = make(r, (12, 3, 64), dtype)
        out = K.wide(K.attend(cache, b, q, scale=0.125))
        assert (out[:4] == 0).all() and (out[9:] == 0).all()
        k, v = ref.tokens(tables[0], 5)
        want, tol = O.attention(K.wide(q[4:9]), k, v, O.sees(5, 5, True, 0), 0.125)
        np.testing.assert_array_less(np.abs(out[4:9] - want), tol + (2 * BF if dtype == "bf16" else 1e-6) *
                                     (np.abs(v).max() + 1e-9))
        # keys before the first position, not causal: all five tokens
        out = K.wide(K.attend(cache, b, q, causal=False, scale=0.125))
        assert (out[9:] == 0).all() and np.isfinite(out[:9]).all() and (out[:9] != 0).all()
        b.free()
        cache.free()


def test_attention_nan_stays_where_it_is_seen(ctx, spare):
    """A NaN value or key that some rows of a tile see and others do not reaches those that do, in its dims (values) or
    whole (keys); NaN codes behind a length reach nobody (every cache here begins with them)."""
    r = rng(8)
    for dtype in ("f32", "bf16"):
        for D in (64, 256):
            n = 200
            blocks, tables = K.tables_for(r, [n])
            cache = K.Cache(ctx, blocks, 1, D)
            k, v = make(r, (n, 1, D), "f32"), make(r, (n, 1, D), "f32")
            v[100, 0, 5] = np.nan
            v[150, 0, 33] = np.inf
            k[180, 0, 1] = -np.inf
            if dtype == "bf16":
                k, v = S.f32_to_bf16(k), S.f32_to_bf16(v)
                k[180, 0, 1] = 0xFF80
            b = K.Batch(ctx, tables, [n], [0, n])
            K.write(cache, b, k, v)
            q = make(r, (n, 3, D), dtype)
            out = K.wide(K.attend(cache, b, q, scale=0.05))
            bad = np.isnan(out)
            want = np.zeros_like(bad)
            want[100:, :, 5] = True
            want[150:, :, 33] = True
            want[180:] = True
            np.testing.assert_array_equal(bad, want)
            out = K.wide(K.attend(cache, b, q, scale=0.05, window=20))
            want[:] = False
            want[100:120, :, 5] = True
            want[150:170, :, 33] = True
            want[180:200] = True
            np.testing.assert_array_equal(np.isnan(out), want)
            b.free()
            cache.free()


def test_attention_nan_among_drafted_tokens(ctx):
    """The same with a tile of few rows: NaN at the positions of the last tokens, seen by those after them."""
    r = rng(18)
    for dtype in ("f32", "bf16"):
        for D, length in ((64, 70), (256, 2000), (512, 131)):
            blocks, tables = K.tables_for(r, [length])
            cache = K.Cache(ctx, blocks, 1, D)
            k, v = make(r, (length, 1, D), "f32"), make(r, (length, 1, D), "f32")
            v[length - 4, 0, 5] = np.nan
            v[length - 2, 0, 40] = -np.inf
            k[length - 1, 0, 1] = np.nan
            if dtype == "bf16":
                k, v = S.f32_to_bf16(k), S.f32_to_bf16(v)
                k[length - 1, 0, 1] = 0x7FC0
            b = K.Batch(ctx, tables, [length], [0, length])
            K.write(cache, b, k, v)
            b.free()
            b = K.Batch(ctx, tables, [length], [0, 5])
            q = make(r, (5, 3, D), dtype)
            out = K.wide(K.attend(cache, b, q, scale=0.05))
            want = np.zeros(out.shape, bool)
            want[1:, :, 5] = True
            want[3:, :, 40] = True
            want[4] = True
            np.testing.assert_array_equal(np.isnan(out), want)
            b.free()
            cache.free()


def test_attention_nan_query_stays_in_its_row(ctx, spare):
    r = rng(9)
    cache, ref, tables = fill(ctx, r, [90], 2, 64)
    b = K.Batch(ctx, tables, [90], [0, 90])
    q = make(r, (90, 4, 64), "f32")
    clean = K.attend(cache, b, q, scale=0.125)
    q[50, 2, 7] = np.nan
    q[51, 0, 0] = np.inf
    out = K.attend(cache, b, q, scale=0.125)
    assert np.isnan(out[50, 2]).all() and np.isnan(out[51, 0]).all()
    keep = np.ones(out.shape[:2], bool)
    keep[50, 2] = keep[51, 0] = False
    np.testing.assert_array_equal(out[keep], clean[keep])
    b.free()
    cache.free()


def test_bad_tables_give_nan_and_touch_nothing(ctx, spare):
    """Entries outside the pool and lengths past the table row: NaN for those that see them, and no write."""
    r = rng(4)
    for dtype in ("f32", "bf16"):
        cache, ref, tables = fill(ctx, r, [200, 100, 65], 2, 64, dtype)
        before = [x.copy() for x in cache.state()]
        t = tables.copy()
        t[0, 1] = cache.blocks
        t[1, 0] = -1
        cu = [0, 200, 300, 301]
        b = K.Batch(ctx, t, [200, 100, 64 * t.shape[1] + 1], cu)
        k, v = K.read(cache, b)
        for x in (k, v):
            nan = np.isnan(x).all((1, 2))
            assert nan[64:128].all() and nan[200:264].all() and nan[300]
            assert np.isfinite(x[:64]).all() and np.isfinite(x[128:200]).all() and np.isfinite(x[264:300]).all()
        q = make(r, (301, 4, 64), dtype)
        out = K.wide(K.attend(cache, b, q, scale=0.125))
        assert np.isfinite(out[:64]).all() and np.isnan(out[64:300]).all() and np.isnan(out[300]).all()
        # single tokens over a split axis see it too
        b2 = K.Batch(ctx, np.concatenate([t, np.full((3, 60), -5, np.int32)], 1), [200, 100, 65], [0, 1, 2, 3])
        out = K.wide(K.attend(cache, b2, q[:3], scale=0.125))
        assert np.isnan(out[:2]).all() and np.isfinite(out[2]).all()
        x = make(r, (301, 2, 64), dtype)
        t[:] = -1
        b3 = K.Batch(ctx, t, [200, 100, 64 * t.shape[1] + 1], cu)
        K.write(cache, b3, x, x)
        for x0, x1 in zip(before, cache.state()):
            np.testing.assert_array_equal(x0, x1)
        for x in (b, b2, b3):
            x.free()
        cache.free()


def test_row_starts_out_of_order_stay_in_bounds(ctx, spare):
    """Device arrays are not checked on the host: whatever row starts they hold, nothing outside the call's rows is
    written."""
    r = rng(6)
    cache, ref, tables = fill(ctx, r, [300, 300, 300], 1, 64)
    before = [x.copy() for x in cache.state()]
    for cu in ([0, 500, 20, 10 ** 9], [-7, -9, -2 ** 31, 4], [100, 50, 2, 1], [2 ** 31 - 1] * 4):
        for rows in (40, 500):
            b = K.Batch(ctx, tables, [300, -5, 300], cu, rows=rows)
            q = make(r, (rows, 2, 64), "f32")
            out = K.attend(cache, b, q, scale=0.125)
            assert out.shape == (rows, 2, 64)
            K.read(cache, b)
            b.free()
    for x0, x1 in zip(before, cache.state()):
        np.testing.assert_array_equal(x0, x1)
    cache.free()


def test_offsets_past_32_bits(ctx):
    """A pool of more than 4 GiB, the sequence in its last blocks."""
    Hkv, D = 8, 512
    blocks = (5 << 30) // (Hkv * 2 * 64 * D) + 1
    c = K.Cache.__new__(K.Cache)
    c.ctx, c.blocks, c.Hkv, c.D, c.Dp = ctx, blocks, Hkv, D, D
    c.codes = K.Buf(ctx, nbytes=N.lib().fa_kv_codes_bytes(blocks, Hkv, D))
    c.scales = K.Buf(ctx, nbytes=blocks * Hkv * 8)
    assert c.codes.nbytes > 5 << 30
    c.c = N.KvCache(c.codes.p, c.scales.p, blocks, Hkv, D)
    r = rng(10)
    tables = np.array([[blocks - 1, 0, blocks - 2]], np.int32)
    k, v = make(r, (150, Hkv, D), "f32"), make(r, (150, Hkv, D), "f32")
    b = K.Batch(ctx, tables, [150], [0, 150])
    K.write(c, b, k, v)
    ref = O.RefCache(3, Hkv, D)
    rt = [[0, 1, 2]]
    ref.write(rt, [150], [0, 150], k, v)
    wk, wv = ref.tokens(rt[0], 150)
    gk, gv = K.read(c, b)
    np.testing.assert_array_equal(gk, wk)
    np.testing.assert_array_equal(gv, wv)
    q = make(r, (150, Hkv, D), "f32")
    got = K.attend(c, b, q, scale=0.05)
    want, tol = O.attention(q[-1:], wk, wv, O.sees(150, 1, True, 0), float(np.float32(0.05)))
    close(got[-1:], want, tol, "pool of 5 GiB")
    b.free()
    c.free()


def test_same_results_every_time(ctx, spare):
    """No order that changes: equal bits from call to call, split axis included."""
    r = rng(12)
    cache, ref, tables = fill(ctx, r, [4000, 100, 1700], 2, 128)
    for ns in ([1, 1, 1], [300, 100, 200]):
        b = K.Batch(ctx, tables, [4000, 100, 1700], K.cu_of(ns))
        q = make(r, (sum(ns), 8, 128), "f32")
        first = K.attend(cache, b, q, scale=0.09)
        for _ in range(5):
            np.testing.assert_array_equal(K.attend(cache, b, q, scale=0.09, work=True).view(np.uint32),
                                          first.view(np.uint32))
        b.free()
    cache.free()


# ---- host entry points and refusals that need a context ------------------------------------

def test_host_entry_points_equal_the_device_ones(ctx):
    r = rng(21)
    lengths, ns, Hkv, H, D = [130, 40, 64], [30, 40, 1], 2, 4, 96
    for dtype in ("f32", "bf16"):
        cache, ref, tables = fill(ctx, r, [100, 0, 63], Hkv, D, dtype, extra=6, width=3)
        free = [i for i in range(cache.blocks) if i not in tables[tables < cache.blocks]]
        for i, l in enumerate(lengths):
            for p in range(-(-l // 64)):
                if tables[i, p] >= cache.blocks:
                    tables[i, p] = free.pop()
        cu = K.cu_of(ns)
        # two rows more than the sequences have
        rows = int(cu[-1]) + 2
        k, v, q = (make(r, (rows, h, D), dtype) for h in (Hkv, Hkv, H))
        b = K.Batch(ctx, tables, lengths, cu, rows=rows)
        hb = b.host()
        L = N.lib()
        N.check(ctx.h, L.fa_kv_write(ctx.h, C.byref(cache.c), C.byref(hb), K.dt(k), k.ctypes.data, *K.st(k),
                                     v.ctypes.data, *K.st(v)))
        host_state = [x.copy() for x in cache.state()]
        K.write(cache, b, k, v)  # the same tokens again: nothing changes
        for x0, x1 in zip(host_state, cache.state()):
            np.testing.assert_array_equal(x0, x1)
        bk, bv = np.zeros((rows, Hkv, D), k.dtype), np.zeros((rows, Hkv, D), k.dtype)
        N.check(ctx.h, L.fa_kv_read(ctx.h, C.byref(cache.c), C.byref(hb), K.dt(k), bk.ctypes.data, bv.ctypes.data))
        dk, dv = K.read(cache, b, k.dtype)
        np.testing.assert_array_equal(bk[:-2], dk[:-2])
        np.testing.assert_array_equal(bv[:-2], dv[:-2])
        assert (bk[-2:] == 0).all() and (bv[-2:] == 0).all()
        out = np.zeros((rows, H, D), k.dtype)
        N.check(ctx.h, L.fa_kv_attention(ctx.h, C.byref(cache.c), C.byref(hb), K.dt(q), q.ctypes.data, *K.st(q), H, 1, 50,
                                         0.2, out.ctypes.data))
        dev = K.attend(cache, b, q, True, 50, 0.2)
        np.testing.assert_array_equal(out[:-2], dev[:-2])
        assert (out[-2:] == 0).all()
        b.free()
        cache.free()


def test_work_is_checked(ctx):
    cache = K.Cache(ctx, 50, 1, 64)
    b = K.Batch(ctx, np.arange(50)[None], [3000], [0, 1])
    need = C.c_size_t(0)
    N.check(ctx.h, N.lib().fa_kv_attention_work(C.byref(cache.c), C.byref(b.b), 1, C.byref(need)))
    assert need.value > 0
    q, w = K.Buf(ctx, nbytes=256, fill=0), K.Buf(ctx, nbytes=need.value + 16)
    for p, n in ((w.p.value, need.value - 1), (w.p.value + 4, need.value)):
        rc = N.lib().fa_kv_attention_dev(ctx.h, C.byref(cache.c), C.byref(b.b), 0, q.p, 64, 64, 1, 1, 0, 1.0, q.p, p, n)
        assert rc == N.FA_ERR_ARG and b"work" in N.lib().fa_last_error(ctx.h)
    for x in (q, w, b, cache):
        x.free()


# ---- a captured step, replayed with other contents -------------------------------------------

def test_captured_step_replays_with_new_contents(ctx):
    """Write, attend and read back captured into one graph; each replay with other tokens, lengths and tables, with
    eager work and synchronisation between, equals the eager calls."""
    hip = C.CDLL("libamdhip64.so")
    hip.hipStreamBeginCapture.argtypes = [C.c_void_p, C.c_int]
    hip.hipStreamEndCapture.argtypes = [C.c_void_p, C.POINTER(C.c_void_p)]
    hip.hipGraphInstantiate.argtypes = [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t]
    hip.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
    hip.hipGraphDestroy.argtypes = [C.c_void_p]
    hip.hipGraphExecDestroy.argtypes = [C.c_void_p]
    L = N.lib()
    r = rng(40)
    Hkv, H, D, B, width = 2, 8, 128, 3, 40
    cache, ref, tables = fill(ctx, r, [1000, 64, 300], Hkv, D, "bf16", extra=8, width=width)
    spare = [i for i in range(cache.blocks) if i not in tables[tables < cache.blocks]]
    for i in range(B):
        for p in range(width):
            if tables[i, p] >= cache.blocks and spare:
                tables[i, p] = spare.pop()
                break
    lengths = [1000, 64, 300]
    b = K.Batch(ctx, tables, [l + 1 for l in lengths], [0, 1, 2, 3])
    bufs = {n: K.Buf(ctx, nbytes=3 * h * D * 2, fill=0) for n, h in
            (("k", Hkv), ("v", Hkv), ("q", H), ("out", H), ("rk", Hkv), ("rv", Hkv))}
    need = C.c_size_t(0)
    N.check(ctx.h, L.fa_kv_attention_work(C.byref(cache.c), C.byref(b.b), H, C.byref(need)))
    work = K.Buf(ctx, nbytes=need.value)

    def step(w, nbytes):
        N.check(ctx.h, L.fa_kv_write_dev(ctx.h, C.byref(cache.c), C.byref(b.b), N.FA_DT_BF16, bufs["k"].p, Hkv * D, D,
                                         bufs["v"].p, Hkv * D, D))
        N.check(ctx.h, L.fa_kv_attention_dev(ctx.h, C.byref(cache.c), C.byref(b.b), N.FA_DT_BF16, bufs["q"].p, H * D, D,
                                             H, 1, 0, 0.09, bufs["out"].p, w, nbytes))
        N.check(ctx.h, L.fa_kv_read_dev(ctx.h, C.byref(cache.c), C.byref(b.b), N.FA_DT_BF16, bufs["rk"].p, bufs["rv"].p))

    graph, ex = C.c_void_p(), C.c_void_p()
    ctx.sync()
    assert hip.hipStreamBeginCapture(ctx.stream, 2) == 0
    rc = L.fa_kv_attention_dev(ctx.h, C.byref(cache.c), C.byref(b.b), N.FA_DT_BF16, bufs["q"].p, H * D, D, H, 1, 0, 0.09,
                               bufs["out"].p, None, 0)
    msg = L.fa_last_error(ctx.h)
    hb = b.host()
    hrc = L.fa_kv_read(ctx.h, C.byref(cache.c), C.byref(hb), N.FA_DT_BF16, np.empty(4096, np.uint8).ctypes.data,
                       np.empty(4096, np.uint8).ctypes.data)
    step(work.p, need.value)
    assert hip.hipStreamEndCapture(ctx.stream, C.byref(graph)) == 0
    assert rc == N.FA_ERR_STATE and b"captured" in msg  # no work of the caller's: refused
    assert hrc == N.FA_ERR_STATE
    assert hip.hipGraphInstantiate(C.byref(ex), graph, None, None, 0) == 0
    for turn in range(4):
        data = {n: make(r, (3, h, D), "bf16") for n, h in (("k", Hkv), ("v", Hkv), ("q", H))}
        for n, x in data.items():
            bufs[n].put(x)
        now = [l + 1 for l in lengths] if turn % 2 else [900 - turn, 65, 301]
        b.bufs[1].put(np.array(now, np.int32))
        state = cache.state()
        assert hip.hipGraphLaunch(ex, ctx.stream) == 0
        ctx.sync()
        got = {n: bufs[n].get((3, h, D), np.uint16) for n, h in (("out", H), ("rk", Hkv), ("rv", Hkv))}
        after = cache.state()
        cache.codes.put(state[0])
        cache.scales.put(state[1])
        step(None, 0)
        ctx.sync()
        for n, h in (("out", H), ("rk", Hkv), ("rv", Hkv)):
            np.testing.assert_array_equal(got[n], bufs[n].get((3, h, D), np.uint16))
        for x0, x1 in zip(after, cache.state()):
            np.testing.assert_array_equal(x0, x1)
        assert np.isfinite(S.bf16_to_f32(got["out"])).all()
    hip.hipGraphExecDestroy(ex)
    hip.hipGraphDestroy(graph)
    for x in (*bufs.values(), work, b, cache):
        x.free()


@pytest.mark.parametrize("dtype,D,H,lengths,ns,window,width", [
    ("bf16", 64, 16, [2000, 1900, 2048, 70], [128, 100, 128, 70], 0, 64),  # long enough to be split
    ("bf16", 64, 16, [1000, 900, 64, 200], [128, 100, 64, 128], 0, 64),    # only the tables are
    ("bf16", 64, 16, [2500, 2400, 2048, 2000], [160] * 4, 1700, None),
    ("f32", 80, 16, [2000, 1900, 2048, 1990], [130] * 4, 0, 64),
    ("f32", 80, 9, [1900], [1900], 0, None),                               # a prompt: later tiles see more
    ("f32", 80, 8, [1900], [1900], 500, None)])
def test_tiles_of_many_rows_cut_in_parts(ctx, dtype, D, H, lengths, ns, window, width):
    """128 work items and more of 128 rows, which are cut where the longest sequence is long."""
    attention_case(ctx, 54, dtype, D, H, H, lengths, ns, window=window, width=width, work=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("D,Hkv,G,lengths,ns,causal,window", [
    (64, 16, 4, [400] * 40, [5] * 40, True, 0), (64, 16, 5, [130, 0, 64, 65, 300] * 9, [7, 0, 1, 6, 5] * 9, True, 0),
    (128, 16, 20, [200, 90, 640, 33] * 8, [1] * 32, True, 0), (128, 16, 4, [200, 90, 640, 33] * 8, [8, 7, 6, 5] * 8, False, 60),
    (72, 8, 33, [4100, 4097] * 4, [1] * 8, True, 0), (70, 2, 16, [4500, 4300] * 12, [3] * 24, True, 4400),
    (192, 8, 24, [90, 300, 65] * 11, [1] * 33, True, 0), (256, 8, 5, [90, 300, 128] * 11, [4, 5, 8] * 11, True, 100),
    (200, 8, 16, [150, 80] * 16, [2] * 32, False, 0)])
def test_tiles_of_32_rows(ctx, D, Hkv, G, lengths, ns, causal, window, dtype):
    """More than 16 rows of a sequence and head on a full card."""
    attention_case(ctx, 58, dtype, D, Hkv * G, Hkv, lengths, ns, causal, window, work=True)


@pytest.mark.parametrize("dtype,D,Hkv", [("bf16", 64, 16), ("f32", 64, 16), ("bf16", 256, 8), ("f32", 200, 8)])
def test_nan_in_tiles_of_32_rows(ctx, dtype, D, Hkv):
    """NaN values among drafted tokens reach the rows that see them and no others."""
    r = rng(59)
    B, G, n = 40, 4, 6
    lengths = [int(x) for x in r.integers(n, 200, B)]
    blocks, tables = K.tables_for(r, lengths)
    cache, ref = K.Cache(ctx, blocks, Hkv, D), O.RefCache(blocks, Hkv, D)
    cu = K.cu_of(lengths)
    k, v = make(r, (int(cu[-1]), Hkv, D), "f32"), make(r, (int(cu[-1]), Hkv, D), "f32")
    bad = [int(x) for x in r.integers(1, n, B)]  # the first of the last n tokens with NaN in dim 3 of its values
    for b in range(B):
        v[cu[b + 1] - n + bad[b], :, 3] = np.nan
    if dtype == "bf16":
        k, v = S.f32_to_bf16(k), S.f32_to_bf16(v)
    full = K.Batch(ctx, tables, lengths, cu)
    K.write(cache, full, k, v)
    ref.write(tables, lengths, cu, K.wide(k), K.wide(v))
    q = make(r, (B * n, Hkv * G, D), dtype)
    b = K.Batch(ctx, tables, lengths, K.cu_of([n] * B))
    got = K.wide(K.attend(cache, b, q, scale=0.125)).reshape(B, n, Hkv * G, D)
    for i in range(B):
        kk, vv = ref.tokens(tables[i], lengths[i])
        nan = np.isnan(got[i])
        assert nan[bad[i]:, :, 3].all() and nan.sum() == (n - bad[i]) * Hkv * G
        vv = np.nan_to_num(vv)
        mask = O.sees(lengths[i], n, True, 0)
        qi = K.wide(q[i * n:(i + 1) * n])
        want, tol = O.attention(qi, kk, vv, mask, 0.125)
        half = BF if dtype == "bf16" else O.U
        tol = tol + half * (O.attention(qi, kk, np.abs(vv), mask, 0.125)[0] + np.abs(want)) + 1e-37
        assert (np.abs(got[i] - want) <= tol)[~nan].all()
    for x in (full, b, cache):
        x.free()


def test_work_suffices_whatever_the_mask(ctx):
    """fa_kv_attention_work knows neither the type nor the mask: its bytes do for each, with the results of the
    context's own scratch."""
    r = rng(61)
    for D, Hkv, G, lengths, ns in ((256, 8, 1, [1900], [1900]), (128, 2, 64, [6000] * 24, [1] * 24), (64, 1, 4, [9000, 70], [1, 9])):
        blocks, tables = K.tables_for(r, lengths)
        cache = K.Cache(ctx, blocks, Hkv, D)
        k = make(r, (max(lengths), Hkv, D), "f32")
        for i, length in enumerate(lengths):
            b = K.Batch(ctx, tables[i:i + 1], [length], [0, length])
            K.write(cache, b, k[:length], k[:length])
            b.free()
        b = K.Batch(ctx, tables, lengths, K.cu_of(ns))
        for dtype in ("f32", "bf16"):
            q = make(r, (sum(ns), Hkv * G, D), dtype)
            for causal, window in ((True, 0), (False, 0), (True, 2000), (True, 100), (False, 700)):
                one, two = (K.attend(cache, b, q, causal, window, 0.1, work) for work in (True, False))
                np.testing.assert_array_equal(one, two)
                assert np.isfinite(K.wide(one)).all()
        b.free()
        cache.free()


@pytest.mark.parametrize("dtype,Hkv,lengths,ns,width", [
    ("bf16", 64, [1300, 0, 100, 700, 1299, 400, 90, 1000, 640, 130, 1300, 257],
     [130, 0, 100, 129, 200, 0, 90, 128, 96, 130, 257, 120], 22),
    ("f32", 32, [90 + 2 * i for i in range(70)], [90 + i for i in range(70)], 8),
    ("bf16", 128, [70 * i for i in range(20)], [70] * 10 + [66] * 10, 30)])
def test_whole_tiles_of_many_rows_go_by_length(ctx, dtype, Hkv, lengths, ns, width):
    """More tiles than the card takes at once, of sequences of many lengths, some without rows or tokens: every tile is
    some workgroup's. Heads have the same keys, values and queries; the first is compared with the reference."""
    r = rng(55)
    D, ns = 64, [min(n, l) for n, l in zip(ns, lengths)]
    blocks, tables = K.tables_for(r, lengths, width=width)
    cache, ref = K.Cache(ctx, blocks, Hkv, D), O.RefCache(blocks, 1, D)
    cu = K.cu_of(lengths)
    k, v = (make(r, (int(cu[-1]), 1, D), dtype) for _ in range(2))
    full = K.Batch(ctx, tables, lengths, cu)
    K.write(cache, full, np.repeat(k, Hkv, 1), np.repeat(v, Hkv, 1))
    ref.write(tables, lengths, cu, K.wide(k), K.wide(v))
    cu = K.cu_of(ns)
    q = make(r, (int(cu[-1]), 1, D), dtype)
    b = K.Batch(ctx, tables, lengths, cu)
    got = K.attend(cache, b, np.repeat(q, Hkv, 1), scale=0.125)
    assert (got == got[:, :1]).all()
    for i, (length, n) in enumerate(zip(lengths, ns)):
        at = slice(cu[i], cu[i + 1])
        kk, vv = ref.tokens(tables[i], length)
        want, tol = O.attention(K.wide(q[at]), kk, vv, O.sees(length, n, True, 0), 0.125)
        if dtype == "bf16":
            tol = tol + BF * O.attention(K.wide(q[at]), kk, np.abs(vv), O.sees(length, n, True, 0), 0.125)[0]
        close(got[at, :1], want, tol, f"sequence {i} of {length}, {n} rows")
    for x in (full, b, cache):
        x.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_weights_on_zero_values_count(ctx, dtype):
    """131071 tokens whose values are zero (their scale is the smallest), each with a weight of 2^-22.5: together they
    take 2 % of a row's sum, in the kernels for many rows and for few. The tokens after the first 64 share one block. A
    lane adds 32 weights of a block to a sum over the blocks, or 16 of every fourth block to one sum: at most tokens / 16
    terms one after another, and of the values those of one block."""
    r = rng(52)
    Hkv, G, D, tokens = 256, 32, 64, 131072  # (as many heads as leave tiles whole)
    k, v = np.zeros((128, Hkv, D), np.float32), np.zeros((128, Hkv, D), np.float32)
    k[0, :, 0] = 1.0
    v[:64] = r.standard_normal((64, 1, D)).astype(np.float32)
    k, v = (S.f32_to_bf16(x) if dtype == "bf16" else x for x in (k, v))
    cache, ref = K.Cache(ctx, 2, Hkv, D), O.RefCache(2, Hkv, D)
    first = K.Batch(ctx, [[0, 1]], [128], [0, 128])
    K.write(cache, first, k, v)
    ref.write([[0, 1]], [128], [0, 128], K.wide(k), K.wide(v))
    assert (ref.exp[1, :, 1] == -80).all()
    table = np.ones((1, tokens // 64), np.int32)
    table[0, 0] = 0
    scale = float(np.float32(22.5 * np.log(2.0)))
    kk, vv = (x[:, :1] for x in ref.tokens(table[0], tokens))
    for n in (4, 1):
        q = np.repeat(make(r, (n, G, D), dtype)[:, None], Hkv, 1).reshape(n, Hkv * G, D)
        q[..., 0] = S.f32_to_bf16(np.ones(1, np.float32)) if dtype == "bf16" else 1.0
        b = K.Batch(ctx, table, [tokens], [0, n])
        got = K.attend(cache, b, q, scale=scale)
        q1, mask = K.wide(q[:, :1]), O.sees(tokens, n, True, 0)
        want, tol = O.attention(q1, kk, vv, mask, scale, chain=tokens // 16)
        if dtype == "bf16":
            tol = tol + BF * O.attention(q1, kk, np.abs(vv), mask, scale)[0]
        close(got[:, :1], want, tol, f"{dtype} n={n}")
        assert (got == got[:, :1]).all()  # (keys are zero where queries differ)
        b.free()
    first.free()
    cache.free()


def test_blocks_behind_the_window_are_not_needed(ctx):
    """The host form with a window: table entries of blocks that no row sees may be outside the pool."""
    r = rng(53)
    cache, ref, tables = fill(ctx, r, [500], 2, 64)
    b = K.Batch(ctx, tables, [500], [0, 3])
    q = make(r, (3, 4, 64), "f32")
    want, tol = O.attention(q, *ref.tokens(tables[0], 500), O.sees(500, 3, True, 100), 0.125)
    b.tables[0, :6] = -1  # the first row, 497, sees 398 .. 497
    hb, out = b.host(), np.empty_like(q)
    N.check(ctx.h, N.lib().fa_kv_attention(ctx.h, C.byref(cache.c), C.byref(hb), 0, q.ctypes.data, *K.st(q), 4, 1, 100,
                                           0.125, out.ctypes.data))
    close(out, want, tol, "behind the window")
    b.free()
    cache.free()


def test_two_contexts_at_once():
    """Calls of two contexts on one pool, enqueued side by side, each with scratch of its own."""
    a, c = N.Context(0), N.Context(0)
    r = rng(50)
    cache, ref, tables = fill(a, r, [3000, 500], 2, 128)
    a.sync()
    jobs = []
    for ctx_ in (a, c, a, c):
        q = make(r, (2, 8, 128), "f32")
        jobs.append((ctx_, q, K.Batch(ctx_, tables, [3000, 500], [0, 1, 2]), K.Buf(ctx_, q), K.Buf(ctx_, nbytes=q.nbytes)))
    for _ in range(20):
        for ctx_, q, b, bq, bo in jobs:
            N.check(ctx_.h, N.lib().fa_kv_attention_dev(ctx_.h, C.byref(cache.c), C.byref(b.b), 0, bq.p, 1024, 128, 8, 1,
                                                        0, 0.09, bo.p, None, 0))
    a.sync()
    c.sync()
    for ctx_, q, b, bq, bo in jobs:
        got = bo.get((2, 8, 128), np.float32)
        for i, length in enumerate((3000, 500)):
            want, tol = O.attention(q[i:i + 1], *ref.tokens(tables[i], length), O.sees(length, 1, True, 0),
                                    float(np.float32(0.09)))
            close(got[i:i + 1], want, tol, "two contexts")
    cache.free()
    c.close()
    a.close()


# ---- the operators together, as a program uses them ------------------------------------------

@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_decoding_run(ctx, dtype):
    """Prompts of several sequences, tokens one by one and a few at a time, a rollback, a freed sequence whose blocks are
    used again: after each step attention equals attention over what the cache reads back, by the 64-bit reference and
    by the framework's attention operator."""
    r = rng(60)
    H, Hkv, D = 6, 2, 64
    scale = float(np.float32(1 / 8))

    def check(cache, seqs, q, counts, out, window):
        at = 0
        for s, n in zip(seqs, counts):
            k, v = cache.Read(s)
            rows = slice(at, at + n)
            mask = O.sees(len(k), n, True, window)
            want, tol = O.attention(K.wide(q[rows]), k.astype(np.float64), v.astype(np.float64), mask, scale)
            if dtype == "bf16":
                tol = tol + BF * O.attention(K.wide(q[rows]), k.astype(np.float64), np.abs(v).astype(np.float64), mask,
                                             scale)[0]
            close(out[rows], want, tol, f"step, sequence {s}")
            if dtype == "f32" and n:
                full = [np.repeat(x.transpose(1, 0, 2), H // Hkv, 0)[None] for x in (k, v)]
                add = np.where(mask, np.float32(0), T.MASK_NEG)[None, None]
                other = T.AttentionScaled(np.ascontiguousarray(q[rows].transpose(1, 0, 2))[None], *full, add, scale,
                                          ctx=ctx)[0].transpose(1, 0, 2)
                np.testing.assert_allclose(out[rows], other, rtol=0, atol=2e-5 * max(1.0, np.abs(v).max()))
            at += n

    with KVCache(Hkv, D, 1200, ctx=ctx) as cache:
        a, b, c = cache.Add(), cache.Add(), cache.Add()
        plan = [([a, b], [150, 63]), ([a, b], [1, 1]), ([c, a], [64, 3]), ([a, b, c], [1, 1, 1]), ([b], [200])]
        for seqs, counts in plan:
            n = sum(counts)
            cache.Append(seqs, make(r, (n, Hkv, D), dtype), make(r, (n, Hkv, D), dtype, 3.0), counts)
            q = make(r, (n, H, D), dtype)
            check(cache, seqs, q, counts, cache.Attention(seqs, q, counts), 0)
            check(cache, seqs, q, counts, cache.Attention(seqs, q, counts, window=50), 50)
        room = cache.Room()
        cache.Truncate(a, 130)
        cache.Free(b)
        assert cache.Room() > room and cache.Len(a) == 130
        d = cache.Add()
        cache.Append([d, a], make(r, (310, Hkv, D), dtype), make(r, (310, Hkv, D), dtype), [305, 5])
        q = make(r, (310, H, D), dtype)
        check(cache, [d, a], q, [305, 5], cache.Attention([d, a], q, [305, 5]), 0)
        with pytest.raises(T.TensorError, match="free"):
            cache.Append([d], make(r, (1200, Hkv, D), dtype), make(r, (1200, Hkv, D), dtype), [1200])
        assert cache.Len(d) == 305
        for bad in (lambda: cache.Append([b], q[:1, :Hkv], q[:1, :Hkv]), lambda: cache.Append([d, d], q[:2, :Hkv], q[:2, :Hkv]),
                    lambda: cache.Attention([d], q[:, :5]), lambda: cache.Truncate(d, 400), lambda: cache.Read(d, 400),
                    lambda: cache.Append([d], q[:1], q[:1]), lambda: cache.Attention([d], q, [3])):
            with pytest.raises(T.TensorError):
                bad()
