"""Attention over the 8-bit key/value cache: how many bits its operands keep.

bf16 tensors: outputs are rounded to bf16 once, and nothing before them is. A
weight enters as two bf16 terms: rounded to bf16 it leaves at most 2^-8 of
itself, which is rounded again, so it is off by at most 2^-16 of itself, and a
sum by 2^-16 of sum p |v|; the rest of the bound is float32's (kv_oracle).
float32 tensors: three exact bf16 terms of queries and weights, in every kernel."""
import numpy as np
import pytest

import kv_lib as K
import kv_oracle as O
import test_gpu_kvcache as G

pytestmark = pytest.mark.gpu

TWO = 2.0 ** -16  # of a weight in two bf16 terms


def bf16_case(ctx, seed, D, H, Hkv, lengths, ns, causal=True, window=0, width=None, scale=None):
    r = G.rng(seed)
    cache, ref, tables = G.fill(ctx, r, lengths, Hkv, D, "bf16", width=width)
    scale = float(np.float32(1 / np.sqrt(D) if scale is None else scale))
    cu = K.cu_of(ns)
    q = G.make(r, (int(cu[-1]), H, D), "bf16")
    b = K.Batch(ctx, tables, lengths, cu)
    got = K.attend(cache, b, q, causal, window, scale)
    for i, (length, n) in enumerate(zip(lengths, ns)):
        if not n:
            continue
        k, v = ref.tokens(tables[i], length)
        rows = slice(cu[i], cu[i + 1])
        mask = O.sees(length, n, causal, window)
        want, tol = O.attention(K.wide(q[rows]), k, v, mask, scale)
        tol = (tol + TWO * O.attention(K.wide(q[rows]), k, np.abs(v), mask, scale)[0]) * (1 + G.BF)
        G.close(got[rows], want, tol, f"D={D} H={H}/{Hkv} len={length} n={n}")
    b.free()
    cache.free()


@pytest.mark.parametrize("D,H,Hkv,lengths,ns,width", [
    (64, 6, 2, [1, 65, 700], [1, 3, 2], None), (128, 4, 1, [900], [1], 400), (256, 3, 1, [500, 90], [1, 7], None),
    (512, 2, 2, [300], [2], None), (320, 2, 1, [200], [40], None),                       # tiles of 16 rows
    (64, 64, 16, [400] * 40, [5] * 40, None), (192, 192, 8, [90, 300, 65] * 11, [1] * 33, None),  # of 32
    (64, 4, 4, [300] * 3, [257, 300, 128], 20000), (128, 8, 2, [700, 333], [640, 333], 20000),    # of 128
    (192, 1, 1, [1000], [129], 20000), (256, 3, 1, [500, 129], [400, 129], 20000)])
def test_bf16_outputs_are_rounded_once(ctx, D, H, Hkv, lengths, ns, width):
    bf16_case(ctx, D + H, D, H, Hkv, lengths, ns, width=width)
    bf16_case(ctx, D + H + 1, D, H, Hkv, lengths, ns, causal=False, window=150, width=width)


def test_bf16_value_scales_far_apart(ctx):
    """Two terms of weights that carry block scales from 2^-80 (values of zero beside them) to 2^110."""
    r = G.rng(31)
    D, n = 64, 320
    blocks, tables = K.tables_for(r, [n], width=20000)
    cache, ref = K.Cache(ctx, blocks, 1, D), O.RefCache(blocks, 1, D)
    k, v = G.make(r, (n, 1, D), "bf16"), G.make(r, (n, 1, D), "f32")
    for i, e in enumerate((0, 30, -30, 110, -70)):
        v[i * 64:(i + 1) * 64] *= np.float32(2.0 ** e)
    v = G.S.f32_to_bf16(v)
    b = K.Batch(ctx, tables, [n], [0, n])
    K.write(cache, b, k, v)
    ref.write(tables, [n], [0, n], K.wide(k), K.wide(v))
    wk, wv = ref.tokens(tables[0], n)
    for heads in (1, 2):
        q = G.make(r, (n, heads, D), "bf16")
        for window in (64, 20):
            got = K.attend(cache, b, q, True, window, 0.125)
            mask = O.sees(n, n, True, window)
            want, tol = O.attention(K.wide(q), wk, wv, mask, 0.125)
            tol = (tol + TWO * O.attention(K.wide(q), wk, np.abs(wv), mask, 0.125)[0]) * (1 + G.BF)
            G.close(got, want, tol, f"value scales, {heads} heads, window {window}")
    b.free()
    cache.free()


def f32_bound(q, k, v, mask, scale):
    """The reference's output and float32's bound without any loss of a query's bits: products of three bf16 terms are
    exact, their sums of 3 D terms and the factors in float32 (as kv_oracle.attention states, whose bound grows with the
    row's largest query value, too; this one only with the products)."""
    n, H, D = q.shape
    q = q.astype(np.float64)
    with np.errstate(over="ignore"):  # (its bound)
        out, tol = O.attention(q, k, v, mask, scale)
        absv = O.attention(q, k, np.abs(v), mask, scale)[0]
    for h in range(H):
        kh = np.abs(k[:, h // (H // k.shape[1])])
        mag = np.where(mask, np.abs(q[:, h]) @ kh.T, 0).max(1) * abs(scale)
        ds = (3 * D + 4) * O.U * mag
        rel = np.expm1(2 * ds) + 2.0 ** -22 + 2 * 150 * O.U + (3 * mask.sum(1) + 64) * O.U
        tol[:, h] = rel[:, None] * absv[:, h]
    return out, tol


@pytest.mark.parametrize("D,H,Hkv,length,n,width", [(64, 2, 1, 200, 5, None), (64, 4, 1, 300, 257, 20000),
                                                    (128, 2, 2, 300, 300, 20000), (256, 3, 1, 200, 200, 20000)])
@pytest.mark.parametrize("large", [2.0 ** 30, 2.0 ** -60, 2.0 ** 90])
def test_f32_queries_keep_their_bits(ctx, D, H, Hkv, length, n, width, large):
    """A channel of the queries is far from the others and meets zero keys (2^-60: the others do, and it meets ones of
    2^60): every other channel's 24 bits count, whichever kernel takes the call."""
    r = G.rng(D + n)
    blocks, tables = K.tables_for(r, [length], width=width)
    cache, ref = K.Cache(ctx, blocks, Hkv, D), O.RefCache(blocks, Hkv, D)
    k, v = G.make(r, (length, Hkv, D), "f32"), G.make(r, (length, Hkv, D), "f32")
    q = G.make(r, (n, H, D), "f32")
    if large > 1:
        q[:, :, 3] *= np.float32(large)
        k[:, :, 3] = 0
    else:
        q[:, :, :4] *= np.float32(large)
        k[:, :, 4:] = 0
        k *= np.float32(1 / large)
    b = K.Batch(ctx, tables, [length], [0, length])
    K.write(cache, b, k, v)
    ref.write(tables, [length], [0, length], k, v)
    b.free()
    b = K.Batch(ctx, tables, [length], [0, n])
    got = K.attend(cache, b, q, scale=0.125)
    want, tol = f32_bound(q, *ref.tokens(tables[0], length), O.sees(length, n, True, 0), 0.125)
    G.close(got, want, tol, f"D={D} n={n} large={large:g}")
    b.free()
    cache.free()


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n,width", [(5, None), (150, 20000), (150, 1000)])
def test_scales_near_zero(ctx, dtype, n, width):
    """Queries of 2^110 and scales down to 0, whose product with a block's key scale is below float32's normal numbers:
    scores are that product's, in the kernel for many rows too."""
    r = G.rng(70 + n)
    D, H, length = 64, 2, 300
    cache, ref, tables = G.fill(ctx, r, [length], 1, D, dtype, width=width)
    wk, wv = ref.tokens(tables[0], length)
    q = G.make(r, (n, H, D), "f32", 2.0 ** 112)
    q = G.S.f32_to_bf16(q) if dtype == "bf16" else q
    b = K.Batch(ctx, tables, [length], [0, n])
    mask = O.sees(length, n, True, 0)
    for scale in (0.0, 2.0 ** -122, -2.0 ** -120, 1e-45, 2.0 ** -114):
        got = K.attend(cache, b, q, scale=scale)
        want, tol = f32_bound(K.wide(q), wk, wv, mask, scale)
        if dtype == "bf16":
            tol = (tol + TWO * O.attention(K.wide(q), wk, np.abs(wv), mask, scale)[0]) * (1 + G.BF)
        if 0 < abs(scale) < 2.0 ** -116:  # a factor with fewer than 24 bits: at most 2^-149 of a product under 2^128
            tol = tol + 2.0 ** -20 * O.attention(K.wide(q), wk, np.abs(wv), mask, scale)[0]
        G.close(got, want, tol, f"{dtype} n={n} scale={scale:g}")
    b.free()
    cache.free()
