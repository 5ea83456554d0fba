"""Attention over the 8-bit key/value cache: how many bits its operands keep.

bf16 tensors: outputs are rounded to bf16 once, and nothing before them is. A
weight enters as two bf16 terms: rounded to bf16 it leaves at most 2^-8 of
itself, which is rounded again, so it is off by at most 2^-16 of itself, and a
sum by 2^-16 of sum p |v|; the rest of the bound is float32's (kv_oracle)."""
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
