"""Sampling where sums meet their bounds exactly: equal logits, whose weights
are 1, so that the definition's sums have no rounding and say which tokens stay
and which is drawn."""
import numpy as np
import pytest

import test_gpu_kvcache as G
import test_gpu_sample as T
from ai_amd import synth as S

pytestmark = pytest.mark.gpu
INF = np.inf


def some_equal(r, rows, n, vocab, dtype, spread=3.0):
    """Rows of n equal logits at places of their own, -inf elsewhere."""
    l = np.full((rows, vocab), -INF, np.float32)
    for x in l:
        x[r.permutation(vocab)[:n]] = np.float32(r.standard_normal() * spread)
    return S.f32_to_bf16(l) if dtype == "bf16" else l


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("n", [2, 4, 8, 1000])
def test_top_p_of_equal_logits(ctx, n, dtype):
    """A share of n tokens that is a whole number of them is reached by that many."""
    r = G.rng(n)
    rows = 240
    l = some_equal(r, rows, n, n + 37, dtype)
    top_p = r.choice([0.25, 0.5, 0.75], rows).astype(np.float32)
    temperature = r.choice([1e-3, 0.2, 0.7, 1.0, 1.7], rows).astype(np.float32)
    for u in (0.0, 0.3, 0.9, 1 - 2.0 ** -24):
        u = np.full(rows, u, np.float32)
        T.check(T.draw(ctx, l, u, top_p=top_p, temperature=temperature), l, u, top_p=top_p, temperature=temperature)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_shares_where_logits_are_many_steps_from_zero(ctx, dtype):
    """Logits that are up to 2^39 steps of 1/32 of the temperature from zero share the weight as others do."""
    r = G.rng(5)
    rows, n = 120, 6
    l = some_equal(r, rows, n, 90, dtype, spread=1000.0)
    temperature = (10.0 ** r.uniform(-7, 0, rows)).astype(np.float32)
    u = (np.arange(rows) % n / n + 0.01).astype(np.float32)
    for s in (dict(min_p=0.5), dict(top_p=0.999), dict(top_p=0.5), dict(top_k=20, min_p=0.1)):
        s = {k: np.full(rows, v, np.int32 if k == "top_k" else np.float32) for k, v in s.items()}
        T.check(T.draw(ctx, l, u, temperature=temperature, **s), l, u, temperature=temperature, **s)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("s", [dict(min_p=0.5), dict(top_p=0.999), dict(top_k=16), {}])
@pytest.mark.parametrize("n", [2, 4, 16])
def test_numbers_on_the_border_of_two_tokens(ctx, n, s, dtype):
    """u times the sum equal to a running sum draws the token after it: the sum does not exceed it."""
    r = G.rng(n + 100)
    rows = 160
    l = some_equal(r, rows, n, n + 50, dtype)
    u = (np.arange(rows) % n / n).astype(np.float32)
    s = {k: np.full(rows, v, np.int32 if k == "top_k" else np.float32) for k, v in s.items()}
    s["temperature"] = r.choice([0.3, 0.7, 1.0, 1.9], rows).astype(np.float32)
    T.check(T.draw(ctx, l, u, **s), l, u, **s)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("s", [{}, dict(min_p=0.5), dict(top_p=0.5), dict(top_k=2 ** 19 + 8192)])
def test_numbers_on_the_border_of_two_slices(ctx, s, dtype):
    """Rows of 128 slices, all logits equal: slices found by different waves, at each border, beside it and within."""
    rows, vocab = 24, 2 ** 20
    keep = vocab if "min_p" in s or not s else 2 ** 19 if "top_p" in s else s["top_k"]
    at = np.concatenate([np.arange(8) * 8192 * 16, np.arange(8) * 8192 * 16 + 8191, np.arange(8) * 65536 + 70000]) % keep
    l = np.full((rows, vocab), -2.5, np.float32)
    l = S.f32_to_bf16(l) if dtype == "bf16" else l
    u = (at / np.float64(keep)).astype(np.float32)
    want = np.floor(np.float64(u) * keep).astype(np.int32)  # (u rounds where keep is no power of two)
    s = {k: np.full(rows, v, np.int32 if k == "top_k" else np.float32) for k, v in s.items()}
    ids, logp = T.draw(ctx, l, u, temperature=np.full(rows, 0.7, np.float32), **s)
    np.testing.assert_array_equal(ids, want)
    assert np.abs(logp + np.log(keep)).max() <= 2.0 ** -24 * np.log(keep) + 1e-9


# ---- rows of many slices ---------------------------------------------------------------------


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [600001, 4300001, 2 ** 24])
def test_very_large_vocabularies(ctx, vocab, dtype):
    """More than 64 and than 512 slices, and slices of 16384: all filters, tokens that stay near both ends."""
    r = G.rng(vocab)
    rows = 3
    l = T.logits(r, rows, vocab, "f32", "tail")
    l[0, [0, 1, vocab - 2, vocab - 1]] = l[0].max() + np.float32(0.5)
    l[1] = r.standard_normal(vocab) * 0.05
    l = S.f32_to_bf16(l) if dtype == "bf16" else l
    settings = [dict(temperature=[0.7, 1.0, 0.5], top_k=[50, vocab // 3, 0], top_p=[0.9, 0.5, 0.99], min_p=[0, 0, 0.01]),
                dict(top_p=[0.999, 0.3, 0.5]), dict(temperature=[1.3] * 3)]
    for s, u in zip(settings, ([0.99, 0.5, 0.7], [0.0, 0.999, 0.4], [0.25, 1 - 2.0 ** -24, 0.6])):
        s = {k: np.asarray(v, np.int32 if k == "top_k" else np.float32) for k, v in s.items()}
        T.check(T.draw(ctx, l, u, work=True, **s), l, u, **s)
        print(f"{vocab} {dtype} {list(s)}", flush=True)


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab", [600001, 4300001, 2 ** 24])
def test_very_large_vocabularies_of_equal_logits(ctx, vocab, dtype):
    """Every token listed at once; draws at the ends of what stays."""
    l = np.full((4, vocab), -2.5, np.float32)
    l = S.f32_to_bf16(l) if dtype == "bf16" else l
    u = np.array([0, 0.25, 0.7, 1 - 2.0 ** -24], np.float32)
    for s, keep in ((dict(top_p=0.5), (vocab + 1) // 2), (dict(top_k=vocab - 5), vocab - 5), (dict(min_p=1.0), vocab),
                    (dict(top_k=vocab // 2, top_p=0.25), -(-(vocab // 2) // 4)), ({}, vocab)):
        s = {k: np.full(4, v, np.int32 if k == "top_k" else np.float32) for k, v in s.items()}
        ids, logp = T.draw(ctx, l, u, temperature=np.full(4, 0.7, np.float32), **s)
        np.testing.assert_array_equal(ids, np.floor(u.astype(np.float64) * keep).astype(np.int32))
        assert np.abs(logp + np.log(keep)).max() <= 2.0 ** -24 * np.log(keep) + 1e-9


@pytest.mark.parametrize("dtype", ["f32", "bf16"])
@pytest.mark.parametrize("vocab,rows", [(32000, 300), (8000, 700), (60000, 130)])
def test_rows_cut_otherwise_agree(ctx, vocab, rows, dtype):
    """A row by itself is cut in slices of half the size that it has among many: the same token, and the log of its share
    to its rounding."""
    r = G.rng(vocab)
    l, u, s = T.logits(r, rows, vocab, dtype), T.numbers(r, rows), T.settings(r, rows)
    equal = some_equal(r, rows // 2, 1000, vocab, dtype)
    l[:len(equal)] = equal
    s["top_p"][:len(equal) // 2] = 0.5
    many = T.draw(ctx, l, u, **s)
    for i in range(0, rows, 9):
        one = T.draw(ctx, l[i:i + 1], u[i:i + 1], **{k: v[i:i + 1] for k, v in s.items()})
        assert one[0][0] == many[0][i], (i, {k: v[i] for k, v in s.items()}, u[i])
        assert abs(float(one[1][0]) - float(many[1][i])) <= 2.0 ** -23 * abs(float(many[1][i])) + 1e-9
