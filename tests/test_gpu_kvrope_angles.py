"""Cosines and sines of the rotary append: float64's rounded to float32, to the
bit. A query of ones and zeros is turned into them."""
import numpy as np
import pytest

import kv_lib as K
import test_gpu_kvcache as G
import test_gpu_kvrope as R

pytestmark = pytest.mark.gpu

# (position, base, pair of 64) where a cosine or sine in float64 lies within 2^-37 of the middle of two float32 numbers
NEAR_MIDDLES = [(7485698, 5e5, 43), (33945, 1e6, 24), (61517, 1e4, 15), (5093596, 1e4, 20), (7029092, 1e6, 48),
                (65726, 1e6, 7), (1959542, 1e4, 53), (35583, 5e5, 47), (61517, 1e6, 10), (9192579, 1e6, 1),
                (163, 5e5, 1), (6692761, 1e6, 58), (5732059, 1e6, 42), (65160, 1e6, 5), (3930282, 1e4, 12),
                (7621303, 1e4, 43), (8407696, 1e6, 45), (620306, 1e4, 1), (19137, 1e6, 22), (15657, 1e6, 23),
                (7717755, 1e6, 13), (3813646, 1e4, 49), (98137, 1e4, 26), (84461, 1e4, 1)]


def turned(ctx, positions, base, D):
    """Cosines and sines [rows, D / 2] of the positions' angles as queries turn by them."""
    n = len(positions)
    r = G.rng(1)
    blocks, tables = K.tables_for(r, [n])
    cache = K.Cache(ctx, blocks, 1, D)
    k, v = (G.make(r, (n, 1, D), "f32") for _ in range(2))
    q = np.zeros((n, 1, D), np.float32)
    q[:, :, :D // 2] = 1
    b = K.Batch(ctx, tables, [n], [0, n])
    s = R.Step(ctx, q, k, v, positions)
    out = s.run(cache, b, base, D)[:, 0]
    for x in (s, b, cache):
        x.free()
    return out[:, :D // 2], out[:, D // 2:]


def angles(positions, base, D):
    inv = np.array([base ** (-(2.0 * i) / D) for i in range(D // 2)])
    return np.asarray(positions, np.float64)[:, None] * inv


@pytest.mark.parametrize("base", [1e4, 5e5, 1e6])
def test_angles_near_the_middle_of_two_numbers(ctx, base):
    near = [(p, i) for p, b, i in NEAR_MIDDLES if b == base]
    c, s = turned(ctx, [p for p, _ in near], base, 128)
    a = angles([p for p, _ in near], base, 128)
    at = np.arange(len(near)), [i for _, i in near]
    np.testing.assert_array_equal(c[at], np.cos(a).astype(np.float32)[at])
    np.testing.assert_array_equal(s[at], np.sin(a).astype(np.float32)[at])


@pytest.mark.parametrize("base", [1.0, 1e4, 1e6])
def test_angles_of_many_positions(ctx, base):
    """The device's cosine and the host's are within 2^-52 of the value: they round to two numbers of float32 once in 2^27."""
    r = G.rng(2)
    pos = np.concatenate([np.arange(2000), r.integers(-2 ** 31, 2 ** 31, 1000), r.integers(0, 10 ** 6, 3000)])
    c, s = turned(ctx, pos, base, 256)
    a = angles(pos, base, 256)
    differ = (c != np.cos(a).astype(np.float32)).sum() + (s != np.sin(a).astype(np.float32)).sum()
    assert differ <= 2, differ
