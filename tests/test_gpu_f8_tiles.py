"""Products with 8-bit weights in tiles of 256 rows by 256 columns (bf16 results, 256 such tiles and more): several
groups of four blocks and what is left of them, remainders of rows and columns."""
import numpy as np
import pytest

import decode_oracle as O
import kv_lib as K
import test_gpu_f8 as F
import test_gpu_kvcache as G
from ai_amd import synth as S

pytestmark = pytest.mark.gpu

# blocks of 128 columns: 9, 10, 11, 12
SIZES = [(4000, 4090, 1100), (300, 32700, 1153), (2000, 8200, 1400), (300, 32700, 1500)]


def some(r, n, edge):
    """Places among n: some of every part, the ends and the last tile's."""
    return np.unique(np.concatenate([[0, 1, n - 1, n // edge * edge, n // edge * edge - 1], r.integers(0, n, 200),
                                     np.arange(n // edge * edge, n)[::7]]).clip(0, n - 1))


@pytest.mark.parametrize("epi", [(), ("bias", 2, "mul"), ("row_scale", "residual")])
@pytest.mark.parametrize("m,n,k", SIZES)
def test_products(ctx, m, n, k, epi):
    r = G.rng(m + n + k)
    a = (r.standard_normal((m, k)) * np.exp(0.5 * r.standard_normal((m, 1)))).astype(np.float32)
    a = S.f32_to_bf16(a)
    w = (r.standard_normal((n, k)) / np.sqrt(k)).astype(np.float32)
    e = {}
    for x in epi:
        if x == 2:
            e["act"] = x
        else:
            shape = {"bias": (n,), "row_scale": (m,), "mul": (m, n), "residual": (m, n)}[x]
            e[x] = r.standard_normal(shape).astype(np.float32)
    held = F.Held(ctx, n, k).write(w)
    got = F.product(ctx, held, a, "bf16", e if epi else None, pad=3)
    np.testing.assert_array_equal(F.product(ctx, held, a, "bf16", e if epi else None, work=True), got)
    held.free()
    rows, cols = some(r, m, 256), some(r, n, 256)
    part = {x: v if x == "act" else v[cols] if x == "bias" else v[rows] if x == "row_scale" else v[np.ix_(rows, cols)]
            for x, v in e.items()}
    want, tol = O.product(K.wide(a[rows]).astype(np.float64), w[cols].astype(np.float64), True, **part)
    F.check(got[np.ix_(rows, cols)], want, tol, f"{m}x{n}x{k} {epi}")


@pytest.mark.parametrize("m,n,k", SIZES)
def test_exact_sums(ctx, m, n, k):
    """Operands of -1, 0 and 1 with a block's scale of its own: a term lost or read twice, or a scale of another block
    or row, shows in every element."""
    r = G.rng(m + n + k + 1)
    kb = -(-k // 128)
    mine = np.arange(k) // 128
    a, w = (r.integers(-1, 2, (x, k)).astype(np.float32) for x in (m, n))
    a[:, ::128], w[:, ::128] = 1, 1
    a *= (2.0 ** r.integers(-3, 4, (m, kb)))[:, mine].astype(np.float32)
    w *= (2.0 ** r.integers(-3, 4, (n, kb)))[:, mine].astype(np.float32)
    want = a @ w.T  # (sums of at most 2^11 multiples of 2^-6 up to 2^6: exact in float32, whatever the order)
    held = F.Held(ctx, n, k).write(w)
    got = F.product(ctx, held, a, "bf16")
    np.testing.assert_array_equal(got, S.f32_to_bf16(want))
    held.free()


@pytest.mark.parametrize("m,n", [(4000, 4090), (300, 32700)])
def test_nan_stays_in_its_row_and_column(ctx, m, n):
    r = G.rng(m)
    k = 1100
    a, w = r.standard_normal((m, k)).astype(np.float32), r.standard_normal((n, k)).astype(np.float32)
    a[m - 2, 1099], w[n - 3, 700] = np.inf, np.nan
    held = F.Held(ctx, n, k).write(w)
    got = np.isnan(K.wide(F.product(ctx, held, a, "bf16")))
    want = np.zeros((m, n), bool)
    want[m - 2], want[:, n - 3] = True, True
    np.testing.assert_array_equal(got, want)
    held.free()
