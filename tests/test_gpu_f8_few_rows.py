"""Products of up to 16 rows on both sides of the bounds between the kernel for few rows and tiles: up to 2^24 weights
bf16 results are float32's, rounded once."""
import numpy as np
import pytest

import decode_oracle as O
import kv_lib as K
import test_gpu_f8 as F
import test_gpu_kvcache as G
from ai_amd import synth as S

pytestmark = pytest.mark.gpu


@pytest.mark.parametrize("cdt", ["f32", "bf16"])
@pytest.mark.parametrize("m", [1, 3, 16])
@pytest.mark.parametrize("n,k", [(8192, 300), (8193, 300), (16384, 1024), (40000, 257), (131072, 128), (100, 6144), (100, 6145),
                                 (1024, 16384), (7, 200001), (2730, 6144)])
def test_both_sides_of_the_bounds(ctx, n, k, m, cdt):
    r = G.rng(m * 100 + n + k)
    a = (r.standard_normal((m, k)) * np.exp(1.5 * r.standard_normal((m, k)))).astype(np.float32)
    w = (r.standard_normal((n, k)) / np.sqrt(k)).astype(np.float32)
    bias = r.standard_normal(n).astype(np.float32)
    held = F.Held(ctx, n, k).write(w)
    got = F.product(ctx, held, a, cdt, dict(bias=bias), pad=3, work=True)
    np.testing.assert_array_equal(F.product(ctx, held, a, cdt, dict(bias=bias)), got)
    held.free()
    cols = np.unique(np.concatenate([[0, 1, n - 1, n - 2], r.integers(0, n, 2000)]).clip(0, n - 1))
    want, tol = O.product(a.astype(np.float64), w[cols].astype(np.float64), False, bias=bias[cols])
    if cdt == "bf16":
        tol = tol + O.BF * (np.abs(want) + tol)
    F.check(got[:, cols], want, tol, f"{m}x{n}x{k} {cdt}")
