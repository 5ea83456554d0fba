"""64-bit references of a decoding step's operators: rotary positions, products
with 8-bit weights, sampling. From their definitions, with tolerances."""
import numpy as np

import kv_oracle as KO

U32 = 2.0 ** -24  # half a step of float32, relative
BF = 2.0 ** -8    # of bf16


def rotate(x, positions, base, dims):
    """x [rows, heads, D] in float32, turned: float32 as the definition has it (products of float32 exact in float64)."""
    half = dims // 2
    inv = np.array([float(base) ** (-(2.0 * i) / dims) for i in range(half)])
    angle = np.asarray(positions, np.float64)[:, None] * inv
    c, s = (f(angle).astype(np.float32).astype(np.float64)[:, None, :] for f in (np.cos, np.sin))
    x = x.astype(np.float64)
    out = x.copy()
    lo, hi = x[..., :half], x[..., half:dims]
    with np.errstate(invalid="ignore", over="ignore"):
        out[..., :half] = lo * c - hi * s
        out[..., half:dims] = hi * c + lo * s
        return out.astype(np.float32)


# ---- products ------------------------------------------------------------------------------


def quantize(x):
    """x [n, k] -> (values in units of the scale, exponents), [n, kb, 128] (NaN kept, zeros past k) and [n, kb]."""
    n, k = x.shape
    kb = -(-k // 128)
    p = np.zeros((n, kb * 128))
    p[:, :k] = x
    p = p.reshape(n, kb, 128)
    fin = np.isfinite(p)
    big = np.where(fin, np.abs(p), 0).max(2, initial=0)
    with np.errstate(divide="ignore"):
        e = np.ceil(np.log2(big / 448))
    e = np.clip(np.where(big > 0, e, KO.E_MIN), KO.E_MIN, KO.E_MAX)
    e = np.where((e < KO.E_MAX) & (big > 448 * 2.0 ** e), e + 1, e)  # (log2 rounds)
    e = np.where((e > KO.E_MIN) & (big <= 448 * 2.0 ** (e - 1)), e - 1, e)
    top = np.where(e == KO.E_MAX, 240.0, 448.0)[:, :, None]
    v = np.clip(np.where(fin, p, np.nan) * 2.0 ** -e[:, :, None], -top, top)
    return KO.round_e4m3(v), e


def values(q, e, k):
    return (q * 2.0 ** e[:, :, None]).reshape(len(q), -1)[:, :k]


def gelu(v):
    with np.errstate(over="ignore"):
        return 0.5 * v * (1 + np.tanh(np.sqrt(2 / np.pi) * (v + 0.044715 * v ** 3)))


def product(a, w, c_bf16, bias=None, row_scale=None, act=0, mul=None, residual=None):
    """epilogue(A^ . W^T) of a [m, k] and w [n, k] (values before quantising), and how far the kernel may be from it.

    float32 results: products exact, K sums in float32 by units that may cut instead of rounding: at most K 2^-23 of the
    sum of magnitudes, whatever their order. bf16 results, as the header states: each product cut to a multiple of 2^-13
    of the power of two below the largest of its group of eight (seven of them: the largest has eight bits itself), and
    the same sums. Epilogue: a rounding of float32 for each operation, GELU off by 2^-21 of its argument and with a slope
    of at most 1.13; tanh by 2^-21, slope 1; the result's own rounding."""
    qa, ea = quantize(a)
    qw, ew = quantize(w)
    k = a.shape[1]
    A, W = values(qa, ea, k), values(qw, ew, k)
    if k == 0:
        A, W = np.zeros((len(a), 1)), np.zeros((len(w), 1))
    v = A @ W.T
    mag = np.abs(A) @ np.abs(W).T
    tol = (k + 8) * 2.0 ** -23 * mag
    if c_bf16 and k:
        kp = -(-k // 8) * 8
        pa, pw = (np.pad(np.nan_to_num(np.abs(x)), ((0, 0), (0, kp - k))).reshape(len(x), -1, 8) for x in (A, W))
        for g in range(kp // 8):
            tol += 7 * 2.0 ** -13 * (pa[:, None, g] * pw[None, :, g]).max(2)
    if bias is not None:
        v = v + bias
        tol = tol + 2 * U32 * (np.abs(v) + tol)
    if row_scale is not None:
        v = v * row_scale[:, None]
        tol = tol * np.abs(row_scale[:, None]) + 2 * U32 * np.abs(v)
    if act == 1:
        v = np.maximum(v, 0)
    elif act == 2:
        tol = 1.13 * tol + 2.0 ** -21 * np.abs(v)
        v = gelu(v)
    elif act == 3:
        v = np.tanh(v)
        tol = tol + 2.0 ** -21
    if mul is not None:
        v = v * mul
        tol = tol * np.abs(mul) + 2 * U32 * np.abs(v)
    if residual is not None:
        v = v + residual
        tol = tol + 2 * U32 * (np.abs(v) + tol)
    return v, tol + (BF if c_bf16 else U32) * (np.abs(v) + tol) + 1e-38


# ---- sampling ---------------------------------------------------------------------------------


def sample(l, u, temperature=1.0, top_k=0, top_p=1.0, min_p=0.0):
    """(id, log of its share) of one row; settings as float32 values."""
    l = np.where(np.isnan(l), -np.inf, l.astype(np.float64))
    M = l.max()
    if M == -np.inf:
        return -1, np.nan
    order = np.lexsort((np.arange(len(l)), -l))
    if temperature == 0:
        return int(order[0]), 0.0
    with np.errstate(invalid="ignore"):
        w = np.where(l == M, 1.0, 0.0) if M == np.inf else np.exp((l - M) / np.float64(temperature))
    n = len(l) if top_k <= 0 else min(int(top_k), len(l))
    run = np.cumsum(w[order[:n]])
    if top_p < 1:
        n = min(n, int(np.searchsorted(run, np.float64(top_p) * run[-1], side="left")) + 1)
    keep = np.zeros(len(l))
    keep[order[:n]] = w[order[:n]]
    keep[keep < np.float64(min_p)] = 0
    run = np.cumsum(keep)
    at = int(np.searchsorted(run, np.float64(u) * run[-1], side="right"))
    at = min(at, int(np.nonzero(keep)[0][-1]))
    return at, float(np.log(keep[at] / run[-1]))
