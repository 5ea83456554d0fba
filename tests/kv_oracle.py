"""64-bit reference of the 8-bit key/value cache, from its definition, with
the tolerances of attention over it."""
import numpy as np

BLOCK = 64
E_MIN, E_MAX = -80, 120
U = 2.0 ** -24  # half a step of float32, relative


def decode_table():
    """The 256 values of e4m3 (bias 7, three bits of mantissa, 0x7F and 0xFF NaN)."""
    t = np.empty(256)
    for b in range(256):
        e, m = (b >> 3) & 15, b & 7
        x = m * 2.0 ** -9 if e == 0 else (1 + m / 8) * 2.0 ** (e - 7)
        if b & 127 == 127:
            x = np.nan
        t[b] = -x if b >= 128 else x
    return t


DECODE = decode_table()


def round_e4m3(x):
    """x rounded to a value of e4m3, ties to even (|x| <= 448, NaN kept)."""
    a = np.abs(x)
    with np.errstate(invalid="ignore", divide="ignore"):
        e = np.floor(np.log2(np.maximum(a, 2.0 ** -6)))
        step = 2.0 ** (e - 3)
        return np.sign(x) * np.round(a / step) * step


def scale_exp(x):
    """The smallest e with every finite |x| <= 448 * 2^e, in the allowed range."""
    a = np.abs(x[np.isfinite(x)])
    big = a.max() if a.size else 0.0
    e = E_MIN
    while e < E_MAX and big > 448 * 2.0 ** e:
        e += 1
    return e


class RefCache:
    """Values and scale exponents of [blocks][kv_heads][2][64][head_dim]."""

    def __init__(self, blocks, kv_heads, D):
        self.val = np.full((blocks, kv_heads, 2, BLOCK, D), np.nan)  # in units of the scale
        self.exp = np.full((blocks, kv_heads, 2), np.nan)

    def write(self, tables, lengths, cu, k, v):
        for b, length in enumerate(lengths):
            n = cu[b + 1] - cu[b]
            first = length - n
            pos = first
            while pos < length:
                slot, place = divmod(pos, BLOCK)
                m = min(BLOCK - place, length - pos)
                r = cu[b] + pos - first
                block = tables[b][slot]
                for part, x in enumerate((k, v)):
                    for h in range(x.shape[1]):
                        new = x[r:r + m, h].astype(np.float64)
                        e = scale_exp(new)
                        if place:
                            old = self.exp[block, h, part]
                            e = max(e, old)
                            self.val[block, h, part, :place] = round_e4m3(
                                self.val[block, h, part, :place] * 2.0 ** (old - e))
                        top = 240.0 if e == E_MAX else 448.0  # 256 * 2^120 is past float32
                        self.val[block, h, part, place:place + m] = round_e4m3(
                            np.clip(np.where(np.isfinite(new), new, np.nan) * 2.0 ** -float(e), -top, top))
                        self.exp[block, h, part] = e
                pos += m

    def tokens(self, table, length):
        """Keys and values [length, kv_heads, D] of a sequence."""
        got, used = [], np.asarray(table[:-(-length // BLOCK)], int)
        for part in (0, 1):
            x = self.val[used, :, part] * 2.0 ** self.exp[used, :, part][:, :, None, None]  # [blocks, heads, 64, D]
            got.append(x.transpose(0, 2, 1, 3).reshape(-1, x.shape[1], x.shape[3])[:length])
        return got


def sees(length, n, causal, window):
    """[n, length]: whether query i (position length - n + i) sees token j."""
    p = np.arange(length - n, length)[:, None]
    j = np.arange(length)[None, :]
    m = np.ones((n, length), bool)
    if causal:
        m &= j <= p
    if window:
        m &= np.abs(p - j) < window
    return m


def attention(q, k, v, mask, scale, chain=None):
    """q [n, H, D] on k, v [S, Hkv, D] -> out [n, H, D] and, elementwise, how far the kernel may be from it before its
    output is rounded (float32 queries); the second bound is for bf16 tensors, whose weights are rounded to bf16.

    Scores: exact products of bf16 terms, sums of at most 3 D terms and three factors in float32, so off by at most
    (3 D + 4) U times the sum of magnitudes (two fp16 terms leave 2^-22 = 4 U of a query value, with sums of 2 D terms:
    no more from D = 4 on, and below that the bound of D = 4 is taken; or 2^-39 of the row's largest); the largest such error among a row's tokens, dS, moves every weight by a
    factor within e^(+-2 dS) (weight and sum), the hardware's exp2 by 2^-22 at most (its argument is rounded, too: U
    times its size, at most 150 where a weight counts). The sums over S tokens, of three terms each, and the joining of
    waves and parts add at most (3 S + 64) U (chain: terms that are added one after another, if not S). All relative to
    sum p |v|."""
    n, H, D = q.shape
    S, Hkv, _ = k.shape
    out = np.zeros((n, H, D))
    tol = np.zeros((n, H, D))
    q = q.astype(np.float64)
    for h in range(H):
        kh, vh = k[:, h // (H // Hkv)], v[:, h // (H // Hkv)]
        s = q[:, h] @ kh.T * scale
        mag = np.abs(q[:, h]) @ np.abs(kh).T * abs(scale)
        for i in range(n):
            on = mask[i]
            if not on.any():
                continue
            x = s[i, on]
            p = np.exp(x - x.max())
            p /= p.sum()
            out[i, h] = p @ vh[on]
            ds = (3 * max(D, 4) + 4) * U * mag[i, on].max()
            ds += 2.0 ** -39 * np.abs(q[i, h]).max() * np.abs(kh[on]).sum(1).max() * abs(scale)
            rel = np.expm1(2 * ds) + 2.0 ** -22 + 2 * 150 * U + (3 * (chain or on.sum()) + 64) * U
            tol[i, h] = rel * (p @ np.abs(vh[on]))
    return out, tol
