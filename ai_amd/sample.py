"""The next token of each row of logits (fa_sample of include/fa_rocm.h), for
programs that add tokens one after another (kvcache.KVCache).

    ids, logp = Sample(logits, rng.random(len(logits)), temperature=0.7, top_k=50, top_p=0.9)
"""
from __future__ import annotations

import numpy as np

from . import _native as N
from .tensor import TensorError, _call, default_context


def Sample(logits, u, *, temperature=None, top_k=None, top_p=None, min_p=None,
           ctx: N.Context | None = None) -> tuple[np.ndarray, np.ndarray]:
    """Draws a token from each row of logits [rows, vocab] (float32, or bfloat16 as uint16 bits) with the row's number u
    in [0, 1): int32 ids and the float32 logs of their shares of what the filters left. Settings are numbers, or arrays
    [rows]; temperature 0 takes the largest logit, top_k 0 and top_p 1 leave all."""
    logits = np.asarray(logits)
    if logits.dtype != np.uint16 and logits.dtype != np.float32:
        logits = logits.astype(np.float32)
    if logits.ndim != 2 or logits.shape[1] < 1:
        raise TensorError("Sample", f"want logits [rows, vocab], got {list(logits.shape)}")
    rows, vocab = logits.shape
    size = logits.itemsize
    if rows and (logits.strides[1] != size or logits.strides[0] < vocab * size or logits.strides[0] % size):
        logits = np.ascontiguousarray(logits)
    ld = logits.strides[0] // size if rows > 1 else vocab

    def setting(x, name, dtype):
        if x is None:
            return None
        x = np.asarray(x)
        if dtype == np.int32:
            if x.dtype.kind not in "iu":
                raise TensorError("Sample", f"{name} is {x.dtype}, not a whole number")
            x = np.clip(x, 0, vocab)
        if x.ndim == 0:
            x = np.full(rows, x)
        if x.shape != (rows,):
            raise TensorError("Sample", f"{name} has shape {list(x.shape)}, want [{rows}]")
        return np.ascontiguousarray(x, dtype)

    if u is None:
        raise TensorError("Sample", "no numbers u")
    below = np.asarray(u) < 1
    u = setting(u, "u", np.float32)
    u = np.where(below & (u == 1), np.float32(1 - 2.0 ** -24), u)  # (float64 numbers just below 1 round to it)
    got = [setting(temperature, "temperature", np.float32), setting(top_k, "top_k", np.int32),
           setting(top_p, "top_p", np.float32), setting(min_p, "min_p", np.float32)]
    s = N.Sampling(*(None if x is None else x.ctypes.data for x in got))
    ids, logp = np.empty(rows, np.int32), np.empty(rows, np.float32)
    ctx = ctx or default_context()
    _call("Sample", ctx, N.lib().fa_sample(
        ctx.h, rows, vocab, N.FA_DT_BF16 if logits.dtype == np.uint16 else N.FA_DT_F32, logits.ctypes.data, ld,
        N.C.byref(s), u.ctypes.data, N.ptr(ids), N.ptr(logp)))
    return ids, logp
