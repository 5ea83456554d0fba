"""Products with weights held in 8 bits (fa_f8_*, fa_matmul_f8 of
include/fa_rocm.h): beside tensor.MatMulFused, for layers that are bound by
reading their weights or by the matrix units.

A matrix is held on the GPU as e4m3 codes with a power of two for each 128
columns of a row; the left operand is rounded by the same rule on the way.
Tensors are numpy arrays, float32 or bfloat16 (uint16 bits); there is no CPU
fallback. A shape error raises tensor.TensorError.

    w = F8Matrix(weight)                       # [out, in]
    y = w.MatMul(x, Fused(Act=GELUAct))        # x [rows, in] -> [rows, out]
"""
from __future__ import annotations

import numpy as np

from . import _native as N
from .tensor import Fused, TensorError, _call, default_context

_OP = "MatMulF8"


def _fail(msg: str):
    raise TensorError(_OP, msg)


def _matrix(x, what: str) -> np.ndarray:
    """x as float32 or bf16 (uint16), 2-D, rows contiguous."""
    x = np.asarray(x)
    if x.dtype != np.uint16 and x.dtype != np.float32:
        x = x.astype(np.float32)
    if x.ndim != 2:
        _fail(f"{what}: want a 2-D array, got {list(x.shape)}")
    if x.size and (x.strides[1] != x.itemsize or x.strides[0] < x.shape[1] * x.itemsize or x.strides[0] % x.itemsize):
        x = np.ascontiguousarray(x)
    return x


def _ld(x: np.ndarray) -> int:
    return x.strides[0] // x.itemsize if x.size and x.shape[0] > 1 else max(x.shape[1], 1)


def _dtype(dtype) -> int:
    return N.FA_DT_BF16 if dtype == np.uint16 else N.FA_DT_F32


class F8Matrix:
    """w [n, k] (float32, or bfloat16 as uint16 bits) in 8 bits in device memory."""

    def __init__(self, w, *, ctx: N.Context | None = None):
        self._codes, self._scales = N.vp(), N.vp()
        w = _matrix(w, "F8Matrix")
        self.n, self.k = w.shape
        L = N.lib()
        sizes = [f(self.n, self.k) for f in (L.fa_f8_codes_bytes, L.fa_f8_scales_bytes)]
        if w.size and not all(sizes):
            _fail(f"F8Matrix: {list(w.shape)} is larger than a matrix can be")
        self.ctx = ctx or default_context()
        N.own(self)
        for p, size in zip((self._codes, self._scales), sizes):
            N.check(self.ctx.h, L.fa_device_alloc(self.ctx.h, size, N.C.byref(p)))
        self.matrix = N.F8Matrix(self._codes, self._scales, self.n, self.k)
        _call("F8Write", self.ctx, L.fa_f8_write(self.ctx.h, N.C.byref(self.matrix), _dtype(w.dtype), w.ctypes.data,
                                                 _ld(w)))

    def close(self) -> None:
        """Frees the device memory (also when the matrix is dropped, with its context, and at interpreter exit)."""
        codes, scales = self._codes, self._scales
        self._codes, self._scales = N.vp(), N.vp()
        for p in (codes, scales):
            if p and self.ctx.h:
                N.lib().fa_device_free(self.ctx.h, p)

    def __del__(self):
        try:
            self.close()
        except Exception:  # (a matrix whose constructor raised has nothing to free)
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    def _open(self):
        if not self._codes:
            _fail("the matrix is closed")

    def Values(self, *, dtype=np.float32) -> np.ndarray:
        """The values that the matrix holds, [n, k]."""
        self._open()
        out = np.empty((self.n, self.k), np.dtype(dtype))
        if out.dtype not in (np.float32, np.uint16):
            _fail(f"Values: dtype {out.dtype}")
        _call("F8Read", self.ctx, N.lib().fa_f8_read(self.ctx.h, N.C.byref(self.matrix), _dtype(out.dtype), N.ptr(out),
                                                     max(self.k, 1)))
        return out

    def MatMul(self, x, f: Fused | None = None, *, dtype=None) -> np.ndarray:
        """x [m, k] times the matrix's transpose, [m, n], with MatMulFused's epilogue f; dtype: float32 or uint16
        (bfloat16), x's by default."""
        self._open()
        x = _matrix(x, "MatMul")
        if x.shape[1] != self.k:
            _fail(f"MatMul: [{x.shape[0]} x {x.shape[1]}] times the transpose of [{self.n} x {self.k}]")
        m, n = x.shape[0], self.n
        out = np.empty((m, n), x.dtype if dtype is None else np.dtype(dtype))
        if out.dtype not in (np.float32, np.uint16):
            _fail(f"MatMul: dtype {out.dtype}")
        e, keep = None, []
        if f is not None:
            def operand(a, shape, name):
                if a is None:
                    return None
                a = np.ascontiguousarray(a, np.float32)
                if a.shape != shape:
                    _fail(f"MatMul: {name} has shape {list(a.shape)}, want {list(shape)}")
                keep.append(a)
                return a.ctypes.data
            e = N.Epilogue(operand(f.Bias, (n,), "Bias"), operand(f.RowScale, (m,), "RowScale"), int(f.Act),
                           operand(f.Mul, (m, n), "Mul"), max(n, 1), operand(f.Residual, (m, n), "Residual"), max(n, 1))
        _call(_OP, self.ctx, N.lib().fa_matmul_f8(
            self.ctx.h, m, _dtype(x.dtype), x.ctypes.data, _ld(x), N.C.byref(self.matrix),
            None if e is None else N.C.byref(e), _dtype(out.dtype), N.ptr(out), max(n, 1)))
        del keep
        return out
