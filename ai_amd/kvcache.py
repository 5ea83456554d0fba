"""Key/value cache in 8 bits (fa_kv_* of include/fa_rocm.h): what a program
that adds tokens one after another keeps of the tokens before them.

The reference's nn package has a float32 KVCache for its attention module;
this one holds e4m3 codes with a power-of-two scale for every 64 tokens of a
head, in blocks that sequences of any length share. Tensors are numpy arrays,
float32 or bfloat16 (uint16 bits); computation and the cache are on the GPU,
there is no CPU fallback. A shape error raises tensor.TensorError.

    cache = KVCache(kv_heads=1, head_dim=256, tokens=100_000)
    seq = cache.Add()
    cache.Append([seq], k, v, [len(k)])              # a prompt's keys and values
    out = cache.Attention([seq], q, [len(q)])        # and its queries
    cache.Append([seq], k1, v1)                      # the next token
    out1 = cache.Attention([seq], q1)
"""
from __future__ import annotations

import math

import numpy as np

from . import _native as N
from .tensor import TensorError, _call, default_context

BLOCK = N.FA_KV_BLOCK
_I32 = 2 ** 31 - 1


def _fail(msg: str):
    raise TensorError("KVCache", msg)


def _rows(x, what: str, heads: int | None, dim: int) -> np.ndarray:
    """x as float32 or bf16 [rows, heads, dim] whose rows of dim are contiguous."""
    x = np.asarray(x)
    if x.dtype != np.uint16 and x.dtype != np.float32:
        x = x.astype(np.float32)
    if x.ndim != 3 or x.shape[2] != dim or (heads is not None and x.shape[1] != heads):
        _fail(f"{what}: want [rows, {heads or 'heads'}, {dim}], got {list(x.shape)}")
    size = x.itemsize
    if x.size and (x.strides[2] != size or any(s < 0 or s % size for s in x.strides[:2])):
        x = np.ascontiguousarray(x)
    return x


def _strides(x: np.ndarray) -> tuple[int, int]:
    return (x.strides[0] // x.itemsize, x.strides[1] // x.itemsize) if x.size else (0, 0)


def _dtype(x: np.ndarray) -> int:
    return N.FA_DT_BF16 if x.dtype == np.uint16 else N.FA_DT_F32


class KVCache:
    """A pool of blocks for `tokens` tokens (in whole blocks) and the sequences that hold them."""

    def __init__(self, kv_heads: int, head_dim: int, tokens: int, *, ctx: N.Context | None = None):
        self.kv_heads, self.head_dim = int(kv_heads), int(head_dim)
        self.blocks = -(-int(tokens) // BLOCK)
        L = N.lib()
        sizes = (self.blocks, self.kv_heads, self.head_dim)
        size = L.fa_kv_codes_bytes(*sizes) if all(0 < x <= _I32 for x in sizes) else 0
        if size == 0:
            _fail(f"{kv_heads} heads of {head_dim} dims for {tokens} tokens")
        self.ctx = ctx or default_context()
        self._codes, self._scales = N.vp(), N.vp()
        N.check(self.ctx.h, L.fa_device_alloc(self.ctx.h, size, N.C.byref(self._codes)))
        rc = L.fa_device_alloc(self.ctx.h, self.blocks * self.kv_heads * 8, N.C.byref(self._scales))
        if rc != N.FA_OK:
            L.fa_device_free(self.ctx.h, self._codes)
            self._codes = N.vp()
            N.check(self.ctx.h, rc)
        self.cache = N.KvCache(self._codes, self._scales, self.blocks, self.kv_heads, self.head_dim)
        self._free = list(range(self.blocks - 1, -1, -1))
        self._tables: dict[int, list[int]] = {}
        self._lengths: dict[int, int] = {}
        self._next = 0
        N.own(self)

    def close(self) -> None:
        """Frees the device memory (also when the cache is dropped, with its context, and at interpreter exit)."""
        codes, scales = self._codes, self._scales
        self._codes, self._scales = N.vp(), N.vp()
        if codes and self.ctx.h:
            N.lib().fa_device_free(self.ctx.h, codes)
            N.lib().fa_device_free(self.ctx.h, scales)

    def __del__(self):
        try:
            self.close()
        except Exception:  # (a cache whose constructor raised has nothing to free)
            pass

    def __enter__(self):
        return self

    def __exit__(self, *exc):
        self.close()

    # ---- sequences ---------------------------------------------------------------

    def Add(self) -> int:
        """A new, empty sequence."""
        seq, self._next = self._next, self._next + 1
        self._tables[seq], self._lengths[seq] = [], 0
        return seq

    def Len(self, seq: int) -> int:
        """Tokens of a sequence."""
        self._known(seq)
        return self._lengths[seq]

    def Room(self) -> int:
        """Tokens that free blocks have room for."""
        return len(self._free) * BLOCK

    def Truncate(self, seq: int, length: int) -> None:
        """Drops the tokens from position `length` on."""
        self._known(seq)
        if not 0 <= length <= self._lengths[seq]:
            _fail(f"Truncate: length {length} of a sequence of {self._lengths[seq]}")
        table = self._tables[seq]
        used = -(-length // BLOCK)
        self._free.extend(reversed(table[used:]))
        del table[used:]
        self._lengths[seq] = length

    def Free(self, seq: int) -> None:
        """Drops a sequence."""
        self.Truncate(seq, 0)
        del self._tables[seq], self._lengths[seq]

    def _known(self, seq: int) -> None:
        if seq not in self._lengths:
            _fail(f"no sequence {seq}")

    def _counts(self, seqs, rows: int, counts, what: str) -> list[int]:
        if not self._codes:
            _fail(f"{what}: the cache is closed")
        for s in seqs:
            self._known(s)
        counts = [1] * len(seqs) if counts is None else [int(c) for c in counts]
        if len(counts) != len(seqs) or any(c < 0 for c in counts) or sum(counts) != rows:
            _fail(f"{what}: {rows} rows for {len(seqs)} sequences with counts {counts[:8]}")
        return counts

    def _batch(self, seqs, counts) -> tuple[N.KvBatch, list]:
        width = max([len(self._tables[s]) for s in seqs], default=0)
        tables = np.zeros((len(seqs), max(width, 1)), np.int32)
        for i, s in enumerate(seqs):
            tables[i, :len(self._tables[s])] = self._tables[s]
        lengths = np.array([self._lengths[s] for s in seqs], np.int32)
        cu = np.concatenate([[0], np.cumsum(counts)]).astype(np.int32)
        keep = [tables, lengths, cu]
        return N.KvBatch(tables.ctypes.data, tables.shape[1], lengths.ctypes.data, cu.ctypes.data, len(seqs),
                         int(cu[-1])), keep

    # ---- operators ----------------------------------------------------------------

    def Append(self, seqs, k, v, counts=None) -> None:
        """Adds k and v [rows, kv_heads, head_dim], counts[i] rows to sequence seqs[i] (one each by default)."""
        seqs = list(seqs)
        k, v = (_rows(x, "Append", self.kv_heads, self.head_dim) for x in (k, v))
        if len(k) != len(v) or k.dtype != v.dtype:
            _fail(f"Append: k is {list(k.shape)} {k.dtype}, v is {list(v.shape)} {v.dtype}")
        counts = self._counts(seqs, len(k), counts, "Append")
        if len(set(seqs)) != len(seqs):
            _fail("Append: a sequence is given twice")
        need = [-(-(self._lengths[s] + c) // BLOCK) - len(self._tables[s]) for s, c in zip(seqs, counts)]
        if sum(need) > len(self._free):
            _fail(f"Append: {sum(need)} blocks needed, {len(self._free)} free")
        before = {s: self._lengths[s] for s in seqs}
        try:
            for s, c, u in zip(seqs, counts, need):
                self._tables[s].extend(self._free.pop() for _ in range(u))
                self._lengths[s] += c
            batch, keep = self._batch(seqs, counts)
            _call("KVWrite", self.ctx, N.lib().fa_kv_write(
                self.ctx.h, N.C.byref(self.cache), N.C.byref(batch), _dtype(k), k.ctypes.data, *_strides(k),
                v.ctypes.data, *_strides(v)))
        except BaseException:
            for s in reversed(seqs):
                self.Truncate(s, before[s])
            raise
        del keep

    def Attention(self, seqs, q, counts=None, *, causal: bool = True, window: int = 0,
                  scale: float | None = None) -> np.ndarray:
        """softmax(scale * q . k^T) . v of q [rows, heads, head_dim], the last counts[i] tokens of each sequence, over
        the cached tokens each sees (causal: up to its own; window > 0: fewer than window positions away)."""
        seqs = list(seqs)
        q = _rows(q, "Attention", None, self.head_dim)
        counts = self._counts(seqs, len(q), counts, "Attention")
        if not 0 <= int(window) <= _I32:
            _fail(f"Attention: window {window}")
        scale = float(np.float32(1.0 / math.sqrt(self.head_dim))) if scale is None else float(scale)
        out = np.empty(q.shape, q.dtype)
        batch, keep = self._batch(seqs, counts)
        _call("KVAttention", self.ctx, N.lib().fa_kv_attention(
            self.ctx.h, N.C.byref(self.cache), N.C.byref(batch), _dtype(q), q.ctypes.data, *_strides(q), q.shape[1],
            int(bool(causal)), int(window), scale, N.ptr(out)))
        del keep
        return out

    def Read(self, seq: int, count: int | None = None, *, dtype=np.float32) -> tuple[np.ndarray, np.ndarray]:
        """Keys and values of a sequence's last count tokens (all by default), [count, kv_heads, head_dim]."""
        self._known(seq)
        count = self._lengths[seq] if count is None else int(count)
        if not 0 <= count <= self._lengths[seq]:
            _fail(f"Read: {count} tokens of a sequence of {self._lengths[seq]}")
        self._counts([seq], count, [count], "Read")
        k = np.empty((count, self.kv_heads, self.head_dim), np.dtype(dtype))
        if k.dtype not in (np.float32, np.uint16):
            _fail(f"Read: dtype {k.dtype}")
        v = np.empty_like(k)
        batch, keep = self._batch([seq], [count])
        _call("KVRead", self.ctx, N.lib().fa_kv_read(self.ctx.h, N.C.byref(self.cache), N.C.byref(batch), _dtype(k),
                                                     N.ptr(k), N.ptr(v)))
        del keep
        return k, v
