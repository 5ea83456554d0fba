"""A decoding step's operators as a program runs them together: a product with
8-bit weights, the rotary append to the key/value cache, attention over it, the
products behind it, a drawn token. Every stage against its 64-bit definition from
what the stage before gave; the step captured and replayed; two contexts at once."""
import ctypes as C

import numpy as np
import pytest

import decode_oracle as O
import kv_lib as K
import kv_oracle as KO
import test_gpu_f8 as F
import test_gpu_kvcache as G
import test_gpu_kvrope as R
from ai_amd import _native as N
from ai_amd import synth as S
from ai_amd.f8 import F8Matrix
from ai_amd.kvcache import KVCache
from ai_amd.sample import Sample

pytestmark = pytest.mark.gpu
H, HKV, D, DM, VOCAB = 6, 2, 64, 200, 1500
BASE, DIMS, SCALE = 1e6, 48, 0.125
QKV = (H + 2 * HKV) * D


class Step:
    """Buffers and weights of a step; run() is the step, with the caller's work or without."""

    def __init__(self, ctx, r, lengths, dtype):
        self.ctx, self.dtype, self.lengths = ctx, dtype, lengths
        self.B = len(lengths)
        self.cache, self.ref, self.tables = G.fill(ctx, r, lengths, HKV, D, dtype, extra=4, width=20)
        spare = [i for i in range(self.cache.blocks) if i not in self.tables]
        for i, l in enumerate(lengths):  # room for three more tokens
            if (l + 2) // 64 > (l - 1) // 64:
                self.tables[i, (l + 2) // 64] = spare.pop()
        self.batch = K.Batch(ctx, self.tables, [l + 1 for l in lengths], np.arange(self.B + 1))
        self.mats = {n: F.Held(ctx, *shape).write((r.standard_normal(shape) / np.sqrt(shape[1])).astype(np.float32))
                     for n, shape in (("qkv", (QKV, DM)), ("o", (DM, H * D)), ("vocab", (VOCAB, DM)))}
        size = 2 if dtype == "bf16" else 4
        self.np = F.NP[dtype]
        self.bufs = {n: K.Buf(ctx, nbytes=self.B * k * s, fill=0x5A) for n, k, s in (
            ("x", DM, size), ("res", DM, 4), ("qkv", QKV, size), ("q", H * D, size), ("att", H * D, size), ("y", DM, size),
            ("logits", VOCAB, 4), ("u", 1, 4), ("temperature", 1, 4), ("top_p", 1, 4), ("top_k", 1, 4), ("ids", 1, 4),
            ("logp", 1, 4))}
        L = N.lib()
        self.work = {}
        for n, m in self.mats.items():
            need = C.c_size_t(0)
            N.check(ctx.h, L.fa_matmul_f8_work(self.B, C.byref(m.w), C.byref(need)))
            self.work[n] = need.value
        need = C.c_size_t(0)
        N.check(ctx.h, L.fa_kv_attention_work(C.byref(self.cache.c), C.byref(self.batch.b), H, C.byref(need)))
        self.work["attention"] = need.value
        N.check(ctx.h, L.fa_sample_work(self.B, VOCAB, C.byref(need)))
        self.work["sample"] = need.value
        # one buffer for all: calls of one stream use it in turn
        self.space = K.Buf(ctx, nbytes=max(*self.work.values(), 16), fill=0xFF)

    def put(self, r):
        x = G.make(r, (self.B, DM), self.dtype)
        self.bufs["x"].put(x)
        self.bufs["res"].put(r.standard_normal((self.B, DM)).astype(np.float32))
        self.bufs["u"].put(r.random(self.B).astype(np.float32))
        self.bufs["temperature"].put(r.choice([0.0, 0.7, 1.3], self.B).astype(np.float32))
        self.bufs["top_p"].put(r.choice([0.5, 0.9, 1.0], self.B).astype(np.float32))
        self.bufs["top_k"].put(r.choice([0, 3, 50], self.B).astype(np.int32))

    def matmul(self, name, a, lda, c, cdt, work, residual=None):
        m = self.mats[name]
        e = N.Epilogue(None, None, 0, None, m.n, residual, m.n)
        return N.lib().fa_matmul_f8_dev(self.ctx.h, self.B, F.DT[self.dtype], self.bufs[a].p, lda, C.byref(m.w),
                                        C.byref(e) if residual else None, F.DT[cdt], self.bufs[c].p, m.n,
                                        self.space.p if work else None, self.work[name] if work else 0)

    def calls(self, work):
        """The step's calls in order."""
        L, h, b, size = N.lib(), self.ctx.h, self.bufs, self.np().itemsize
        rope = N.KvRope(BASE, DIMS, None)
        dt = F.DT[self.dtype]
        yield self.matmul("qkv", "x", DM, "qkv", self.dtype, work)
        q, k, v = (b["qkv"].p.value + i * D * size for i in (0, H, H + HKV))
        yield L.fa_kv_write_rope_dev(h, C.byref(self.cache.c), C.byref(self.batch.b), C.byref(rope), dt, q, QKV, D, H,
                                     b["q"].p, k, QKV, D, v, QKV, D)
        yield L.fa_kv_attention_dev(h, C.byref(self.cache.c), C.byref(self.batch.b), dt, b["q"].p, H * D, D, H, 1, 0, SCALE,
                                    b["att"].p, self.space.p if work else None, self.work["attention"] if work else 0)
        yield self.matmul("o", "att", H * D, "y", self.dtype, work, b["res"].p)
        yield self.matmul("vocab", "y", DM, "logits", "f32", work)
        s = N.Sampling(b["temperature"].p, b["top_k"].p, b["top_p"].p, None)
        yield L.fa_sample_dev(h, self.B, VOCAB, N.FA_DT_F32, b["logits"].p, VOCAB, C.byref(s), b["u"].p, b["ids"].p,
                              b["logp"].p, self.space.p if work else None, self.work["sample"] if work else 0)

    def run(self, work):
        for rc in self.calls(work):
            N.check(self.ctx.h, rc)

    def state(self):
        kind = {"qkv": (QKV, self.np), "q": (H * D, self.np), "att": (H * D, self.np), "y": (DM, self.np),
                "logits": (VOCAB, np.float32), "ids": (1, np.int32), "logp": (1, np.float32)}
        return {n: self.bufs[n].get((self.B, k), t).copy() for n, (k, t) in kind.items()}

    def free(self):
        for x in (*self.bufs.values(), *self.mats.values(), self.space, self.batch, self.cache):
            x.free()


def same(a, b):
    for n in a:
        np.testing.assert_array_equal(a[n].view(np.uint8), b[n].view(np.uint8), err_msg=n)


@pytest.mark.parametrize("work", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_every_stage(ctx, dtype, work):
    r = G.rng(61)
    lengths = [1, 63, 64, 300, 1000]  # (new tokens at the end of a block and at the start of one)
    s = Step(ctx, r, lengths, dtype)
    B, bf = s.B, dtype == "bf16"
    for turn in range(3):
        s.put(r)
        s.run(work)
        ctx.sync()
        got = s.state()
        x = s.bufs["x"].get((B, DM), s.np)
        held = {n: m.read().astype(np.float64) for n, m in s.mats.items()}

        def near(c, a, name, c_bf16, residual=None):
            want, tol = O.product(K.wide(a).astype(np.float64), held[name], c_bf16, residual=residual)
            d = np.abs(K.wide(c).astype(np.float64) - want)
            assert (d <= tol).all(), (name, (d / tol).max())

        near(got["qkv"], x, "qkv", bf)
        qkv = got["qkv"].reshape(B, H + 2 * HKV, D)
        q, k, v = qkv[:, :H], qkv[:, H:H + HKV], qkv[:, H + HKV:]
        now = [l + 1 + turn for l in lengths]
        pos = np.array(now) - 1
        R.check_queries(got["q"].reshape(B, H, D), q, pos, BASE, DIMS)
        s.ref.write(s.tables, now, np.arange(B + 1), O.rotate(K.wide(k), pos, BASE, DIMS), K.wide(v))
        R.check_cache(s.cache, s.ref, D)
        for i in range(B):
            kk, vv = s.ref.tokens(s.tables[i], now[i])
            one = K.wide(got["q"][i].reshape(1, H, D))
            sees = KO.sees(now[i], 1, True, 0)
            want, tol = KO.attention(one, kk, vv, sees, SCALE)
            if bf:
                tol = tol + G.BF * KO.attention(one, kk, np.abs(vv), sees, SCALE)[0]
            G.close(got["att"][i].reshape(1, H, D), want, tol, f"sequence {i}")
        near(got["y"], got["att"], "o", bf, s.bufs["res"].get((B, DM), np.float32).astype(np.float64))
        near(got["logits"], got["y"], "vocab", False)
        for i in range(B):
            one = {n: s.bufs[n].get((B,), t)[i] for n, t in (("temperature", np.float32), ("top_k", np.int32),
                                                            ("top_p", np.float32))}
            want, lp = O.sample(got["logits"][i], s.bufs["u"].get((B,), np.float32)[i], **one)
            assert got["ids"][i, 0] == want
            assert abs(float(got["logp"][i, 0]) - lp) <= 2.0 ** -24 * abs(lp) + 1e-9
        # the next turn's tokens follow (every sequence stays in a block that its table has)
        s.batch.bufs[1].put(np.array([l + 1 for l in now], np.int32))
    s.free()


def hip():
    h = C.CDLL("libamdhip64.so")
    h.hipStreamBeginCapture.argtypes = [C.c_void_p, C.c_int]
    h.hipStreamEndCapture.argtypes = [C.c_void_p, C.POINTER(C.c_void_p)]
    h.hipGraphInstantiate.argtypes = [C.POINTER(C.c_void_p), C.c_void_p, C.c_void_p, C.c_void_p, C.c_size_t]
    h.hipGraphLaunch.argtypes = [C.c_void_p, C.c_void_p]
    h.hipGraphDestroy.argtypes = [C.c_void_p]
    h.hipGraphExecDestroy.argtypes = [C.c_void_p]
    return h


@pytest.mark.parametrize("eager_first", [False, True])
@pytest.mark.parametrize("dtype", ["f32", "bf16"])
def test_captured_step(ctx, dtype, eager_first):
    """A captured step on the caller's work, replayed with new contents and lengths between eager steps, equals them;
    calls without work are refused under capture, also where the context's own has grown before."""
    h, r = hip(), G.rng(62)
    lengths = [5, 63, 64, 700]
    s = Step(ctx, r, lengths, dtype)
    s.put(r)
    if eager_first:
        s.run(False)
        ctx.sync()
    graph, ex = C.c_void_p(), C.c_void_p()
    ctx.sync()
    assert h.hipStreamBeginCapture(ctx.stream, 2) == 0
    refused = []
    for name, rc in zip(("qkv", "rope", "attention", "o", "vocab", "sample"), s.calls(False)):
        refused.append((name, rc, N.lib().fa_last_error(ctx.h) if rc else b""))
    assert h.hipStreamEndCapture(ctx.stream, C.byref(graph)) == 0
    h.hipGraphDestroy(graph)
    assert h.hipStreamBeginCapture(ctx.stream, 2) == 0
    codes = list(s.calls(True))
    assert h.hipStreamEndCapture(ctx.stream, C.byref(graph)) == 0
    assert codes == [0] * 6
    for name, rc, text in refused:
        if name == "rope" or s.work[name] == 0:
            assert rc == 0, (name, rc, text)
        elif name != "attention":  # (which may need less than it says for any lengths)
            assert rc == N.FA_ERR_STATE and b"captured" in text, (name, rc, text)
    assert s.work["sample"] > 0
    assert h.hipGraphInstantiate(C.byref(ex), graph, None, None, 0) == 0
    for turn in range(4):
        s.put(r)
        s.batch.bufs[1].put(np.array([l + 1 - turn for l in lengths], np.int32))
        before = s.cache.state()
        assert h.hipGraphLaunch(ex, ctx.stream) == 0
        ctx.sync()
        got, after = s.state(), s.cache.state()
        s.cache.codes.put(before[0])
        s.cache.scales.put(before[1])
        s.run(turn % 2 == 0)
        ctx.sync()
        same(got, s.state())
        for x, y in zip(after, s.cache.state()):
            np.testing.assert_array_equal(x, y)
    h.hipGraphExecDestroy(ex)
    h.hipGraphDestroy(graph)
    s.free()


def test_two_contexts_at_once(ctx):
    """Steps of two contexts, their streams side by side, give what each gives alone."""
    other = N.Context(0)
    a, b = Step(ctx, G.rng(63), [10, 700, 64], "bf16"), Step(other, G.rng(64), [900, 3], "f32")
    want = []
    for s in (a, b):
        s.put(G.rng(65))
        s.state0 = s.cache.state()
        s.run(False)
        s.ctx.sync()
        want.append(s.state())
        s.cache.codes.put(s.state0[0])
        s.cache.scales.put(s.state0[1])
    for turn in range(10):
        a.run(turn % 2 == 0)
        b.run(turn % 2 == 1)
    for s, w in zip((a, b), want):
        s.ctx.sync()
        same(s.state(), w)
    a.free()
    b.free()
    other.close()


def test_from_python(ctx):
    """The same step through F8Matrix, KVCache and Sample: a prompt, then tokens one by one."""
    r = G.rng(66)
    w = {n: (r.standard_normal(shape) / np.sqrt(shape[1])).astype(np.float32)
         for n, shape in (("qkv", (QKV, DM)), ("o", (DM, H * D)), ("vocab", (VOCAB, DM)))}
    m = {n: F8Matrix(x, ctx=ctx) for n, x in w.items()}
    emb = r.standard_normal((VOCAB, DM)).astype(np.float32)
    with KVCache(HKV, D, 400, ctx=ctx) as cache:
        seq = cache.Add()
        tokens = r.integers(0, VOCAB, 70).tolist()
        new, kept = list(tokens), []
        for turn in range(4):
            x = emb[new]
            qkv = m["qkv"].MatMul(x).reshape(len(new), H + 2 * HKV, D)
            q = cache.AppendRoPE([seq], qkv[:, :H], qkv[:, H:H + HKV], qkv[:, H + HKV:], [len(new)], base=BASE, dims=DIMS)
            pos = np.arange(len(tokens) - len(new), len(tokens))
            R.check_queries(q, np.ascontiguousarray(qkv[:, :H]), pos, BASE, DIMS)
            kept.append(O.rotate(qkv[:, H:H + HKV], pos, BASE, DIMS))
            att = cache.Attention([seq], q, [len(new)], causal=True, scale=SCALE)
            y = x[-1:] + m["o"].MatMul(np.ascontiguousarray(att[-1:].reshape(1, H * D)))
            logits = m["vocab"].MatMul(y)
            u = np.array([r.random()], np.float32)
            ids, logp = Sample(logits, u, temperature=0.8, top_k=40, top_p=0.9, ctx=ctx)
            want, lp = O.sample(logits[0], u[0], np.float32(0.8), 40, np.float32(0.9))
            assert ids[0] == want and abs(float(logp[0]) - lp) <= 2.0 ** -24 * abs(lp) + 1e-9
            new = [int(ids[0])]
            tokens += new
        assert cache.Len(seq) == len(tokens) - 1
        k, _ = cache.Read(seq)
        full = np.concatenate(kept)
        assert k.shape == full.shape
        # a block's scale is at most twice what its largest value needs, and codes are off by half a step: 2^-4 of the
        # value, and 2^-10 of the scale below the normal codes, where 448 / 2 of the scale is below the largest value
        for at in range(0, len(k), 64):
            rows = slice(at, at + 64)
            top = np.abs(full[rows]).max((0, 2), keepdims=True)
            assert (np.abs(k[rows] - full[rows]) <= 2.0 ** -3 * np.abs(full[rows]) + top * 2.0 ** -8).all()
    for x in m.values():
        x.close()
