"""The work of the key/value cache held in 8 bits, through the C ABI of
include/fa_rocm.h: keys and values quantised as they are written and read
back, and attention of new tokens over the cached ones.

A cache is a pool of blocks of 64 tokens. Each block holds, for every
key/value head, the e4m3 codes of 64 keys and 64 values and one power of two
for the keys and one for the values: a value is code * scale. A sequence is a
list of blocks (its row of the block table) and a length. A batch's rows
cu[b] .. cu[b + 1] are the last tokens of sequence b.

Writing: a block that receives new tokens takes the smallest scale 2^e
(-80 <= e <= 120) under which the largest finite magnitude among them is at
most 448, or its own where tokens already in the block need a larger one; if
it grows, the codes already there are rounded again. Rounding is to nearest,
ties to even. Attention: softmax(scale * q . k) . v over the tokens a query
sees: those up to its own position (causal) or all of the sequence, and with
a window only those fewer than window positions away.

listed() are the fixed cases, draw(rng) another one of the same ranges;
prepare / run / work / exact take one case each. With own the framework's
calls are made, else the plain forms below.
"""
import math

import torch

own = False

DEV = "cuda"
BLOCK = 64
BF16, F32 = "bf16", "f32"


def listed():
    return [
        # One user's next token at this repository's own head shape (3 query heads on one of 256 dims): pure latency.
        dict(name="next token 1x1000", kind="attend", dtype=F32, B=1, H=3, Hkv=1, D=256, lo=1000, hi=1000, nlo=1,
             nhi=1, causal=True, window=0),
        # A small serving batch with ragged contexts, grouped queries: the ordinary decoding step.
        dict(name="next token 16x2048", kind="attend", dtype=BF16, B=16, H=32, Hkv=8, D=128, lo=200, hi=2048, nlo=1,
             nhi=1, causal=True, window=0),
        # A full serving batch with long ragged contexts: bound by reading the cache.
        dict(name="next token 64x8192", kind="attend", dtype=BF16, B=64, H=32, Hkv=8, D=128, lo=1024, hi=8192, nlo=1,
             nhi=1, causal=True, window=0),
        # One very long context: the token axis has to be split over the card.
        dict(name="next token 1x131072", kind="attend", dtype=BF16, B=1, H=32, Hkv=8, D=128, lo=131072, hi=131072,
             nlo=1, nhi=1, causal=True, window=0),
        # A sliding-window layer: a few drafted tokens each, only the window of a long cache is read.
        dict(name="drafts 32x6000 window", kind="attend", dtype=BF16, B=32, H=8, Hkv=2, D=256, lo=600, hi=6000, nlo=2,
             nhi=5, causal=True, window=512),
        # The next chunk of long prompts against what is cached of them.
        dict(name="chunk 4x512 on 8192", kind="attend", dtype=BF16, B=4, H=32, Hkv=8, D=128, lo=6000, hi=8704,
             nlo=384, nhi=512, causal=True, window=0),
        # Whole passages in float32 at this repository's own head shape, ragged.
        dict(name="prompt 8x1100 f32", kind="attend", dtype=F32, B=8, H=3, Hkv=1, D=256, lo=300, hi=1100, nlo=300,
             nhi=1100, causal=True, window=0),
        # One long prompt from its first token: the largest product.
        dict(name="prompt 1x8192", kind="attend", dtype=BF16, B=1, H=32, Hkv=8, D=128, lo=8192, hi=8192, nlo=8192,
             nhi=8192, causal=True, window=0),
        # The cache side of a decoding step: one token each, into blocks that hold others, and back.
        dict(name="store 64x1", kind="store", dtype=F32, B=64, H=8, Hkv=8, D=128, lo=100, hi=2000, nlo=1, nhi=1,
             causal=True, window=0),
        # The cache side of prompts: whole blocks and ragged ends, bound by memory.
        dict(name="store prompts 16x2048", kind="store", dtype=BF16, B=16, H=32, Hkv=8, D=128, lo=700, hi=2048,
             nlo=700, nhi=2048, causal=True, window=0),
        # Sequences read back whole, in float32, as a program does that hands them to another operator.
        dict(name="read 32x2000 f32", kind="read", dtype=F32, B=32, H=8, Hkv=8, D=64, lo=500, hi=2000, nlo=500,
             nhi=2000, causal=True, window=0),
        # The last hundred tokens of two conversations, to be looked at or moved: latency.
        dict(name="read 2x100", kind="read", dtype=BF16, B=2, H=32, Hkv=8, D=128, lo=150, hi=333, nlo=90, nhi=100,
             causal=True, window=0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    most_bytes, most_flops = 5e8, 5e11
    while True:
        kind = rng.choice(["attend"] * 6 + ["store"] * 2 + ["read"])
        dtype = rng.choice([BF16, BF16, F32])
        Hkv = rng.choice([1, 1, 2, 4, 8])
        G = rng.choice([1, 2, 3, 4, 4, 8])
        D = rng.choice([64, 64, 128, 128, 256, 256, 40, 80, 96, 192, 512])
        hi = _log(rng, 2, 60000)
        lo = max(1, int(hi * rng.choice([0.1, 0.5, 0.9])))
        B = _log(rng, 1, 96)
        what = rng.choice(["token", "token", "few", "chunk", "prompt"]) if kind != "read" else "prompt"
        if what == "token":
            nlo = nhi = 1
        elif what == "few":
            nlo, nhi = 1, rng.randint(2, 12)
        elif what == "chunk":
            nhi = _log(rng, 16, 1024)
            nlo = max(1, nhi // 2)
        else:
            nlo, nhi = lo, hi
        causal = rng.random() < 0.85
        window = 0 if rng.random() < 0.7 else _log(rng, 16, 2000)
        case = dict(kind=kind, dtype=dtype, B=B, H=Hkv * G, Hkv=Hkv, D=D, lo=lo, hi=hi, nlo=nlo, nhi=nhi,
                    causal=causal, window=window)
        w = work(case)
        lens, ns = _sizes(case)
        plain = 4 * B * Hkv * max(lens) * D + 4 * B * max(ns) * Hkv * G * max(lens)  # what the plain form holds
        if w["bytes"] <= most_bytes and w["flops"] * (4 if dtype == F32 else 1) <= most_flops and plain < 6e9:
            return case


# ---- a batch's sizes: the same for each seed, in another order -----------------------


def _spread(lo, hi, B):
    """B whole numbers over lo .. hi, hi among them."""
    return [hi - int((hi - lo) * ((i * 0.6180339887) % 1.0)) for i in range(B)]


def _sizes(case):
    lens = _spread(case["lo"], case["hi"], case["B"])
    if (case["nlo"], case["nhi"]) == (case["lo"], case["hi"]):
        return lens, list(lens)
    ns = _spread(case["nlo"], case["nhi"], case["B"])
    return lens, [min(n, l) for n, l in zip(ns, lens)]


def _pairs(case, length, n):
    """Query-token pairs of a sequence of which the last n tokens ask."""
    w = case["window"]
    first = length - n
    if case["causal"]:
        if not w:
            return n * first + n * (n + 1) // 2
        full = max(0, min(n, length - max(first, w - 1)))  # queries that see w tokens
        rest = n - full
        return full * w + rest * first + rest * (rest + 1) // 2
    if not w:
        return n * length
    return sum(min(length - 1, p + w - 1) - max(0, p - w + 1) + 1 for p in range(first, length))


def _seen(case, length, n):
    """Tokens of a sequence that some query sees."""
    return length if not case["window"] else min(length, n + case["window"] - 1)


def work(case):
    D, H, Hkv = case["D"], case["H"], case["Hkv"]
    size = 4 if case["dtype"] == F32 else 2
    lens, ns = _sizes(case)
    rows = sum(ns)
    if case["kind"] == "attend":
        seen = sum(_seen(case, l, n) for l, n in zip(lens, ns))
        pairs = sum(_pairs(case, l, n) for l, n in zip(lens, ns))
        return {"bytes": seen * Hkv * 2 * (D + 4 / BLOCK) + 2 * rows * H * D * size, "flops": 4 * pairs * H * D}
    per = rows * Hkv * D * 2
    if case["kind"] == "read":
        return {"bytes": per * (1 + size), "flops": per}
    return {"bytes": per * (size + 1 + 1 + size), "flops": 3 * per}


# ---- inputs ------------------------------------------------------------------------


def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 1000003 + salt)
    return g


def _dtype(case):
    return torch.float32 if case["dtype"] == F32 else torch.bfloat16


def _keys_values(g, case, rows):
    """Keys with a few strong channels, as rotary models have them, and values whose magnitude differs by token."""
    Hkv, D = case["Hkv"], case["D"]
    k = torch.randn(rows, Hkv, D, generator=g, device=DEV)
    strong = (torch.rand(Hkv, D, generator=g, device=DEV) < 0.03).float()
    k = k * (1 + 5 * strong) + 2 * strong
    v = torch.randn(rows, Hkv, D, generator=g, device=DEV)
    v = v * torch.exp(0.7 * torch.randn(rows, 1, 1, generator=g, device=DEV))
    return k.to(_dtype(case)), v.to(_dtype(case))


def prepare(case, seed):
    lens, ns = _sizes(case)
    order = torch.randperm(case["B"], generator=torch.Generator().manual_seed(seed)).tolist()
    lens, ns = [lens[i] for i in order], [ns[i] for i in order]
    g = _gen(seed, 1)
    Hkv, D = case["Hkv"], case["D"]
    width = -(-max(lens) // BLOCK)
    used = [-(-l // BLOCK) for l in lens]
    blocks = sum(used) + 3
    perm = torch.randperm(blocks, generator=g, device=DEV).to(torch.int32)
    tables = torch.zeros(case["B"], width, dtype=torch.int32, device=DEV)
    at = 0
    for b, u in enumerate(used):
        tables[b, :u] = perm[at:at + u]
        at += u
    padded = -(-D // 64) * 64

    def ints(v):
        return torch.tensor(v, dtype=torch.int32, device=DEV)

    def cu(v):
        return ints([sum(v[:i]) for i in range(len(v) + 1)])

    st = dict(case=case, codes=torch.zeros(blocks, Hkv, 2, 64 * padded, dtype=torch.uint8, device=DEV),
              scales=torch.zeros(blocks, Hkv, 2, device=DEV), tables=tables, lengths=ints(lens), cu=cu(ns),
              rows=sum(ns), most=max(ns))
    # what the sequences hold before the call; for store cases without the new tokens
    old = lens if case["kind"] != "store" else [l - n for l, n in zip(lens, ns)]
    k, v = _keys_values(g, case, sum(old))
    _plain_write(dict(st, lengths=ints(old), cu=cu(old), rows=sum(old), k=k, v=v))
    del k, v
    if case["kind"] == "store":
        st["k"], st["v"] = _keys_values(g, case, st["rows"])
    if case["kind"] == "attend":
        st["q"] = torch.randn(st["rows"], case["H"], D, generator=g, device=DEV).to(_dtype(case))
        st["out"] = torch.empty_like(st["q"])
    else:
        st["k_back"] = torch.empty(st["rows"], Hkv, D, dtype=_dtype(case), device=DEV)
        st["v_back"] = torch.empty_like(st["k_back"])
    torch.cuda.synchronize()  # the inputs come from torch's stream, a context's calls run on its own
    return st


# ---- the framework's calls -------------------------------------------------------------

_ctx = None


def _arguments(st):
    """The context and the call's descriptors, which a program keeps."""
    global _ctx
    from ai_amd import _native as N
    if _ctx is None:
        _ctx = N.Context(0)
    if "args" not in st:
        c = st["case"]
        cache = N.KvCache(st["codes"].data_ptr(), st["scales"].data_ptr(), st["codes"].shape[0], c["Hkv"], c["D"])
        batch = N.KvBatch(st["tables"].data_ptr(), st["tables"].shape[1], st["lengths"].data_ptr(),
                          st["cu"].data_ptr(), c["B"], st["rows"])
        st["args"] = (N, N.lib(), N.C.byref(cache), N.C.byref(batch), N.FA_DT_F32 if c["dtype"] == F32 else N.FA_DT_BF16)
    return _ctx, st["args"]


def _own_run(st):
    c = st["case"]
    ctx, (N, L, cache, batch, dt) = _arguments(st)
    H, Hkv, D = c["H"], c["Hkv"], c["D"]
    if c["kind"] == "attend":
        N.check(ctx.h, L.fa_kv_attention_dev(ctx.h, cache, batch, dt, st["q"].data_ptr(), H * D, D, H, c["causal"],
                                             c["window"], 1 / math.sqrt(D), st["out"].data_ptr(), None, 0))
        return st["out"]
    if c["kind"] == "store":
        N.check(ctx.h, L.fa_kv_write_dev(ctx.h, cache, batch, dt, st["k"].data_ptr(), Hkv * D, D, st["v"].data_ptr(),
                                         Hkv * D, D))
    N.check(ctx.h, L.fa_kv_read_dev(ctx.h, cache, batch, dt, st["k_back"].data_ptr(), st["v_back"].data_ptr()))
    return {"keys": st["k_back"], "values": st["v_back"], "scales": st["scales"]}


# ---- the plain forms -----------------------------------------------------------------


def _places(st):
    """Of every row: its sequence, position, block and place in the block."""
    row = torch.arange(st["rows"], device=DEV)
    seq = torch.searchsorted(st["cu"][1:].long(), row, right=True)
    pos = st["lengths"].long()[seq] - st["cu"].long()[seq + 1] + row
    return seq, pos, st["tables"].long()[seq, pos // BLOCK], pos % BLOCK


def _views(codes, D):
    """The codes as [blocks, heads, token, dim] for keys and values. Keys lie in slices of 64 dims, a slice's tokens
    64 bytes apart; a value dim's 64 tokens lie together, token 16 a + 4 b + c at place 16 b + 4 a + c."""
    n, Hkv = codes.shape[:2]
    padded = codes.shape[3] // 64
    k = codes[:, :, 0].view(n, Hkv, padded // 64, 64, 64).permute(0, 1, 3, 2, 4)  # [.., token, slice, dim]
    v = codes[:, :, 1].view(n, Hkv, padded, 4, 4, 4).permute(0, 1, 4, 3, 5, 2)  # [.., a, b, c, dim]
    return k.reshape(n, Hkv, 64, padded)[..., :D], v.reshape(n, Hkv, 64, padded)[..., :D]


def _values_of(codes):
    return codes.contiguous().view(torch.float8_e4m3fn).float()


def _round(x):
    return x.to(torch.float8_e4m3fn).view(torch.uint8)


def _plain_write(st):
    if not st["rows"]:
        return
    codes, scales = st["codes"], st["scales"]
    n, Hkv = codes.shape[:2]
    D = st["k"].shape[2]
    padded = codes.shape[3] // 64
    _, _, block, place = _places(st)
    first = torch.full((n,), BLOCK, device=DEV).scatter_reduce_(0, block, place, "amin")
    touched = (first < BLOCK).nonzero()[:, 0]
    old_codes = _views(codes[touched], D)
    where = torch.zeros(n, dtype=torch.long, device=DEV)
    where[touched] = torch.arange(len(touched), device=DEV)
    kept = torch.arange(BLOCK, device=DEV)[None, :] < first[touched][:, None]  # tokens there before
    out = []
    for part, x in enumerate((st["k"].float(), st["v"].float())):
        size = torch.where(x.isfinite(), x.abs(), 0).amax(2)
        largest = torch.zeros(n, Hkv, device=DEV).scatter_reduce_(0, block[:, None].expand(-1, Hkv), size, "amax")
        m, e = torch.frexp(largest[touched])  # m in [0.5, 1)
        e = torch.where(m > 0, e - 9 + (m > 0.875).int(), -80).clamp(-80, 120).float()
        before = scales[touched][:, :, part]
        e = torch.where(kept[:, :1], torch.maximum(e, torch.log2(before).clamp(-80, 120)), e)
        scale = torch.exp2(e)
        back = _values_of(old_codes[part]) * (before / scale)[:, :, None, None]
        new = torch.where(kept[:, None, :, None], _round(back), old_codes[part])
        x = torch.where(x.isfinite(), x, math.nan) / scale[where[block]][:, :, None]
        new[where[block], :, place] = _round(x)
        scales[touched, :, part] = scale
        out.append(new)
    k, v = (torch.nn.functional.pad(t, (0, padded - D)) for t in out)
    k = k.view(-1, Hkv, 64, padded // 64, 64).permute(0, 1, 3, 2, 4).reshape(-1, Hkv, 64 * padded)
    v = v.view(-1, Hkv, 4, 4, 4, padded).permute(0, 1, 5, 3, 2, 4).reshape(-1, Hkv, 64 * padded)
    codes[touched] = torch.stack((k, v), 2)


def _plain_read(st):
    D = st["case"]["D"]
    _, _, block, place = _places(st)
    got = []
    for part, codes in enumerate(_views(st["codes"], D)):
        got.append(_values_of(codes[block, :, place]) * st["scales"][block, :, part][:, :, None])
    return got


def _plain_attend(st):
    c = st["case"]
    B, H, Hkv, D = c["B"], c["H"], c["Hkv"], c["D"]
    G, S, n = H // Hkv, st["tables"].shape[1] * BLOCK, st["most"]
    cached = []
    for part, codes in enumerate(_views(st["codes"], D)):
        x = _values_of(codes) * st["scales"][:, :, part][:, :, None, None]
        x = x[st["tables"].long()]  # [B, blocks, Hkv, 64, D]
        cached.append(x.permute(0, 2, 1, 3, 4).reshape(B, Hkv, S, D))
    seq, pos, _, _ = _places(st)
    index = torch.arange(st["rows"], device=DEV) - st["cu"].long()[seq]
    q = torch.zeros(B, n, H, D, device=DEV)
    q[seq, index] = st["q"].float()
    q = q.view(B, n, Hkv, G, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, G * n, D)
    s = torch.matmul(q, cached[0].transpose(2, 3).contiguous()).view(B, Hkv, G, n, S) / math.sqrt(D)
    at = torch.full((B, n), -1, device=DEV)
    at[seq, index] = pos
    j = torch.arange(S, device=DEV)
    see = (j < st["lengths"].long()[:, None])[:, None, :]
    if c["causal"]:
        see = see & (j <= at[:, :, None])
    if c["window"]:
        see = see & ((j - at[:, :, None]).abs() < c["window"])
    see = see[:, None, None].expand(B, 1, 1, n, S)
    s = s.masked_fill(~see, -math.inf)
    p = torch.exp(s - s.amax(-1, keepdim=True).clamp_min(-1e30))
    p = p / p.sum(-1, keepdim=True).clamp_min(1e-30)
    out = torch.matmul(p.view(B, Hkv, G * n, S), cached[1]).view(B, Hkv, G, n, D)
    out = out.permute(0, 3, 1, 2, 4).reshape(B, n, H, D)[seq, index]
    return out.to(_dtype(c))


def run(st):
    if own:
        return _own_run(st)
    kind = st["case"]["kind"]
    if kind == "attend":
        return _plain_attend(st)
    if kind == "store":
        _plain_write(st)
    k, v = _plain_read(st)
    return {"keys": k.to(_dtype(st["case"])), "values": v.to(_dtype(st["case"])), "scales": st["scales"]}


# ---- 64 bits, one sequence at a time -----------------------------------------------------


def _exact_code(byte):
    """The values of e4m3 codes from their bits: sign, four exponent bits (bias 7), three of mantissa."""
    byte = byte.long()
    e, m = (byte >> 3) & 15, (byte & 7).double()
    x = torch.where(e == 0, m * 2.0 ** -9, (1 + m / 8) * torch.exp2(e.double() - 7))
    x = torch.where((byte & 127) == 127, math.nan, x)
    return torch.where(byte >= 128, -x, x)


def _exact_nearest(x):
    """x rounded to a value of e4m3, ties to even; |x| <= 448."""
    a = x.abs()
    step = torch.exp2(torch.floor(torch.log2(a.clamp_min(2.0 ** -6))) - 3)
    return torch.sign(x) * torch.round(a / step) * step


def _exact_tokens(st, b, length):
    """Keys and values [heads, length, D] of sequence b, and of each token its block's two scales."""
    D = st["case"]["D"]
    j = torch.arange(length, device=DEV)
    block, t = st["tables"][b].long()[j // 64], j % 64
    d = torch.arange(D, device=DEV)
    got = []
    for part, at in enumerate(((d[None] // 64) * 4096 + t[:, None] * 64 + d[None] % 64,
                               d[None] * 64 + (t[:, None] // 4 % 4) * 16 + (t[:, None] // 16) * 4 + t[:, None] % 4)):
        rows = st["codes"][:, :, part].permute(1, 0, 2)  # [heads, blocks, bytes]
        scale = st["scales"][block, :, part].double().t()
        got.append((_exact_code(rows[:, block[:, None], at]) * scale[:, :, None], scale))
    return got


def exact(case, seed):
    st = prepare(case, seed)
    lens, cu = st["lengths"].tolist(), st["cu"].tolist()
    H, Hkv, D, w = case["H"], case["Hkv"], case["D"], case["window"]
    if case["kind"] == "attend":
        out = torch.empty(st["rows"], H, D, dtype=torch.float64, device=DEV)
        for b, length in enumerate(lens):
            (k, _), (v, _) = _exact_tokens(st, b, length)
            j = torch.arange(length, device=DEV)
            for r in range(cu[b], cu[b + 1], 2048):
                r1 = min(cu[b + 1], r + 2048)
                pos = torch.arange(length - cu[b + 1] + r, length - cu[b + 1] + r1, device=DEV)[:, None]
                hide = torch.zeros(r1 - r, length, dtype=torch.bool, device=DEV)
                if case["causal"]:
                    hide |= j > pos
                if w:
                    hide |= (j - pos).abs() >= w
                for h in range(H):
                    s = (st["q"][r:r1, h].double() @ k[h // (H // Hkv)].t()) / math.sqrt(D)
                    out[r:r1, h] = torch.softmax(s.masked_fill(hide, -math.inf), 1) @ v[h // (H // Hkv)]
        return out
    keys = torch.empty(st["rows"], Hkv, D, dtype=torch.float64, device=DEV)
    values = torch.empty_like(keys)
    scales = st["scales"].double().clone()
    for b, length in enumerate(lens):
        r0, r1 = cu[b], cu[b + 1]
        if case["kind"] == "read":
            (k, _), (v, _) = _exact_tokens(st, b, length)
            first = length - (r1 - r0)
            keys[r0:r1], values[r0:r1] = k[:, first:].transpose(0, 1), v[:, first:].transpose(0, 1)
            continue
        first = length - (r1 - r0)
        for slot in range(first // 64, (length - 1) // 64 + 1):
            lo, hi = max(first, slot * 64), min(length, slot * 64 + 64)
            block = int(st["tables"][b, slot])
            for part, (x, to) in enumerate(((st["k"], keys), (st["v"], values))):
                x = x[r0 + lo - first:r0 + hi - first].double()  # [tokens, heads, D]
                e = torch.ceil(torch.log2(x.abs().amax((0, 2)) / 448)).clamp(-80, 120)
                if lo > slot * 64:
                    e = torch.maximum(e, torch.log2(scales[block, :, part]))
                scale = torch.exp2(e)
                scales[block, :, part] = scale
                to[r0 + lo - first:r0 + hi - first] = _exact_nearest(x / scale[:, None]) * scale[:, None]
    return {"keys": keys, "values": values, "scales": scales}
