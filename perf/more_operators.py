"""The work of one step of a program that adds tokens one after another, through
the C ABI of include/fa_rocm.h, around the attention over the 8-bit key/value
cache: products with weights held in 8 bits, keys and values rotated and written
into the cache, and the next tokens drawn from logits.

Product: C = epilogue(A^ . W^T). Of every row of A and of W each block of 128
columns (the last may be shorter) is held as e4m3 codes times one scale 2^e, the
smallest (-80 <= e <= 120) under which the block's largest finite magnitude is at
most 448; A^ and W^ are those values. W is held so by the program, A is rounded
within the call. Codes [n][kp], kp = k in whole blocks, zeros past k; scales
[n][ks] bytes e + 127, ks = kp / 128 rounded up to 4. The epilogue adds a bias,
applies tanh-GELU, multiplies and adds a matrix, each if given.

Append: pair i of the first `dims` of a head (dims i and i + dims / 2) turns by
the angle p base^(-2 i / dims), p the token's position; the angle in float64, its
cosine and sine rounded to float32, the turned values to float32. Queries are
returned in the tensors' type, keys and values go into the cache as they do
without rotation: blocks of 64 tokens, per head e4m3 codes times a power of two.

Sampling: with M the largest logit and T the temperature, w = exp((l - M) / T).
Of the tokens ordered by logit, falling, ties by the lower id, those stay that
are among the first top_k, of these the shortest run whose weights make at
least top_p of theirs, and of these the ones with w >= min_p. The token drawn is
the first, by id, up to which the weights of those that stay exceed u times
their sum; with it goes the log of its share of that sum. T = 0 takes the first
of the order. NaN and -inf logits are never drawn; a row of nothing else gives
the id -1 and NaN.

listed() are the fixed cases, draw(rng) another one of the same ranges;
prepare / run / work / exact take one case each. With own the framework's
calls are made, else the plain forms below.
"""
import math

import torch

own = False

DEV = "cuda"
BF16, F32 = "bf16", "f32"


def listed():
    return [
        # One user's next token against the whole vocabulary at this repository's widths: reading the weights.
        dict(name="product 1x262144x768 f32", kind="product", a=F32, c=F32, m=1, n=262144, k=768, epi=""),
        # A layer of a small serving batch: few rows, latency and the weights.
        dict(name="product 16x4096x4096", kind="product", a=BF16, c=BF16, m=16, n=4096, k=4096, epi=""),
        # This repository's gated layer on a ragged batch, in float32, with its epilogue.
        dict(name="product 777x1152x768 f32", kind="product", a=F32, c=F32, m=777, n=1152, k=768, epi="gelu mul"),
        # The prompts of a large batch through a wide layer: the largest product.
        dict(name="product 8192x8192x8192", kind="product", a=BF16, c=BF16, m=8192, n=8192, k=8192, epi="residual"),
        # One user's next token at this repository's own head shape: pure latency.
        dict(name="append 1 token f32", kind="append", dtype=F32, B=1, H=3, Hkv=1, D=256, dims=256, base=1e6, lo=1000,
             hi=1000, nlo=1, nhi=1, far=0),
        # The next tokens of a full serving batch.
        dict(name="append 64x1", kind="append", dtype=BF16, B=64, H=32, Hkv=8, D=128, dims=128, base=1e6, lo=1024,
             hi=8192, nlo=1, nhi=1, far=0),
        # Chunks whose positions are given, far from zero, half of each head turning.
        dict(name="append chunk 4x512 far f32", kind="append", dtype=F32, B=4, H=16, Hkv=4, D=128, dims=64, base=5e5,
             lo=900, hi=2000, nlo=384, nhi=512, far=1000000),
        # Whole prompts, ragged: bound by memory.
        dict(name="append prompts 16x2048", kind="append", dtype=BF16, B=16, H=32, Hkv=8, D=128, dims=128, base=1e4,
             lo=700, hi=2048, nlo=700, nhi=2048, far=0),
        # One user's next token from this repository's vocabulary: latency.
        dict(name="sample 1x262144 f32", kind="sample", dtype=F32, rows=1, vocab=262144, filters="k p", masked=0.0),
        # A serving batch of users with settings of their own.
        dict(name="sample 64x32000", kind="sample", dtype=BF16, rows=64, vocab=32000, filters="k p m t", masked=0.01),
        # Odd rows, no order to find: plain draws, as in scoring by samples.
        dict(name="sample 37x49999 f32", kind="sample", dtype=F32, rows=37, vocab=49999, filters="", masked=0.0),
        # Many draws at once over a large vocabulary, cut by their mass alone.
        dict(name="sample 256x262144 f32", kind="sample", dtype=F32, rows=256, vocab=262144, filters="p", masked=0.0),
    ]


def _log(rng, lo, hi):
    return max(lo, min(hi, int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))))


def draw(rng):
    kind = rng.choice(["product", "append", "sample"])
    most = {c["name"]: work(c) for c in listed() if c["kind"] == kind}
    most_bytes, most_flops = (max(w[x] for w in most.values()) for x in ("bytes", "flops"))
    while True:
        if kind == "product":
            a = rng.choice([BF16, BF16, F32])
            case = dict(kind=kind, a=a, c=rng.choice([a, a, F32, BF16]),
                        m=rng.choice([_log(rng, 1, 64), _log(rng, 1, 8192)]), n=_log(rng, 8, 32768),
                        k=rng.choice([_log(rng, 16, 16384), 128 * _log(rng, 1, 128)]),
                        epi=rng.choice(["", "", "bias", "gelu", "gelu mul", "residual", "bias residual"]))
        elif kind == "append":
            Hkv, D = rng.choice([1, 1, 2, 4, 8]), rng.choice([64, 128, 128, 256, 256, 40, 80, 96, 192, 512, 66])
            hi = _log(rng, 2, 30000)
            lo = max(1, int(hi * rng.choice([0.1, 0.5, 0.9])))
            what = rng.choice(["token", "token", "few", "chunk", "prompt"])
            nlo, nhi = 1, 1
            if what == "few":
                nhi = rng.randint(2, 12)
            elif what == "chunk":
                nhi = _log(rng, 16, 1024)
                nlo = max(1, nhi // 2)
            elif what == "prompt":
                nlo, nhi = lo, hi
            case = dict(kind=kind, dtype=rng.choice([BF16, BF16, F32]), B=_log(rng, 1, 96),
                        H=Hkv * rng.choice([1, 2, 3, 4, 4, 8]), Hkv=Hkv, D=D,
                        dims=rng.choice([D, D, D, D // 4 * 2, 2]), base=rng.choice([1e4, 5e5, 1e6]), lo=lo, hi=hi,
                        nlo=nlo, nhi=nhi, far=rng.choice([0, 0, _log(rng, 1, 10000000)]))
        else:
            case = dict(kind=kind, dtype=rng.choice([F32, F32, BF16]), rows=_log(rng, 1, 1024),
                        vocab=_log(rng, 2, 262144), masked=rng.choice([0.0, 0.0, 0.01, 0.9]),
                        filters=rng.choice(["", "k", "p", "m", "t", "k p", "p m", "k p m t", "k p m t"]))
        w = work(case)
        if w["bytes"] > most_bytes or w["flops"] > most_flops:
            continue
        if kind == "append" and sum(_sizes(case)[0]) * case["Hkv"] * case["D"] > 6e8:  # the pool behind the call
            continue
        return case


# ---- sizes and work ---------------------------------------------------------------------


def _spread(lo, hi, B):
    """B whole numbers over lo .. hi, hi among them."""
    return [hi - int((hi - lo) * ((i * 0.6180339887) % 1.0)) for i in range(B)]


def _sizes(case):
    """Lengths of an append's sequences, the new tokens included, and how many are new."""
    lens = _spread(case["lo"], case["hi"], case["B"])
    if (case["nlo"], case["nhi"]) == (case["lo"], case["hi"]):
        return lens, list(lens)
    ns = _spread(case["nlo"], case["nhi"], case["B"])
    return lens, [min(n, l) for n, l in zip(ns, lens)]


def _bytes_of(dtype):
    return 4 if dtype == F32 else 2


def work(case):
    if case["kind"] == "product":
        m, n, k = case["m"], case["n"], case["k"]
        more = 4 * n * ("bias" in case["epi"]) + 4 * m * n * (("mul" in case["epi"]) + ("residual" in case["epi"]))
        return {"bytes": m * k * _bytes_of(case["a"]) + n * k + n * -(-k // 128) + m * n * _bytes_of(case["c"]) + more,
                "flops": 2 * m * n * k}
    if case["kind"] == "append":
        rows, size = sum(_sizes(case)[1]), _bytes_of(case["dtype"])
        H, Hkv, D = case["H"], case["Hkv"], case["D"]
        return {"bytes": rows * D * (2 * H * size + 2 * Hkv * (size + 1)),
                "flops": rows * (3 * (H + Hkv) * case["dims"] + 3 * 2 * Hkv * D)}
    size = case["rows"] * case["vocab"]
    return {"bytes": size * _bytes_of(case["dtype"]) + 28 * case["rows"], "flops": 4 * size}


# ---- inputs ------------------------------------------------------------------------------


def _gen(seed, salt):
    g = torch.Generator(device=DEV)
    g.manual_seed(seed * 1000003 + salt)
    return g


def _type(name):
    return torch.float32 if name == F32 else torch.bfloat16


def _ints(v):
    return torch.tensor(v, dtype=torch.int32, device=DEV)


def prepare(case, seed):
    st = {"product": _prepare_product, "append": _prepare_append, "sample": _prepare_sample}[case["kind"]](case, seed)
    torch.cuda.synchronize()  # the inputs come from torch's stream, a context's calls run on its own
    return st


def _prepare_product(case, seed):
    g = _gen(seed, 1)
    m, n, k = case["m"], case["n"], case["k"]

    def randn(*shape):
        return torch.randn(*shape, generator=g, device=DEV)

    # activations with a few strong channels and rows of their own size, as layers see them
    strong = 1 + 12 * (torch.rand(k, generator=g, device=DEV) < 0.01).float()
    a = (randn(m, k) * strong * torch.exp(0.5 * randn(m, 1))).to(_type(case["a"]))
    codes, scales = _plain_quantize(randn(n, k) / math.sqrt(k))
    st = dict(case=case, a=a, codes=codes, scales=scales, c=torch.empty(m, n, dtype=_type(case["c"]), device=DEV))
    if "bias" in case["epi"]:
        st["bias"] = randn(n)
    if "mul" in case["epi"]:
        st["mul"] = randn(m, n)
    if "residual" in case["epi"]:
        st["residual"] = randn(m, n)
    return st


def _keys_values(g, case, rows):
    """Keys with a few strong channels, as rotary models have them, and values whose magnitude differs by token."""
    Hkv, D = case["Hkv"], case["D"]
    k = torch.randn(rows, Hkv, D, generator=g, device=DEV)
    strong = (torch.rand(Hkv, D, generator=g, device=DEV) < 0.03).float()
    k = k * (1 + 5 * strong) + 2 * strong
    v = torch.randn(rows, Hkv, D, generator=g, device=DEV)
    v = v * torch.exp(0.7 * torch.randn(rows, 1, 1, generator=g, device=DEV))
    return k.to(_type(case["dtype"])), v.to(_type(case["dtype"]))


def _prepare_append(case, seed):
    lens, ns = _sizes(case)
    order = torch.randperm(case["B"], generator=torch.Generator().manual_seed(seed)).tolist()
    lens, ns = [lens[i] for i in order], [ns[i] for i in order]
    g = _gen(seed, 2)
    Hkv, D = case["Hkv"], case["D"]
    used = [-(-l // 64) for l in lens]
    blocks = sum(used) + 3
    perm = torch.randperm(blocks, generator=g, device=DEV).to(torch.int32)
    tables = torch.zeros(case["B"], max(used), dtype=torch.int32, device=DEV)
    at = 0
    for b, u in enumerate(used):
        tables[b, :u] = perm[at:at + u]
        at += u

    def cu(v):
        return _ints([sum(v[:i]) for i in range(len(v) + 1)])

    st = dict(case=case, codes=torch.zeros(blocks, Hkv, 2, 64 * (-(-D // 64) * 64), dtype=torch.uint8, device=DEV),
              scales=torch.zeros(blocks, Hkv, 2, device=DEV), tables=tables, lengths=_ints(lens), cu=cu(ns),
              rows=sum(ns))
    # what lies in the block that a sequence's new tokens continue, already rotated
    old = [(l - n) % 64 for l, n in zip(lens, ns)]
    k, v = _keys_values(g, case, sum(old))
    _plain_write(dict(st, lengths=_ints([l - n for l, n in zip(lens, ns)]), cu=cu(old), rows=sum(old)), k.float(),
                 v.float())
    st["k"], st["v"] = _keys_values(g, case, st["rows"])
    st["q"] = torch.randn(st["rows"], case["H"], D, generator=g, device=DEV).to(_type(case["dtype"]))
    st["q_out"] = torch.empty_like(st["q"])
    if case["far"]:
        st["positions"] = (_places(st)[1] + case["far"]).to(torch.int32)
    return st


def _prepare_sample(case, seed):
    g = _gen(seed, 3)
    rows, vocab, what = case["rows"], case["vocab"], case["filters"].split()

    def pick(values, dtype):
        at = torch.randint(len(values), (rows,), generator=g, device=DEV)
        return torch.tensor(values, dtype=dtype, device=DEV)[at]

    # logits whose shares fall with a power of the rank, as a language's words do, steeper in some rows than in others
    l = -torch.log(torch.rand(rows, vocab, generator=g, device=DEV).clamp_min(1e-9))
    l = l * (0.7 + 0.9 * torch.rand(rows, 1, generator=g, device=DEV)) + 8 * torch.rand(rows, 1, generator=g, device=DEV)
    if case["masked"]:
        l = torch.where(torch.rand(rows, vocab, generator=g, device=DEV) < case["masked"], -math.inf, l)
    st = dict(case=case, logits=l.to(_type(case["dtype"])), u=torch.rand(rows, generator=g, device=DEV),
              ids=torch.empty(rows, dtype=torch.int32, device=DEV), logp=torch.empty(rows, device=DEV))
    if "k" in what:
        st["top_k"] = pick([1, 10, 40, 50, 200, 1000, 0], torch.int32)
    if "p" in what:
        st["top_p"] = pick([0.5, 0.8, 0.9, 0.95, 0.99], torch.float32)
    if "m" in what:
        st["min_p"] = pick([0.0, 0.02, 0.05, 0.1], torch.float32)
    if "t" in what:
        st["temperature"] = pick([0.0, 0.3, 0.7, 1.0, 1.5], torch.float32)
    return st


# ---- the framework's calls -----------------------------------------------------------------

_ctx = None


def _context():
    global _ctx
    from ai_amd import _native as N
    if _ctx is None:
        _ctx = N.Context(0)
    return N, N.lib(), _ctx


def _dt(N, name):
    return N.FA_DT_F32 if name == F32 else N.FA_DT_BF16


def _at(x):
    return None if x is None else x.data_ptr()


def _own_product(st):
    """The descriptors are what a program keeps."""
    c = st["case"]
    N, L, ctx = _context()
    n, k = c["n"], c["k"]
    if "args" not in st:
        w = N.F8Matrix(st["codes"].data_ptr(), st["scales"].data_ptr(), n, k)
        e = N.Epilogue(_at(st.get("bias")), None, N.FA_ACT_GELU if "gelu" in c["epi"] else N.FA_ACT_NONE,
                       _at(st.get("mul")), n, _at(st.get("residual")), n)
        st["args"] = (w, e, N.C.byref(w), N.C.byref(e) if c["epi"] else None)
    N.check(ctx.h, L.fa_matmul_f8_dev(ctx.h, c["m"], _dt(N, c["a"]), st["a"].data_ptr(), k, st["args"][2],
                                      st["args"][3], _dt(N, c["c"]), st["c"].data_ptr(), n, None, 0))
    return st["c"]


def _own_append(st):
    c = st["case"]
    N, L, ctx = _context()
    H, Hkv, D = c["H"], c["Hkv"], c["D"]
    if "args" not in st:
        cache = N.KvCache(st["codes"].data_ptr(), st["scales"].data_ptr(), st["codes"].shape[0], Hkv, D)
        batch = N.KvBatch(st["tables"].data_ptr(), st["tables"].shape[1], st["lengths"].data_ptr(),
                          st["cu"].data_ptr(), c["B"], st["rows"])
        rope = N.KvRope(c["base"], c["dims"], _at(st.get("positions")))
        st["args"] = (cache, batch, rope, *(N.C.byref(x) for x in (cache, batch, rope)))
    N.check(ctx.h, L.fa_kv_write_rope_dev(ctx.h, *st["args"][3:], _dt(N, c["dtype"]), st["q"].data_ptr(), H * D, D, H,
                                          st["q_out"].data_ptr(), st["k"].data_ptr(), Hkv * D, D, st["v"].data_ptr(),
                                          Hkv * D, D))
    return {"q": st["q_out"], "codes": st["codes"].view(torch.float8_e4m3fn), "scales": st["scales"]}


def _own_sample(st):
    c = st["case"]
    N, L, ctx = _context()
    if "args" not in st:
        s = N.Sampling(_at(st.get("temperature")), _at(st.get("top_k")), _at(st.get("top_p")), _at(st.get("min_p")))
        st["args"] = (s, N.C.byref(s))
    N.check(ctx.h, L.fa_sample_dev(ctx.h, c["rows"], c["vocab"], _dt(N, c["dtype"]), st["logits"].data_ptr(),
                                   c["vocab"], st["args"][1], st["u"].data_ptr(), st["ids"].data_ptr(),
                                   st["logp"].data_ptr(), None, 0))
    return {"ids": st["ids"], "logp": st["logp"]}


# ---- the plain forms -------------------------------------------------------------------------


def _exponent(largest):
    """The smallest e with largest <= 448 * 2^e, in -80 .. 120."""
    m, e = torch.frexp(largest)  # m in [0.5, 1)
    return torch.where(m > 0, e - 9 + (m > 0.875).int(), -80).clamp(-80, 120)


def _plain_quantize(x):
    """Codes [n][kp] and scale bytes [n][ks] of x [n][k]."""
    n, k = x.shape
    kb = -(-k // 128)
    x = torch.nn.functional.pad(x.float(), (0, kb * 128 - k)).view(n, kb, 128)
    e = _exponent(torch.where(x.isfinite(), x.abs(), 0).amax(2))
    x = torch.where(x.isfinite(), x, math.nan) / torch.exp2(e.float())[:, :, None]
    x = torch.where(e[:, :, None] == 120, x.clamp(-240, 240), x)
    scales = torch.nn.functional.pad((e + 127).to(torch.uint8), (0, -kb % 4), value=127)
    return x.to(torch.float8_e4m3fn).view(torch.uint8).view(n, kb * 128), scales


def _plain_values(codes, scales):
    n, kp = codes.shape
    e = scales[:, :kp // 128].float() - 127
    return (codes.view(torch.float8_e4m3fn).float().view(n, kp // 128, 128) * torch.exp2(e)[:, :, None]).view(n, kp)


def _plain_product(st):
    c = torch.matmul(_plain_values(*_plain_quantize(st["a"])), _plain_values(st["codes"], st["scales"]).t())
    if "bias" in st:
        c = c + st["bias"]
    if "gelu" in st["case"]["epi"]:
        c = 0.5 * c * (1 + torch.tanh(math.sqrt(2 / math.pi) * (c + 0.044715 * c * c * c)))
    if "mul" in st:
        c = c * st["mul"]
    if "residual" in st:
        c = c + st["residual"]
    return c.to(_type(st["case"]["c"]))


def _places(st):
    """Of every row: its sequence, position, block and place in the block."""
    row = torch.arange(st["rows"], device=DEV)
    seq = torch.searchsorted(st["cu"][1:].long(), row, right=True)
    pos = st["lengths"].long()[seq] - st["cu"].long()[seq + 1] + row
    return seq, pos, st["tables"].long()[seq, pos // 64], pos % 64


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


def _plain_write(st, k, v):
    """k and v in float32 into the cache of 8 bits."""
    if not st["rows"]:
        return
    codes, scales = st["codes"], st["scales"]
    n, Hkv = codes.shape[:2]
    D = k.shape[2]
    padded = codes.shape[3] // 64
    _, _, block, place = _places(st)
    first = torch.full((n,), 64, device=DEV).scatter_reduce_(0, block, place, "amin")
    touched = (first < 64).nonzero()[:, 0]
    old_codes = _views(codes[touched], D)
    where = torch.zeros(n, dtype=torch.long, device=DEV)
    where[touched] = torch.arange(len(touched), device=DEV)
    kept = torch.arange(64, device=DEV)[None, :] < first[touched][:, None]  # tokens there before
    out = []
    for part, x in enumerate((k, v)):
        size = torch.where(x.isfinite(), x.abs(), 0).amax(2)
        largest = torch.zeros(n, Hkv, device=DEV).scatter_reduce_(0, block[:, None].expand(-1, Hkv), size, "amax")
        e = _exponent(largest[touched]).float()
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


def _plain_rotate(st, x):
    """x [rows, heads, D] turned, in float32 (the products of two float32 values are exact in 64 bits)."""
    c = st["case"]
    half = c["dims"] // 2
    pos = st["positions"].long() if "positions" in st else _places(st)[1]
    turn = torch.tensor([c["base"] ** (-2 * i / c["dims"]) for i in range(half)], dtype=torch.float64, device=DEV)
    angle = pos.double()[:, None] * turn
    cos, sin = (f(angle).float().double()[:, None, :] for f in (torch.cos, torch.sin))
    lo, hi = x[..., :half].double(), x[..., half:2 * half].double()
    return torch.cat(((lo * cos - hi * sin).float(), (hi * cos + lo * sin).float(), x[..., 2 * half:].float()), 2)


def _plain_append(st):
    _plain_write(st, _plain_rotate(st, st["k"]), st["v"].float())
    return {"q": _plain_rotate(st, st["q"]).to(st["q"].dtype), "codes": st["codes"].view(torch.float8_e4m3fn),
            "scales": st["scales"]}


def _setting(st, name, default):
    x = st.get(name)
    rows = st["case"]["rows"]
    return (torch.full((rows,), default, device=DEV) if x is None else x).double()[:, None]


def _plain_sample(st):
    vocab = st["case"]["vocab"]
    l = st["logits"].double()
    l = torch.where(l.isnan(), -math.inf, l)
    l, order = torch.sort(l, dim=1, descending=True, stable=True)
    t = _setting(st, "temperature", 1.0)
    none = l[:, 0] == -math.inf
    off = torch.where(none[:, None], 0.0, l - l[:, :1])
    w = torch.where(t > 0, torch.exp(off / torch.where(t > 0, t, 1.0)), 0.0)
    w[:, 0] = 1.0  # (all of it where the temperature is 0)
    k = _setting(st, "top_k", 0.0)
    rank = torch.arange(vocab, device=DEV)
    w = torch.where((rank < k) | (k <= 0), w, 0.0)
    p = _setting(st, "top_p", 1.0)
    run = torch.cumsum(w, 1)
    before = torch.nn.functional.pad(run[:, :-1], (1, 0))
    w = torch.where((before < p * run[:, -1:]) | (p >= 1) | (rank == 0), w, 0.0)
    w = torch.where(w >= _setting(st, "min_p", 0.0), w, 0.0)
    w = torch.zeros_like(w).scatter_(1, order, w)
    run = torch.cumsum(w, 1)
    ids = ((run > st["u"].double()[:, None] * run[:, -1:]) & (w > 0)).int().argmax(1)
    share = torch.log(torch.gather(w, 1, ids[:, None]) / run[:, -1:])[:, 0]
    return {"ids": torch.where(none, -1, ids).to(torch.int32), "logp": torch.where(none, math.nan, share).float()}


def run(st):
    kind = st["case"]["kind"]
    if own:
        return {"product": _own_product, "append": _own_append, "sample": _own_sample}[kind](st)
    return {"product": _plain_product, "append": _plain_append, "sample": _plain_sample}[kind](st)


# ---- 64 bits ------------------------------------------------------------------------------------


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


def _exact_product(case, seed):
    st = prepare(case, seed)
    m, n, k = case["m"], case["n"], case["k"]
    a, w = st["a"].double(), torch.empty(n, k, dtype=torch.float64, device=DEV)
    for at in range(0, k, 128):
        to = min(k, at + 128)
        scale = torch.exp2(torch.ceil(torch.log2(a[:, at:to].abs().amax(1, keepdim=True) / 448)).clamp(-80, 120))
        a[:, at:to] = _exact_nearest(a[:, at:to] / scale) * scale
        w[:, at:to] = _exact_code(st["codes"][:, at:to]) * torch.exp2(st["scales"][:, at // 128].double() - 127)[:, None]
    c = a @ w.t()
    if "bias" in st:
        c += st["bias"].double()
    if "gelu" in case["epi"]:
        c = c * torch.sigmoid(2 * math.sqrt(2 / math.pi) * (c + 0.044715 * c ** 3))
    if "mul" in st:
        c *= st["mul"].double()
    if "residual" in st:
        c += st["residual"].double()
    return c


def _exact_append(case, seed):
    st = prepare(case, seed)
    lens, cu, D = st["lengths"].tolist(), st["cu"].tolist(), case["D"]
    half = case["dims"] // 2
    d = torch.arange(D, device=DEV)
    partner = torch.where(d < half, d + half, torch.where(d < 2 * half, d - half, d))
    sign = torch.where(d < half, -1.0, 1.0).double()
    turn = torch.exp2(torch.where(d < 2 * half, d % half, 0).double() * (-2 / case["dims"]) * math.log2(case["base"]))
    turn = torch.where(d < 2 * half, turn, 0.0)  # an angle of zero: kept as it is
    first = [l - (b - a) for l, a, b in zip(lens, cu, cu[1:])]
    pos = torch.cat([torch.arange(f, l, device=DEV) for f, l in zip(first, lens)]).double() + case["far"]

    def rotated(x):
        angle = pos[:, None] * turn
        cos, sin = torch.cos(angle).float().double(), (torch.sin(angle) * sign).float().double()
        return x.double() * cos[:, None] + x.double()[..., partner] * sin[:, None]

    k, v = rotated(st["k"]).float().double(), st["v"].double()
    codes = _exact_code(st["codes"])
    scales = st["scales"].double().clone()
    for b, length in enumerate(lens):
        for slot in range(first[b] // 64, (length - 1) // 64 + 1):
            lo, hi = max(first[b], slot * 64), min(length, slot * 64 + 64)
            block = int(st["tables"][b, slot])
            t = torch.arange(slot * 64, hi, device=DEV) % 64
            for part, x in enumerate((k, v)):
                x = x[cu[b] + lo - first[b]:cu[b] + hi - first[b]].transpose(0, 1)  # [heads, tokens, D]
                e = torch.ceil(torch.log2(x.abs().amax((1, 2)) / 448)).clamp(-80, 120)
                if part == 0:
                    at = (d // 64) * 4096 + t[:, None] * 64 + d % 64
                else:
                    at = d * 64 + (t[:, None] // 4 % 4) * 16 + (t[:, None] // 16) * 4 + t[:, None] % 4
                kept = lo - slot * 64  # tokens there before
                old = codes[block, :, part][:, at[:kept]] * scales[block, :, part][:, None, None]
                if kept:
                    e = torch.maximum(e, torch.log2(scales[block, :, part]))
                scale = torch.exp2(e)
                scales[block, :, part] = scale
                codes[block, :, part][:, at] = _exact_nearest(torch.cat((old, x), 1) / scale[:, None, None])
    return {"q": rotated(st["q"]), "codes": codes, "scales": scales}


def _exact_sample(case, seed):
    st = prepare(case, seed)
    ids, logp = [], []
    for r in range(case["rows"]):
        l, u = st["logits"][r].double(), float(st["u"][r])

        def of(name, default):
            return float(st[name][r]) if name in st else default

        t, k, p, least = of("temperature", 1.0), int(of("top_k", 0)), of("top_p", 1.0), of("min_p", 0.0)
        if not torch.any(l > -math.inf):
            ids.append(-1)
            logp.append(math.nan)
            continue
        if t == 0:
            ids.append(int((l == l.max()).nonzero()[0, 0]))
            logp.append(0.0)
            continue
        w = torch.exp((l - l.max()) / t)
        order = torch.sort(l, descending=True, stable=True).indices
        stay = len(order) if k <= 0 else min(k, len(order))
        run = torch.cumsum(w[order[:stay]], 0)
        if p < 1:
            stay = min(stay, int(torch.searchsorted(run, p * run[-1])) + 1)
        kept = torch.zeros_like(w)
        kept[order[:stay]] = w[order[:stay]]
        kept[kept < least] = 0
        run = torch.cumsum(kept, 0)
        at = int(torch.searchsorted(run, u * run[-1], right=True))
        ids.append(at)
        logp.append(float(torch.log(kept[at] / run[-1])))
    return {"ids": torch.tensor(ids, dtype=torch.int32), "logp": torch.tensor(logp, dtype=torch.float64)}


def exact(case, seed):
    return {"product": _exact_product, "append": _exact_append, "sample": _exact_sample}[case["kind"]](case, seed)
