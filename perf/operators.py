"""The operators that a decoder's serving step needs next to the dynamically quantized linear:

  linear     int8 matrix product with a scale for each token and each output channel, the tokens
             quantized on the way in (ops.gpu_token_qlinear over an ops.TokenWeight)
  shared     the same for several weights over one quantized activation (ops.gpu_quantize_tokens,
             then ops.gpu_token_qlinear of its int8 rows)
  write      keys and values quantized into a paged cache of 4 or 8 bits and read back
             (ops.gpu_kv_cache_write, ops.gpu_kv_cache_read over an ops.KvCache)
  read       cached tokens read back alone (ops.gpu_kv_cache_read)
  attention  attention over such a cache, from one token a sequence to whole prompts
             (ops.gpu_kv_cache_attention)

Definitions.  A token x of K values has the scale s = max(max|x| / 127, 2^-126) and the bytes
q = rne(x / s) (the quotient's exact value); the product is (sum_k q_mk w_kn) (s_m w_n) + bias_n.

A cached head of D values is cut into blocks of 32 with a power-of-two scale 2^e each.  4 bits hold
the magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6 and a sign; 8 bits hold a sign, 4 bits of exponent (bias 7)
and 3 of mantissa, up to 448.  e is the least exponent for which no value of the block rounds past
the largest magnitude, kept in [-125, 125] (4 bits) or [-117, 119] (8 bits); codes round to nearest,
ties to the even code, and past the largest magnitude become it.

Row i of the n rows of a sequence of L cached tokens has the position p = L - n + i and attends to
the tokens j <= p (and j > p - window): softmax over j of cap(scale q.k_j) + slope_h (j - p), with
cap(s) = softcap tanh(s / softcap) where a cap is given.
"""
import functools
import math

import torch

own = False

_T = {"float32": torch.float32, "float16": torch.float16, "bfloat16": torch.bfloat16}


def listed():
    return [
        # one decoding step of 8 sequences through an attention projection: latency and one walk of the weight
        dict(name="linear_decode", kind="linear", M=8, K=4096, N=4096, dtype="bfloat16", bias=False),
        # a ragged batch of short texts, sizes that fit no tile
        dict(name="linear_ragged", kind="linear", M=333, K=1000, N=1500, dtype="float16", bias=True),
        # the three projections of a 6-layer encoder's attention over 16 texts of 128 tokens, quantized once
        dict(name="linear_qkv", kind="shared", M=2048, K=768, N=768, products=3, dtype="float32", bias=True),
        # the largest product: 16384 tokens by 4096 x 4096
        dict(name="linear_prompt", kind="linear", M=16384, K=4096, N=4096, dtype="bfloat16", bias=False),
        # one step of 64 sequences: one token each into its own page
        dict(name="write_step", kind="write", T=64, heads=8, D=128, bits=4, page=16, dtype="bfloat16", fused=False),
        # prompts written at once, keys and values being slices of the fused projection's output
        dict(name="write_prompts", kind="write", T=12289, heads=12, D=64, bits=8, page=64, dtype="float16", fused=True),
        # a cached prefix read back for a layer that wants it in float32
        dict(name="read_prefix", kind="read", T=517, heads=16, D=64, bits=4, page=16, dtype="float32"),
        # a long shared prefix read back
        dict(name="read_long", kind="read", T=65536, heads=8, D=128, bits=8, page=128, dtype="bfloat16"),
        # one text of at most 128 tokens, the next token's attention alone: nothing but latency
        dict(name="attention_one_text", kind="attention", B=1, Hq=12, Hkv=12, D=64, length=128, rows=1, bits=4, page=16,
             dtype="float32", softcap=0.0, window=0, slopes=True),
        # a decoding step of a full server: 64 sequences of up to 8192 tokens, 4 query heads a cached head
        dict(name="attention_decode", kind="attention", B=64, Hq=32, Hkv=8, D=128, length=8192, rows=1, bits=4, page=16,
             dtype="bfloat16", softcap=0.0, window=0, slopes=False),
        # chunks of prompts beside decoding rows, capped scores and a window
        dict(name="attention_chunks", kind="attention", B=6, Hq=16, Hkv=4, D=96, length=2500, rows=300, bits=8, page=32,
             dtype="float16", softcap=30.0, window=1024, slopes=False),
        # the second half of a prompt of 8192 tokens
        dict(name="attention_prompt", kind="attention", B=1, Hq=32, Hkv=8, D=128, length=8192, rows=4096, bits=4, page=64,
             dtype="bfloat16", softcap=0.0, window=0, slopes=False),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng):
    kind = rng.choice(["linear", "shared", "write", "read", "attention", "attention"])
    dtype = rng.choice(["bfloat16", "bfloat16", "float16", "float32"])
    if kind in ("linear", "shared"):
        c = dict(kind=kind, M=_log(rng, 1, 8192), K=_log(rng, 64, 4096), N=_log(rng, 64, 4096), dtype=dtype,
                 bias=rng.random() < 0.5)
        if rng.random() < 0.5:
            c["K"], c["N"] = -(-c["K"] // 64) * 64, -(-c["N"] // 64) * 64
        if kind == "shared":
            c["products"] = rng.randint(2, 4)
        return c
    heads, D, page = rng.randint(1, 16), 32 * rng.choice([2, 2, 3, 4, 4, 4, 5, 8]), 16 * rng.choice([1, 2, 3, 4, 8])
    bits = rng.choice([4, 8])
    if kind in ("write", "read"):
        c = dict(kind=kind, T=_log(rng, 1, 16384), heads=heads, D=D, bits=bits, page=page, dtype=dtype)
        if kind == "write":
            c["fused"] = rng.random() < 0.5
        return c
    group = rng.choice([1, 1, 2, 3, 4, 7, 8])
    heads = min(heads, 32 // group)
    many = rng.random() < 0.5
    length = _log(rng, 1, 4096)
    return dict(kind="attention", B=rng.randint(1, 4) if many else _log(rng, 1, 48), Hq=heads * group, Hkv=heads, D=D,
                length=length, rows=min(length, _log(rng, 2, 1024)) if many else min(length, rng.choice([1, 1, 1, 4])),
                bits=bits, page=page, dtype=dtype, softcap=rng.choice([0.0, 0.0, 20.0, 50.0]),
                window=rng.choice([0, 0, 0, _log(rng, 1, 2048)]), slopes=rng.random() < 0.3)


def _lengths(case):
    """(tokens cached, query rows) of each sequence: the first has the most of both."""
    out = []
    for b in range(case["B"]):
        n = case["length"] - (b * 37 * case["length"] // 100) % (case["length"] // 2 + 1)
        out.append((n, min(n, 1 + (case["rows"] - 1 + 131 * b) % case["rows"])))
    return out


# ---- inputs -------------------------------------------------------------------------------
def _inputs(case, seed):
    """What the definitions take, on the GPU (on the CPU where there is none)."""
    dev = "cuda" if torch.cuda.is_available() else "cpu"
    g = torch.Generator(device=dev).manual_seed(seed)
    t = _T[case["dtype"]]

    def normal(*shape):
        return torch.randn(shape, generator=g, device=dev)

    def channels(n):  # activations and keys have a few channels far above the others
        return 1.0 + 7.0 * (torch.rand(n, generator=g, device=dev) < 0.02)

    kind = case["kind"]
    if kind in ("linear", "shared"):
        M, K, N = case["M"], case["K"], case["N"]
        d = dict(x=(normal(M, K) * channels(K)).to(t), w=[], ws=[], bias=[])
        for _ in range(case.get("products", 1)):
            d["w"].append(torch.randint(-127, 128, (K, N), generator=g, device=dev, dtype=torch.int8))
            d["ws"].append((0.5 + torch.rand(N, generator=g, device=dev)) / (73.0 * math.sqrt(K)))
            d["bias"].append(normal(N) if case["bias"] else None)
        return d
    if kind in ("write", "read"):
        T, H, D, page = case["T"], case["heads"], case["D"], case["page"]
        step = kind == "write" and T <= 256  # a token a page: a step of many sequences
        pages = (T if step else -(-T // page)) + 3
        order = torch.randperm(pages, generator=g, device=dev)
        if step:
            slots = order[:T] * page + torch.randint(0, page, (T,), generator=g, device=dev)
        else:
            at = torch.arange(T, device=dev)
            slots = order[at // page] * page + at % page
        qkv = normal(T, 3, H, D)
        qkv[:, 1] *= channels(H * D).view(H, D)
        qkv = qkv.to(t)
        k, v = (qkv[:, 1], qkv[:, 2]) if case.get("fused") else (qkv[:, 1].contiguous(), qkv[:, 2].contiguous())
        return dict(k=k, v=v, slots=slots, pages=pages)
    lens = _lengths(case)
    H, D, page = case["Hkv"], case["D"], case["page"]
    width = -(-case["length"] // page)
    need = [-(-n // page) for n, _ in lens]
    pages = sum(need) + 2
    order = torch.randperm(pages, generator=g, device=dev)
    table = torch.zeros(case["B"], width, dtype=torch.int32)
    at = 0
    for b, n in enumerate(need):
        table[b, :n] = torch.arange(at, at + n, dtype=torch.int32)
        at += n
    table = order.to(torch.int32)[table.to(dev).long()]
    starts = [0]
    for _, r in lens:
        starts.append(starts[-1] + r)
    q = (normal(starts[-1], case["Hq"], D) * 1.5).to(t)
    k = (normal(pages * page, H, D) * channels(H * D).view(H, D)).to(t)
    v = normal(pages * page, H, D).to(t)
    slopes = torch.tensor([2.0 ** (-8.0 * (h + 1) / case["Hq"]) for h in range(case["Hq"])], device=dev)
    return dict(q=q, k=k, v=v, pages=pages, table=table, lengths=torch.tensor([n for n, _ in lens], dtype=torch.int32).to(dev),
                starts=torch.tensor(starts, dtype=torch.int32).to(dev), slopes=slopes if case["slopes"] else None)


def prepare(case, seed):
    d = _inputs(case, seed)
    kind = case["kind"]
    if own:
        from iconnx_amd import ops
        if kind in ("linear", "shared"):
            w = [ops.TokenWeight(a, s) for a, s in zip(d["w"], d["ws"])]
            return dict(kind=kind, dtype=_T[case["dtype"]], x=d["x"], w=w, bias=d["bias"])
        cache = ops.KvCache(d["pages"], case["page"], case.get("heads") or case["Hkv"], case["D"], bits=case["bits"])
        if kind == "write":
            return dict(kind=kind, dtype=d["k"].dtype, cache=cache, k=d["k"], v=d["v"], slots=d["slots"])
        if kind == "read":
            ops.gpu_kv_cache_write(cache, d["k"], d["v"], d["slots"])
            return dict(kind=kind, dtype=d["k"].dtype, cache=cache, slots=d["slots"])
        ops.gpu_kv_cache_write(cache, d["k"], d["v"], torch.arange(len(d["k"]), device=d["k"].device))
    else:
        if kind in ("linear", "shared"):
            return dict(kind=kind, dtype=_T[case["dtype"]], x=d["x"], w=list(zip(d["w"], d["ws"])), bias=d["bias"])
        bits = case["bits"]
        if kind == "write":
            cache = [x for y in (d["k"], d["v"]) for x in _blank(y, d["pages"] * case["page"], bits)]
            return dict(kind=kind, bits=bits, dtype=d["k"].dtype, cache=cache, k=d["k"], v=d["v"], slots=d["slots"])
        cache = [x for y in (d["k"], d["v"]) for x in _encode(y, bits)]
        if kind == "read":
            cache = [torch.zeros((d["pages"] * case["page"],) + x.shape[1:], dtype=x.dtype, device=x.device).index_copy_(
                0, d["slots"], x) for x in cache]
            return dict(kind=kind, bits=bits, dtype=d["k"].dtype, cache=cache, slots=d["slots"])
    return dict(kind=kind, bits=case["bits"], page=case["page"], cache=cache, q=d["q"], table=d["table"], lengths=d["lengths"],
                starts=None if case["rows"] == 1 else d["starts"], rows=case["rows"], scale=case["D"] ** -0.5,
                softcap=case["softcap"], window=case["window"], slopes=d["slopes"])


# ---- the plain form -------------------------------------------------------------------------
def _tokens(x):
    x = x.double()  # the quotient decides between neighbouring bytes
    s = (x.abs().amax(-1).float() / 127.0).clamp_min(2.0 ** -126)
    return torch.round(x / s.double()[:, None]).float(), s


def _product(q, s, w, ws, bias, dtype):
    y = (q @ w.float()) * (s[:, None] * ws)
    return (y if bias is None else y + bias).to(dtype)


def _exponents(blocks, bits):
    m, e = torch.frexp(blocks.abs().amax(-1))  # max = m 2^e, m in [0.5, 1)
    if bits == 4:
        return (e - 3 + (m >= 0.875).int()).clamp(-125, 125)
    return (e - 9 + (m > 0.90625).int()).clamp(-117, 119)


def _encode(x, bits):
    """(codes uint8 [..., D / 2 or D], biased exponents uint8 [..., D / 32])"""
    b = x.float().unflatten(-1, (-1, 32))
    e = _exponents(b, bits)
    a = torch.ldexp(b.abs(), -e[..., None])
    if bits == 4:
        c = (a > 0.25).byte() + (a >= 0.75) + (a > 1.25) + (a >= 1.75) + (a > 2.5) + (a >= 3.5) + (a > 5.0)
        c = (c + 8 * (b < 0)).byte().flatten(-2)
        return c[..., 0::2] + 16 * c[..., 1::2], (e + 127).byte()
    step = (torch.frexp(a)[1] - 4).clamp_min(-9)  # the exponent of one step of the mantissa
    n = torch.round(torch.ldexp(a, -step)).int()
    c = (n + 8 * (step + 9)).clamp_max(126)
    return (c + 128 * (b < 0).int()).byte().flatten(-2), (e + 127).byte()


def _blank(x, n, bits):
    D = x.shape[-1]
    return (torch.zeros((n, x.shape[1], D * bits // 8), dtype=torch.uint8, device=x.device),
            torch.zeros((n, x.shape[1], D // 32), dtype=torch.uint8, device=x.device))


@functools.lru_cache(None)
def _magnitudes(bits, device):
    if bits == 4:
        t = [0.0, 0.5, 1.0, 1.5, 2.0, 3.0, 4.0, 6.0]
    else:
        t = [m / 512.0 if e == 0 else (8 + m) * 2.0 ** (e - 10) for e in range(16) for m in range(8)]
    return torch.tensor(t + [-x for x in t], device=device)


def _decode(codes, exps, bits):
    if bits == 4:
        codes = torch.stack([codes & 15, codes >> 4], -1).flatten(-2)
    v = _magnitudes(bits, codes.device)[codes.int()].unflatten(-1, (-1, 32))
    return torch.ldexp(v, exps.int()[..., None] - 127).flatten(-2)


def _attend(s):
    q, bits, page = s["q"], s["bits"], s["page"]
    B, width = s["table"].shape
    at = (s["table"].long()[:, :, None] * page + torch.arange(page, device=q.device)).flatten(1)
    L = at.shape[1]
    kc, ke, vc, ve = s["cache"]
    k = _decode(kc[at], ke[at], bits).transpose(1, 2)  # [B, Hkv, L, D]
    v = _decode(vc[at], ve[at], bits).transpose(1, 2)
    Hq, D = q.shape[1:]
    Hkv, R = k.shape[1], s["rows"]
    starts = torch.arange(B + 1, device=q.device) if s["starts"] is None else s["starts"].long()
    i = torch.arange(R, device=q.device)
    n = starts[1:] - starts[:-1]
    there = i < n[:, None]  # [B, R]: rows that are
    pick = (starts[:-1, None] + i).clamp_max(len(q) - 1)
    qp = q.float()[pick].view(B, R, Hkv, Hq // Hkv, D).permute(0, 2, 3, 1, 4).reshape(B, Hkv, -1, D)
    sc = ((qp * s["scale"]) @ k.transpose(2, 3)).view(B, Hq, R, L)
    if s["softcap"]:
        sc = s["softcap"] * torch.tanh(sc / s["softcap"])
    p = s["lengths"].long()[:, None] - n[:, None] + i  # [B, R]
    off = torch.arange(L, device=q.device) - p[:, :, None]  # [B, R, L]: j - p
    if s["slopes"] is not None:
        sc = sc + s["slopes"][:, None, None] * off[:, None].float()
    hidden = off > 0
    if s["window"]:
        hidden |= off <= -s["window"]
    sc = sc.masked_fill(hidden[:, None], -math.inf)
    w = torch.exp(sc - sc.amax(-1, keepdim=True))
    w = w / w.sum(-1, keepdim=True)
    w = w.nan_to_num(0.0)  # a row without tokens
    o = (w.view(B, Hkv, -1, L) @ v).view(B, Hq, R, D).permute(0, 2, 1, 3)
    return o[there].to(q.dtype)


def run(s):
    kind = s["kind"]
    if own:
        from iconnx_amd import ops
        if kind == "linear":
            return ops.gpu_token_qlinear(s["x"], s["w"][0], bias=s["bias"][0])
        if kind == "shared":
            q, scale = ops.gpu_quantize_tokens(s["x"])
            return [ops.gpu_token_qlinear(q, w, x_scale=scale, bias=b, dtype=s["dtype"]) for w, b in zip(s["w"], s["bias"])]
        if kind == "write":
            ops.gpu_kv_cache_write(s["cache"], s["k"], s["v"], s["slots"])
        if kind in ("write", "read"):
            return ops.gpu_kv_cache_read(s["cache"], s["slots"], dtype=s["dtype"])
        return ops.gpu_kv_cache_attention(s["q"], s["cache"], s["table"], s["lengths"], q_starts=s["starts"], max_rows=s["rows"],
                                          scale=s["scale"], softcap=s["softcap"], window=s["window"], slopes=s["slopes"])
    if kind in ("linear", "shared"):
        q, scale = _tokens(s["x"])
        y = [_product(q, scale, w, ws, b, s["dtype"]) for (w, ws), b in zip(s["w"], s["bias"])]
        return y[0] if kind == "linear" else y
    if kind == "write":
        for x, into in ((s["k"], s["cache"][:2]), (s["v"], s["cache"][2:])):
            for a, b in zip(into, _encode(x, s["bits"])):
                a.index_copy_(0, s["slots"], b)
    if kind in ("write", "read"):
        kc, ke, vc, ve = (a[s["slots"]] for a in s["cache"])
        return [_decode(kc, ke, s["bits"]).to(s["dtype"]), _decode(vc, ve, s["bits"]).to(s["dtype"])]
    return _attend(s)


# ---- the definitions in 64 bits ---------------------------------------------------------------
def _exact_cached(x, bits):
    """The values that a cache holds in the place of x: the nearest of the format's, by distance."""
    x = x.double()
    shape = x.shape
    b = x.reshape(-1, 32)
    top = b.abs().amax(1)
    if bits == 4:
        grid = [0, 0.5, 1, 1.5, 2, 3, 4, 6]
        limit, lo, hi = 7.0, -125, 125
        past = lambda r: r >= limit  # noqa: E731  (half way to the next magnitude goes there: its code is even)
    else:
        grid = [m / 8.0 * 2.0 ** -6 for m in range(8)] + [(1 + m / 8.0) * 2.0 ** e for e in range(-6, 9) for m in range(8)][:-1]
        limit, lo, hi = 464.0, -117, 119
        past = lambda r: r > limit  # noqa: E731
    e = torch.floor(torch.log2(top.clamp_min(1e-300) / limit)) - 1
    for _ in range(3):
        e = torch.where(past(top * torch.exp2(-e)), e + 1, e)
    e = e.clamp(lo, hi)
    a = (b.abs() * torch.exp2(-e)[:, None])
    grid = torch.tensor(grid, dtype=torch.float64, device=x.device)
    i = torch.searchsorted(grid, a).clamp(1, len(grid) - 1)  # grid[i - 1] < a <= grid[i]
    below, above = a - grid[i - 1], grid[i] - a
    i = torch.where((below < above) | ((below == above) & (i % 2 == 1)), i - 1, i)
    return (torch.sign(b) * grid[i] * torch.exp2(e)[:, None]).reshape(shape)


def exact(case, seed):
    d = _inputs(case, seed)
    if case["kind"] in ("linear", "shared"):
        x = d["x"].double()
        s = (x.abs().max(1).values / 127.0).float().double()
        s = torch.where(s < 2.0 ** -126, torch.full_like(s, 2.0 ** -126), s)
        q = (x / s.unsqueeze(1)).round()
        out = []
        for w, ws, b in zip(d["w"], d["ws"], d["bias"]):
            y = torch.mm(q, w.double()) * s.unsqueeze(1) * ws.double()
            out.append(y + b.double() if b is not None else y)
        return out[0] if case["kind"] == "linear" else out
    if case["kind"] in ("write", "read"):
        return [torch.cat([_exact_cached(c, case["bits"]) for c in x.split(4096)]) for x in (d["k"], d["v"])]
    out, at, page, group = [], 0, case["page"], case["Hq"] // case["Hkv"]
    for b, (n, rows) in enumerate(_lengths(case)):
        j = torch.arange(n, device=d["q"].device)
        slot = d["table"][b, j // page].long() * page + j % page
        p = n - rows + torch.arange(rows, device=j.device)
        seen = j[None, :] <= p[:, None]
        if case["window"]:
            seen &= j[None, :] > p[:, None] - case["window"]
        res = torch.zeros(rows, case["Hq"], case["D"], dtype=torch.float64, device=j.device)
        for g in range(case["Hkv"]):
            k, v = _exact_cached(d["k"][slot, g], case["bits"]), _exact_cached(d["v"][slot, g], case["bits"])
            for h in range(g * group, (g + 1) * group):
                t = torch.mm(d["q"][at:at + rows, h].double(), k.t()) * case["D"] ** -0.5
                if case["softcap"]:
                    t = torch.tanh(t / case["softcap"]) * case["softcap"]
                if d["slopes"] is not None:
                    t = t + d["slopes"][h].double() * (j[None, :] - p[:, None])
                res[:, h] = torch.mm(torch.softmax(torch.where(seen, t, float("-inf")), 1), v)
        out.append(res)
        at += rows
    return torch.cat(out)


# ---- what a pass cannot do without --------------------------------------------------------------
def work(case):
    size = 4 if case["dtype"] == "float32" else 2
    if case["kind"] in ("linear", "shared"):
        M, K, N, n = case["M"], case["K"], case["N"], case.get("products", 1)
        return {"bytes": M * K * size + n * (K * N + 4 * N * (2 if case["bias"] else 1) + M * N * size), "flops": 2 * M * K * N * n}
    if case["kind"] in ("write", "read"):
        n = 2 * case["T"] * case["heads"] * case["D"]
        held = n * case["bits"] // 8 + n // 32
        times = 2 if case["kind"] == "write" else 1
        return {"bytes": times * (n * size + held + 8 * case["T"]), "flops": 2 * n * times}
    D, tokens, pairs, total = case["D"], 0, 0, 0
    for n, rows in _lengths(case):
        w = case["window"] or n
        first = max(0, n - rows - w + 1)
        tokens += n - first
        pairs += sum(min(w, n - rows + i + 1) for i in range(rows))
        total += rows
    held = 2 * tokens * case["Hkv"] * (D * case["bits"] // 8 + D // 32)
    return {"bytes": held + 2 * total * case["Hq"] * D * size, "flops": 4 * pairs * case["Hq"] * D}
