"""The quantised KV cache (its writers, its read-back) and the attention that reads caches for single tokens and for
trees of drafted tokens: each operator's plain form, the framework's call, and cases to time and compare them on.

A cache row is one token of one KV head. e4m3 rows have a power-of-two scale 2^E, E the smallest integer >= -126 with
max|x| <= 448 * 2^E, and codes x * 2^-E rounded to e4m3; int8 rows have the scale d / 127, d = max(max|x|, 127 * 2^-126),
and codes 127 x / d rounded half to even. Codes lie in [blocks, block_size, Hkv, D], scales in [blocks, Hkv, block_size].
"""
import math
import os
import random
import sys

import torch

# The package's folder, so that `import nanovllm_b200` works from a checkout.
sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "nano-vllm-triton-kernels_b200"))

own = False

E4M3, INT8 = torch.float8_e4m3fn, torch.int8
DTYPES = {"bf16": torch.bfloat16, "fp16": torch.float16, "e4m3": E4M3, "int8": INT8}


# ---------------------------------------------------------------------------------------------------------------
# Cases.

def listed():
    return [
        # The cache write of one decode step: 32 sequences, one token each (Qwen3-0.6B's 8 KV heads).
        dict(name="store_decode32", op="store", T=32, hkv=8, d=128, dtype="bf16", cache="e4m3", bs=256),
        # The cache write of a long prefill, an odd number of tokens, fp16 model.
        dict(name="store_prefill", op="store", T=8191, hkv=8, d=128, dtype="fp16", cache="e4m3", bs=256),
        # Chunked prefill: the chunk's keys and values are written, then each sequence's whole context is read back
        # for the prefill attention.
        dict(name="chunk_int8", op="store_load", B=6, new=341, L=5000, hkv=8, d=128, dtype="bf16", cache="int8", bs=64),
        # Read-back of long shared prefixes, ragged.
        dict(name="load_prefix", op="load", B=16, L=11000, hkv=8, d=128, dtype="bf16", cache="e4m3", bs=256),
        # Fused norm + rotation + quantising write: a decode step (Qwen3-0.6B) and a prefill (Qwen3-8B heads).
        dict(name="fused_decode32", op="fused", T=32, hq=16, hkv=8, d=128, cache="e4m3", bs=256),
        dict(name="fused_prefill", op="fused", T=8192, hq=32, hkv=8, d=128, cache="e4m3", bs=256),
        # Decode attention: one short chat; the framework's decode step (32 sequences of 1024 keys); ragged long
        # contexts on an int8 cache.
        dict(name="decode_single", op="decode", B=1, L=611, ragged=False, hq=16, hkv=8, d=128, dtype="bf16", cache="e4m3", bs=256),
        dict(name="decode_step", op="decode", B=32, L=1024, ragged=False, hq=16, hkv=8, d=128, dtype="bf16", cache="e4m3", bs=256),
        dict(name="decode_long", op="decode", B=24, L=32768, ragged=True, hq=32, hkv=8, d=128, dtype="bf16", cache="int8", bs=64),
        # Verifying trees of drafted tokens: 8 drafts of one chat on the plain cache, 16 drafts (ragged) for a batch
        # on the quantised cache, large trees over long contexts on the plain cache.
        dict(name="tree_single", op="tree", B=1, n=8, L=777, ragged=False, hq=16, hkv=8, d=128, dtype="bf16", cache="bf16", bs=256),
        dict(name="tree_batch", op="tree", B=32, n=16, L=2048, ragged=True, hq=32, hkv=8, d=128, dtype="bf16", cache="e4m3", bs=256),
        dict(name="tree_large", op="tree", B=8, n=64, L=16384, ragged=True, hq=32, hkv=8, d=128, dtype="bf16", cache="bf16", bs=256),
    ]


def _log(rng, lo, hi):
    return int(round(math.exp(rng.uniform(math.log(lo), math.log(hi)))))


def draw(rng: random.Random):
    op = rng.choice(["store", "store_load", "load", "fused", "decode", "decode", "tree", "tree"])
    hkv, d = rng.choice([1, 2, 4, 8]), rng.choice([64, 128, 128])
    quant = rng.choice(["e4m3", "int8"])
    dtype = rng.choice(["bf16", "bf16", "fp16"])
    bs = rng.choice([16, 32, 64, 80, 256])
    if op == "store":
        return dict(op=op, T=_log(rng, 1, 8191), hkv=hkv, d=d, dtype=dtype, cache="e4m3", bs=bs)
    if op == "store_load":
        L = _log(rng, 2, 5000)
        return dict(op=op, B=_log(rng, 1, 6), new=_log(rng, 1, L), L=L, hkv=hkv, d=d, dtype=dtype, cache=quant, bs=bs)
    if op == "load":
        return dict(op=op, B=_log(rng, 1, 16), L=_log(rng, 1, 11000), hkv=hkv, d=d, dtype=dtype, cache=quant, bs=bs)
    if op == "fused":
        return dict(op=op, T=_log(rng, 1, 8192), hq=hkv * rng.choice([1, 2, 4]), hkv=hkv, d=d, cache="e4m3", bs=bs)
    group = rng.choice([1, 2, 4, 8])
    c = dict(op=op, B=_log(rng, 1, 64), n=1, L=1, ragged=rng.random() < 0.7, hq=hkv * group, hkv=hkv, d=d, dtype=dtype,
             cache=quant, bs=bs)
    if op == "tree":
        c["n"] = rng.randint(2, 64)
        c["cache"] = rng.choice([dtype, quant])
    else:
        del c["n"]
    n = c.get("n", 1)
    most = min(32768, 400000 // c["B"], 1000000 // (c["B"] * hkv), 150000000 // (c["B"] * n * c["hq"]))
    c["L"] = _log(rng, n, max(n + 1, most))
    return c


# ---------------------------------------------------------------------------------------------------------------
# Inputs.

def _lengths(c):
    """Tokens in the cache of each sequence: the case's own, the same for every seed. The first is the longest."""
    rng = random.Random(repr(sorted((k, v) for k, v in c.items() if k != "name")))
    n, L = c.get("n", 1), c["L"]
    if c["op"] in ("load", "store_load"):
        return [L] + [rng.randint(max(1, L // 4), L) for _ in range(c["B"] - 1)]
    return [L] + [rng.randint(max(n, L // 8), L) if c["ragged"] else L for _ in range(c["B"] - 1)]


def _rows(gen, n, hkv, d, dtype):
    """Keys or values: unit normals under a token-and-head magnitude and a few louder channels, as projections give."""
    x = torch.randn(n, hkv, d, device="cuda", generator=gen)
    x *= torch.exp(0.5 * torch.randn(n, hkv, 1, device="cuda", generator=gen))
    x *= 1 + 4 * (torch.rand(d, device="cuda", generator=gen) < 0.03)
    return x.to(dtype)


def _pages(rng, lens, bs):
    """Block tables over a shuffled pool of pages, and the pool's size."""
    need = [max(1, -(-n // bs)) for n in lens]
    pool = list(range(sum(need) + 2))
    rng.shuffle(pool)
    width, table, at = max(need), [], 0
    for k in need:
        table.append(pool[at:at + k] + [0] * (width - k))
        at += k
    return torch.tensor(table, dtype=torch.int32, device="cuda"), len(pool)


def _filled_cache(gen, blocks, bs, hkv, d, dtype):
    """A cache (and scales) whose every slot holds rows of _rows."""
    if dtype not in (E4M3, INT8):
        return _rows(gen, blocks * bs, hkv, d, dtype).view(blocks, bs, hkv, d), None
    codes, scale = _quantise(_rows(gen, blocks * bs, hkv, d, torch.bfloat16), dtype)
    return codes.view(blocks, bs, hkv, d), scale.view(blocks, bs, hkv).transpose(1, 2).contiguous()


def _trees(rng, B, n):
    """Ancestor masks [B, n, n] of random trees: token i's parent is an earlier token (or the context), and it sees
    its ancestors and itself."""
    parent = torch.tensor([[rng.randint(max(-1, i - 6), i - 1) for i in range(n)] for _ in range(B)]).reshape(B, n)
    mask = torch.zeros(B, n, n, dtype=torch.bool)
    every = torch.arange(B)
    for i in range(n):
        has = parent[:, i] >= 0
        mask[:, i] = mask[every, parent[:, i].clamp(min=0)] & has[:, None]
        mask[:, i, i] = True
    return mask.cuda()


def prepare(case, seed):
    c = case
    gen = torch.Generator(device="cuda").manual_seed(seed)
    rng = random.Random(seed * 7919 + 1)
    s = dict(op=c["op"], cache=c["cache"])
    hkv, d, bs = c["hkv"], c["d"], c["bs"]
    cdt = DTYPES[c["cache"]]
    if c["op"] in ("store", "fused"):
        T = c["T"]
        blocks = -(-T // bs) + 1
        slots = torch.randperm(blocks * bs, device="cuda", generator=gen)[:T].to(torch.int32)
        if T >= 20:
            slots[torch.randperm(T, device="cuda", generator=gen)[:T // 20]] = -1
        s |= dict(slots=slots, k_cache=torch.zeros(blocks, bs, hkv, d, device="cuda").to(cdt),
                  v_cache=torch.zeros(blocks, bs, hkv, d, device="cuda").to(cdt),
                  k_scale=torch.zeros(blocks, hkv, bs, device="cuda"), v_scale=torch.zeros(blocks, hkv, bs, device="cuda"))
        if c["op"] == "store":
            s |= dict(k=_rows(gen, T, hkv, d, DTYPES[c["dtype"]]), v=_rows(gen, T, hkv, d, DTYPES[c["dtype"]]))
            return s
        hq = c["hq"]
        qkv = torch.randn(T, (hq + 2 * hkv) * d, device="cuda", generator=gen).to(torch.bfloat16)
        q, k, v = qkv.split([hq * d, hkv * d, hkv * d], dim=-1)
        pos = torch.arange(8192, device="cuda", dtype=torch.float64)
        ang = pos[:, None] * 1e6 ** (-torch.arange(0, d, 2, device="cuda", dtype=torch.float64) / d)
        s |= dict(q=q.view(T, hq, d), k=k.view(T, hkv, d), v=v.view(T, hkv, d),
                  positions=torch.randint(0, 8192, (T,), device="cuda", generator=gen),
                  q_w=(1 + 0.1 * torch.randn(d, device="cuda", generator=gen)).to(torch.bfloat16),
                  k_w=(1 + 0.1 * torch.randn(d, device="cuda", generator=gen)).to(torch.bfloat16), eps=1e-6,
                  cos_sin=torch.cat([ang.cos(), ang.sin()], -1).float().unsqueeze(1))
        return s
    B, n = c["B"], c.get("n", 1)
    lens = _lengths(c)
    table, blocks = _pages(rng, lens, bs)
    s["table"] = table
    s["k_cache"], s["k_scale"] = _filled_cache(gen, blocks, bs, hkv, d, cdt)
    s["v_cache"], s["v_scale"] = _filled_cache(gen, blocks, bs, hkv, d, cdt)
    if c["op"] in ("load", "store_load"):
        s["cu"] = torch.tensor([0] + lens, device="cuda").cumsum(0).to(torch.int32)
        s["total"], s["dtype"] = sum(lens), DTYPES[c["dtype"]]
        if c["op"] == "store_load":
            new = [min(c["new"], m) for m in lens]
            at = [(b, j) for b in range(B) for j in range(lens[b] - new[b], lens[b])]
            bb, jj = (torch.tensor(x, device="cuda") for x in zip(*at))
            s["slots"] = (table[bb, jj // bs].long() * bs + jj % bs).to(torch.int32)
            s["k"] = _rows(gen, len(at), hkv, d, s["dtype"])
            s["v"] = _rows(gen, len(at), hkv, d, s["dtype"])
        return s
    s["lens"] = torch.tensor(lens, dtype=torch.int32, device="cuda")
    # Queries of norm about sqrt(d), as normalised heads have; softmax over scores of a few units.
    s["q"] = torch.randn(B, n, c["hq"], d, device="cuda", generator=gen).to(DTYPES[c["dtype"]])
    s["softmax_scale"] = d ** -0.5
    if c["op"] == "tree":
        s["mask"] = _trees(rng, B, n)
        s["drafts"] = torch.tensor([n] + [rng.randint(1, n) if c["ragged"] else n for _ in range(B - 1)],
                                   dtype=torch.int32, device="cuda")
    return s


# ---------------------------------------------------------------------------------------------------------------
# Plain forms, in 32 bits.

def _quantise(x, dtype):
    """Codes and scales of rows x [..., d]."""
    x = x.float()
    a = x.abs().amax(-1)
    if dtype == E4M3:
        m, e = torch.frexp(a)
        e = torch.where(m <= 0.875, e - 9, e - 8)  # 448 = 0.875 * 2^9
        e = torch.where(a == 0, torch.full_like(e, -126), e.clamp(min=-126))
        scale = torch.ldexp(torch.ones_like(a), e)
        codes = x * torch.ldexp(torch.ones_like(a), -e)[..., None]
    else:
        den = a.clamp(min=127 * 2.0 ** -126)
        scale = den / 127
        h = torch.where(den > 2.0 ** 100, 2.0 ** -8, 1.0)  # keeps 127 x below the largest fp32
        codes = torch.round((x * h[..., None] * 127) / (den * h)[..., None])
    good = torch.isfinite(a)
    codes = torch.where(good[..., None], codes, torch.zeros_like(codes))
    return codes.to(dtype), torch.where(good, scale, torch.full_like(scale, math.nan))


def _put(cache, scale, slots, codes, row_scale):
    keep = slots >= 0
    at = slots[keep].long()
    blocks, bs, hkv, d = cache.shape
    cache.view(torch.uint8).view(blocks * bs, hkv, d)[at] = codes[keep].view(torch.uint8)
    scale.view(blocks, hkv, bs)[at // bs, :, at % bs] = row_scale[keep]


def _store(s):
    for x, name in (("k", "k"), ("v", "v")):
        codes, scale = _quantise(s[x], s[name + "_cache"].dtype)
        _put(s[name + "_cache"], s[name + "_scale"], s["slots"], codes, scale)


def _load(s):
    cu = s["cu"].long()
    t = torch.arange(s["total"], device=cu.device)
    b = torch.searchsorted(cu, t, right=True) - 1
    j = t - cu[b]
    bs = s["k_cache"].shape[1]
    page = s["table"][b, j // bs].long()
    out = []
    for name in ("k", "v"):
        rows = s[name + "_cache"].view(torch.uint8)[page, j % bs].view(s[name + "_cache"].dtype).float()
        out.append((rows * s[name + "_scale"][page, :, j % bs][..., None]).to(s["dtype"]))
    return out


def _norm_rope(x, w, positions, cos_sin, eps):
    x = x.float()
    x = x * torch.rsqrt((x * x).mean(-1, keepdim=True) + eps)
    x = (x.to(torch.bfloat16).float() * w.float()).to(torch.bfloat16).float()
    cos, sin = cos_sin[positions].chunk(2, -1)
    x1, x2 = x.chunk(2, -1)
    return torch.cat([x1 * cos - x2 * sin, x2 * cos + x1 * sin], -1).to(torch.bfloat16)


def _gather(s, name):
    cache, scale, table = s[name + "_cache"], s[name + "_scale"], s["table"].long()
    B, width = table.shape
    _, bs, hkv, d = cache.shape
    if scale is None:
        return cache[table].view(B, width * bs, hkv, d).float()
    rows = cache.view(torch.uint8)[table].view(cache.dtype).float()
    return (rows * scale[table].transpose(2, 3)[..., None]).view(B, width * bs, hkv, d)


def _attention(s):
    q = s["q"].float()
    B, n, hq, d = q.shape
    k, v = _gather(s, "k"), _gather(s, "v")
    hkv, keys = k.shape[2], k.shape[1]
    at = torch.arange(keys, device=q.device)
    lens = s["lens"].long()
    drafts = s["drafts"].long() if "drafts" in s else torch.full_like(lens, n)
    rel = at[None, :] - (lens - drafts)[:, None]                       # [B, keys]: index among the drafted tokens
    if "mask" in s:
        cols = rel.clamp(0, n - 1)[:, None, :].expand(B, n, keys)
        seen = torch.gather(s["mask"], 2, cols) | (rel < 0)[:, None, :]
        seen &= (torch.arange(n, device=q.device)[None, :] < drafts[:, None])[..., None]
    else:
        seen = rel[:, None, :] <= torch.arange(n, device=q.device)[None, :, None]
    seen &= (at[None, :] < lens[:, None])[:, None, :]
    qh = q.view(B, n, hkv, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(B, hkv, -1, d)
    scores = torch.matmul(qh * s["softmax_scale"], k.permute(0, 2, 3, 1)).view(B, hkv, n, hq // hkv, keys)
    scores = torch.where(seen[:, None, :, None, :], scores, torch.full_like(scores, -math.inf))
    m = scores.amax(-1, keepdim=True)
    p = torch.exp(scores - torch.where(m == -math.inf, torch.zeros_like(m), m))
    total = p.sum(-1, keepdim=True)
    p = p / torch.where(total > 0, total, torch.ones_like(total))
    out = torch.matmul(p.view(B, hkv, -1, keys), v.permute(0, 2, 1, 3))
    return out.view(B, hkv, n, hq // hkv, d).permute(0, 2, 1, 3, 4).reshape(B, n, hq, d).to(s["q"].dtype)


def run(s):
    op = s["op"]
    if own:
        from nanovllm_b200 import (decode_attention_quant, load_kvcache_quant, qk_norm_rope_kv_quant, store_kvcache_quant,
                                   tree_attention)
        cache = [s[x] for x in ("k_cache", "v_cache", "k_scale", "v_scale")]
        if op == "store":
            store_kvcache_quant(s["k"], s["v"], *cache, s["slots"])
            return cache
        if op == "store_load":
            store_kvcache_quant(s["k"], s["v"], *cache, s["slots"])
        if op in ("load", "store_load"):
            return load_kvcache_quant(*cache, s["table"], s["cu"], s["total"], dtype=s["dtype"])
        if op == "fused":
            q, _ = qk_norm_rope_kv_quant(s["q"], s["k"], s["v"], s["positions"], s["q_w"], s["k_w"], s["eps"],
                                         s["cos_sin"], *cache, s["slots"], False)
            return [q] + cache
        if op == "decode":
            return decode_attention_quant(s["q"], *cache, s["lens"], block_table=s["table"],
                                          softmax_scale=s["softmax_scale"], causal=True)
        return tree_attention(s["q"], s["k_cache"], s["v_cache"], s["lens"], s["mask"], block_table=s["table"],
                              draft_lens=s["drafts"], softmax_scale=s["softmax_scale"], k_scale=s["k_scale"],
                              v_scale=s["v_scale"])
    cache = [s[x] for x in ("k_cache", "v_cache", "k_scale", "v_scale")]
    if op == "store":
        _store(s)
        return cache
    if op == "store_load":
        _store(s)
    if op in ("load", "store_load"):
        return _load(s)
    if op == "fused":
        q = _norm_rope(s["q"], s["q_w"], s["positions"], s["cos_sin"], s["eps"])
        k = _norm_rope(s["k"], s["k_w"], s["positions"], s["cos_sin"], s["eps"])
        _store(dict(s, k=k))
        return [q] + cache
    return _attention(s)


# ---------------------------------------------------------------------------------------------------------------
# What a pass cannot do without.

def work(case):
    c = case
    hkv, d = c["hkv"], c["d"]
    quant = c["cache"] in ("e4m3", "int8")
    row = 2 * hkv * (d + 4) if quant else 2 * hkv * d * 2  # a token's K and V in the cache
    plain = 2 * hkv * d * 2                                 # and outside it, in 16 bits
    if c["op"] == "store":
        return {"bytes": c["T"] * (plain + row + 4), "flops": 4 * c["T"] * hkv * d}
    if c["op"] == "fused":
        heads = c["hq"] + 2 * hkv
        return {"bytes": c["T"] * (heads * d * 2 + c["hq"] * d * 2 + row + 12 + 4 * d), "flops": 12 * c["T"] * heads * d}
    lens = _lengths(c)
    tokens = sum(lens)
    if c["op"] in ("load", "store_load"):
        new = sum(min(c["new"], m) for m in lens) if c["op"] == "store_load" else 0
        return {"bytes": tokens * (row + plain) + new * (plain + row), "flops": 2 * tokens * hkv * d}
    rows = c.get("n", 1) * c["hq"]
    return {"bytes": tokens * row + 2 * c["B"] * rows * d * 2, "flops": 4 * tokens * rows * d}


# ---------------------------------------------------------------------------------------------------------------
# The same results in 64 bits, from the definitions.

def _exact_row_codes(x, cache):
    x = x.double()
    a = x.abs().amax(-1, keepdim=True)
    if cache == "int8":
        d = a.clamp(min=127 * 2.0 ** -126)
        return torch.round(127 * x / d), d / 127
    e = torch.ceil(torch.log2(a / 448)).clamp(min=-126)
    e = torch.where(a > 448 * torch.exp2(e), e + 1, e)
    e = torch.where((a <= 448 * torch.exp2(e - 1)) & (e > -126), e - 1, e)
    y = x / torch.exp2(e)
    # Steps of e4m3: 2^-9 below 2^-6, an eighth of the power of two below |y| above it.
    step = torch.exp2(torch.floor(torch.log2(y.abs().clamp(min=2.0 ** -6))) - 3)
    return torch.round(y / step) * step, torch.exp2(e)


def exact(case, seed):
    s = prepare(case, seed)
    op, cache = s["op"], s["cache"]
    bs = case["bs"]
    if op in ("store", "fused", "store_load"):
        k, v = s["k"].double(), s["v"].double()
        q = None
        if op == "fused":
            cos, sin = s["cos_sin"][s["positions"]].double().chunk(2, -1)

            def turned(x, w):
                x = x.double()
                x = x / torch.sqrt((x ** 2).sum(-1, keepdim=True) / x.shape[-1] + s["eps"]) * w.double()
                a, b = x[..., :x.shape[-1] // 2], x[..., x.shape[-1] // 2:]
                return torch.cat([a * cos - b * sin, b * cos + a * sin], -1)
            q, k = turned(s["q"], s["q_w"]), turned(s["k"], s["k_w"])
        filled = []
        for x, name in ((k, "k"), (v, "v")):
            codes = s[name + "_cache"].to(torch.float32).double()
            scale = s[name + "_scale"].double()
            c, sc = _exact_row_codes(x, cache)
            for t, slot in enumerate(s["slots"].tolist()) if len(s["slots"]) <= 64 else ():
                if slot >= 0:
                    codes[slot // bs, slot % bs], scale[slot // bs, :, slot % bs] = c[t], sc[t, :, 0]
            if len(s["slots"]) > 64:
                on = torch.nonzero(s["slots"] >= 0).flatten()
                at = s["slots"][on].long()
                codes[torch.div(at, bs, rounding_mode="floor"), torch.remainder(at, bs)] = c[on]
                scale.transpose(1, 2)[torch.div(at, bs, rounding_mode="floor"), torch.remainder(at, bs)] = sc[on, :, 0]
            filled.append((codes, scale))
        (kc, ks), (vc, vs) = filled
        if op == "store":
            return [kc, vc, ks, vs]
        if op == "fused":
            # The stored rows are quantised from bf16 values, so a code's exact value depends on that rounding.
            return [q, None, vc, None, vs]
    if op in ("load", "store_load"):
        if op == "load":
            filled = [(s[x + "_cache"].to(torch.float32).double(), s[x + "_scale"].double()) for x in ("k", "v")]
        out = []
        cu = s["cu"].tolist()
        for codes, scale in filled:
            values = codes * scale.transpose(1, 2)[..., None]
            parts = []
            for b in range(len(cu) - 1):
                m = cu[b + 1] - cu[b]
                parts.append(values[s["table"][b].long()].flatten(0, 1)[:m])
            out.append(torch.cat(parts))
        return out
    # Attention, one sequence at a time, keys in the order of the context.
    q = s["q"].double()
    B, n, hq, d = q.shape
    out = torch.zeros_like(q)
    for b, L in enumerate(s["lens"].tolist()):
        kv = []
        for name in ("k", "v"):
            pages = s["table"][b].long()
            x = s[name + "_cache"].view(torch.uint8)[pages].view(s[name + "_cache"].dtype).double()
            if s[name + "_scale"] is not None:
                x = x * s[name + "_scale"][pages].double().transpose(1, 2)[..., None]
            kv.append(x.flatten(0, 1)[:L])
        hkv = kv[0].shape[1]
        k, v = (x.repeat_interleave(hq // hkv, 1) for x in kv)
        m = int(s["drafts"][b]) if "drafts" in s else n
        see = torch.ones(m, L, dtype=torch.bool, device=q.device)
        see[:, L - m:] = s["mask"][b, :m, :m] if "mask" in s else torch.ones(m, m, device=q.device).tril().bool()
        scores = torch.einsum("ihd,khd->hik", q[b, :m], k) * s["softmax_scale"]
        p = torch.softmax(scores.masked_fill(~see, -math.inf), -1)
        out[b, :m] = torch.einsum("hik,khd->ihd", p, v)
    return out
