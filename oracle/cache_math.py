"""Plain implementations, in 64 bits, of the 8-bit KV cache and of attention with a tree mask over a paged cache.

TEST INFRASTRUCTURE ONLY. Written from the definitions in include/nvb200.h, apart from the kernels; the reference has no
counterpart (its cache is 16-bit and its drafts are linear).
"""
import math

import torch


def quantise_rows(x: torch.Tensor, dtype: torch.dtype):
    """Codes (dtype, x's shape) and fp32 scales (x.shape[:-1]) of rows x [..., d] of bf16, fp16 or fp32 elements."""
    x = x.double()
    a = x.abs().amax(-1)  # NaN where the row has one
    good = torch.isfinite(a)
    a = torch.where(good, a, torch.zeros_like(a))
    y = torch.where(good[..., None], x, torch.zeros_like(x))
    if dtype == torch.int8:
        d = a.clamp(min=127 * 2.0 ** -126)
        scale = d.float() / 127  # one fp32 division
        codes = torch.round(127 * y / d[..., None])  # 127 y is exact; no quotient that is not a tie rounds to one
    else:
        m, e = torch.frexp(a)  # a = m 2^e, m in [0.5, 1); 448 = 0.875 * 2^9
        e = torch.where(m <= 0.875, e - 9, e - 8)
        e = torch.where(a == 0, torch.full_like(e, -126), e.clamp(min=-126)).double()
        scale = torch.exp2(e).float()
        z = y * torch.exp2(-e)[..., None]
        step = torch.exp2(torch.floor(torch.log2(z.abs().clamp(min=2.0 ** -6))) - 3)  # e4m3: 3 bits, 2^-9 at the bottom
        codes = torch.round(z / step) * step
    scale = torch.where(good, scale, torch.full_like(scale, math.nan))
    return codes.float().to(dtype), scale


def row_values(codes: torch.Tensor, scale: torch.Tensor) -> torch.Tensor:
    """fp64 values of an 8-bit cache [blocks, block_size, Hkv, D] with scales [blocks, Hkv, block_size]."""
    return codes.float().double() * scale.double().transpose(1, 2)[..., None]


def cache_attention(q, k, v, lens, table, mask, drafts, scale, causal=True):
    """q [B, n, Hq, D]; k, v [blocks, block_size, Hkv, D] in any type (row_values for 8-bit caches); lens, drafts: lists.
    mask: bool [B, n, n] or None (causal: the chain, else every key). Returns (out, sum_j p_j |v_j|, the largest
    sum_d |q_d k_jd| scale of the row's keys [B, n, Hq, 1]) in fp64.
    A key that a row does not see is left out of its sums."""
    B, n, hq, d = q.shape
    hkv = k.shape[2]
    out = torch.zeros(B, n, hq, d, dtype=torch.float64, device=q.device)
    spread, reach = torch.zeros_like(out), torch.zeros_like(out[..., :1])
    for b in range(B):
        L, m = int(lens[b]), int(drafts[b])
        if table is None:
            kk, vv = k[b, :L].double(), v[b, :L].double()
        else:
            bs = k.shape[1]
            pages = table[b, :(L + bs - 1) // bs].long()
            kk, vv = (x[pages].reshape(-1, hkv, d)[:L].double() for x in (k, v))
        for i in range(m):
            j = torch.arange(L, device=q.device)
            rel = j - (L - m)
            if mask is not None:
                see = (rel < 0) | mask[b, i, rel.clamp(0, n - 1)]
            else:
                see = (rel <= i) if causal else torch.ones_like(rel, dtype=torch.bool)
            if not bool(see.any()):
                continue
            ks = kk[see].repeat_interleave(hq // hkv, 1)  # [keys, Hq, D]
            vs = vv[see].repeat_interleave(hq // hkv, 1)
            qi = q[b, i].double()
            s = torch.einsum("hd,khd->hk", qi, ks) * scale
            p = torch.softmax(s, -1)
            out[b, i] = torch.einsum("hk,khd->hd", p, vs)
            spread[b, i] = torch.einsum("hk,khd->hd", p, vs.abs())
            reach[b, i, :, 0] = torch.einsum("hd,khd->hk", qi.abs(), ks.abs()).amax(-1) * abs(scale)
    return out, spread, reach
