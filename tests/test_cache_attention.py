"""tree_attention and decode_attention_quant (nanovllm_b200.kernels.cache_attention) against the 64-bit oracle.

Tolerance, per output element, from the roundings the kernel makes (u = half a step: bf16 2^-8, fp16 2^-11):
  * the output: u |out|;
  * each weight, rounded to the type the matrix instructions take: u_w sum_j p_j |v_j|, u_w = 2^-8 for bf16 caches and 2^-11
    for fp16 and 8-bit ones, and for those fp16's smallest step: each weight is off by at most 2^-25 of the largest possible
    weight, which is at most 4 times the largest one there is, over `keys` keys of at most max|v|: 2^-23 keys max|v|;
  * each score: fp32 sums of D products, with up to 8 more roundings of the score: (D + 8) 2^-24 max_j sum_d |q_d k_jd| scale,
    as a relative error of a weight, twice (numerator and sum): 2 of them times sum_j p_j |v_j|;
  * 2^-18 sum_j p_j |v_j| for exp2 and the fp32 sums of weights and outputs.
"""
import ctypes
import os
import shutil
import subprocess

import pytest
import torch

from oracle import cache_math as cm
from oracle import reference_math as om

E4M3, I8, B16, H16 = torch.float8_e4m3fn, torch.int8, torch.bfloat16, torch.float16


def _tolerance(ref, spread, reach, qdt, cdt, keys, vmax, d):
    u = 2.0 ** -8 if qdt == B16 else 2.0 ** -11
    uw = 2.0 ** -8 if cdt == B16 else 2.0 ** -11
    tol = u * ref.abs() + spread * (uw + 2.0 ** -18 + 2 * (d + 8) * 2.0 ** -24 * reach)
    if cdt != B16:
        tol = tol + 2.0 ** -23 * keys * vmax * (spread > 0)
    return tol + 1e-30


def _problem(B, n, lens, hq, hkv, d, bs, qdt, cdt, device, seed=0, drafts=None, mask="tree", paged=True):
    g = torch.Generator().manual_seed(seed)
    pages = max(1, max(-(-L // bs) for L in lens)) if paged else 1
    blocks = B * pages + 2 if paged else B
    if not paged:
        bs = max(1, max(lens))
    shape = (blocks, bs, hkv, d)
    if cdt in (E4M3, I8):
        codes = [torch.randint(-127, 128, shape, generator=g) for _ in range(2)]
        codes = [c.to(I8) if cdt == I8 else c.float().to(E4M3) for c in codes]
        sc = [torch.exp(torch.randn(blocks, hkv, bs, generator=g) - 4) for _ in range(2)]
        if cdt == E4M3:
            sc = [torch.exp2(torch.round(torch.log2(s))) for s in sc]
        kv = [cm.row_values(c, s) for c, s in zip(codes, sc)]
        cache = [x.to(device) for x in codes + sc]
    else:
        codes = [torch.randn(shape, generator=g).to(cdt) for _ in range(2)]
        kv, cache = codes, [x.to(device) for x in codes] + [None, None]
    q = torch.randn(B, n, hq, d, generator=g).to(qdt)
    table = torch.randperm(blocks, generator=g)[:B * pages].view(B, pages).int() if paged else None
    m = None
    if mask == "tree":
        m = torch.rand(B, n, n, generator=g) < 0.4
        if n > 1:
            m[:, n - 1] = False  # a row that sees the context only (or nothing)
    drafts = [n] * B if drafts is None else drafts
    return q, kv, cache, table, m, drafts


def _check(got, q, kv, table, lens, m, drafts, scale, cdt, causal=True):
    ref, spread, reach = cm.cache_attention(q, kv[0], kv[1], lens, table, m, drafts, scale, causal)
    vmax = float(torch.nan_to_num(kv[1].double(), 0, 0, 0).abs().max())
    tol = _tolerance(ref, spread, reach, q.dtype, cdt, max(lens), vmax, q.shape[-1])
    err = (got.double().cpu() - ref).abs()
    assert got.dtype == q.dtype and bool((err <= tol).all()), float((err / tol).max())


# ---------------------------------------------------------------------------------------------------------------
# CPU.

def test_oracle_chain_is_the_decode_oracle():
    g = torch.Generator().manual_seed(0)
    q, kc, vc = (torch.randn(s, generator=g) for s in ((2, 3, 4, 64), (8, 16, 2, 64), (8, 16, 2, 64)))
    table = torch.randperm(8, generator=g)[:4].view(2, 2).int()
    lens = torch.tensor([20, 2], dtype=torch.int32)
    a = om.paged_decode_attention(q, kc, vc, lens, table, 0.1, True)
    chain = torch.ones(3, 3).tril().bool()[None].expand(2, 3, 3)
    for mask in (None, chain):
        b, _, _ = cm.cache_attention(q, kc, vc, [20, 2], table, mask, [3, 3], 0.1)
        assert torch.allclose(a.double(), b, atol=1e-6)


@pytest.mark.skipif(shutil.which("gcc") is None, reason="gcc not available")
@pytest.mark.parametrize("name", ["CacheAttentionArgs", "QuantCache"])
def test_struct_layout_matches_header(tmp_path, name):
    from nanovllm_b200 import _lib
    ctype = getattr(_lib, name)
    cname = {"CacheAttentionArgs": "nvb200_cache_attention_args", "QuantCache": "nvb200_quant_cache"}[name]
    fields = [f[0] for f in ctype._fields_]
    src = tmp_path / "layout.c"
    body = "\n".join(f'  printf("{f} %zu\\n", offsetof({cname}, {f}));' for f in fields)
    src.write_text('#include <stddef.h>\n#include <stdio.h>\n#include "nvb200.h"\nint main(void) {\n' + body +
                   f'\n  printf("sizeof %zu\\n", sizeof({cname}));\n  return 0;\n}}\n')
    include = os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))), "include")
    subprocess.run(["gcc", "-I", include, str(src), "-o", str(tmp_path / "layout")], check=True)
    out = dict(x.split() for x in subprocess.run([str(tmp_path / "layout")], capture_output=True, text=True,
                                                 check=True).stdout.splitlines())
    assert all(int(out[f]) == getattr(ctype, f).offset for f in fields) and int(out["sizeof"]) == ctypes.sizeof(ctype)


def test_refusals():
    from nanovllm_b200 import decode_attention_quant, tree_attention
    q = torch.zeros(1, 2, 4, 64, dtype=B16)
    kc = torch.zeros(3, 16, 2, 64, dtype=B16)
    lens, table = torch.ones(1, dtype=torch.int32), torch.zeros(1, 2, dtype=torch.int32)
    q8 = torch.zeros(3, 16, 2, 64, dtype=torch.int8)
    sc = torch.ones(3, 2, 16)
    with pytest.raises(AssertionError):  # CPU tensors
        tree_attention(q, kc, kc, lens, block_table=table)
    with pytest.raises(AssertionError):
        decode_attention_quant(q, q8, q8, None, None, lens, table)
    with pytest.raises(AssertionError):
        decode_attention_quant(q, q8, q8, sc, sc, lens, table)


def test_entry_point_checks_arguments_without_a_gpu():
    from nanovllm_b200 import _lib
    f = _lib.lib().nvb200_cache_attention
    assert f(None, None, 0, None) == _lib.ERR_ARG

    def args(**kw):
        a = _lib.CacheAttentionArgs()
        for p in ("out", "q", "k_cache", "v_cache", "k_scale", "v_scale", "block_table", "seqlens"):
            setattr(a, p, 16)
        a.num_blocks, a.batch, a.queries_per_seq, a.num_q_heads, a.num_kv_heads, a.head_dim = 4, 1, 1, 4, 2, 128
        a.cache_block_stride, a.cache_token_stride, a.cache_head_stride = 4096, 256, 128
        a.block_size, a.max_blocks_per_seq, a.dtype, a.cache_dtype, a.softmax_scale = 16, 4, _lib.BF16, _lib.BF16, 0.1
        for k, v in kw.items():
            setattr(a, k, v)
        assert (_lib.lib().nvb200_cache_attention_workspace_size(a) == -1) == (f(a, None, 0, None) in (_lib.ERR_ARG, _lib.ERR_UNSUPPORTED))
        return f(a, None, 0, None)
    for bad in (dict(num_q_heads=3), dict(num_kv_heads=0), dict(batch=-1), dict(block_size=0), dict(causal=2),
                dict(num_splits=9), dict(num_splits=-1), dict(dtype=_lib.F32), dict(cache_dtype=_lib.F16), dict(q=None),
                dict(softmax_scale=float("nan")), dict(cache_dtype=_lib.E4M3, k_scale=None), dict(seqlens=None),
                dict(block_table=None, num_blocks=0), dict(max_blocks_per_seq=-1)):
        assert args(**bad) == _lib.ERR_ARG, bad
    for no in (dict(head_dim=96), dict(k_cache=8), dict(cache_token_stride=257), dict(queries_per_seq=4097),
               dict(max_blocks_per_seq=1 << 28)):
        assert args(**no) == _lib.ERR_UNSUPPORTED, no
    assert args(batch=0) == _lib.OK and args(queries_per_seq=0) == _lib.OK


# ---------------------------------------------------------------------------------------------------------------
# GPU.

@pytest.mark.gpu
@pytest.mark.parametrize("qdt,cdt", [(B16, B16), (H16, H16), (B16, E4M3), (B16, I8), (H16, E4M3), (H16, I8)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,hq,hkv,bs,lens", [
    (1, 1, 1, 16, [1]), (2, 2, 2, 16, [2, 17]), (5, 8, 2, 48, [300, 5, 6, 63]), (8, 16, 8, 256, [777]),
    (16, 8, 1, 7, [16, 99, 1025]), (33, 12, 4, 32, [40, 200]), (64, 8, 2, 64, [64, 65, 2100]), (3, 28, 4, 1, [130, 31])])
def test_tree(cuda, qdt, cdt, d, n, hq, hkv, bs, lens):
    import nanovllm_b200
    q, kv, cache, table, m, drafts = _problem(len(lens), n, lens, hq, hkv, d, bs, qdt, cdt, cuda, seed=n)
    scale = d ** -0.5
    nanovllm_b200.status(cuda, clear=True)
    got = nanovllm_b200.tree_attention(q.to(cuda), cache[0], cache[1], torch.tensor(lens, dtype=torch.int32, device=cuda),
                                       m.to(cuda), block_table=table.to(cuda), k_scale=cache[2], v_scale=cache[3])
    _check(got, q, kv, table, lens, m, drafts, scale, cdt)
    assert nanovllm_b200.status(cuda) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("cdt", [B16, E4M3])
@pytest.mark.parametrize("n,lens,drafts", [(6, [50, 6, 3, 0, 9], [6, 2, 3, 0, 1]), (40, [41, 700, 12, 5], [40, 17, 12, 0]),
                                           (4, [2, 3, 1], [4, 4, 4])])
@pytest.mark.parametrize("mask", ["tree", "chain"])
def test_ragged_drafts_and_short_contexts(cuda, cdt, n, lens, drafts, mask):
    """Padding tokens give zeros; lengths below the draft count leave the first drafts out of the cache; rows whose mask
    leaves nothing give zeros."""
    import nanovllm_b200
    q, kv, cache, table, m, _ = _problem(len(lens), n, lens, 4, 2, 128, 16, B16, cdt, cuda, drafts=drafts, mask=mask)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    got = nanovllm_b200.tree_attention(q.to(cuda), cache[0], cache[1], i32(lens), None if m is None else m.to(cuda),
                                       table.to(cuda), i32(drafts), k_scale=cache[2], v_scale=cache[3])
    _check(got, q, kv, table, lens, m, drafts, 128 ** -0.5, cdt)
    for b, k in enumerate(drafts):
        assert not bool(got[b, k:].float().any())


@pytest.mark.gpu
@pytest.mark.parametrize("qdt,cdt", [(B16, E4M3), (H16, I8)])
@pytest.mark.parametrize("n,causal", [(1, True), (1, False), (3, True), (3, False)])
@pytest.mark.parametrize("hq,hkv,d", [(16, 8, 128), (32, 4, 128), (6, 6, 64), (16, 1, 64)])
def test_decode_quant(cuda, qdt, cdt, n, causal, hq, hkv, d):
    import nanovllm_b200
    lens = [1024, 1, 0, 311, 4097]
    q, kv, cache, table, _, drafts = _problem(5, n, lens, hq, hkv, d, 64, qdt, cdt, cuda, mask=None)
    got = nanovllm_b200.decode_attention_quant(q.to(cuda), *cache, torch.tensor(lens, dtype=torch.int32, device=cuda),
                                               block_table=table.to(cuda), softmax_scale=0.2, causal=causal)
    _check(got, q, kv, table, lens, None, drafts, 0.2, cdt, causal)


@pytest.mark.gpu
@pytest.mark.parametrize("splits", range(1, 9))
@pytest.mark.parametrize("cdt", [H16, I8])
def test_every_split(cuda, splits, cdt):
    import nanovllm_b200
    lens, n = [1500, 40, 0, 129], 9
    q, kv, cache, table, m, drafts = _problem(4, n, lens, 6, 2, 128, 32, H16, cdt, cuda, drafts=[9, 9, 0, 5])
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    got = nanovllm_b200.tree_attention(q.to(cuda), cache[0], cache[1], i32(lens), m.to(cuda), table.to(cuda),
                                       i32([9, 9, 0, 5]), k_scale=cache[2], v_scale=cache[3], num_splits=splits)
    _check(got, q, kv, table, lens, m, [9, 9, 0, 5], 128 ** -0.5, cdt)


@pytest.mark.gpu
@pytest.mark.parametrize("cdt", [B16, H16, E4M3, I8])
@pytest.mark.parametrize("n", [4, 48])
def test_values_in_unseen_places_have_no_effect(cuda, cdt, n):
    """Infinities and NaN in keys and values that a row does not see (drafts off its branch, slots behind the sequence, other
    sequences' pages) change nothing; in ones that it sees they reach it."""
    import nanovllm_b200
    qdt = H16 if cdt == H16 else B16
    hq, hkv, d, bs, L = 4, 2, 64, 16, 100 + n
    q, kv, cache, table, m, drafts = _problem(2, n, [L, L], hq, hkv, d, bs, qdt, cdt, cuda)
    m[:] = torch.eye(n, dtype=torch.bool)
    bad = 1  # the draft that only row 1 sees
    clean = [None if x is None else x.clone() for x in cache]
    lens = torch.tensor([L, L], dtype=torch.int32, device=cuda)
    run = lambda c: nanovllm_b200.tree_attention(q.to(cuda), c[0], c[1], lens, m.to(cuda), table.to(cuda),  # noqa: E731
                                                 k_scale=c[2], v_scale=c[3])
    want = run(clean)
    slot = [(int(table[b, (L - n + bad) // bs]), (L - n + bad) % bs) for b in range(2)]
    behind = [(int(table[b, j // bs]), j % bs) for b in range(2) for j in range(L, table.shape[1] * bs)]
    for t, at in [(t, at) for t in (0, 1) for at in behind]:
        if cdt in (E4M3, I8):
            cache[2 + t][at[0], :, at[1]] = float("nan")
            cache[t].view(torch.uint8)[at] = 0x7F
        else:
            cache[t][at] = float("nan")
    assert torch.equal(run(cache), want)
    if cdt in (E4M3, I8):
        cache[3][slot[0][0], :, slot[0][1]] = float("nan")
        cache[2][slot[1][0], :, slot[1][1]] = float("nan")
    else:
        cache[1][slot[0]] = float("inf")
        cache[1][slot[0]][0, 3] = -float("inf")
        cache[1][slot[0]][0, 4] = float("nan")
        cache[0][slot[1]] = float("nan")
    got = run(cache)
    keep = [i for i in range(n) if i != bad]
    assert torch.equal(got[:, keep], want[:, keep])
    if cdt in (E4M3, I8):
        assert bool(got[:, bad].isnan().all())
        if cdt == E4M3:
            cache[3].copy_(clean[3]), cache[2].copy_(clean[2])
            cache[1].view(torch.uint8)[slot[0]][:, 7] = 0xFF  # e4m3's NaN, in one column
            got = run(cache)
            assert torch.equal(got[:, keep], want[:, keep])
            assert bool(got[0, bad, :, 7].isnan().all()) and torch.equal(got[0, bad, :, :7], want[0, bad, :, :7])
    else:
        inf = float("inf")
        per = hq // hkv
        assert bool((got[0, bad, :per, :3] == inf).all()) and bool((got[0, bad, :per, 3] == -inf).all())
        assert bool(got[0, bad, :per, 4].isnan().all()) and bool((got[0, bad, per:] == inf).all())
        assert bool(got[1, bad].isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("cdt", [B16, E4M3])
def test_values_in_seen_places_reach_every_row(cuda, cdt):
    import nanovllm_b200
    n, L = 3, 70
    q, kv, cache, table, m, _ = _problem(1, n, [L], 4, 2, 64, 16, B16, cdt, cuda)
    at = (int(table[0, 1]), 5)
    if cdt == B16:
        cache[1][at] = float("inf")
    else:
        cache[3][at[0], :, at[1]] = float("nan")
    got = nanovllm_b200.tree_attention(q.to(cuda), cache[0], cache[1], torch.tensor([L], dtype=torch.int32, device=cuda),
                                       m.to(cuda), table.to(cuda), k_scale=cache[2], v_scale=cache[3])
    assert bool((got == float("inf")).all() if cdt == B16 else got.isnan().all())


@pytest.mark.gpu
@pytest.mark.parametrize("cdt", [E4M3, I8])
def test_row_scales_of_any_range(cuda, cdt):
    """Value rows many binades apart, the loud ones on unlikely keys: weights times row scales, and both sums, keep their
    precision."""
    import nanovllm_b200
    n, L, d = 2, 90, 64
    q, kv, cache, table, m, drafts = _problem(1, n, [L], 2, 1, d, 16, B16, cdt, cuda)
    g = torch.Generator().manual_seed(5)
    cache[3].copy_(torch.exp2(torch.randint(-100, 90, cache[3].shape, generator=g).float()))
    cache[2].copy_(cache[2] * 8)
    kv = [cm.row_values(cache[0].cpu(), cache[2].cpu()), cm.row_values(cache[1].cpu(), cache[3].cpu())]
    got = nanovllm_b200.tree_attention(q.to(cuda), cache[0], cache[1], torch.tensor([L], dtype=torch.int32, device=cuda),
                                       m.to(cuda), table.to(cuda), k_scale=cache[2], v_scale=cache[3])
    ref, spread, reach = cm.cache_attention(q, kv[0], kv[1], [L], table, m, drafts, d ** -0.5)
    # The smallest-step term of the tolerance, relative to the largest weight times value that the row has.
    tol = 2.0 ** -8 * ref.abs() + (spread + 4 * spread.amax(-1, keepdim=True) * L * 2.0 ** -14) * (
        2.0 ** -11 + 2.0 ** -18 + 2 * (d + 8) * 2.0 ** -24 * reach)
    assert bool(((got.double().cpu() - ref).abs() <= tol).all())
    # All-zero value rows keep their share of the softmax.
    cache[1].zero_()
    cache[3].fill_(2.0 ** -126)
    cache[1].view(torch.uint8)[int(table[0, 0]), 0] = 0x38 if cdt == E4M3 else 1  # key 0: ones
    cache[3][int(table[0, 0]), 0, 0] = 1.0
    kv[1] = cm.row_values(cache[1].cpu(), cache[3].cpu())
    # The only value row that counts is 1 and its weight p may be any number in (0, 1]: below fp32's normal range, 2^-126,
    # exp2 gives it no precision (and below 2^-149 zero), so an absolute 2^-125 joins the relative terms. At the second
    # scale every weight is far above that.
    for scale in (d ** -0.5, d ** -0.5 / 64):
        got = nanovllm_b200.tree_attention(q.to(cuda), cache[0], cache[1], torch.tensor([L], dtype=torch.int32, device=cuda),
                                           m.to(cuda), table.to(cuda), softmax_scale=scale, k_scale=cache[2],
                                           v_scale=cache[3])
        ref, spread, reach = cm.cache_attention(q, kv[0], kv[1], [L], table, m, drafts, scale)
        tol = spread * (2.0 ** -8 + 2.0 ** -11 + 2.0 ** -18 + 2 * (d + 8) * 2.0 ** -24 * reach) + 2.0 ** -125
        assert bool(((got.double().cpu() - ref).abs() <= tol).all())
    assert float(ref[ref > 0].min()) > 2.0 ** -60


@pytest.mark.gpu
@pytest.mark.parametrize("cdt", [B16, I8])
@pytest.mark.parametrize("factor", [0.0, 1e-30, 300.0, 1e30])
def test_queries_of_any_size(cuda, cdt, factor):
    """Queries outside fp16's range; scores of hundreds; zeros."""
    import nanovllm_b200
    n, L, d = 3, 60, 128
    q, kv, cache, table, m, drafts = _problem(1, n, [L], 4, 2, d, 16, B16, cdt, cuda)
    q = (q.float() * factor).to(B16)
    scale = d ** -0.5 if factor < 1e3 else d ** -0.5 / factor
    got = nanovllm_b200.tree_attention(q.to(cuda), cache[0], cache[1], torch.tensor([L], dtype=torch.int32, device=cuda),
                                       m.to(cuda), table.to(cuda), softmax_scale=scale, k_scale=cache[2], v_scale=cache[3])
    _check(got, q, kv, table, [L], m, drafts, scale, cdt)


@pytest.mark.gpu
@pytest.mark.parametrize("cdt", [B16, E4M3])
def test_strides_masks_and_no_block_table(cuda, cdt):
    """Queries as a view of a qkv buffer; a mask shared by the batch, transposed, or a slice; caches by sequence."""
    import nanovllm_b200
    B, n, hq, hkv, d, lens = 3, 5, 4, 2, 128, [30, 9, 17]
    q, kv, cache, _, m, drafts = _problem(B, n, lens, hq, hkv, d, 16, B16, cdt, cuda, paged=False)
    wide = torch.zeros(B, n, (hq + 2) * d + 3, dtype=B16)
    wide[..., 3:3 + hq * d] = q.view(B, n, hq * d)
    view = torch.as_strided(wide.to(cuda), (B, n, hq, d), (n * wide.shape[2], wide.shape[2], d, 1), 3)
    tl = torch.tensor([9, 1, 1, 30, 2, 9, 17, 1], dtype=torch.int32, device=cuda)[3:]  # not contiguous below
    sl = torch.stack([torch.tensor(lens), torch.zeros(3, dtype=torch.int64)], 1).int().to(cuda)[:, 0]
    assert tl.numel() and not sl.is_contiguous()
    for mask in (m, m[:1].expand(B, n, n), m.transpose(1, 2), m[0]):
        dev_mask = mask.to(cuda) if mask is not m else torch.zeros(B, n + 2, n + 4, dtype=torch.bool, device=cuda)
        if mask is m:
            dev_mask = dev_mask[:, 1:1 + n, 2:2 + n]
            dev_mask.copy_(m.to(cuda))
        got = nanovllm_b200.tree_attention(view, cache[0], cache[1], sl, dev_mask, k_scale=cache[2], v_scale=cache[3])
        full = mask if mask.dim() == 3 else mask[None].expand(B, n, n)
        _check(got, q, kv, None, lens, full, drafts, d ** -0.5, cdt)


@pytest.mark.gpu
def test_cache_views(cuda):
    """A cache that is a strided slice: every second block, heads of a wider cache."""
    import nanovllm_b200
    q, kv, cache, table, m, drafts = _problem(2, 4, [50, 20], 4, 2, 64, 16, B16, B16, cuda)
    wide = [torch.randn(2 * c.shape[0], 16, 5, 64, device=cuda).to(B16) for c in cache[:2]]
    views = [w[::2, :, 1:3] for w in wide]
    for view, c in zip(views, cache):
        view.copy_(c)
    got = nanovllm_b200.tree_attention(q.to(cuda), *views, torch.tensor([50, 20], dtype=torch.int32, device=cuda),
                                       m.to(cuda), table.to(cuda))
    _check(got, q, kv, table, [50, 20], m, drafts, 64 ** -0.5, B16)


@pytest.mark.gpu
@pytest.mark.parametrize("cdt", [B16, I8])
def test_bad_pages_and_lengths_are_flagged(cuda, cdt):
    """Keys on pages that cannot be followed are seen by no row; lengths beyond the table and draft counts beyond n are
    clamped."""
    import nanovllm_b200
    n, d, lens = 2, 64, [40, 33, 60]
    q, kv, cache, table, m, drafts = _problem(3, n, lens, 2, 1, d, 16, B16, cdt, cuda)
    bad = table.clone()
    bad[0, 1], bad[1, 0] = table.numel() + 2, -1
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    nanovllm_b200.status(cuda, clear=True)
    got = nanovllm_b200.tree_attention(q.to(cuda), cache[0], cache[1], i32([40, 33, 1000]), m.to(cuda), bad.to(cuda),
                                       i32([2, 2, 7]), k_scale=cache[2], v_scale=cache[3])
    assert nanovllm_b200.status(cuda, clear=True) == 2
    # The oracle with those keys taken out of the sequence (the third one is 64 keys long).
    keep = [[j for j in range(40) if j // 16 != 1], [j for j in range(33) if j // 16 != 0], list(range(64))]
    seqs = [[x[table[b].long()].flatten(0, 1)[keep[b]] for b in range(3)] for x in kv]
    flat = [torch.zeros(3, 64, 1, d, dtype=torch.float64) for _ in range(2)]
    for x, seq in zip(flat, seqs):
        for b in range(3):
            x[b, :len(keep[b])] = seq[b].double()
    _check(got, q, flat, None, [len(k) for k in keep], m, [2, 2, 2], d ** -0.5, cdt)
    got = nanovllm_b200.tree_attention(q.to(cuda), cache[0], cache[1], i32([-3, 33, 60]), m.to(cuda), table.to(cuda),
                                       i32([2, -1, 2]), k_scale=cache[2], v_scale=cache[3])
    assert nanovllm_b200.status(cuda, clear=True) == 2
    assert not bool(got[:2].float().any()) and bool(got[2].float().any())


@pytest.mark.gpu
def test_refusals_on_the_device(cuda):
    import nanovllm_b200
    q = torch.zeros(2, 2, 4, 64, dtype=B16, device=cuda)
    kc = torch.zeros(3, 16, 2, 64, dtype=B16, device=cuda)
    lens, table = torch.ones(2, dtype=torch.int32, device=cuda), torch.zeros(2, 2, dtype=torch.int32, device=cuda)
    run = lambda q=q, k=kc, v=None, l=lens, **kw: nanovllm_b200.tree_attention(  # noqa: E731
        q, k, k if v is None else v, l, **{**dict(block_table=table), **kw})
    run()
    yes = torch.ones(2, 2, dtype=torch.bool, device=cuda)
    for bad in (dict(l=lens.long()), dict(l=lens[:1]), dict(block_table=table.long()), dict(block_table=table[:1]),
                dict(block_table=table[:, :0]), dict(tree_mask=yes.int()), dict(tree_mask=yes[:1]), dict(tree_mask=yes.cpu()),
                dict(draft_lens=lens.long()), dict(num_splits=9), dict(k=kc[:, :, :1].expand(3, 16, 3, 64)), dict(v=kc[:2]),
                dict(k_scale=torch.ones(3, 2, 16, device=cuda)), dict(k=kc.view(torch.int8)), dict(q=q[..., ::2]),
                dict(q=q[0]), dict(k=kc[:1], block_table=None), dict(l=lens.cpu())):
        with pytest.raises(AssertionError):
            run(**bad)
    sc = torch.ones(3, 16, 2, device=cuda)
    with pytest.raises(AssertionError):  # scales of another layout
        run(k=kc[..., :64].to(torch.int8), k_scale=sc, v_scale=sc)
    for no in (dict(q=q.float(), k=kc.float()), dict(k=kc.half()), dict(q=q[..., :32].contiguous(), k=kc[..., :32].contiguous()),
               dict(k=torch.zeros(3, 16, 2, 68, dtype=B16, device=cuda)[..., :64])):
        with pytest.raises(NotImplementedError):
            run(**no)
    with pytest.raises(ValueError):
        run(softmax_scale=float("inf"))
    assert run(q=q[:0], l=lens[:0], block_table=table[:0]).shape == (0, 2, 4, 64)
    assert run(q=q[:, :0]).shape == (2, 0, 4, 64)


@pytest.mark.gpu
def test_capture_streams_and_repeats(cuda):
    """A captured step of writer and readers replays to the eager step's bits, on another stream too, and two graphs of
    different sizes replayed in turn do not disturb each other."""
    import nanovllm_b200
    hq, hkv, d, bs = 8, 2, 128, 16
    g = torch.Generator().manual_seed(0)
    steps = []
    for B, n, L in ((3, 4, 200), (2, 7, 1900)):
        pages = -(-L // bs)
        cache = nanovllm_b200.empty_quant_cache(B * pages, bs, hkv, d, I8, cuda)
        table = torch.randperm(B * pages, generator=g).view(B, pages).int().to(cuda)
        k = torch.randn(B * L, hkv, d, generator=g).to(B16).to(cuda)
        j = torch.arange(L, device=cuda)
        slots = (table[:, j // bs] * bs + j % bs).flatten().int()
        q = torch.randn(B, n, hq, d, generator=g).to(B16).to(cuda)
        lens = torch.full((B,), L, dtype=torch.int32, device=cuda)
        mask = (torch.rand(B, n, n, generator=g) < 0.5).to(cuda)

        def step(k=k, cache=cache, slots=slots, q=q, lens=lens, mask=mask, table=table):
            nanovllm_b200.store_kvcache_quant(k, -k, *cache, slots)
            a = nanovllm_b200.tree_attention(q, cache[0], cache[1], lens, mask, table, k_scale=cache[2], v_scale=cache[3])
            return a, nanovllm_b200.decode_attention_quant(a[:, :1], *cache, lens, table)
        want = [t.clone() for t in step()]
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            got = step()
        torch.cuda.current_stream().wait_stream(side)
        assert all(torch.equal(a, b) for a, b in zip(got, want))
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph):
            got = step()
        steps.append((graph, got, want, step))  # the step's inputs live as long as its graph
    for _ in range(3):
        for graph, *_ in steps:
            graph.replay()
    torch.cuda.synchronize()
    for _, got, want, _ in steps:
        assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
def test_a_draft_verification_step(cuda):
    """The operators together, as a verification step uses them: the tree's q/k/v through the fused quantising write, the
    tree attention on the cache, then the accepted path read back; against the same step in 64 bits on the cache's values."""
    import nanovllm_b200
    B, n, hq, hkv, d, bs, ctx = 2, 6, 8, 2, 128, 16, [37, 90]
    g = torch.Generator().manual_seed(2)
    pages = 7
    cache = nanovllm_b200.empty_quant_cache(B * pages, bs, hkv, d, E4M3, cuda)
    table = torch.randperm(B * pages, generator=g).view(B, pages).int()
    slot = lambda b, j: int(table[b, j // bs]) * bs + j % bs  # noqa: E731
    for b in range(B):
        k = torch.randn(ctx[b], hkv, d, generator=g).to(B16).to(cuda)
        nanovllm_b200.store_kvcache_quant(k, k * 2, *cache, torch.tensor([slot(b, j) for j in range(ctx[b])], device=cuda))
    qkv = torch.randn(B * n, (hq + 2 * hkv) * d, generator=g).to(B16).to(cuda)
    q, k, v = (x.view(B * n, -1, d) for x in qkv.split([hq * d, hkv * d, hkv * d], -1))
    parent = [-1, 0, 0, 1, 2, 2]
    depth, mask = [], torch.zeros(n, n, dtype=torch.bool)
    for i, p in enumerate(parent):
        depth.append(0 if p < 0 else depth[p] + 1)
        if p >= 0:
            mask[i] = mask[p]
        mask[i, i] = True
    pos = torch.tensor([c + x for c in ctx for x in depth], device=cuda)
    w = torch.ones(d, dtype=B16, device=cuda)
    ang = torch.arange(200)[:, None] * 1e4 ** (-torch.arange(0, d, 2) / d)
    cs = torch.cat([ang.cos(), ang.sin()], -1).to(cuda)
    slots = torch.tensor([slot(b, ctx[b] + i) for b in range(B) for i in range(n)], dtype=torch.int32, device=cuda)
    q_out, _ = nanovllm_b200.qk_norm_rope_kv_quant(q, k, v, pos, w, w, 1e-6, cs, *cache, slots, False)
    lens = [c + n for c in ctx]
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    out = nanovllm_b200.tree_attention(q_out.view(B, n, hq, d), cache[0], cache[1], i32(lens), mask.to(cuda),
                                       table.to(cuda), k_scale=cache[2], v_scale=cache[3])
    kv = [cm.row_values(cache[0].cpu(), cache[2].cpu()), cm.row_values(cache[1].cpu(), cache[3].cpu())]
    _check(out, q_out.cpu().view(B, n, hq, d), kv, table, lens, mask[None].expand(B, n, n), [n] * B, d ** -0.5, E4M3)
    k_back, v_back = nanovllm_b200.load_kvcache_quant(*cache, table.to(cuda), i32([0, lens[0], sum(lens)]), sum(lens))
    for got, values in ((k_back, kv[0]), (v_back, kv[1])):
        want = torch.cat([values[table[b].long()].flatten(0, 1)[:lens[b]] for b in range(B)])
        assert torch.equal(got.cpu(), want.to(B16))


@pytest.mark.gpu
@pytest.mark.parametrize("cdt", [B16, E4M3])
def test_offsets_past_32_bits(cuda, cdt):
    """Pages whose element offsets lie past 2^32 in the cache, a long sequence across both ends of it."""
    import nanovllm_b200
    hkv, d, bs, n, L = 8, 128, 256, 4, 5000
    blocks = 16400  # 4.3e9 elements
    pages = -(-L // bs)
    table = torch.stack([torch.arange(pages), blocks - 1 - torch.arange(pages)]).int()
    g = torch.Generator().manual_seed(0)
    used = torch.cat([table[0], table[1]]).long()
    cache = [torch.zeros(blocks, bs, hkv, d, dtype=torch.uint8 if cdt == E4M3 else B16, device=cuda) for _ in range(2)]
    small = [torch.randn(len(used), bs, hkv, d, generator=g).to(cdt) for _ in range(2)]
    scales, kw = [], {}
    for c, s in zip(cache, small):
        c[used.to(cuda)] = (s.view(torch.uint8) if cdt == E4M3 else s).to(cuda)
    if cdt == E4M3:
        cache = [c.view(E4M3) for c in cache]
        scales = [torch.zeros(blocks, hkv, bs, device=cuda) for _ in range(2)]
        for x in scales:
            x[used.to(cuda)] = 0.5
        kw = dict(k_scale=scales[0], v_scale=scales[1])
    q = torch.randn(2, n, 8, d, generator=g).to(B16)
    m = torch.ones(n, n).tril().bool()
    got = nanovllm_b200.tree_attention(q.to(cuda), *cache, torch.tensor([L, L - 7], dtype=torch.int32, device=cuda),
                                       m.to(cuda), table.to(cuda), **kw)
    kv = [s.float() * (0.5 if cdt == E4M3 else 1.0) for s in small]
    at = torch.arange(len(used)).view(2, pages).int()
    _check(got, q, kv, at, [L, L - 7], m[None].expand(2, n, n), [n, n], d ** -0.5, cdt)


@pytest.mark.gpu
@pytest.mark.parametrize("qdt,cdt", [(B16, B16), (H16, H16), (B16, E4M3), (H16, I8)])
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("n,hq,hkv,lens,drafts", [
    (1, 8, 2, [4500, 1, 0, 700, 2100], None), (3, 8, 2, [5000, 2, 0, 700, 2100], [3, 2, 0, 1, 3]),
    (6, 8, 1, [5000, 64, 47, 0, 129], None), (12, 8, 2, [4300, 11, 900], [12, 12, 7]),
    (34, 8, 2, [3000, 34, 0, 5], [34, 30, 0, 34]), (100, 4, 2, [4200, 101, 100], None)])
def test_shares_of_long_tables(cuda, qdt, cdt, d, n, hq, hkv, lens, drafts):
    """Block tables long enough for the keys of all sequences to be dealt out evenly, in each size of row block: 1 to 8, 16,
    several blocks of 16, 64 (16-bit caches) and 128."""
    import nanovllm_b200
    q, kv, cache, table, m, dr = _problem(len(lens), n, lens, hq, hkv, d, 64, qdt, cdt, cuda, seed=n, drafts=drafts)
    i32 = lambda x: torch.tensor(x, dtype=torch.int32, device=cuda)  # noqa: E731
    nanovllm_b200.status(cuda, clear=True)
    run = lambda splits=0: nanovllm_b200.tree_attention(  # noqa: E731
        q.to(cuda), cache[0], cache[1], i32(lens), m.to(cuda), table.to(cuda), None if drafts is None else i32(drafts),
        k_scale=cache[2], v_scale=cache[3], num_splits=splits)
    got = run()
    _check(got, q, kv, table, lens, m, dr, d ** -0.5, cdt)
    assert torch.equal(run(), got)
    _check(run(3), q, kv, table, lens, m, dr, d ** -0.5, cdt)
    assert nanovllm_b200.status(cuda) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("cdt", [B16, E4M3])
@pytest.mark.parametrize("n,hq", [(1, 4), (4, 4), (30, 4), (80, 4)])
def test_many_short_sequences_in_wide_tables(cuda, cdt, n, hq):
    """Shares that hold many sequences of a tile or less, pages of several sizes; the table's unused entries are never read."""
    import nanovllm_b200
    g = torch.Generator().manual_seed(n)
    lens = [n + int(x) for x in torch.randint(0, 90, (70,), generator=g)]
    q, kv, cache, table, m, drafts = _problem(70, n, lens, hq, 2, 64, 32, B16, cdt, cuda, seed=n)
    wide = torch.full((70, 150), -7, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    nanovllm_b200.status(cuda, clear=True)
    got = nanovllm_b200.tree_attention(q.to(cuda), cache[0], cache[1], torch.tensor(lens, dtype=torch.int32, device=cuda),
                                       m.to(cuda), wide.to(cuda), k_scale=cache[2], v_scale=cache[3])
    _check(got, q, kv, table, lens, m, drafts, 64 ** -0.5, cdt)
    assert nanovllm_b200.status(cuda) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("cdt", [B16, I8])
@pytest.mark.parametrize("n", [2, 40, 80])
def test_workspaces(cuda, cdt, n):
    """The C call: a workspace that is too small or misaligned is refused, none at all gives the result by another form, and
    nothing outside the stated bytes is written."""
    import nanovllm_b200
    from nanovllm_b200 import _lib
    lens, d, scale = [4500, n], 128, 0.1
    q, kv, cache, table, _, drafts = _problem(2, n, lens, 4, 2, d, 64, B16, cdt, cuda, mask=None)
    qd, td, ld = q.to(cuda), table.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda)
    out = torch.zeros_like(qd)
    s, k = qd.stride(), cache[0].stride()
    a = _lib.CacheAttentionArgs.pack(
        out.data_ptr(), qd.data_ptr(), s[0], s[1], s[2], cache[0].data_ptr(), cache[1].data_ptr(), k[0], k[1], k[2],
        cache[2].data_ptr() if cdt == I8 else 0, cache[3].data_ptr() if cdt == I8 else 0, cache[0].shape[0], td.data_ptr(),
        td.stride(0), ld.data_ptr(), 0, 0, 0, 0, 2, n, 4, 2, d, 64, td.shape[1], 1, 0, _lib.BF16,
        _lib.I8 if cdt == I8 else _lib.BF16, scale, _lib.status_word(cuda).data_ptr())
    L = _lib.lib()
    need = L.nvb200_cache_attention_workspace_size(a)
    assert need > 0
    ws = torch.full((need + 64,), 77, dtype=torch.uint8, device=cuda)
    stream = _lib.stream_of(qd)
    assert L.nvb200_cache_attention(a, ws.data_ptr(), need - 1, stream) == _lib.ERR_ARG
    assert L.nvb200_cache_attention(a, ws.data_ptr() + 8, need, stream) == _lib.ERR_ARG
    assert L.nvb200_cache_attention(a, ws.data_ptr(), -1, stream) == _lib.ERR_ARG
    assert not bool(out.any()) and bool((ws == 77).all())
    for pointer, size in ((ws.data_ptr(), need), (None, 0)):
        out.zero_()
        assert L.nvb200_cache_attention(a, pointer, size, stream) == _lib.OK
        _check(out, q, kv, table, lens, None, drafts, scale, cdt)
    assert bool((ws[need:] == 77).all())


@pytest.mark.gpu
@pytest.mark.parametrize("n", [1, 40, 80])
def test_two_calls_at_once(cuda, n):
    """Calls in flight on two streams, eager and captured, keep to their own workspaces."""
    import nanovllm_b200
    lens = [4500, 300, 2000]
    runs = []
    for seed, cdt in ((1, B16), (2, E4M3)):
        q, kv, cache, table, m, _ = _problem(3, n, lens, 8, 2, 128, 64, B16, cdt, cuda, seed=seed)
        q, table, m, ld = q.to(cuda), table.to(cuda), m.to(cuda), torch.tensor(lens, dtype=torch.int32, device=cuda)
        runs.append(lambda q=q, cache=cache, table=table, m=m, ld=ld: nanovllm_b200.tree_attention(
            q, cache[0], cache[1], ld, m, table, k_scale=cache[2], v_scale=cache[3]))
    want = [f().clone() for f in runs]
    graphs, got = [], []
    for f in runs:
        graphs.append(torch.cuda.CUDAGraph())
        with torch.cuda.graph(graphs[-1]):
            got.append(f())
    torch.cuda.synchronize()
    streams, eager = [torch.cuda.Stream() for _ in runs], [[], []]
    for _ in range(5):
        for i, s in enumerate(streams):
            with torch.cuda.stream(s):
                graphs[i].replay()
                eager[i].append(runs[i]())
    torch.cuda.synchronize()
    for i in range(2):
        assert torch.equal(got[i], want[i]) and all(torch.equal(x, want[i]) for x in eager[i])


@pytest.mark.gpu
@pytest.mark.parametrize("cdt", [B16, H16, E4M3])
@pytest.mark.parametrize("n", [2, 30, 80])
@pytest.mark.parametrize("pages", [12, 300])
def test_context_values_beside_the_drafts_reach_every_row(cuda, cdt, n, pages):
    """An infinity (e4m3: a NaN code) of V in the context, in the same tile of keys as the first drafts, reaches every row;
    beside one in a draft that only one row sees. In short and long block tables."""
    import nanovllm_b200
    qdt = H16 if cdt == H16 else B16
    ctx, hq, hkv, d, bs = 100, 4, 2, 64, 16
    q, kv, cache, table, m, _ = _problem(1, n, [ctx + n], hq, hkv, d, bs, qdt, cdt, cuda, seed=n)
    wide = torch.zeros(1, pages, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    m[:] = torch.eye(n, dtype=torch.bool)
    run = lambda causal_mask: nanovllm_b200.tree_attention(  # noqa: E731
        q.to(cuda), cache[0], cache[1], torch.tensor([ctx + n], dtype=torch.int32, device=cuda), causal_mask, wide.to(cuda),
        k_scale=cache[2], v_scale=cache[3])
    masks = (m.to(cuda), None)
    want = [run(x) for x in masks]
    for j, col in ((ctx - 2, 3), (ctx + 1, 5)):
        at = (int(table[0, j // bs]), j % bs)
        if cdt == E4M3:
            cache[1].view(torch.uint8)[at][0, col] = 0x7F
        else:
            cache[1][at][0, col] = float("inf")
    hit = (lambda x: x.isnan()) if cdt == E4M3 else (lambda x: x == float("inf"))
    for x, w, sees in zip(map(run, masks), want, ([1], range(1, n))):
        assert bool(hit(x[0, :, :2, 3]).all())
        assert [i for i in range(n) if bool(hit(x[0, i, :2, 5]).all())] == list(sees)
        rest = torch.ones_like(x, dtype=torch.bool)
        rest[0, :, :2, 3] = False
        rest[0, list(sees), :2, 5] = False
        assert torch.equal(x[rest], w[rest])


# ---------------------------------------------------------------------------------------------------------------
# Row scales at any address.

def _host_args(**kw):
    """nvb200_cache_attention_args of 2 x 4 tokens, 8 query heads over one KV head, for host-side queries (nothing runs)."""
    from nanovllm_b200 import _lib
    a = _lib.CacheAttentionArgs()
    for p in ("out", "q", "k_cache", "v_cache", "block_table", "seqlens", "k_scale", "v_scale"):
        setattr(a, p, 1 << 20)
    a.num_blocks, a.batch, a.queries_per_seq, a.num_q_heads, a.num_kv_heads, a.head_dim = 64, 2, 4, 8, 1, 128
    a.q_batch_stride, a.q_token_stride, a.q_head_stride = 4096, 1024, 128
    a.cache_block_stride, a.cache_token_stride, a.cache_head_stride = 64 * 128, 128, 128
    a.block_size, a.max_blocks_per_seq, a.dtype, a.cache_dtype, a.softmax_scale = 64, 16, _lib.BF16, _lib.E4M3, 0.1
    a.causal = 1
    for k, v in kw.items():
        setattr(a, k, v)
    return a


@pytest.mark.parametrize("field", ["k_scale", "v_scale"])
@pytest.mark.parametrize("offset", [4, 8, 12])
def test_scales_off_a_16_byte_boundary_do_not_take_the_wide_kernel(field, offset):
    """The wide kernel brings row scales by bulk copies, whose sources are 16-byte aligned. In a short block table it is the
    only form that needs a workspace, so the size tells which kernel a call takes."""
    from nanovllm_b200 import _lib
    size = _lib.lib().nvb200_cache_attention_workspace_size
    many = dict(queries_per_seq=40)  # 320 rows
    assert size(_host_args(**many)) > 0
    assert size(_host_args(**many, **{field: (1 << 20) + offset})) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("cdt", [E4M3, I8])
@pytest.mark.parametrize("n,width", [(1, 0), (3, 0), (40, 0), (40, 80), (80, 0)])
@pytest.mark.parametrize("offset", [1, 2, 3])
def test_scales_at_any_address(cuda, cdt, n, width, offset):
    """Scales carved out of a larger buffer: written, read back and attended as at the buffer's start."""
    import nanovllm_b200
    lens, hq, hkv, d, bs = [n + 130, n + 7], 4, 1, 128, 64
    q, kv, cache, table, m, drafts = _problem(2, n, lens, hq, hkv, d, bs, B16, cdt, cuda, seed=n)
    table = torch.cat([table, table.new_zeros(2, max(0, width - table.shape[1]))], 1)
    for i in (2, 3):
        pool = torch.full((cache[i].numel() + 8,), -1.0, device=cuda)
        view = pool[offset:offset + cache[i].numel()].view(cache[i].shape)
        view.copy_(cache[i])
        cache[i] = view
        assert view.data_ptr() % 16 == 4 * offset
    nanovllm_b200.status(cuda, clear=True)
    got = nanovllm_b200.tree_attention(q.to(cuda), cache[0], cache[1], torch.tensor(lens, dtype=torch.int32, device=cuda),
                                       m.to(cuda), table.to(cuda), k_scale=cache[2], v_scale=cache[3])
    _check(got, q, kv, table, lens, m, drafts, d ** -0.5, cdt)
    cu = torch.tensor([0, lens[0], sum(lens)], dtype=torch.int32, device=cuda)
    back = nanovllm_b200.load_kvcache_quant(*cache, table.to(cuda), cu, sum(lens), dtype=torch.float32)
    for x, values in zip(back, kv):
        want = torch.cat([values[table[b].long()].flatten(0, 1)[:lens[b]] for b in range(2)])
        assert torch.equal(x.cpu(), want.float())
    slot = int(table[0, 0]) * bs
    nanovllm_b200.store_kvcache_quant(back[0][5:6], back[1][5:6], *cache, torch.tensor([slot], device=cuda))
    again = nanovllm_b200.load_kvcache_quant(*cache, table.to(cuda), cu, sum(lens), dtype=torch.float32)
    # Values that came from a row of the cache: quantised again by the definition.
    for x, y in zip(back, again):
        codes, scale = cm.quantise_rows(x[5:6].cpu(), cdt)
        assert torch.equal(y[0].cpu(), codes.float()[0] * scale[0][:, None]) and torch.equal(x[1:], y[1:])
    assert nanovllm_b200.status(cuda) == 0


# ---------------------------------------------------------------------------------------------------------------
# Infinities and NaN of V among the drafts, in large trees and beside other sequences.

def _same_nonfinite(got, ref):
    """got has ref's infinities and NaN where ref has any; the finite places are left to _check's tolerance."""
    got, bad = got.double().cpu(), ~torch.isfinite(ref)
    assert torch.equal(torch.nan_to_num(got[bad], nan=7.0, posinf=1.0, neginf=-1.0),
                       torch.nan_to_num(ref[bad], nan=7.0, posinf=1.0, neginf=-1.0))
    return bad


@pytest.mark.gpu
@pytest.mark.parametrize("cdt", [B16, H16, E4M3])
@pytest.mark.parametrize("n,group,pages", [(5, 2, 20), (20, 2, 200), (30, 4, 20), (160, 1, 20), (90, 3, 200)])
@pytest.mark.parametrize("mask", ["tree", "chain"])
def test_infinities_of_several_drafts(cuda, cdt, n, group, pages, mask):
    """Several drafts with infinities of both signs and NaN in some columns, in both kernels and their merges: each row has the
    sum of those it sees."""
    import nanovllm_b200
    hkv, d, bs, lens = 2, 64, 16, [n + 75, n + 3]
    qdt = H16 if cdt == H16 else B16
    q, kv, cache, table, m, drafts = _problem(2, n, lens, group * hkv, hkv, d, bs, qdt, cdt, cuda, seed=n, mask=mask)
    wide = torch.zeros(2, pages, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    g = torch.Generator().manual_seed(3)
    values = kv[1].double().clone()
    for b in range(2):
        for k in [0, n - 1] + torch.randint(0, n, (6,), generator=g).tolist():
            j = lens[b] - n + k
            at = (int(table[b, j // bs]), j % bs, int(torch.randint(0, hkv, (1,), generator=g)))
            for col in torch.randint(0, d, (5,), generator=g).tolist():
                x = [float("inf"), -float("inf"), float("nan")][int(torch.randint(0, 3, (1,), generator=g))]
                if cdt == E4M3:
                    x = float("nan")
                    cache[1].view(torch.uint8)[at][col] = 0x7F if col % 2 else 0xFF
                else:
                    cache[1][at][col] = x
                values[at][col] = x
    nanovllm_b200.status(cuda, clear=True)
    got = nanovllm_b200.tree_attention(q.to(cuda), cache[0], cache[1], torch.tensor(lens, dtype=torch.int32, device=cuda),
                                       None if m is None else m.to(cuda), wide.to(cuda), k_scale=cache[2], v_scale=cache[3])
    assert nanovllm_b200.status(cuda) == 0
    # Column by column with and without the values that are not finite: a sum over the seen drafts' ones.
    ref, spread, reach = cm.cache_attention(q, kv[0], values, lens, table, m, drafts, d ** -0.5)
    bad = _same_nonfinite(got, ref)
    assert bool(bad.any()) and not bool(bad.all())
    clean = torch.nan_to_num(values, nan=0.0, posinf=0.0, neginf=0.0)
    ref, spread, reach = cm.cache_attention(q, kv[0], clean, lens, table, m, drafts, d ** -0.5)
    tol = _tolerance(ref, spread, reach, qdt, cdt, max(lens), float(clean.abs().max()), d)
    assert bool(((got.double().cpu() - ref).abs() <= tol)[~bad].all())


@pytest.mark.gpu
@pytest.mark.parametrize("cdt", [B16, E4M3])
@pytest.mark.parametrize("n,pages", [(3, 8), (24, 8), (40, 130), (140, 8)])
def test_one_sequence_with_infinities_among_many(cuda, cdt, n, pages):
    """More units than the GPU holds, so that a CTA has several, and one sequence whose drafts hold infinities or NaN: the
    other sequences' results keep their bits, and its own are the definition's."""
    import nanovllm_b200
    B, hq, hkv, d, bs = 260, 4, 2, 64, 32
    g = torch.Generator().manual_seed(n)
    lens = [n + int(x) for x in torch.randint(0, 60, (B,), generator=g)]
    q, kv, cache, table, m, drafts = _problem(B, n, lens, hq, hkv, d, bs, B16, cdt, cuda, seed=n)
    wide = torch.zeros(B, pages, dtype=torch.int32)
    wide[:, :table.shape[1]] = table
    args = (q.to(cuda), cache[0], cache[1], torch.tensor(lens, dtype=torch.int32, device=cuda), m.to(cuda), wide.to(cuda))
    run = lambda: nanovllm_b200.tree_attention(*args, k_scale=cache[2], v_scale=cache[3])  # noqa: E731
    want = run()
    sick = 101
    values = kv[1].double().clone()
    for k in range(0, n, 2):
        j = lens[sick] - n + k
        at = (int(table[sick, j // bs]), j % bs)
        if cdt == E4M3:
            cache[1].view(torch.uint8)[at][:, 9] = 0x7F
        else:
            cache[1][at][:, 9] = float("inf")
        values[at][:, 9] = float("nan") if cdt == E4M3 else float("inf")
    nanovllm_b200.status(cuda, clear=True)
    got = run()
    assert nanovllm_b200.status(cuda) == 0
    well = [b for b in range(B) if b != sick]
    assert torch.equal(got[well], want[well])
    one = [x[sick:sick + 1] for x in (q, table, m)]
    ref, _, _ = cm.cache_attention(one[0], kv[0], values, lens[sick:sick + 1], one[1], one[2], [n], d ** -0.5)
    bad = _same_nonfinite(got[sick:sick + 1], ref)
    assert bool(bad.any()) and torch.equal(got[sick:sick + 1].cpu()[~bad], want[sick:sick + 1].cpu()[~bad])


@pytest.mark.gpu
@pytest.mark.parametrize("cdt", [B16, E4M3])
@pytest.mark.parametrize("bs", [12, 64])
def test_the_largest_tree_with_every_value_infinite(cuda, cdt, bs):
    """4096 drafts whose values are all infinite (e4m3: NaN): what rows pick up from them ends well inside the waits' limit, in
    the warp-level kernel (pages of 12 tokens) and the wide one."""
    import nanovllm_b200
    n, d, ctx = 4096, 128, 100
    pages = -(-(ctx + n) // bs)
    table = torch.arange(pages, dtype=torch.int32, device=cuda)[None]
    cache = [torch.zeros(pages, bs, 1, d, dtype=torch.uint8 if cdt == E4M3 else cdt, device=cuda) for _ in range(2)]
    flat = cache[1].view(-1, d)
    flat[ctx:ctx + n] = 0x7F if cdt == E4M3 else float("inf")
    kw = {}
    if cdt == E4M3:
        cache = [c.view(E4M3) for c in cache]
        kw = dict(k_scale=torch.ones(pages, 1, bs, device=cuda), v_scale=torch.ones(pages, 1, bs, device=cuda))
    q = torch.ones(1, n, 1, d, dtype=B16, device=cuda)
    nanovllm_b200.status(cuda, clear=True)
    lens = torch.tensor([ctx + n], dtype=torch.int32, device=cuda)
    got = nanovllm_b200.tree_attention(q, *cache, lens, None, table, **kw)
    assert nanovllm_b200.status(cuda) == 0
    assert bool(got.isnan().all()) if cdt == E4M3 else bool((got == float("inf")).all())
    none = torch.zeros(n, n, dtype=torch.bool, device=cuda)
    none[7, 4000] = True
    got = nanovllm_b200.tree_attention(q, *cache, lens, none, table, **kw)
    assert nanovllm_b200.status(cuda) == 0
    hit = got.isnan() if cdt == E4M3 else got == float("inf")
    assert bool(hit[0, 7].all()) and int(hit.sum()) == d and not bool(got[~hit].any())


# ---------------------------------------------------------------------------------------------------------------
# A key that takes almost the whole softmax, over a long context.

@pytest.mark.gpu
@pytest.mark.parametrize("qdt,cdt", [(B16, B16), (H16, H16), (B16, E4M3), (H16, I8)])
@pytest.mark.parametrize("B,n,splits", [(1, 1, 0), (1, 1, 5), (1, 12, 0), (1, 70, 0), (1300, 1, 0), (320, 70, 0)])
@pytest.mark.parametrize("gap", [23.6, 26.0, 29.3])
def test_many_small_weights_beside_a_large_one(cuda, qdt, cdt, B, n, splits, gap):
    """The first key's score is `gap` binades above those of 20000 others, and its value is zero: the output is what the small
    weights leave. Types of 16 bits hold weights relative to the largest one or two binades above it; fp16, whose step is
    2^-24 from 2^-14 down, must have them far enough up. Both kernels keep the largest weight at 2^5 or above (2^13 in the
    warp-level one), so a weight is off by 2^-30 of it at most, and half a step of its own type. Batches (of one sequence
    over and over), so that a warp or a CTA holds much of a sequence."""
    import nanovllm_b200
    L, hq, d, bs = 20000, 2, 64, 64
    g = torch.Generator().manual_seed(1)
    pages = -(-L // bs)
    table = torch.arange(pages, dtype=torch.int32)[None]
    k, v = torch.zeros(pages, bs, 1, d), torch.randint(64, 128, (pages, bs, 1, d), generator=g).float()
    k[0, 0, 0, 0], v[0, 0] = 64.0, 0.0
    kv = [x.to(cdt) for x in (k, v)]
    cache = [x.to(cuda) for x in kv]
    kw = {}
    if cdt in (E4M3, I8):
        scale = torch.full((pages, 1, bs), 1.0 / 64)
        kw = dict(k_scale=scale.to(cuda), v_scale=scale.to(cuda))
        kv = [cm.row_values(x, scale) for x in kv]
    q = torch.zeros(1, n, hq, d, dtype=qdt)
    q[..., 0] = 1.0
    of_batch = lambda x: x.expand(B, *x.shape[1:]).to(cuda)  # noqa: E731
    top = 1.0 if cdt in (E4M3, I8) else 64.0
    got = nanovllm_b200.tree_attention(of_batch(q), *cache, torch.full((B,), L, dtype=torch.int32, device=cuda), None,
                                       of_batch(table), softmax_scale=gap * 0.6931471805599453 / top, num_splits=splits, **kw)
    ref, spread, reach = cm.cache_attention(q, kv[0], kv[1], [L], table, None, [n], gap * 0.6931471805599453 / top)
    u, uw = (2.0 ** -8 if t == B16 else 2.0 ** -11 for t in (qdt, cdt))
    tol = u * ref.abs() + spread * (uw + 2.0 ** -18 + 2 * (d + 8) * 2.0 ** -24 * reach)
    if cdt != B16:
        tol = tol + 2.0 ** -30 * L * float(kv[1].double().abs().max())
    assert float(ref.min()) > 0 and float((tol / ref).max()) < 1
    err = (got.double().cpu() - ref).abs()
    assert bool((err <= tol).all()), float((err / ref).max())


# ---------------------------------------------------------------------------------------------------------------
# Limits.

def test_limits_are_refused_by_size_and_call_alike():
    """workspace_size says -1 for sizes that the call refuses, whatever form they would take."""
    from nanovllm_b200 import _lib
    L = _lib.lib()
    for kw in (dict(queries_per_seq=4096, num_q_heads=17), dict(queries_per_seq=4097), dict(max_blocks_per_seq=(1 << 25)),
               # 16 x 4096 blocks of 16 rows, kept from the many-row kernel by its split count, its page size or its alignment
               dict(queries_per_seq=4096, num_q_heads=256, num_kv_heads=16, num_splits=1),
               dict(queries_per_seq=4096, num_q_heads=256, num_kv_heads=16, block_size=12),
               dict(queries_per_seq=4096, num_q_heads=256, num_kv_heads=16, k_scale=(1 << 20) + 4)):
        a = _host_args(**kw)
        assert L.nvb200_cache_attention_workspace_size(a) == -1, kw
        assert L.nvb200_cache_attention(a, None, 0, None) == _lib.ERR_UNSUPPORTED, kw
    for kw in (dict(queries_per_seq=4096, num_q_heads=16), dict(queries_per_seq=4096, num_q_heads=256, num_kv_heads=16),
               dict(batch=1 << 20), dict(batch=1 << 20, num_splits=3)):
        assert L.nvb200_cache_attention_workspace_size(_host_args(**kw)) >= 0, kw


@pytest.mark.gpu
def test_row_limit_is_named(cuda):
    import nanovllm_b200
    q = torch.zeros(1, 4096, 17, 64, dtype=B16, device=cuda)
    kc = torch.zeros(1, 64, 1, 64, dtype=B16, device=cuda)
    with pytest.raises(NotImplementedError, match="65536 query rows"):
        nanovllm_b200.tree_attention(q, kc, kc, torch.ones(1, dtype=torch.int32, device=cuda))


@pytest.mark.gpu
@pytest.mark.parametrize("cdt", [B16, I8])
@pytest.mark.parametrize("splits", [0, 2])
def test_more_sequences_than_a_grid_holds(cuda, cdt, splits):
    """65600 sequences: the bits of the same sequences in a call of their own, and the oracle's values on both sides of the
    65535th."""
    import nanovllm_b200
    B, n, hq, hkv, d, bs = 65600, 2, 2, 1, 64, 16
    g = torch.Generator().manual_seed(0)
    q, kv, cache, table, _, _ = _problem(30, n, [20] * 30, hq, hkv, d, bs, B16, cdt, cuda, mask=None)
    q = torch.randn(B, n, hq, d, generator=g).to(B16)
    table = torch.randint(0, cache[0].shape[0], (B, 2), generator=g).int()
    lens, drafts = (torch.randint(0, hi, (B,), generator=g).int() for hi in (33, 3))
    mask = torch.rand(B, n, n, generator=g) < 0.5
    dev = [x.to(cuda) for x in (q, lens, mask, table, drafts)]
    run = lambda at: nanovllm_b200.tree_attention(  # noqa: E731
        dev[0][at], cache[0], cache[1], dev[1][at], dev[2][at], dev[3][at], dev[4][at], k_scale=cache[2], v_scale=cache[3],
        num_splits=splits)
    nanovllm_b200.status(cuda, clear=True)
    got = run(slice(None))
    assert nanovllm_b200.status(cuda) == 0
    assert torch.equal(got[:40000], run(slice(0, 40000))) and torch.equal(got[40000:], run(slice(40000, B)))
    at = list(range(65520, 65550)) + [0, 1, B - 1]
    _check(got[at], q[at], kv, table[at], lens[at].tolist(), mask[at], drafts[at].tolist(), d ** -0.5, cdt)


@pytest.mark.gpu
def test_one_length_for_all_sequences(cuda):
    """cache_seqlens as an int, as the 16-bit decode attention takes it."""
    import nanovllm_b200
    q, kv, cache, table, m, drafts = _problem(3, 2, [37] * 3, 4, 2, 64, 16, B16, E4M3, cuda)
    got = nanovllm_b200.decode_attention_quant(q.to(cuda), *cache, 37, table.to(cuda), causal=True)
    _check(got, q, kv, table, [37] * 3, None, drafts, 64 ** -0.5, E4M3)
    got = nanovllm_b200.tree_attention(q.to(cuda), cache[0], cache[1], 37, m.to(cuda), table.to(cuda), k_scale=cache[2],
                                       v_scale=cache[3])
    _check(got, q, kv, table, [37] * 3, m, drafts, 64 ** -0.5, E4M3)
    nanovllm_b200.status(cuda, clear=True)
    nanovllm_b200.decode_attention_quant(q.to(cuda), *cache, 49, table.to(cuda))  # a key more than the table holds
    assert nanovllm_b200.status(cuda, clear=True) == 2
