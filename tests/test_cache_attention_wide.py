"""The many-row kernel of nvb200_cache_attention (up to 128 query rows a CTA) where its own code can go wrong: pages of all
sizes it takes, strided caches, misaligned queries, negative scales, pages that cannot be followed, value scales far apart,
queries of any size, NaN in unseen places, offsets past 32 bits. Oracle and tolerances as in test_cache_attention.py.

In block tables of at most 2048 keys only this kernel needs a workspace, so the workspace's size tells that a case reaches it.
"""
import pytest
import torch

from oracle import cache_math as cm
from test_cache_attention import B16, E4M3, H16, I8, _check, _host_args, _problem

TYPES = [(B16, B16), (H16, H16), (B16, E4M3), (H16, I8)]


def _reaches_wide(n, hq, hkv, d, bs, pages, qdt, cdt, **kw):
    from nanovllm_b200 import _lib
    code = {B16: _lib.BF16, H16: _lib.F16, E4M3: _lib.E4M3, I8: _lib.I8}
    assert bs * pages <= 2048
    a = _host_args(queries_per_seq=n, num_q_heads=hq, num_kv_heads=hkv, head_dim=d, block_size=bs, max_blocks_per_seq=pages,
                   dtype=code[qdt], cache_dtype=code[cdt], cache_token_stride=hkv * d, cache_block_stride=bs * hkv * d,
                   cache_head_stride=d, **kw)
    return _lib.lib().nvb200_cache_attention_workspace_size(a) > 0


def _i32(x, device):
    return torch.tensor(x, dtype=torch.int32, device=device)


def _attend(q, cache, lens, mask, table, cuda, **kw):
    import nanovllm_b200
    nanovllm_b200.status(cuda, clear=True)
    out = nanovllm_b200.tree_attention(q.to(cuda), cache[0], cache[1], _i32(lens, cuda), None if mask is None else mask.to(cuda),
                                       None if table is None else table.to(cuda), k_scale=cache[2], v_scale=cache[3], **kw)
    return out, nanovllm_b200.status(cuda, clear=True)


def test_which_calls_reach_the_kernel():
    for qdt, cdt in TYPES:
        for bs in (8, 24, 40, 64, 256):
            assert _reaches_wide(80, 4, 2, 128, bs, 4, qdt, cdt)
        for kw in (dict(num_splits=1), dict(out=(1 << 20) + 8), dict(softmax_scale=0.0)):
            assert not _reaches_wide(80, 4, 2, 128, 64, 4, qdt, cdt, **kw)
        assert not _reaches_wide(80, 4, 2, 128, 12, 4, qdt, cdt) and not _reaches_wide(3, 4, 2, 128, 64, 4, qdt, cdt)
        assert _reaches_wide(80, 4, 2, 128, 64, 4, qdt, cdt, softmax_scale=-0.1)


@pytest.mark.gpu
@pytest.mark.parametrize("qdt,cdt", TYPES)
@pytest.mark.parametrize("d", [64, 128])
@pytest.mark.parametrize("bs", [8, 24, 40, 32, 128])
@pytest.mark.parametrize("scale", [0.09, -0.09])
def test_page_sizes_and_negative_scales(cuda, qdt, cdt, d, bs, scale):
    n, hq, hkv, lens, drafts = 80, 4, 2, [300, 80, 127, 83], [80, 80, 70, 0]
    q, kv, cache, table, m, _ = _problem(4, n, lens, hq, hkv, d, bs, qdt, cdt, cuda, seed=bs, drafts=drafts)
    assert _reaches_wide(n, hq, hkv, d, bs, table.shape[1], qdt, cdt)
    got, status = _attend(q, cache, lens, m, table, cuda, draft_lens=_i32(drafts, cuda), softmax_scale=scale)
    _check(got, q, kv, table, lens, m, drafts, scale, cdt)
    assert status == 0


@pytest.mark.gpu
@pytest.mark.parametrize("qdt,cdt", TYPES)
def test_negative_scales_in_the_warp_level_kernel(cuda, qdt, cdt):
    n, lens = 6, [90, 7]
    q, kv, cache, table, m, drafts = _problem(2, n, lens, 4, 2, 128, 16, qdt, cdt, cuda)
    got, _ = _attend(q, cache, lens, m, table, cuda, softmax_scale=-0.09)
    _check(got, q, kv, table, lens, m, drafts, -0.09, cdt)


@pytest.mark.gpu
@pytest.mark.parametrize("cdt", [B16, E4M3, I8])
@pytest.mark.parametrize("factor", [0.0, 1e-30, 300.0, 1e28])
def test_queries_of_any_size(cuda, cdt, factor):
    n, lens, d = 70, [400, 71], 128
    q, kv, cache, table, m, drafts = _problem(2, n, lens, 4, 2, d, 16, B16, cdt, cuda)
    q = (q.float() * factor).to(B16)
    scale = d ** -0.5 if factor < 1e3 else d ** -0.5 / factor
    assert _reaches_wide(n, 4, 2, d, 16, table.shape[1], B16, cdt, softmax_scale=scale)
    got, _ = _attend(q, cache, lens, m, table, cuda, softmax_scale=scale)
    _check(got, q, kv, table, lens, m, drafts, scale, cdt)


@pytest.mark.gpu
@pytest.mark.parametrize("cdt", [E4M3, I8])
@pytest.mark.parametrize("lo,hi", [(-100, 90), (-6, 3), (-12, 0)])
def test_row_scales_of_any_range(cuda, cdt, lo, hi):
    """Value rows up to 190 binades apart, within the 8 that one reference serves, and just past them, in tiles that every row
    sees whole and in the drafts' own."""
    n, L, d = 140, 700, 64
    q, kv, cache, table, m, drafts = _problem(1, n, [L], 2, 1, d, 16, B16, cdt, cuda)
    g = torch.Generator().manual_seed(hi)
    cache[3].copy_(torch.exp2(torch.randint(lo, hi, cache[3].shape, generator=g).float()))
    if lo == -12:  # the loud rows come late, to sequences that have begun quietly
        for page in table[0, :20].tolist():
            cache[3][page].mul_(2.0 ** -9)
    cache[2].mul_(8)
    kv = [cm.row_values(cache[0].cpu(), cache[2].cpu()), cm.row_values(cache[1].cpu(), cache[3].cpu())]
    assert _reaches_wide(n, 2, 1, d, 16, table.shape[1], B16, cdt)
    got, status = _attend(q, cache, [L], m, table, cuda)
    assert status == 0
    ref, spread, reach = cm.cache_attention(q, kv[0], kv[1], [L], table, m, drafts, d ** -0.5)
    # Weights times row scales are off by half a step of fp16, and by 2^-25 where the largest of them is 2^-3 or more (its own
    # reference, or one that row scales at most 2^8 apart share): 2^-22 of the largest weight times value, for each key.
    tol = 2.0 ** -8 * ref.abs() + spread * (2.0 ** -11 + 2.0 ** -18 + 2 * (d + 8) * 2.0 ** -24 * reach)
    tol = tol + spread.amax(-1, keepdim=True) * L * 2.0 ** -22
    # A weight p_j <= 1 below fp32's normal range is zero, as exp2 gives it: p_j |v_j| < 2^-126 max|v| for each key, which counts
    # beside likelier keys where their values lie more than 2^126 below max|v| (they span 2^197 here; a key 2^-138 as likely as
    # the first, with a value of 2^67 beside one of 2^-88, is the first case met).
    tol = tol + L * 2.0 ** -126 * float(kv[1].abs().max())
    assert bool(((got.double().cpu() - ref).abs() <= tol).all())


@pytest.mark.gpu
@pytest.mark.parametrize("cdt", [B16, E4M3, I8])
def test_value_rows_of_zeros(cuda, cdt):
    """Rows of zeros, whose scales are the smallest there are, keep their share of the softmax."""
    n, L, d, bs = 140, 500, 128, 16
    q, kv, cache, table, m, drafts = _problem(1, n, [L], 2, 1, d, bs, B16, cdt, cuda)
    for page in table[0, ::2].tolist():
        cache[1].view(torch.uint8)[page].zero_()
        if cdt != B16:
            cache[3][page] = 2.0 ** -126
    kv = [x.cpu() for x in cache[:2]] if cdt == B16 else [cm.row_values(cache[i].cpu(), cache[2 + i].cpu()) for i in (0, 1)]
    got, _ = _attend(q, cache, [L], m, table, cuda)
    _check(got, q, kv, table, [L], m, drafts, d ** -0.5, cdt)


@pytest.mark.gpu
@pytest.mark.parametrize("qdt,cdt", TYPES)
@pytest.mark.parametrize("pages", [0, 200])
def test_pages_that_cannot_be_followed(cuda, qdt, cdt, pages):
    """Keys on such pages, in the middle, at the start and among the drafts, are seen by no row; lengths beyond the table and
    draft counts beyond n are clamped."""
    n, d, bs, lens = 90, 64, 16, [500, 333, 320]
    q, kv, cache, table, m, drafts = _problem(3, n, lens, 4, 2, d, bs, qdt, cdt, cuda)
    gone = [[3, 4, 9], [0, 15], []]
    bad = table.clone()
    for b, g in enumerate(gone):
        for k, page in enumerate(g):
            bad[b, page] = -5 if k % 2 else table.numel() + 2
    length = list(lens)
    if pages:  # unused entries behind the sequences' own
        bad = torch.cat([bad, torch.zeros(3, pages - bad.shape[1], dtype=torch.int32)], 1)
    else:
        assert _reaches_wide(n, 4, 2, d, bs, table.shape[1], qdt, cdt)
        length[2] = 5000  # the table has 32 pages: 512 keys
        lens = lens[:2] + [512]
    got, status = _attend(q, cache, length, m, bad, cuda, draft_lens=_i32([n, n, n + 7], cuda))
    assert status == 2
    # Rows of the oracle see a sequence without those keys: context and drafts are told apart by the mask.
    for b in range(3):
        L = lens[b]
        keep = [j for j in range(L) if j // bs not in gone[b]]
        seq = [x[table[b].long()].flatten(0, 1)[keep][None] for x in kv]
        own = [j - (L - n) for j in keep if j >= L - n]  # the drafts that are there
        assert own == list(range(n - len(own), n))  # the last ones of them: the oracle's are the last keys, too
        one = torch.zeros(1, n, n, dtype=torch.bool)
        one[0, :, :len(own)] = m[b][:, own]
        # As many drafts for the oracle as there are, asked by all n rows: blocks of rows of that many.
        k = len(own)
        for r0 in range(0, n, k):
            rows = list(range(r0, min(n, r0 + k)))
            qq, mm = q[b:b + 1, rows], one[:, rows][:, :, :k]
            pad = k - len(rows)
            if pad:
                qq = torch.cat([qq, qq[:, :1].expand(1, pad, *qq.shape[2:])], 1)
                mm = torch.cat([mm, mm[:, :1].expand(1, pad, k)], 1)
            out = torch.cat([got[b:b + 1, rows], got[b:b + 1, rows[:1]].expand(1, pad, *got.shape[2:])], 1)
            _check(out, qq, seq, None, [len(keep)], mm, [k], d ** -0.5, cdt)


@pytest.mark.gpu
@pytest.mark.parametrize("qdt,cdt", [(B16, E4M3), (B16, I8), (H16, E4M3)])
@pytest.mark.parametrize("pages", [0, 200])
def test_nan_in_unseen_places_of_an_8_bit_cache(cuda, qdt, cdt, pages):
    """NaN scales and codes behind the sequence, on pages of nobody's, and in drafts that a row does not see."""
    n, hq, hkv, d, bs, L = 80, 4, 2, 64, 16, 333
    q, kv, cache, table, m, drafts = _problem(2, n, [L, L], hq, hkv, d, bs, qdt, cdt, cuda)
    assert _reaches_wide(n, hq, hkv, d, bs, table.shape[1], qdt, cdt)
    m[:] = torch.eye(n, dtype=torch.bool)
    wide = torch.cat([table, torch.full((2, max(0, pages - table.shape[1])), -1, dtype=torch.int32)], 1)
    want, _ = _attend(q, cache, [L, L], m, wide, cuda)
    for b in range(2):
        for j in range(L, table.shape[1] * bs):
            at = (int(table[b, j // bs]), j % bs)
            for t in (0, 1):
                cache[t].view(torch.uint8)[at] = 0x7F
                cache[2 + t][at[0], :, at[1]] = float("nan")
    nobody = sorted(set(range(cache[0].shape[0])) - set(table.flatten().tolist()))
    cache[3][nobody], cache[2][nobody] = float("nan"), float("nan")
    got, status = _attend(q, cache, [L, L], m, wide, cuda)
    assert status == 0 and torch.equal(got, want)
    sick = {0: 5, 1: n - 2}  # draft of each sequence, seen by its own row only
    for b, k in sick.items():
        j = L - n + k
        at = (int(table[b, j // bs]), j % bs)
        cache[3 if b == 0 else 2][at[0], :, at[1]] = float("nan")
    got, status = _attend(q, cache, [L, L], m, wide, cuda)
    assert status == 0
    for b, k in sick.items():
        keep = [i for i in range(n) if i != k]
        assert torch.equal(got[b, keep], want[b, keep]) and bool(got[b, k].isnan().all())
    # One in the context reaches every row.
    at = (int(table[0, 1]), 3)
    cache[3][at[0], 0, at[1]] = float("nan")
    got, _ = _attend(q, cache, [L, L], m, wide, cuda)
    assert bool(got[0, :, :2].isnan().all()) and torch.equal(got[0, [0], 2:], want[0, [0], 2:])


@pytest.mark.gpu
@pytest.mark.parametrize("qdt,cdt", TYPES)
@pytest.mark.parametrize("shift", [1, 3, 4, 8])
def test_strides_masks_and_no_block_table(cuda, qdt, cdt, shift):
    """Queries as a view of a qkv buffer at any 2-byte address; a mask shared by the batch, transposed, or a slice; caches by
    sequence."""
    B, n, hq, hkv, d, lens = 3, 70, 4, 2, 128, [200, 70, 104]
    q, kv, cache, _, m, drafts = _problem(B, n, lens, hq, hkv, d, 16, qdt, cdt, cuda, paged=False)
    assert _reaches_wide(n, hq, hkv, d, 200, 1, qdt, cdt)
    wide = torch.zeros(B, n, (hq + 2) * d + shift, dtype=qdt)
    wide[..., shift:shift + hq * d] = q.view(B, n, hq * d)
    view = torch.as_strided(wide.to(cuda), (B, n, hq, d), (n * wide.shape[2], wide.shape[2], d, 1), shift)
    for mask in (m, m[:1].expand(B, n, n), m.transpose(1, 2), m[0]):
        dev_mask = mask.to(cuda) if mask is not m else torch.zeros(B, n + 2, n + 4, dtype=torch.bool, device=cuda)
        if mask is m:
            dev_mask = dev_mask[:, 1:1 + n, 2:2 + n]
            dev_mask.copy_(m.to(cuda))
        got, status = _attend(view, cache, lens, dev_mask, None, cuda)
        full = mask if mask.dim() == 3 else mask[None].expand(B, n, n)
        _check(got, q, kv, None, lens, full, drafts, d ** -0.5, cdt)
        assert status == 0


@pytest.mark.gpu
@pytest.mark.parametrize("qdt", [B16, H16])
@pytest.mark.parametrize("d", [64, 128])
def test_cache_views(cuda, qdt, d):
    """Caches that are strided slices (every second block, heads of a wider cache, rows of wider tokens), or have their heads
    before their tokens."""
    n, lens = 70, [300, 75]
    q, kv, cache, table, m, drafts = _problem(2, n, lens, 4, 2, d, 16, qdt, qdt, cuda)
    blocks = cache[0].shape[0]
    sliced = [torch.full((2 * blocks, 16, 5, d + 16), 9.0, dtype=qdt, device=cuda)[::2, :, 1:3, 8:8 + d] for _ in range(2)]
    turned = [torch.zeros(blocks, 2, 16, d, dtype=qdt, device=cuda).transpose(1, 2) for _ in range(2)]
    for views in (sliced, turned):
        for view, c in zip(views, cache):
            view.copy_(c)
        got, status = _attend(q, [*views, None, None], lens, m, table, cuda)
        _check(got, q, kv, table, lens, m, drafts, d ** -0.5, qdt)
        assert status == 0


@pytest.mark.gpu
@pytest.mark.parametrize("cdt", [B16, E4M3])
def test_offsets_past_32_bits(cuda, cdt):
    """Pages whose element offsets lie past 2^32 in the cache, a long sequence across both ends of it."""
    hkv, d, bs, n, L = 8, 128, 256, 70, 2040
    blocks = 16400  # 4.3e9 elements
    pages = 8
    table = torch.stack([torch.arange(pages), blocks - 1 - torch.arange(pages)]).int()
    assert _reaches_wide(n, 16, hkv, d, bs, pages, B16, cdt)
    g = torch.Generator().manual_seed(0)
    used = torch.cat([table[0], table[1]]).long()
    cache = [torch.zeros(blocks, bs, hkv, d, dtype=torch.uint8 if cdt == E4M3 else B16, device=cuda) for _ in range(2)]
    small = [torch.randn(len(used), bs, hkv, d, generator=g).to(cdt) for _ in range(2)]
    for c, s in zip(cache, small):
        c[used.to(cuda)] = (s.view(torch.uint8) if cdt == E4M3 else s).to(cuda)
    cache += [None, None]
    if cdt == E4M3:
        cache = [c.view(E4M3) for c in cache[:2]] + [torch.zeros(blocks, hkv, bs, device=cuda) for _ in range(2)]
        for x in cache[2:]:
            x[used.to(cuda)] = 0.5
    q = torch.randn(2, n, 16, d, generator=g).to(B16)
    m = torch.ones(n, n).tril().bool()
    got, status = _attend(q, cache, [L, L - 7], m, table, cuda)
    kv = [s.float() * (0.5 if cdt == E4M3 else 1.0) for s in small]
    at = torch.arange(len(used)).view(2, pages).int()
    _check(got, q, kv, at, [L, L - 7], m[None].expand(2, n, n), [n, n], d ** -0.5, cdt)
    assert status == 0


@pytest.mark.gpu
@pytest.mark.parametrize("qdt,cdt", TYPES)
@pytest.mark.parametrize("n,lens,drafts", [(80, [2, 40, 79, 1], [80, 80, 80, 80]), (130, [131, 64, 300, 0], [130, 70, 1, 5])])
def test_drafts_not_in_the_cache_and_ragged(cuda, qdt, cdt, n, lens, drafts):
    """Lengths below the draft count leave the first drafts out of the cache; few or no drafts of many; empty sequences."""
    for mask in ("tree", "chain"):
        q, kv, cache, table, m, _ = _problem(4, n, lens, 4, 2, 128, 64, qdt, cdt, cuda, drafts=drafts, mask=mask)
        got, status = _attend(q, cache, lens, m, table, cuda, draft_lens=_i32(drafts, cuda))
        _check(got, q, kv, table, lens, m, drafts, 128 ** -0.5, cdt)
        for b, k in enumerate(drafts):
            assert not bool(got[b, k:].float().any())
        assert status == 0
