"""The 8-bit KV cache (nanovllm_b200.kernels.kv_quant): store_kvcache_quant, qk_norm_rope_kv_quant, load_kvcache_quant.

Codes and scales are compared bit for bit with the oracle's 64-bit quantiser (oracle/cache_math.py): each code is one
rounding of an exactly scaled element (e4m3), or the correctly rounded quotient of exact operands (int8, whose operands
are exact for bf16 and fp16 inputs; fp32 inputs are multiples of 2^-12 here, which keeps them so). The fused op is compared with
its two steps, the read-back with code * scale in fp32, rounded once.
"""
import ctypes

import pytest
import torch

from oracle import cache_math as cm

E4M3, I8 = torch.float8_e4m3fn, torch.int8
FMTS = [E4M3, I8]


def _bits(t):
    return t.contiguous().view(torch.uint8) if t.dtype in FMTS else t


def _cache(blocks, bs, hkv, d, fmt, device, seed=0):
    """A cache with arbitrary finite codes and scales everywhere, so that untouched slots show."""
    g = torch.Generator().manual_seed(seed)
    out = []
    for _ in range(2):
        codes = torch.randint(-100, 100, (blocks, bs, hkv, d), generator=g).to(torch.int8)
        out.append((codes if fmt == I8 else codes.float().to(E4M3)).to(device))
    return out + [torch.rand(blocks, hkv, bs, generator=g).to(device) for _ in range(2)]


def _rows(T, hkv, d, dtype, seed=0):
    g = torch.Generator().manual_seed(seed)
    x = torch.randn(T, hkv, d, generator=g) * torch.exp(2 * torch.randn(T, hkv, 1, generator=g))
    if dtype == torch.float32:
        x = torch.round(x * 4096).clamp(-2 ** 16, 2 ** 16) / 4096
    return x.to(dtype)


def _expect_store(cache, k, v, slots, bs):
    kc, vc, ks, vs = (_bits(x).clone().cpu() for x in cache)
    for x, codes, scale in ((k, kc, ks), (v, vc, vs)):
        c, s = cm.quantise_rows(x.cpu(), cache[0].dtype)
        c = _bits(c)
        for t, slot in enumerate(slots.tolist()):
            if 0 <= slot < codes.shape[0] * bs:
                codes[slot // bs, slot % bs] = c[t]
                scale[slot // bs, :, slot % bs] = s[t]
    return kc, vc, ks, vs


def _same(got, want):
    for a, b in zip(got, want):
        assert torch.equal(torch.nan_to_num(_bits(a).cpu().float(), nan=-7.0), torch.nan_to_num(b.float(), nan=-7.0))


# ---------------------------------------------------------------------------------------------------------------
# CPU.

@pytest.mark.parametrize("fmt", FMTS)
def test_oracle_quantiser_known_rows(fmt):
    top = 448.0 if fmt == E4M3 else 127.0
    codes, scale = cm.quantise_rows(torch.tensor([[top, -top / 2, 0.0, 1.0]]), fmt)
    assert scale.item() == 1.0
    assert codes.float().tolist() == [[top, -top / 2 if fmt == E4M3 else -64.0, 0.0, 1.0]]
    codes, scale = cm.quantise_rows(torch.tensor([[0.0, 0.0], [float("inf"), 1.0], [float("nan"), 1.0]]), fmt)
    assert scale[0].item() == 2.0 ** -126 and bool(scale[1:].isnan().all())
    assert not bool(codes.float().any())


def test_oracle_e4m3_is_the_nearest_code():
    """Every fp16 value up to 448, against torch's own conversion."""
    x = torch.arange(0, 1 << 15, dtype=torch.int32).to(torch.int16).view(torch.float16)
    x = x[x.float() <= 448].float()
    rows = torch.stack([torch.full_like(x, 448.0), x], -1)  # the first element fixes the scale at 1
    codes, scale = cm.quantise_rows(rows, E4M3)
    assert bool((scale == 1).all())
    assert torch.equal(codes[:, 1].view(torch.uint8), x.to(E4M3).view(torch.uint8))


def test_empty_quant_cache_shapes():
    from nanovllm_b200 import empty_quant_cache
    kc, vc, ks, vs = empty_quant_cache(3, 16, 2, 64, device="cpu")
    assert kc.shape == vc.shape == (3, 16, 2, 64) and kc.dtype == vc.dtype == E4M3
    assert ks.shape == vs.shape == (3, 2, 16) and ks.dtype == torch.float32
    with pytest.raises(AssertionError):
        empty_quant_cache(3, 16, 2, 64, dtype=torch.float16, device="cpu")


def test_refusals():
    """Argument checks come before anything touches a device."""
    from nanovllm_b200 import load_kvcache_quant, qk_norm_rope_kv_quant, store_kvcache_quant
    cache = _cache(2, 4, 2, 8, E4M3, "cpu")
    x, slots = torch.zeros(3, 2, 8), torch.zeros(3, dtype=torch.int32)
    bad_store = [
        (x[..., ::2], x[..., ::2], cache, slots),                        # heads not contiguous
        (x, x.half(), cache, slots),                                     # two dtypes
        (x.double(), x.double(), cache, slots),
        (x, x, cache, slots[:2]),
        (x, x, cache, slots.short()),
        (x, x, [cache[0].view(torch.uint8)] + cache[1:], slots),         # not an 8-bit cache type
        (x, x, [cache[0], cache[1].view(torch.int8)] + cache[2:], slots),
        (x, x, cache[:2] + [cache[2].transpose(1, 2)] + cache[3:], slots),  # scales [blocks, block_size, Hkv]
        (x, x, [c[:, :, :1] for c in cache[:2]] + cache[2:], slots),     # a strided slice of a cache
        (x, x, cache, slots),                                            # CPU tensors
    ]
    for k, v, c, s in bad_store:
        with pytest.raises(AssertionError):
            store_kvcache_quant(k, v, *c, s)
    table, cu = torch.zeros(1, 2, dtype=torch.int32), torch.tensor([0, 3], dtype=torch.int32)
    for t, c, n, dt in [(table.long(), cu, 3, torch.bfloat16), (table, cu[:1], 3, torch.bfloat16),
                        (table, cu.long(), 3, torch.bfloat16), (table, cu, -1, torch.bfloat16),
                        (table[:, :0], cu, 3, torch.bfloat16), (table, cu, 3, torch.float64),
                        (table, cu, 3, torch.bfloat16)]:
        with pytest.raises(AssertionError):
            load_kvcache_quant(*cache, t, c, n, dtype=dt)
    b = torch.bfloat16
    q, k = torch.zeros(3, 4, 8, dtype=b), torch.zeros(3, 2, 8, dtype=b)
    w, cs, pos = torch.ones(8, dtype=b), torch.zeros(5, 8), torch.zeros(3, dtype=torch.int64)
    for args in [(q.float(), k, k, pos, w, w, 1e-6, cs), (q[:, :3], k, k, pos, w, w, 1e-6, cs),
                 (q, k, k, pos.int(), w, w, 1e-6, cs), (q, k, k, pos, w.float(), w, 1e-6, cs),
                 (q, k, k, pos, w, w, 1e-6, cs.double()), (q, k, k, pos, w, w, 1e-6, cs)]:
        with pytest.raises(AssertionError):
            qk_norm_rope_kv_quant(*args, *cache, slots, False)


def test_entry_points_check_arguments_without_a_gpu():
    from nanovllm_b200 import _lib
    L = _lib.lib()
    c = _lib.QuantCache(16, 16, 16, 16, 2, 4, 2, 8, _lib.E4M3)
    store = lambda cache, n=1, dt=_lib.BF16, sb=4, key=16: L.nvb200_store_kvcache_quant(  # noqa: E731
        key, 16, 16, 16, 16, sb, n, dt, cache, None, None)
    assert store(None) == _lib.ERR_ARG
    assert store(c, n=-1) == _lib.ERR_ARG and store(c, dt=_lib.E4M3) == _lib.ERR_ARG and store(c, sb=2) == _lib.ERR_ARG
    assert store(c, key=None) == _lib.ERR_ARG
    assert store(c, n=0, key=None) == _lib.OK
    assert store(c, n=1 << 31) == _lib.ERR_UNSUPPORTED  # rows are counted in 32 bits
    for field, value in [("dtype", _lib.BF16), ("block_size", 0), ("num_kv_heads", 0), ("head_dim", 0),
                         ("num_blocks", -1)]:
        bad = _lib.QuantCache(16, 16, 16, 16, 2, 4, 2, 8, _lib.E4M3)
        setattr(bad, field, value)
        assert store(bad) == _lib.ERR_ARG, field
    big = _lib.QuantCache(16, 16, 16, 16, 1 << 31, 4, 2, 8, _lib.E4M3)
    assert store(big) == _lib.ERR_UNSUPPORTED  # slots are divided in 32 bits
    load = lambda cache, total=1, table=16, zero=1, batch=1: L.nvb200_load_kvcache_quant(  # noqa: E731
        16, 16, cache, table, 2, 2, 16, batch, total, _lib.BF16, zero, None, None)
    assert load(None) == _lib.ERR_ARG and load(c, total=-1) == _lib.ERR_ARG and load(c, table=None) == _lib.ERR_ARG
    assert load(c, zero=2) == _lib.ERR_ARG and load(c, batch=-1) == _lib.ERR_ARG and load(c, total=0) == _lib.OK
    a = _lib.QkNormRopeKvArgs()
    fused = lambda: L.nvb200_qk_norm_rope_kv_quant(a, c, None)  # noqa: E731
    assert L.nvb200_qk_norm_rope_kv_quant(None, c, None) == _lib.ERR_ARG and fused() == _lib.ERR_ARG
    a.num_q_heads, a.num_kv_heads, a.head_dim, a.num_positions = 4, 2, 8, 5
    assert fused() == _lib.OK  # no tokens
    a.num_tokens = 1
    assert fused() == _lib.ERR_ARG  # null pointers
    for f in ("q", "k", "v", "q_out", "positions", "slot_mapping", "q_weight", "k_weight", "cos_sin"):
        setattr(a, f, 16)
    assert fused() == _lib.ERR_UNSUPPORTED  # head_dim 8
    a.head_dim = 16
    assert fused() == _lib.ERR_ARG  # not the cache's


# ---------------------------------------------------------------------------------------------------------------
# GPU.

@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("T,hkv,d,bs", [(1, 1, 8, 1), (37, 8, 128, 16), (300, 2, 64, 48), (129, 3, 256, 7),
                                        (65, 2, 72, 16), (33, 5, 20, 256), (9, 1, 264, 16), (2049, 4, 128, 256)])
def test_store_bitwise(cuda, fmt, dtype, T, hkv, d, bs):
    import nanovllm_b200
    blocks = (T + T // 3 + bs) // bs + 1
    cache = _cache(blocks, bs, hkv, d, fmt, cuda)
    g = torch.Generator().manual_seed(1)
    slots = torch.randperm(blocks * bs, generator=g)[:T].to(torch.int64 if T % 2 else torch.int32)
    slots[torch.randperm(T, generator=g)[:T // 10]] = -1
    k, v = _rows(T, hkv, d, dtype, 2), _rows(T, hkv, d, dtype, 3)
    want = _expect_store(cache, k, v, slots, bs)
    nanovllm_b200.status(cuda, clear=True)
    nanovllm_b200.store_kvcache_quant(k.to(cuda), v.to(cuda), *cache, slots.to(cuda))
    _same(cache, want)
    assert nanovllm_b200.status(cuda) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("d", [64, 128, 12])
def test_store_rows_where_the_quantiser_can_go_wrong(cuda, fmt, d):
    """Zeros, infinities, NaN, the largest and smallest magnitudes, maxima at and next to the e4m3 range's end, exact ties."""
    import nanovllm_b200
    inf, nan = float("inf"), float("nan")
    heads = [[0.0], [-0.0], [inf, 1.0], [-inf], [nan, 3.0], [1.0, nan, inf], [3.3e38, -1e38, 1.0], [-3.38e38, 1e-3],
             [2.0 ** 100, 2.0 ** 93], [2.0 ** 101, -2.0 ** 95, 2.0 ** 94], [1e-38, -2e-39], [1e-40], [9e-41, 1e-40], [2.0 ** -133],
             [448.0, 447.0, 7.0], [450.0, 449.0, 1.0], [1.75, 0.109375], [1.7578125, 0.11], [1.7421875, 0.1],
             [127.0, 0.5, 1.5, 2.5, -0.5, -3.5], [254.0, 1.0, 3.0, 5.0, -7.0], [1.0, 2.0 ** -10, 2.0 ** -17, 2.0 ** -18],
             [448.0, 2.0 ** -10, 3 * 2.0 ** -10, 17.0, 19.0, 2.0 ** -9]]
    x = torch.zeros(len(heads), 1, d)
    for i, h in enumerate(heads):
        x[i, 0, d - len(h):] = torch.tensor(h)  # the last lane's elements
    k = x.to(torch.bfloat16)
    v = k.flip(-1).contiguous()
    cache = _cache(4, 8, 1, d, fmt, cuda)
    slots = torch.randperm(32, generator=torch.Generator().manual_seed(0))[:len(heads)].int()
    want = _expect_store(cache, k, v, slots, 8)
    nanovllm_b200.store_kvcache_quant(k.to(cuda), v.to(cuda), *cache, slots.to(cuda))
    _same(cache, want)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
def test_store_every_bf16_against_every_maximum(cuda, fmt):
    """Rows of one maximum (every bf16 fraction) and the 1270 bf16 values up to it, almost 10 binades."""
    import nanovllm_b200
    frac = torch.arange(0x3F80, 0x4000, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)  # [1, 2)
    low = torch.arange(0x4000 - 10 * 127, 0x4000, dtype=torch.int32).to(torch.int16).view(torch.bfloat16)
    rows = low[None, :].expand(128, -1).clone()
    rows = torch.where(rows <= frac[:, None], rows, torch.zeros_like(rows)).view(128, -1, 127)[:, :, :127]
    rows = torch.cat([frac[:, None, None].expand(-1, rows.shape[1], 1), rows], -1)  # [128, n, 128]: heads as rows
    T, hkv, d = rows.shape
    cache = _cache(1, 128, hkv, d, fmt, cuda)
    want = _expect_store(cache, rows, -rows, torch.arange(T), 128)
    nanovllm_b200.store_kvcache_quant(rows.to(cuda), -rows.to(cuda), *cache, torch.arange(T, device=cuda))
    _same(cache, want)


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("pad", [0, 1, 4, 8])
def test_store_strided_and_misaligned(cuda, fmt, pad):
    """Views of a qkv buffer whose token pitch, or base, is not a multiple of 16 bytes."""
    import nanovllm_b200
    T, hq, hkv, d, bs = 45, 4, 2, 64, 16
    width = (hq + 2 * hkv) * d + pad
    buf = _rows(T, 1, width, torch.bfloat16, 4).view(T, width).to(cuda)
    k = torch.as_strided(buf, (T, hkv, d), (width, d, 1), hq * d + pad)
    v = torch.as_strided(buf, (T, hkv, d), (width, d, 1), (hq + hkv) * d)
    cache = _cache(5, bs, hkv, d, fmt, cuda)
    slots = torch.randperm(80, generator=torch.Generator().manual_seed(5))[:T].int()
    want = _expect_store(cache, k.cpu(), v.cpu(), slots, bs)
    nanovllm_b200.store_kvcache_quant(k, v, *cache, slots.to(cuda))
    _same(cache, want)


@pytest.mark.gpu
def test_store_bad_slots_are_reported_and_skipped(cuda):
    import nanovllm_b200
    cache = _cache(2, 8, 2, 64, E4M3, cuda)
    k = _rows(6, 2, 64, torch.bfloat16)
    slots = torch.tensor([3, -1, 16, -2, 15, 2 ** 31 - 1], dtype=torch.int32)
    want = _expect_store(cache, k, k, slots, 8)
    nanovllm_b200.status(cuda, clear=True)
    nanovllm_b200.store_kvcache_quant(k.to(cuda), k.to(cuda), *cache, slots.to(cuda))
    _same(cache, want)
    assert nanovllm_b200.status(cuda, clear=True) == 2


def _fused_inputs(T, hq, hkv, d, device, seed=0, pad=0):
    g = torch.Generator().manual_seed(seed)
    width = (hq + 2 * hkv) * d + pad
    qkv = torch.randn(T, width, generator=g).bfloat16().to(device)
    at = lambda h, off: torch.as_strided(qkv, (T, h, d), (width, d, 1), off)  # noqa: E731
    w = [(1 + 0.1 * torch.randn(d, generator=g)).bfloat16().to(device) for _ in range(2)]
    ang = torch.arange(50)[:, None] * 1e4 ** (-torch.arange(0, d, 2) / d)
    cs = torch.cat([ang.cos(), ang.sin()], -1).unsqueeze(1).to(device)
    pos = torch.randint(0, 50, (T,), generator=g).to(device)
    return at(hq, 0), at(hkv, hq * d), at(hkv, (hq + hkv) * d), pos, w[0], w[1], 1e-6, cs


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("T,hq,hkv,d,pad", [(1, 16, 8, 128, 0), (33, 16, 8, 128, 0), (700, 32, 8, 128, 8), (70, 3, 1, 64, 0),
                                            (21, 4, 2, 256, 0), (19, 4, 2, 96, 0), (25, 8, 2, 128, 3), (0, 4, 2, 64, 0)])
@pytest.mark.parametrize("write_k", [False, True])
def test_fused_equals_its_two_steps(cuda, fmt, T, hq, hkv, d, pad, write_k):
    import nanovllm_b200
    x = _fused_inputs(T, hq, hkv, d, cuda, pad=pad)
    a, b = _cache(6, 144, hkv, d, fmt, cuda), _cache(6, 144, hkv, d, fmt, cuda)
    slots = torch.randperm(864, generator=torch.Generator().manual_seed(7))[:T].int()
    slots[::7] = -1
    slots = slots.to(cuda)
    none = x[0].new_empty(0)
    q1, k1 = nanovllm_b200.qk_norm_rope_kv(*x, none, none, None, True)
    nanovllm_b200.store_kvcache_quant(k1, x[2], *a, slots)
    nanovllm_b200.status(cuda, clear=True)
    q2, k2 = nanovllm_b200.qk_norm_rope_kv_quant(*x, *b, slots, write_k)
    assert torch.equal(q1, q2) and (torch.equal(k1, k2) if write_k else k2 is None)
    _same(a, [_bits(t).cpu() for t in b])
    assert nanovllm_b200.status(cuda) == 0


@pytest.mark.gpu
def test_fused_bad_positions_and_slots(cuda):
    import nanovllm_b200
    x = list(_fused_inputs(4, 4, 2, 128, cuda))
    x[3] = torch.tensor([0, 50, -1, 3], device=cuda)
    cache = _cache(2, 8, 2, 128, I8, cuda)
    before = [_bits(t).clone() for t in cache]
    nanovllm_b200.status(cuda, clear=True)
    q, _ = nanovllm_b200.qk_norm_rope_kv_quant(*x, *cache, torch.tensor([16, -5, -1, 99], dtype=torch.int32, device=cuda), False)
    assert nanovllm_b200.status(cuda, clear=True) == 3
    _same(cache, [t.cpu() for t in before])
    assert bool(torch.isfinite(q.float()).all())


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16, torch.float32])
@pytest.mark.parametrize("lens,hkv,d,bs", [([1], 1, 8, 1), ([5, 0, 40, 0, 17], 2, 64, 16), ([300, 7], 8, 128, 48),
                                           ([33, 65, 1], 3, 256, 7), ([19], 2, 20, 16), ([0, 0, 3], 1, 72, 256)])
def test_load_bitwise_and_rows_behind(cuda, fmt, dtype, lens, hkv, d, bs):
    import nanovllm_b200
    width = max(1, max(-(-n // bs) for n in lens)) + 1
    blocks = len(lens) * width + 1
    cache = _cache(blocks, bs, hkv, d, fmt, cuda)
    cache[2][0, 0, 0] = float("nan")
    table = torch.randperm(blocks, generator=torch.Generator().manual_seed(3))[:len(lens) * width].view(-1, width).int()
    cu = torch.tensor([0] + lens).cumsum(0).int()
    n, more = int(cu[-1]), 3
    want = []
    for codes, scale in ((cache[0], cache[2]), (cache[1], cache[3])):
        values = (codes.float() * scale.transpose(1, 2)[..., None]).to(dtype).cpu()
        want.append(torch.cat([values[table[b].long()].flatten(0, 1)[:m] for b, m in enumerate(lens)]))
    nanovllm_b200.status(cuda, clear=True)
    got = nanovllm_b200.load_kvcache_quant(*cache, table.to(cuda), cu.to(cuda), n + more, dtype=dtype)
    for x, y in zip(got, want):
        assert torch.equal(torch.nan_to_num(x[:n].cpu().float(), nan=-7.0), torch.nan_to_num(y.float(), nan=-7.0))
        assert not bool(x[n:].float().any())
    out = tuple(torch.full((n + more, hkv, d), 5.0, dtype=dtype, device=cuda) for _ in range(2))
    got2 = nanovllm_b200.load_kvcache_quant(*cache, table.to(cuda), cu.to(cuda), n + more, dtype=dtype, out=out)
    for x, y, z in zip(out, got, got2):
        assert x is z and torch.equal(torch.nan_to_num(x[:n].float(), nan=-7.0), torch.nan_to_num(y[:n].float(), nan=-7.0))
        assert bool((x[n:] == 5.0).all())
    assert nanovllm_b200.status(cuda) == 0


@pytest.mark.gpu
def test_load_pages_that_cannot_be_followed(cuda):
    import nanovllm_b200
    cache = _cache(3, 4, 1, 64, I8, cuda)
    table = torch.tensor([[1, 7], [-1, 2]], dtype=torch.int32, device=cuda)
    cu = torch.tensor([0, 6, 18], dtype=torch.int32, device=cuda)  # 6 tokens; 12 tokens, 4 beyond the table's row
    nanovllm_b200.status(cuda, clear=True)
    k, v = nanovllm_b200.load_kvcache_quant(*cache, table, cu, 18)
    assert nanovllm_b200.status(cuda, clear=True) == 2
    ok = list(range(4)) + list(range(10, 14))
    assert bool(k[ok].float().any(-1).all()) and not bool(k[[4, 5, 6, 7, 8, 9, 14, 15, 16, 17]].float().any())
    assert not bool(v[[4, 5, 6, 7, 8, 9, 14, 15, 16, 17]].float().any())


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
def test_write_then_read_back(cuda, fmt):
    """The round trip's error: half a step of e4m3 (2^-4 relative, or 2^-10 steps of the scale at the bottom), half a step of int8
    (scale / 2), plus the fp32 product and int8's rounded scale (2^-23 together)."""
    import nanovllm_b200
    T, hkv, d, bs = 200, 4, 128, 16
    x = _rows(T, hkv, d, torch.bfloat16, 9).to(cuda)
    cache = nanovllm_b200.empty_quant_cache(16, bs, hkv, d, fmt, cuda)
    table = torch.randperm(16, generator=torch.Generator().manual_seed(1))[None, :13].int().to(cuda)
    t = torch.arange(T, device=cuda)
    slots = (table[0, t // bs] * bs + t % bs).int()
    nanovllm_b200.store_kvcache_quant(x, -x, *cache, slots)
    cu = torch.tensor([0, T], dtype=torch.int32, device=cuda)
    k, v = nanovllm_b200.load_kvcache_quant(*cache, table, cu, T, dtype=torch.float32)
    assert torch.equal(k, -v)
    scale = cache[2][table[0, t // bs].long(), :, t % bs][..., None]
    bound = torch.maximum(x.float().abs() * 2.0 ** -4, scale * 2.0 ** -10) if fmt == E4M3 else scale / 2
    assert bool(((k - x.float()).abs() <= bound + x.float().abs() * 2.0 ** -23).all())


@pytest.mark.gpu
def test_captured_replayed_and_on_another_stream(cuda):
    import nanovllm_b200
    x = _fused_inputs(40, 8, 2, 128, cuda)
    cache = _cache(4, 16, 2, 128, E4M3, cuda)
    slots = torch.arange(40, dtype=torch.int32, device=cuda)
    table = torch.arange(4, dtype=torch.int32, device=cuda)[None]
    cu = torch.tensor([0, 40], dtype=torch.int32, device=cuda)

    def step():
        q, k = nanovllm_b200.qk_norm_rope_kv_quant(*x, *cache, slots, True)
        nanovllm_b200.store_kvcache_quant(k, x[2], *cache, slots)
        return q, *nanovllm_b200.load_kvcache_quant(*cache, table, cu, 40)
    want = [t.clone() for t in step()]
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        got = step()
    torch.cuda.current_stream().wait_stream(side)
    for a, b in zip(got, want):
        assert torch.equal(a, b)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        got = step()
    for t in cache:
        t.view(torch.uint8).zero_()
    for _ in range(2):
        graph.replay()
    for a, b in zip(got, want):
        assert torch.equal(a, b)


@pytest.mark.gpu
def test_offsets_past_32_bits(cuda):
    """A cache of more than 2^32 codes per tensor: the last slots are written and read back, and nothing else changes."""
    import nanovllm_b200
    blocks, bs, hkv, d = 16400, 256, 8, 128  # 4.3e9 codes
    cache = nanovllm_b200.empty_quant_cache(blocks, bs, hkv, d, E4M3, cuda)
    x = _rows(3, hkv, d, torch.bfloat16).to(cuda)
    slots = torch.tensor([blocks * bs - 1, 0, blocks * bs - 256], dtype=torch.int64, device=cuda)
    nanovllm_b200.store_kvcache_quant(x, x, *cache, slots)
    table = torch.tensor([[blocks - 1], [0]], dtype=torch.int32, device=cuda)
    cu = torch.tensor([0, 256, 257], dtype=torch.int32, device=cuda)
    k, v = nanovllm_b200.load_kvcache_quant(*cache, table, cu, 257, dtype=torch.float32)
    assert torch.equal(k, v)
    c, s = cm.quantise_rows(x.cpu(), E4M3)
    want = c.float() * s[..., None]
    assert torch.equal(k[[255, 256, 0]].cpu(), want) and not bool(k[1:255].any())
    assert int((cache[2] != 0).sum()) == 3 * hkv


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float32])
@pytest.mark.parametrize("T,hkv,d,bs", [(50, 3, 512, 16), (41, 2, 320, 5), (60, 1, 48, 16), (3, 7, 16, 256), (12, 2, 528, 8)])
def test_other_row_widths_and_back(cuda, fmt, dtype, T, hkv, d, bs):
    """Head dims that fill a group of lanes in part, and the first one past the widest group; written and read back."""
    import nanovllm_b200
    pages = -(-T // bs)
    cache = _cache(pages + 1, bs, hkv, d, fmt, cuda)
    table = torch.randperm(pages + 1, generator=torch.Generator().manual_seed(9))[:pages].int()
    j = torch.arange(T)
    slots = table[j // bs].long() * bs + j % bs
    k, v = _rows(T, hkv, d, dtype, 4), _rows(T, hkv, d, dtype, 5)
    want = _expect_store(cache, k, v, slots, bs)
    nanovllm_b200.store_kvcache_quant(k.to(cuda), v.to(cuda), *cache, slots.to(cuda))
    _same(cache, want)
    got = nanovllm_b200.load_kvcache_quant(*cache, table.view(1, -1).to(cuda), torch.tensor([0, T], dtype=torch.int32,
                                                                                            device=cuda), T, dtype=dtype)
    for x, codes, scale in ((got[0], cache[0], cache[2]), (got[1], cache[1], cache[3])):
        values = (codes.float() * scale.transpose(1, 2)[..., None]).to(dtype)
        assert torch.equal(x, values[table.long().to(cuda)].flatten(0, 1)[:T])


@pytest.mark.gpu
@pytest.mark.parametrize("fmt", FMTS)
@pytest.mark.parametrize("T,hq,hkv,d", [(1001, 32, 8, 128), (9001, 3, 1, 128), (4500, 16, 2, 64), (3000, 5, 1, 256)])
def test_fused_many_tokens_equals_its_two_steps(cuda, fmt, T, hq, hkv, d):
    """Enough tokens for a lane group to take several heads of one, head counts that they do not divide included."""
    import nanovllm_b200
    x = _fused_inputs(T, hq, hkv, d, cuda)
    blocks = T // 144 + 1
    a, b = _cache(blocks, 144, hkv, d, fmt, cuda), _cache(blocks, 144, hkv, d, fmt, cuda)
    slots = torch.randperm(blocks * 144, generator=torch.Generator().manual_seed(7))[:T].int()
    slots[::7] = -1
    slots = slots.to(cuda)
    none = x[0].new_empty(0)
    q1, k1 = nanovllm_b200.qk_norm_rope_kv(*x, none, none, None, True)
    nanovllm_b200.store_kvcache_quant(k1, x[2], *a, slots)
    nanovllm_b200.status(cuda, clear=True)
    q2, k2 = nanovllm_b200.qk_norm_rope_kv_quant(*x, *b, slots, True)
    assert torch.equal(q1, q2) and torch.equal(k1, k2)
    _same(a, [_bits(t).cpu() for t in b])
    assert nanovllm_b200.status(cuda) == 0


@pytest.mark.gpu
@pytest.mark.parametrize("d", [128, 12])
def test_int8_codes_of_fp32_rows_next_to_ties(cuda, d):
    """fp32 elements at and next to the middle between two codes, for maxima of every size: the code is that of exact
    arithmetic, in the vector kernel and the scalar one. (In 64 bits 127 x is exact, and no quotient of an fp32 pair lies within
    2^-32 of a middle that it does not hit, so the oracle's is.)"""
    import nanovllm_b200
    T, hkv, bs = 600, 2, 16
    g = torch.Generator().manual_seed(d)
    top = torch.rand(T, hkv, 1, generator=g, dtype=torch.float64) + 1
    e = torch.randint(-126, 127, (T, hkv, 1), generator=g).double()
    e[::3] = torch.randint(-4, 5, e[::3].shape, generator=g).double()
    top[::5] = 127 / 64  # exact middles
    top = (top * torch.exp2(e)).float().clamp(min=127 * 2.0 ** -126).double()
    k = torch.randint(0, 127, (T, hkv, d), generator=g).double() + 0.5
    x = (k * top / 127).float()
    bits = x.view(torch.int32) + torch.randint(-1, 2, x.shape, generator=g).int()
    x = bits.view(torch.float32) * (1 - 2 * torch.randint(0, 2, x.shape, generator=g))
    x = torch.minimum(torch.maximum(x, -top.float()), top.float())
    x[..., 0] = top[..., 0].float()
    pages = -(-T // bs)
    cache = _cache(pages, bs, hkv, d, I8, cuda)
    slots = torch.randperm(pages * bs, generator=g)[:T]
    want = _expect_store(cache, x, -x, slots, bs)
    nanovllm_b200.store_kvcache_quant(x.to(cuda), -x.to(cuda), *cache, slots.to(cuda))
    _same(cache, want)
