"""Attention of a few new tokens per sequence over the paged KV cache on B200 (`nvb200_cache_attention`).

* `tree_attention`: the new tokens are drafts of a tree (or any set): each sees the context and those of the others that
  its mask row names. For verifying drafted tokens, beside the chain that `attention.flash_attn_with_kvcache` verifies
  (nanovllm/layers/attention.py:84-91). 16-bit caches, or the 8-bit ones of `kv_quant`.
* `decode_attention_quant`: `attention.decode_attention` (single tokens or a causal chain) over an 8-bit cache.

The new tokens' keys and values are in the cache already (its last rows). Both launch on the current stream of q's
device, allocate their output and workspace with torch (graph-capture safe; nothing is kept between calls), and never read
device data on the host.
Out-of-range block-table entries and lengths are never followed; they are flagged in the device status word
(nanovllm_b200.status()). Types and layouts without a kernel raise NotImplementedError.
"""
import torch

from nanovllm_b200 import _lib
from nanovllm_b200.kernels.kv_quant import check_quant_cache

_QUERY = {torch.bfloat16: _lib.BF16, torch.float16: _lib.F16}
MAX_NEW_TOKENS = 4096
MAX_ROWS = 65536  # query rows per KV head


def _require(cond: bool, msg: str = "") -> None:
    if not cond:
        raise AssertionError(msg)


def _run(what, q, k_cache, v_cache, k_scale, v_scale, cache_seqlens, block_table, tree_mask, draft_lens, softmax_scale,
         causal, num_splits):
    sq = q.stride()
    _require(len(sq) == 4 and sq[3] == 1 and q.is_cuda, "q must be a CUDA tensor [B, n, Hq, D], unit last stride")
    B, n, hq, d = q.shape
    dev, idx = q.device, q.get_device()
    if k_scale is None and v_scale is None:
        _require(k_cache.dim() == 4 and v_cache.shape == k_cache.shape and v_cache.stride() == k_cache.stride()
                 and k_cache.stride(3) == 1, "the caches must be [blocks, block_size, Hkv, D] of equal strides, unit last")
        _require(k_cache.dtype == v_cache.dtype, "the caches must have one dtype")
        _require(k_cache.dtype not in _lib.QUANT_CODE, "an 8-bit cache needs k_scale and v_scale")
        if k_cache.dtype != q.dtype:
            raise NotImplementedError(f"{what}: a 16-bit cache must have q's dtype")
        nb, bs, hkv, dk = k_cache.shape
        code, scales = _QUERY.get(q.dtype), (0, 0)
    else:
        _require(k_scale is not None and v_scale is not None, "k_scale and v_scale come together")
        nb, bs, hkv, dk = check_quant_cache(k_cache, v_cache, k_scale, v_scale)
        code, scales = _lib.QUANT_CODE[k_cache.dtype], (k_scale.data_ptr(), v_scale.data_ptr())
    if q.dtype not in _QUERY:
        raise NotImplementedError(f"{what}: q must be bf16 or fp16")
    _require(dk == d and hkv > 0 and hq > 0 and hq % hkv == 0, "the cache must have q's D, and Hq a multiple of Hkv")
    _require(bs > 0, "block_size must be positive")
    if d not in (64, 128):
        raise NotImplementedError(f"{what}: head_dim must be 64 or 128")
    if n > MAX_NEW_TOKENS:
        raise NotImplementedError(f"{what}: at most {MAX_NEW_TOKENS} new tokens per sequence")
    if n * (hq // hkv) > MAX_ROWS:
        raise NotImplementedError(f"{what}: at most {MAX_ROWS} query rows (n * Hq / Hkv) per KV head")
    _require(0 <= num_splits <= 8, "num_splits must be 0 (automatic) to 8")
    if isinstance(cache_seqlens, int):
        cache_seqlens = torch.full((B,), cache_seqlens, dtype=torch.int32, device=dev)
    _require(cache_seqlens.shape == (B,) and cache_seqlens.dtype == torch.int32, "cache_seqlens must be int32 [B]")
    _require(k_cache.get_device() == v_cache.get_device() == cache_seqlens.get_device() == idx,
             "q, the caches and cache_seqlens must be on one device")
    seqlens = cache_seqlens if cache_seqlens.is_contiguous() else cache_seqlens.contiguous()
    if block_table is not None:
        _require(block_table.dim() == 2 and block_table.shape[0] == B and block_table.shape[1] > 0
                 and block_table.dtype == torch.int32 and block_table.get_device() == idx
                 and (block_table.stride(1) == 1 or block_table.shape[1] == 1),
                 "block_table must be int32 [B, max_blocks] on q's device")
        table, table_stride, pages = block_table.data_ptr(), block_table.stride(0), block_table.shape[1]
    else:
        _require(nb >= B, "without a block_table the cache must have a block for each sequence")
        table, table_stride, pages = 0, 0, 1
    mask, mask_b, mask_r, drafts = 0, 0, 0, 0
    if tree_mask is not None:
        _require(tree_mask.dtype == torch.bool and tree_mask.device == dev, "tree_mask must be bool on q's device")
        if tree_mask.dim() == 2:
            _require(tree_mask.shape == (n, n), "tree_mask must be [n, n] or [B, n, n]")
        else:
            _require(tree_mask.shape == (B, n, n), "tree_mask must be [n, n] or [B, n, n]")
            mask_b = tree_mask.stride(0)
        if n > 1 and tree_mask.stride(-1) != 1:
            tree_mask = tree_mask.contiguous()
            mask_b = tree_mask.stride(0) if tree_mask.dim() == 3 else 0
        mask, mask_r = tree_mask.data_ptr(), tree_mask.stride(-2)
    if draft_lens is not None:
        _require(draft_lens.shape == (B,) and draft_lens.dtype == torch.int32 and draft_lens.device == dev,
                 "draft_lens must be int32 [B] on q's device")
        draft_lens = draft_lens if draft_lens.is_contiguous() else draft_lens.contiguous()
        drafts = draft_lens.data_ptr()
    out = q.new_empty((B, n, hq, d))
    if B == 0 or n == 0:
        return out
    sk = k_cache.stride()
    a = _lib.CacheAttentionArgs.pack(
        out.data_ptr(), q.data_ptr(), sq[0], sq[1], sq[2], k_cache.data_ptr(), v_cache.data_ptr(), sk[0], sk[1], sk[2],
        scales[0], scales[1], nb, table, table_stride, seqlens.data_ptr(), drafts, mask, mask_b, mask_r,
        B, n, hq, hkv, d, bs, pages, int(bool(causal)), int(num_splits), _QUERY[q.dtype], code,
        d ** -0.5 if softmax_scale is None else float(softmax_scale), _lib.status_word(dev).data_ptr())
    L = _lib.lib()
    with _lib.device_of(dev):
        need = L.nvb200_cache_attention_workspace_size(a)
        ws = torch.empty(need, dtype=torch.uint8, device=dev) if need > 0 else None
        rc = L.nvb200_cache_attention(a, _lib.ptr(ws), max(need, 0), _lib.stream_of(q))
    if rc == _lib.ERR_UNSUPPORTED:
        raise NotImplementedError(f"{what}: cache rows must be 16-byte aligned, a sequence's block table address at most "
                                  "2^31 - 65536 keys, and Hkv * ceil(n * Hq / Hkv / 16) be at most 65535")
    _lib.check(rc, what)
    return out


def tree_attention(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, cache_seqlens: torch.Tensor,
                   tree_mask: torch.Tensor | None = None, block_table: torch.Tensor | None = None,
                   draft_lens: torch.Tensor | None = None, softmax_scale: float | None = None,
                   k_scale: torch.Tensor | None = None, v_scale: torch.Tensor | None = None,
                   num_splits: int = 0) -> torch.Tensor:
    """q: [B, n, Hq, D] bf16 or fp16, the new tokens of B sequences. k_cache, v_cache: [blocks, block_size, Hkv, D] (with
    block_table [B, max_blocks] int32) or [B, max_len, Hkv, D] (without), in q's dtype, or 8-bit with k_scale, v_scale
    [blocks, Hkv, block_size]. cache_seqlens: [B] int32 or an int, the keys in the cache per sequence, the new tokens being
    the last draft_lens[b] of them ([B] int32, default n).
    tree_mask: bool [n, n] or [B, n, n]; new token i sees the context (the keys before the new tokens) and new token j
    where tree_mask[..., i, j] (nothing is implied: a token sees itself only if its mask says so). None: the chain, token i
    sees new tokens 0..i. Returns [B, n, Hq, D] in q's dtype; tokens i >= draft_lens[b], and rows that see no key, give
    zeros. A key that a row does not see has no effect on it, infinities and NaN included. softmax_scale: default
    D ** -0.5. num_splits: CTAs sharing one sequence's keys, 1-8, 0 = chosen from the sizes."""
    return _run("tree_attention", q, k_cache, v_cache, k_scale, v_scale, cache_seqlens, block_table, tree_mask,
                draft_lens, softmax_scale, True, num_splits)


def decode_attention_quant(q: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor,
                           v_scale: torch.Tensor, cache_seqlens: torch.Tensor, block_table: torch.Tensor | None = None,
                           softmax_scale: float | None = None, causal: bool = False, num_splits: int = 0) -> torch.Tensor:
    """`attention.decode_attention` over an 8-bit cache (kv_quant): q [B, n, Hq, D] bf16 or fp16 against the
    cache_seqlens[b] keys of each sequence ([B] int32, or an int for all); causal aligns query i of n with key L - n + i. Returns [B, n, Hq, D]."""
    _require(k_scale is not None and v_scale is not None, "decode_attention_quant: an 8-bit cache has scales")
    return _run("decode_attention_quant", q, k_cache, v_cache, k_scale, v_scale, cache_seqlens, block_table, None, None,
                softmax_scale, causal, num_splits)


__all__ = ["tree_attention", "decode_attention_quant"]
