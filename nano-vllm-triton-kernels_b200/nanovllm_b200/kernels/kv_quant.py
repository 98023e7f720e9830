"""The 8-bit paged KV cache on B200: quantised as it is written, and read back.

A cache row (one token of one KV head) is head_dim codes, float8_e4m3fn or int8, and one fp32 scale; its values are
code * scale. Codes lie in [blocks, block_size, Hkv, D], as the 16-bit cache does, scales in [blocks, Hkv, block_size].
e4m3 scales are powers of two, 2^E with E the smallest integer >= -126 for which max|x| <= 448 * 2^E, so a code is one
rounding of its element; int8 scales are d / 127, d = max(max|x|, 127 * 2^-126), codes 127 x / d rounded half to even. A
row with an infinity or NaN reads back as NaN throughout.

* `empty_quant_cache(...)` allocates one; `store_kvcache_quant` writes it as `attention.store_kvcache` writes the 16-bit
  cache (nanovllm/layers/attention.py:34-41); `qk_norm_rope_kv_quant` is the fused q/k RMSNorm + RoPE + cache write
  (nanovllm/kernels/qk_norm_rope_kv.py:92-125) onto it; `load_kvcache_quant` reads sequences back into packed 16- or
  32-bit rows, as a variable-length prefill attention takes them. `cache_attention` has the attention that reads it.
* All launch on the current stream of their tensors' device, allocate outputs with torch (graph-capture safe), and never
  read device data on the host. Out-of-range slots, positions and block-table entries are skipped and flagged in the
  device status word (nanovllm_b200.status()).
* Within one call the slots other than -1 must differ from each other.
"""
import torch

from nanovllm_b200 import _lib
from nanovllm_b200.kernels import qk_norm_rope_kv as _fused

_SLOT_BYTES = {torch.int32: 4, torch.int64: 8}


def _require(cond: bool, msg: str = "") -> None:
    if not cond:
        raise AssertionError(msg)


def empty_quant_cache(num_blocks: int, block_size: int, num_kv_heads: int, head_dim: int,
                      dtype: torch.dtype = torch.float8_e4m3fn, device="cuda"):
    """(k_cache, v_cache, k_scale, v_scale) of an 8-bit cache, every row zero."""
    _require(dtype in _lib.QUANT_CODE, "dtype must be float8_e4m3fn or int8")
    codes = (num_blocks, block_size, num_kv_heads, head_dim)
    scales = (num_blocks, num_kv_heads, block_size)
    return (torch.zeros(codes, dtype=torch.uint8, device=device).view(dtype),
            torch.zeros(codes, dtype=torch.uint8, device=device).view(dtype),
            torch.zeros(scales, dtype=torch.float32, device=device), torch.zeros(scales, dtype=torch.float32, device=device))


def check_quant_cache(k_cache, v_cache, k_scale, v_scale) -> tuple[int, int, int, int]:
    """Checks the four tensors of an 8-bit cache; (blocks, block_size, Hkv, D)."""
    shape = k_cache.shape
    dtype = k_cache.dtype
    _require(len(shape) == 4 and dtype in _lib.QUANT_CODE and v_cache.dtype == dtype and v_cache.shape == shape
             and k_cache.is_contiguous() and v_cache.is_contiguous(),
             "k_cache, v_cache must be contiguous [blocks, block_size, Hkv, D] float8_e4m3fn or int8")
    blocks, bs, hkv, d = shape
    scale_shape = k_scale.shape
    _require(k_scale.dtype is v_scale.dtype is torch.float32 and scale_shape == (blocks, hkv, bs)
             and v_scale.shape == scale_shape and k_scale.is_contiguous() and v_scale.is_contiguous(),
             "k_scale, v_scale must be contiguous fp32 [blocks, Hkv, block_size]")
    _require(k_cache.get_device() == v_cache.get_device() == k_scale.get_device() == v_scale.get_device(),
             "the cache's tensors must be on one device")
    return blocks, bs, hkv, d


def _cache_arg(k_cache, v_cache, k_scale, v_scale, shape):
    return _lib.QuantCache.pack(k_cache.data_ptr(), v_cache.data_ptr(), k_scale.data_ptr(), v_scale.data_ptr(), *shape,
                           _lib.QUANT_CODE[k_cache.dtype])


def store_kvcache_quant(key: torch.Tensor, value: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
                        k_scale: torch.Tensor, v_scale: torch.Tensor, slot_mapping: torch.Tensor) -> None:
    """key, value: [N, Hkv, D] bf16, fp16 or fp32 with contiguous heads (any token stride). The rows of token t are
    quantised into slot slot_mapping[t] (int32 or int64; slot s is token s % block_size of block s // block_size) and slot
    -1 stores nothing. In place."""
    _require(key.dim() == 3 and value.shape == key.shape and value.dtype == key.dtype, "key, value must be [N, Hkv, D]")
    _require(key.dtype in _lib.DTYPE_CODE, "dtype must be bf16, fp16 or fp32")
    n, hkv, d = key.shape
    key_strides, value_strides = key.stride(), value.stride()
    _require(key_strides[1:] == value_strides[1:] == (d, 1),
             "each head must be contiguous: stride(2) == 1, stride(1) == D")
    shape = check_quant_cache(k_cache, v_cache, k_scale, v_scale)
    _require(shape[2:] == (hkv, d), "the cache must hold rows of the key's Hkv and D")
    _require(slot_mapping.shape == (n,) and slot_mapping.dtype in _SLOT_BYTES, "slot_mapping must be int32 or int64 [N]")
    _require(key.is_cuda, "key must be a CUDA tensor")
    _require(key.get_device() == value.get_device() == k_cache.get_device() == slot_mapping.get_device(),
             "key, value, the cache and slot_mapping must be on one device")
    dev = key.device
    if n == 0:
        return
    slots = slot_mapping if slot_mapping.is_contiguous() else slot_mapping.contiguous()
    cache = _cache_arg(k_cache, v_cache, k_scale, v_scale, shape)
    with _lib.device_of(dev):
        _lib.check(_lib.lib().nvb200_store_kvcache_quant(
            key.data_ptr(), key_strides[0], value.data_ptr(), value_strides[0], slots.data_ptr(),
            _SLOT_BYTES[slots.dtype], n, _lib.DTYPE_CODE[key.dtype], cache, _lib.status_word(dev).data_ptr(),
            _lib.stream_of(key)), "store_kvcache_quant")


def qk_norm_rope_kv_quant(
    q: torch.Tensor, k: torch.Tensor, v: torch.Tensor, positions: torch.Tensor, q_weight: torch.Tensor,
    k_weight: torch.Tensor, eps: float, cos_sin_cache: torch.Tensor, k_cache: torch.Tensor, v_cache: torch.Tensor,
    k_scale: torch.Tensor, v_scale: torch.Tensor, slot_mapping: torch.Tensor, write_k: bool,
) -> tuple[torch.Tensor, torch.Tensor | None]:
    """`qk_norm_rope_kv` with the cache write quantised: the same arguments (see there), the 8-bit cache in the place of
    the 16-bit one. Returns (q_out, k_out or None), with that function's bits; the rows stored are those that
    store_kvcache_quant(k_out, v, ...) stores."""
    T, Hq, D = q.shape
    Hkv = k.shape[1]
    _require(q.dtype == k.dtype == v.dtype == torch.bfloat16 and k.shape == v.shape == (T, Hkv, D),
             "q, k, v must be bf16 with k.shape == v.shape == (T, Hkv, D)")
    _require(Hkv > 0 and Hq % Hkv == 0 and D % 2 == 0, "Hq must be a multiple of Hkv and D even")
    sq, sk, sv = q.stride(), k.stride(), v.stride()
    _require(sq[1:] == sk[1:] == sv[1:] == (D, 1), "each head must be contiguous: stride(2) == 1, stride(1) == D")
    _require(positions.shape == (T,) and positions.dtype == torch.int64 and positions.is_contiguous(),
             "positions must be contiguous int64 [T]")
    _require(cos_sin_cache.dtype == torch.float32 and cos_sin_cache.shape[-1] == D and cos_sin_cache.stride(-1) == 1
             and cos_sin_cache.numel() == cos_sin_cache.shape[0] * D,
             "cos_sin_cache must be fp32 [max_pos, D] or [max_pos, 1, D] rows with a unit last stride")
    _require(q_weight.dtype == k_weight.dtype == torch.bfloat16 and q_weight.shape == k_weight.shape == (D,)
             and q_weight.is_contiguous() and k_weight.is_contiguous(), "q/k weights must be contiguous bf16 [D]")
    shape = check_quant_cache(k_cache, v_cache, k_scale, v_scale)
    _require(shape[2:] == (Hkv, D), "the cache must hold rows of k's Hkv and D")
    _require(slot_mapping.shape == (T,) and slot_mapping.dtype == torch.int32 and slot_mapping.is_contiguous(),
             "slot_mapping must be contiguous int32 [T]")
    dev, idx = q.device, q.get_device()
    _require(q.is_cuda, "q must be a CUDA tensor")
    for x in (k, v, positions, q_weight, k_weight, cos_sin_cache, k_cache, slot_mapping):
        _require(x.get_device() == idx, "all tensors must be on one device")
    q_out = q.new_empty((T, Hq, D))
    k_out = q.new_empty((T, Hkv, D)) if write_k else None
    if T == 0:
        return q_out, k_out
    a = _lib.QkNormRopeKvArgs.pack(
        q_out.data_ptr(), 0 if k_out is None else k_out.data_ptr(), q.data_ptr(), k.data_ptr(), v.data_ptr(), sq[0], sk[0], sv[0],
        positions.data_ptr(), slot_mapping.data_ptr(), q_weight.data_ptr(), k_weight.data_ptr(),
        cos_sin_cache.data_ptr(), cos_sin_cache.stride(0), cos_sin_cache.shape[0], 0, 0, 0, T, Hq, Hkv, D, eps,
        _lib.status_word(dev).data_ptr())
    cache = _cache_arg(k_cache, v_cache, k_scale, v_scale, shape)
    with _lib.device_of(dev):
        rc = _lib.lib().nvb200_qk_norm_rope_kv_quant(a, cache, _lib.stream_of(q))
        if rc == _lib.ERR_UNSUPPORTED:
            # Head dims and layouts without a fused kernel: the two steps.
            none = q.new_empty(0)
            q_out, k_out = _fused.qk_norm_rope_kv(q, k, v, positions, q_weight, k_weight, eps, cos_sin_cache, none,
                                                  none, None, True)
            store_kvcache_quant(k_out, v, k_cache, v_cache, k_scale, v_scale, slot_mapping)
            return q_out, k_out if write_k else None
        _lib.check(rc, "qk_norm_rope_kv_quant")
    return q_out, k_out


def load_kvcache_quant(k_cache: torch.Tensor, v_cache: torch.Tensor, k_scale: torch.Tensor, v_scale: torch.Tensor,
                       block_table: torch.Tensor, cu_seqlens: torch.Tensor, total_tokens: int,
                       dtype: torch.dtype = torch.bfloat16, out: tuple[torch.Tensor, torch.Tensor] | None = None,
                       ) -> tuple[torch.Tensor, torch.Tensor]:
    """(key, value) [total_tokens, Hkv, D] in dtype (bf16, fp16 or fp32): row t is token t - cu_seqlens[b] of sequence b
    for cu_seqlens[b] <= t < cu_seqlens[b + 1]. block_table: [B, max_blocks] int32; cu_seqlens: [B + 1] int32, not
    falling. Rows behind the last sequence are zeros, or, with `out` (contiguous tensors of that shape and dtype to
    write to), left as they were."""
    shape = check_quant_cache(k_cache, v_cache, k_scale, v_scale)
    _require(dtype in _lib.DTYPE_CODE, "dtype must be bf16, fp16 or fp32")
    _require(block_table.dim() == 2 and block_table.dtype == torch.int32 and block_table.shape[1] > 0
             and (block_table.stride(1) == 1 or block_table.shape[1] == 1), "block_table must be int32 [B, max_blocks]")
    B = block_table.shape[0]
    _require(cu_seqlens.shape == (B + 1,) and cu_seqlens.dtype == torch.int32 and cu_seqlens.is_contiguous(),
             "cu_seqlens must be contiguous int32 [B + 1]")
    dev = k_cache.device
    _require(k_cache.is_cuda and block_table.device == dev and cu_seqlens.device == dev,
             "the cache, block_table and cu_seqlens must be on one CUDA device")
    _require(total_tokens >= 0, "total_tokens must not be negative")
    want = (total_tokens, shape[2], shape[3])
    if out is None:
        key, value = torch.empty(want, dtype=dtype, device=dev), torch.empty(want, dtype=dtype, device=dev)
    else:
        key, value = out
        for x in (key, value):
            _require(x.shape == want and x.dtype == dtype and x.device == dev and x.is_contiguous(),
                     "out must be two contiguous [total_tokens, Hkv, D] tensors of dtype on the cache's device")
    if total_tokens == 0:
        return key, value
    cache = _cache_arg(k_cache, v_cache, k_scale, v_scale, shape)
    with _lib.device_of(dev):
        _lib.check(_lib.lib().nvb200_load_kvcache_quant(
            key.data_ptr(), value.data_ptr(), cache, block_table.data_ptr(), block_table.stride(0), block_table.shape[1],
            cu_seqlens.data_ptr(), B, total_tokens, _lib.DTYPE_CODE[dtype], int(out is None),
            _lib.status_word(dev).data_ptr(), _lib.stream_of(key)), "load_kvcache_quant")
    return key, value


__all__ = ["empty_quant_cache", "store_kvcache_quant", "qk_norm_rope_kv_quant", "load_kvcache_quant"]
