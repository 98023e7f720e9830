// Shared by the two kernels of nvb200_cache_attention (cache_attention.cu: up to 16 query rows per KV head and CTA;
// cache_attention_wide.cu: up to 128): parameters, cache element types and their conversion.
#pragma once

#include "common.cuh"
#include "kv_quant_math.cuh"

namespace nvb200 {

enum { kBf16 = 0, kF16 = 1, kE4M3 = 2, kI8 = 3 };  // element type of the cache

constexpr int kMaxSplits = 8;  // CTAs sharing one sequence's keys: portable cluster size

struct CacheAttnParams {
  const void *q;
  int64_t q_batch_stride, q_token_stride, q_head_stride;
  const uint8_t *k_cache;
  const uint8_t *v_cache;
  int64_t blk_stride, tok_stride, head_stride;  // elements
  int64_t num_blocks;
  const float *k_scale;  // [blocks, hkv, block_size], 8-bit caches
  const float *v_scale;
  const int32_t *block_table;  // NULL: sequence b is block b
  int64_t bt_stride;
  const int32_t *seqlens;
  const int32_t *draft_lens;  // NULL: n tokens in every sequence
  const uint8_t *mask;        // [batch, n, n] bytes, NULL: chain (causal) or no mask
  int64_t mask_batch_stride, mask_row_stride;
  void *out;                  // [batch, n, hq, D] contiguous
  int n, hq, hkv, group, block_size, bs_shift, max_pages, rows, causal, splits;
  int q_is_f16;
  float scale_log2;
  int32_t *status;
};

namespace {

NVB200_DEVICE uint32_t ld_shared_u32(uint32_t addr) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(addr));
  return v;
}
NVB200_DEVICE void st_shared_u32(uint32_t addr, uint32_t v) {
  asm volatile("st.shared.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

NVB200_DEVICE uint32_t cta_rank_in_cluster() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
NVB200_DEVICE uint32_t map_shared_to(uint32_t addr, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
  return r;
}
NVB200_DEVICE void st_cluster_f32(uint32_t addr, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(addr), "f"(v) : "memory");
}
NVB200_DEVICE void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
NVB200_DEVICE void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

NVB200_DEVICE uint32_t pack_f16x2(float lo, float hi) {
  uint32_t r;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

template <int CT> struct CacheType {
  static constexpr bool kQuant = CT == kE4M3 || CT == kI8;
  static constexpr int kBytes = kQuant ? 1 : 2;
  static constexpr bool kBf16Mma = CT == kBf16;
};

// Bytes 0, 1 (lo) and 2, 3 (hi) of w, codes of an 8-bit cache, as two fp16 pairs.
template <int CT> NVB200_DEVICE void codes_to_f16(uint32_t w, uint32_t &lo, uint32_t &hi) {
  if constexpr (CT == kE4M3) {
    lo = e4m3x2_to_f16x2(static_cast<uint16_t>(w & 0xFFFFu));
    hi = e4m3x2_to_f16x2(static_cast<uint16_t>(w >> 16));
  } else {
    // 0x6400 | u is the fp16 number 1024 + u, u = code + 128: subtracting 1152 leaves the code, exactly.
    const uint32_t u = w ^ 0x80808080u;
    const __half2 off = __halves2half2(__ushort_as_half(0x6480), __ushort_as_half(0x6480));
    const uint32_t a = __byte_perm(u, 0x64646464u, 0x4140), b = __byte_perm(u, 0x64646464u, 0x4342);
    const __half2 x = __hsub2(*reinterpret_cast<const __half2 *>(&a), off);
    const __half2 y = __hsub2(*reinterpret_cast<const __half2 *>(&b), off);
    lo = *reinterpret_cast<const uint32_t *>(&x), hi = *reinterpret_cast<const uint32_t *>(&y);
  }
}
// Bits of the elements of w (two 16-bit elements or four e4m3 codes) that are infinite or NaN, set over the whole
// element. int8 codes are always finite.
template <int CT> NVB200_DEVICE uint32_t nonfinite_bits(uint32_t w) {
  if constexpr (CT == kI8) return 0u;
  if constexpr (CT == kE4M3) return __vcmpeq4(w & 0x7F7F7F7Fu, 0x7F7F7F7Fu);
  constexpr uint32_t kExp = CT == kBf16 ? 0x7F807F80u : 0x7C007C00u;
  return __vcmpeq2(w & kExp, kExp);
}

NVB200_DEVICE int page_of(const CacheAttnParams &p, int j) {
  return p.bs_shift >= 0 ? j >> p.bs_shift : j / p.block_size;
}

// Infinities and NaN of V among the new tokens are taken out of the tiles (0 * inf is NaN in a matrix instruction, and a
// row may not see them); a row that does see one gets it here, where it decides column d whatever its weight. y: the
// row's output without them.
template <int CT>
NVB200_DEVICE float add_nonfinite(const CacheAttnParams &p, const int32_t *bt, int b, int h, int qi, int d, int ctx, int L,
                                  int drafts, float y) {
  for (int k = 0; k < drafts; ++k) {
    const int j = ctx + k;
    if (j < 0 || j >= L || !(p.mask ? p.mask[b * p.mask_batch_stride + qi * p.mask_row_stride + k] != 0 : k <= qi))
      continue;
    const int page = page_of(p, j);
    const int64_t blk = bt ? __ldg(bt + page) : b;
    if (blk < 0 || blk >= p.num_blocks) continue;
    const int64_t at = blk * p.blk_stride + (j - page * p.block_size) * p.tok_stride + h * p.head_stride + d;
    if constexpr (CacheType<CT>::kQuant) {
      if ((__ldg(p.v_cache + at) & 0x7Fu) == 0x7Fu) y = __uint_as_float(0x7FC00000u);
    } else {
      const uint16_t u = __ldg(reinterpret_cast<const uint16_t *>(p.v_cache) + at);
      if (nonfinite_bits<CT>(u))
        y += CT == kBf16 ? __uint_as_float(static_cast<uint32_t>(u) << 16) : __half2float(__ushort_as_half(u));
    }
  }
  return y;
}

}  // namespace

// The wide kernel (cache_attention_wide.cu). NVB200_ERR_UNSUPPORTED where it does not take the call (pages whose size is
// not a multiple of 8 tokens, cache strides that no tensor map describes).
int launch_cache_attention_wide(const CacheAttnParams &p, int ct, int head_dim, int batch, int num_splits,
                                cudaStream_t stream);

}  // namespace nvb200
