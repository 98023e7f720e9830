// Shared by the kernels of nvb200_cache_attention (cache_attention.cu: up to 16 query rows per KV head and CTA;
// cache_attention_wide.cu: up to 128; cache_attention_merge.cu): parameters, cache element types and their conversion.
#pragma once

#include "common.cuh"
#include "kv_quant_math.cuh"

namespace nvb200 {

enum { kBf16 = 0, kF16 = 1, kE4M3 = 2, kI8 = 3 };  // element type of the cache

constexpr int kMaxSplits = 8;  // CTAs sharing one sequence's keys: portable cluster size

// The start of CTA c's range, written by CTA c. A unit is merged by the first end of a range that cuts it.
struct CutInfo {
  int parts;  // records of the unit that this end is the first to cut; 0: nothing to merge here
  int unit_u, T, G;
  int b, unit, blocks, L;
  int drafts, pad[3];
};
static_assert(sizeof(CutInfo) == 48, "whole 16-byte pieces");

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
  int n, hq, hkv, group, block_size, bs_shift, max_pages, rows, causal;
  int batch;
  int splits;      // CTAs of a cluster sharing the keys of a sequence (cluster form)
  int first_batch; // sequence of the grid's first (cluster form: a grid has at most 65535)
  // Workspace of the even-share form: what each CTA says of the start of its range, then [2 * grid] records of
  // [block_rows][D + 4] floats.
  struct CutInfo *cuts;
  float *records;
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
NVB200_DEVICE void st_cluster_v4(uint32_t addr, const float4 &v) {
  asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(addr), "f"(v.x), "f"(v.y), "f"(v.z), "f"(v.w)
               : "memory");
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

// ---------------------------------------------------------------------------------------------------------------
// Even shares of a batch whose lengths the host does not know. The work of a call is a sequence of key tiles, ordered by
// sequence, then unit (KV head, block of query rows), then tile; CTA c of G takes tiles [c T / G, (c + 1) T / G). A
// segment is the part of one unit in one CTA's range. A unit inside one range is finished there; one that a range's end
// cuts leaves a record per CTA in the workspace (only the first and the last segment of a range can be cut: two slots per
// CTA), which a second kernel merges in the order of the CTAs. No CTA waits for another, and nothing outlives the call.

struct SeqInfo {
  int L, drafts;  // keys, and how many of them (the last) are the new tokens
  int tiles;      // of keys
  int blocks;     // of query rows that hold new tokens
};

// `report`: flag lengths that had to be clamped.
NVB200_DEVICE SeqInfo seq_info(const CacheAttnParams &p, int b, int tile_keys, int block_rows, bool report = false) {
  SeqInfo s;
  s.L = __ldg(p.seqlens + b);
  s.drafts = p.draft_lens ? __ldg(p.draft_lens + b) : p.n;
  const int64_t cap = static_cast<int64_t>(p.max_pages) * p.block_size;
  if (s.L < 0 || s.L > cap || s.drafts < 0 || s.drafts > p.n) {
    if (report) set_status(p.status, NVB200_STATUS_BAD_SLOT);
    s.L = s.L < 0 ? 0 : static_cast<int>(min(static_cast<int64_t>(s.L), cap));
    s.drafts = max(0, min(s.drafts, p.n));
  }
  s.tiles = (s.L + tile_keys - 1) / tile_keys;
  s.blocks = s.L > 0 ? (s.drafts * p.group + block_rows - 1) / block_rows : 0;
  if (s.blocks == 0) s.tiles = 0;
  return s;
}

// Tiles of sequence b over all its units.
NVB200_DEVICE int seq_work(const CacheAttnParams &p, int b, int tile_keys, int block_rows) {
  const SeqInfo s = seq_info(p, b, tile_keys, block_rows);
  return s.tiles * s.blocks * p.hkv;
}

// First tile of CTA c, and the CTA that has tile u, of T tiles over G <= T CTAs.
NVB200_DEVICE int range_start(int64_t c, int64_t T, int64_t G) { return static_cast<int>(c * T / G); }
NVB200_DEVICE int range_owner(int64_t u, int64_t T, int64_t G) { return static_cast<int>(((u + 1) * G - 1) / T); }
// Record slot of CTA c for the unit that starts at tile unit_u.
NVB200_DEVICE int record_slot(int c, int unit_u, int64_t T, int64_t G) {
  return 2 * c + (unit_u <= range_start(c, T, G) ? 0 : 1);
}

// The part of one unit in a CTA's range. The same in every thread that walks it.
struct Segment {
  int u;       // global index of its first tile
  int unit_u;  // ... of the unit's first tile
  int unit;    // h * blocks + block
  int t0, n;   // its tiles within the unit; n = 0: the range is exhausted
  int b;
  SeqInfo s;
};

// The segment that holds tile u < T, ending at u1 or with its unit. Warp-wide.
NVB200_DEVICE Segment find_segment(const CacheAttnParams &p, int u, int u1, int tile_keys, int block_rows) {
  const int lane = threadIdx.x & 31;
  Segment g;
  g.u = u;
  int before = 0;
  for (int b0 = 0;; b0 += 32) {
    const int b = b0 + lane;
    int x = b < p.batch ? seq_work(p, b, tile_keys, block_rows) : 0;
    const int mine = x;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int y = __shfl_up_sync(0xffffffffu, x, o);
      if (lane >= o) x += y;
    }
    const unsigned hit = __ballot_sync(0xffffffffu, before + x > u);
    if (hit != 0 || b0 + 32 >= p.batch) {
      const int at = hit ? __ffs(hit) - 1 : 31;
      g.b = b0 + at;
      before += __shfl_sync(0xffffffffu, x - mine, at);
      break;
    }
    before += __shfl_sync(0xffffffffu, x, 31);
  }
  g.s = seq_info(p, g.b, tile_keys, block_rows);
  const int in = u - before;
  g.unit = in / g.s.tiles;
  g.t0 = in - g.unit * g.s.tiles;
  g.unit_u = u - g.t0;
  g.n = min(g.s.tiles - g.t0, u1 - u);
  return g;
}

// Moves on to the next unit of the range [., u1).
NVB200_DEVICE void next_segment(Segment &g, const CacheAttnParams &p, int u1, int tile_keys, int block_rows) {
  g.u += g.n;
  if (g.u >= u1) {
    g.n = 0;
    return;
  }
  if (++g.unit == g.s.blocks * p.hkv) {
    g.unit = 0;
    do {
      g.s = seq_info(p, ++g.b, tile_keys, block_rows);
    } while (g.s.tiles == 0);  // g.u < u1 <= T: there is one with tiles
  }
  g.unit_u = g.u, g.t0 = 0;
  g.n = min(g.s.tiles, u1 - g.u);
}

// T, by a whole warp.
NVB200_DEVICE int total_work(const CacheAttnParams &p, int tile_keys, int block_rows) {
  int x = 0;
  for (int b = threadIdx.x & 31; b < p.batch; b += 32) x += seq_work(p, b, tile_keys, block_rows);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// CTAs that get work: fewer than are launched when the tiles are few.
NVB200_DEVICE int active_ctas(int T, int grid, int min_tiles) { return max(1, min(grid, T / min_tiles)); }

// Says what CTA c's start cuts. One thread of every CTA of the grid, those without work included (g.n = 0).
NVB200_DEVICE void write_cut(const CacheAttnParams &p, int c, const Segment &g, int T, int G) {
  CutInfo x{};
  if (g.n > 0 && g.t0 > 0 && range_start(c - 1, T, G) <= g.unit_u) {
    x.parts = range_owner(g.unit_u + g.s.tiles - 1, T, G) - (c - 1) + 1;
    x.unit_u = g.unit_u, x.T = T, x.G = G, x.b = g.b, x.unit = g.unit, x.blocks = g.s.blocks, x.L = g.s.L, x.drafts = g.s.drafts;
  }
  uint4 *to = reinterpret_cast<uint4 *>(p.cuts + c);
  const uint4 *from = reinterpret_cast<const uint4 *>(&x);
  to[0] = from[0], to[1] = from[1], to[2] = from[2];
}

// Rows of the output that no unit covers (tokens behind draft_lens[b] beyond the last block, sequences without keys):
// zeros, CTA c of `grid` taking every grid-th sequence. Also reports clamped lengths.
NVB200_DEVICE void zero_uncovered_rows(const CacheAttnParams &p, int head_dim, int tile_keys, int block_rows, int c, int grid,
                                       int tid, int threads) {
  for (int b = c; b < p.batch; b += grid) {
    const SeqInfo s = seq_info(p, b, tile_keys, block_rows, tid == 0);
    const int from = min(s.blocks * block_rows, p.n * p.group);
    // Row r of KV head h is token r / group, head h * group + r % group. 16-byte pieces where `out` allows.
    const int rows = p.n * p.group - from;
    const bool wide = (reinterpret_cast<uintptr_t>(p.out) & 15) == 0;
    const int pieces = wide ? head_dim / 8 : head_dim;
    for (int h = 0; h < p.hkv; ++h) {
      for (int e = tid; e < rows * pieces; e += threads) {
        const int r = from + e / pieces, d = e % pieces, qi = r / p.group;
        const int64_t row = ((static_cast<int64_t>(b) * p.n + qi) * p.hq + h * p.group + r - qi * p.group) * head_dim;
        if (wide) *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p.out) + row + 8 * d) = make_uint4(0u, 0u, 0u, 0u);
        else static_cast<uint16_t *>(p.out)[row + d] = 0;
      }
    }
  }
}

NVB200_DEVICE int page_of(const CacheAttnParams &p, int j) {
  return p.bs_shift >= 0 ? j >> p.bs_shift : j / p.block_size;
}

// Infinities and NaN of V among the new tokens are taken out of the tiles (0 * inf is NaN in a matrix instruction, and a
// row may not see them); a row that does see one gets it from here, where it decides a column whatever its weight: what those
// that token qi sees add to columns d .. d + N - 1 of KV head h (d a multiple of N: one piece of the row). Only for segments
// that held one. The loads of eight keys are in flight together, so a call of 4096 new tokens with infinities in all
// of them takes 3.2 ms (wide kernel, one KV head, head_dim 128; 0.09 ms without), far from the second that waiting warps allow.
template <int N> struct Columns {
  float v[N];
};
template <int CT, int N>
__device__ __noinline__ Columns<N> nonfinite_sum(const CacheAttnParams &p, const int32_t *bt, int b, int h, int qi, int d,
                                                 int ctx, int drafts) {
  constexpr int kBatch = 8, kWords = N * CacheType<CT>::kBytes / 4;
  Columns<N> y{};
  const uint8_t *mask = p.mask ? p.mask + b * p.mask_batch_stride + qi * p.mask_row_stride : nullptr;
  for (int k0 = 0; k0 < drafts; k0 += kBatch) {
    int blk[kBatch];
    uint32_t w[kBatch][kWords];
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      const int k = k0 + i;
      const bool seen = k < drafts && ctx + k >= 0 && (mask ? __ldg(mask + k) != 0 : k <= qi);
      blk[i] = !seen ? -1 : (bt ? __ldg(bt + page_of(p, ctx + k)) : b);
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
#pragma unroll
      for (int e = 0; e < kWords; ++e) w[i][e] = 0u;
      if (blk[i] >= 0 && blk[i] < p.num_blocks) {
        const int j = ctx + k0 + i;
        const int64_t at = blk[i] * p.blk_stride + (j - page_of(p, j) * p.block_size) * p.tok_stride + h * p.head_stride + d;
        const uint8_t *from = p.v_cache + at * CacheType<CT>::kBytes;
        if constexpr (kWords == 4) {
          const uint4 u = __ldg(reinterpret_cast<const uint4 *>(from));
          w[i][0] = u.x, w[i][1] = u.y, w[i][2] = u.z, w[i][3] = u.w;
        } else if constexpr (kWords == 2) {
          const uint2 u = __ldg(reinterpret_cast<const uint2 *>(from));
          w[i][0] = u.x, w[i][1] = u.y;
        } else {
          w[i][0] = __ldg(reinterpret_cast<const uint32_t *>(from));
        }
      }
    }
#pragma unroll
    for (int i = 0; i < kBatch; ++i) {
      uint32_t found = 0;
#pragma unroll
      for (int e = 0; e < kWords; ++e) found |= nonfinite_bits<CT>(w[i][e]);
      if (found == 0) continue;
#pragma unroll
      for (int e = 0; e < N; ++e) {
        if constexpr (CacheType<CT>::kQuant) {
          if ((w[i][e / 4] >> (8 * (e % 4)) & 0x7Fu) == 0x7Fu) y.v[e] = __uint_as_float(0x7FC00000u);
        } else {
          const uint32_t u = w[i][e / 2] >> (16 * (e % 2)) & 0xFFFFu;
          if (nonfinite_bits<CT>(u))
            y.v[e] += CT == kBf16 ? __uint_as_float(u << 16) : __half2float(__ushort_as_half(static_cast<unsigned short>(u)));
        }
      }
    }
  }
  return y;
}

}  // namespace

// The wide kernel (cache_attention_wide.cu). NVB200_ERR_UNSUPPORTED where it does not take the call (pages whose size is
// not a multiple of 8 tokens, row scales off a 16-byte boundary, cache strides that no tensor map describes).
bool wide_takes(const CacheAttnParams &p);
int64_t wide_workspace_bytes(const CacheAttnParams &p, int ct, int head_dim);
int launch_cache_attention_wide(const CacheAttnParams &p, int ct, int head_dim, void *workspace, cudaStream_t stream);

// Merges the records of the units that range ends cut, after a grid of `grid` CTAs.
int launch_cache_attention_merge(const CacheAttnParams &p, int ct, int head_dim, int block_rows, int grid,
                                 cudaStream_t stream);
inline int64_t even_share_bytes(int grid, int block_rows, int head_dim) {
  return static_cast<int64_t>(grid) * (sizeof(CutInfo) + 2ll * block_rows * (head_dim + 4) * 4);
}
inline void place_workspace(CacheAttnParams &p, void *workspace, int grid) {
  p.cuts = static_cast<CutInfo *>(workspace);
  p.records = reinterpret_cast<float *>(p.cuts + grid);
}

}  // namespace nvb200
