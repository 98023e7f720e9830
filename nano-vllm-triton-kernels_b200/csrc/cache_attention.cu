// Attention of a few new tokens per sequence over the paged KV cache: single decode tokens, causal chains, and trees of
// drafted tokens (each drafted token sees the context, and of the drafted tokens those its mask row names: its
// ancestors), over 16-bit caches or the 8-bit ones of kv_quant.cu. The reference verifies linear drafts only, through
// flash_attn_with_kvcache (nanovllm/layers/attention.py:84-91); masks and 8-bit caches have no counterpart there.
//
// Mathematics, per query row (token i, query head h) over its visible keys j:
//   s_j = scale * ks_j * (q . k_j),  p_j = 2^(s_j log2 e - m),  out = (sum_j p_j vs_j v_j) / (sum_j p_j)
// with k_j, v_j the stored codes and ks_j, vs_j their row scales (1 for 16-bit caches); one pass over the keys with the
// running maximum m and sum l. Masked keys are selected away (p = 0 by selection, never by adding -inf), so no value of
// a key that a row does not see, infinities and NaN included, reaches it; a row that sees no key gives zeros.
//
// 8-bit caches run on fp16 matrix instructions: e4m3 and int8 codes are exact in fp16 (one conversion per two codes), and
// the query row is brought to fp16 by an exact power of two, so the only roundings are those of p and the output.
// The weights p_j vs_j carry the row scales, whose range fp16 does not have; they are held relative to M, the running
// maximum of s_j log2 e + (binary exponent of vs_j) + 1, which keeps each in [0, 1] with the largest near 1.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "cache_attention.cuh"

namespace nvb200 {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kRows = 16;          // query rows of a CTA: the rows of one m16n8k16 instruction

NVB200_DEVICE void cp_async16(uint32_t dst, const void *src, uint32_t src_bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
}
NVB200_DEVICE void cp_async4(uint32_t dst, const void *src, uint32_t src_bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
}
NVB200_DEVICE void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> NVB200_DEVICE void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

NVB200_DEVICE float2 ld_shared_f2(uint32_t addr) {
  float2 v;
  asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(addr));
  return v;
}
NVB200_DEVICE void mma_16816_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
      "{%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <int CT> NVB200_DEVICE void mma_ct(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (CacheType<CT>::kBf16Mma) mma_16816(d, a, b0, b1);
  else mma_16816_f16(d, a, b0, b1);
}

// The same for the byte pairs (0, 2) and (1, 3).
template <int CT> NVB200_DEVICE void codes_to_f16_even_odd(uint32_t w, uint32_t &even, uint32_t &odd) {
  codes_to_f16<CT>(__byte_perm(w, 0u, 0x3120), even, odd);
}

// Shared-memory geometry of one (cache type, head_dim) pair. A warp streams tiles of kTile keys: kTile K rows, kTile V
// rows, for 8-bit caches their 2 x kTile scales, and one word of flags (bit r: key r exists and its page is valid).
template <int CT, int D> struct Geometry {
  static constexpr int kRowBytes = D * CacheType<CT>::kBytes;  // 64, 128 or 256
  static constexpr int kChunks = kRowBytes / 16;
  static constexpr int kTile = kRowBytes >= 256 ? 16 : 32;
  static constexpr int kStages = 3;
  static constexpr int kKvBytes = kTile * kRowBytes;
  static constexpr int kScaleBytes = CacheType<CT>::kQuant ? 2 * kTile * 4 : 0;
  static constexpr int kStageBytes = 2 * kKvBytes + kScaleBytes + 128;  // a multiple of 128
  static constexpr int kRing = kWarps * kStages * kStageBytes;
  static constexpr int kStride = D + 8;  // floats per record: o[D], m, l, M, flag, padding
  static constexpr int kRecords = kWarps * kRows * kStride * 4;
  static constexpr int kPartials = (kMaxSplits + kRows - 1) * kStride * 4;  // splits * ceil(16 / splits) records
  static constexpr int kSmem = kRing > kRecords + kPartials ? kRing : kRecords + kPartials;
  // Physical 16-byte chunk of logical chunk c of row r: the 8 rows of an 8 x 16-byte matrix at one logical chunk fall
  // in distinct bank groups (two 64-byte rows share a 128-byte line, so their swizzle steps every second row).
  static NVB200_DEVICE int chunk(int r, int c) { return kRowBytes == 64 ? c ^ ((r >> 1) & 3) : c ^ (r & 7); }
};

// One warp's softmax state: lane 4 g + t holds query rows g and g + 8 (index 0, 1). l is the lane's share.
template <int D> struct RowState {
  float m[2], l[2], M[2], o[D / 8][4];
};

// Which keys the rows of this lane see.
struct RowView {
  int qi[2];             // token of rows g and g + 8, -1: a padding row, sees nothing
  const uint8_t *mrow[2];  // its mask row
};

// Folds one tile. kt: the stage's base address. j0: index of its first key. ctx: keys before the drafted tokens;
// every live row sees keys below `open` (ctx with a mask or chain, the length otherwise).
template <int CT, int D>
NVB200_DEVICE void fold_tile(RowState<D> &st, uint32_t kt, const uint32_t (&qa)[D / 16][4], const float (&rs)[2],
                             const RowView &rv, const CacheAttnParams &p, int lane, int j0, int ctx, int open) {
  using G = Geometry<CT, D>;
  using C = CacheType<CT>;
  constexpr int NT = G::kTile / 8;  // key n-tiles of S
  const int t = lane & 3, mq = lane >> 3, rr = lane & 7;
  float s[NT][4];
#pragma unroll
  for (int i = 0; i < NT; ++i) s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
  if constexpr (!C::kQuant) {
#pragma unroll
    for (int np = 0; np < NT / 2; ++np) {
      const int key = np * 16 + (mq >> 1) * 8 + rr;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t b[4];
        ldsm_x4(kt + key * G::kRowBytes + G::chunk(key, 2 * ks + (mq & 1)) * 16, b);
        mma_ct<CT>(s[2 * np], qa[ks], b[0], b[1]);
        mma_ct<CT>(s[2 * np + 1], qa[ks], b[2], b[3]);
      }
    }
  } else {
    // A matrix is 8 keys x 16 codes: one k-step of 16, of which lane (g, t) gets key g's codes 4 t .. 4 t + 3. The
    // instruction's k order (2t, 2t + 1 | 2t + 8, 2t + 9) stands for those four; the query fragments are laid out alike.
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int key = nt * 8 + rr;
#pragma unroll
      for (int k4 = 0; k4 < D / 64; ++k4) {
        uint32_t w[4];
        ldsm_x4(kt + key * G::kRowBytes + G::chunk(key, 4 * k4 + mq) * 16, w);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          uint32_t b0, b1;
          codes_to_f16<CT>(w[i], b0, b1);
          mma_ct<CT>(s[nt], qa[4 * k4 + i], b0, b1);
        }
      }
    }
  }
  const uint32_t scales = kt + 2 * G::kKvBytes;
  const uint32_t live = ld_shared_u32(scales + G::kScaleBytes);
  constexpr uint32_t kAll = G::kTile == 32 ? 0xFFFFFFFFu : (1u << (G::kTile & 31)) - 1u;
  float vs[NT][2], ve[NT][2];  // row scale of V and its exponent bound, for this lane's keys
#pragma unroll
  for (int i = 0; i < NT; ++i) {
    float2 kk = make_float2(1.f, 1.f);
    if constexpr (C::kQuant) {
      kk = ld_shared_f2(scales + (8 * i + 2 * t) * 4);
      const float2 vv = ld_shared_f2(scales + (G::kTile + 8 * i + 2 * t) * 4);
      vs[i][0] = vv.x, vs[i][1] = vv.y;
      ve[i][0] = static_cast<float>(static_cast<int>(__float_as_uint(vv.x) >> 23 & 0xFFu) - 126);
      ve[i][1] = static_cast<float>(static_cast<int>(__float_as_uint(vv.y) >> 23 & 0xFFu) - 126);
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) s[i][e] = s[i][e] * rs[e >> 1] * ((e & 1) ? kk.y : kk.x);
  }
  if (live != kAll || j0 + G::kTile > open) {  // warp-uniform
#pragma unroll
    for (int i = 0; i < NT; ++i) {
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int r = 8 * i + 2 * t + (e & 1), j = j0 + r;
        bool see = ((live >> r) & 1u) && rv.qi[e >> 1] >= 0;
        if (see && j >= open) see = p.mask ? rv.mrow[e >> 1][j - ctx] != 0 : j - ctx <= rv.qi[e >> 1];
        if (!see) s[i][e] = -INFINITY;
      }
    }
  }
  uint32_t pk[NT][2];  // weights as fp16 / bf16 pairs: rows g and g + 8
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float mt = st.m[i], Mt = st.M[i];
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      mt = fmaxf(mt, fmaxf(s[nt][2 * i], s[nt][2 * i + 1]));
      if constexpr (C::kQuant) Mt = fmaxf(Mt, fmaxf(s[nt][2 * i] + ve[nt][0], s[nt][2 * i + 1] + ve[nt][1]));
    }
    mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 1));
    mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, 2));
    const float mu = mt == -INFINITY ? 0.f : mt;  // no key seen yet: any finite reference
    const float al = exp2f(st.m[i] - mu);
    float ao = al, c = 1.f;
    if constexpr (C::kQuant) {
      Mt = fmaxf(Mt, __shfl_xor_sync(0xffffffffu, Mt, 1));
      Mt = fmaxf(Mt, __shfl_xor_sync(0xffffffffu, Mt, 2));
      const float Mu = Mt == -INFINITY ? 0.f : Mt;
      ao = exp2f(st.M[i] - Mu);
      c = exp2f(mu - Mu);
      st.M[i] = Mt;
    }
    st.m[i] = mt;
    float sum = 0.f;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float w[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const float x = s[nt][2 * i + e];
        const float pr = exp2f(x - mu);
        sum += pr;
        w[e] = pr;
        if constexpr (C::kQuant) w[e] = x == -INFINITY ? 0.f : pr * vs[nt][e] * c;
      }
      pk[nt][i] = C::kBf16Mma ? pack_bf16x2(w[0], w[1]) : pack_f16x2(w[0], w[1]);
    }
    st.l[i] = fmaf(st.l[i], al, sum);
    if (__any_sync(0xffffffffu, ao != 1.f)) {
#pragma unroll
      for (int n = 0; n < D / 8; ++n) st.o[n][2 * i] *= ao, st.o[n][2 * i + 1] *= ao;
    }
  }
  const uint32_t vt = kt + G::kKvBytes;
#pragma unroll
  for (int k16 = 0; k16 < NT / 2; ++k16) {
    const uint32_t pa[4] = {pk[2 * k16][0], pk[2 * k16][1], pk[2 * k16 + 1][0], pk[2 * k16 + 1][1]};
    const int key = k16 * 16 + (mq & 1) * 8 + rr;
#pragma unroll
    for (int c2 = 0; c2 < G::kChunks / 2; ++c2) {
      uint32_t b[4];
      ldsm_x4_trans(vt + key * G::kRowBytes + G::chunk(key, 2 * c2 + (mq >> 1)) * 16, b);
      if constexpr (!C::kQuant) {
        mma_ct<CT>(st.o[2 * c2], pa, b[0], b[1]);
        mma_ct<CT>(st.o[2 * c2 + 1], pa, b[2], b[3]);
      } else {
        // A 16-bit unit is two codes of neighbouring columns: the even columns of a chunk make one n-tile, the odd
        // ones the next (record_column undoes it).
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          uint32_t e0, o0, e1, o1;
          codes_to_f16_even_odd<CT>(b[2 * h], e0, o0);
          codes_to_f16_even_odd<CT>(b[2 * h + 1], e1, o1);
          mma_ct<CT>(st.o[2 * (2 * c2 + h)], pa, e0, e1);
          mma_ct<CT>(st.o[2 * (2 * c2 + h) + 1], pa, o0, o1);
        }
      }
    }
  }
  __syncwarp();  // every lane is done with this stage before it is refilled
}

// Replaces every infinity and NaN of the V tile by zero; true if there were any (in any lane).
template <int CT, int D> NVB200_DEVICE bool clean_v_tile(uint32_t kt, int lane) {
  using G = Geometry<CT, D>;
  uint32_t found = 0;
  for (int o = lane * 16; o < G::kKvBytes; o += 512) {
    uint4 u = ld_shared_v4(kt + G::kKvBytes + o);
    uint32_t *w = &u.x;
    uint32_t here = 0;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const uint32_t bad = nonfinite_bits<CT>(w[i]);
      w[i] &= ~bad, here |= bad;
    }
    if (here) st_shared_v4(kt + G::kKvBytes + o, u);
    found |= here;
  }
  __syncwarp();
  return __any_sync(0xffffffffu, found != 0);
}

template <int CT, int D>
__global__ void __launch_bounds__(kThreads) cache_attention_kernel(const __grid_constant__ CacheAttnParams p) {
  using G = Geometry<CT, D>;
  using C = CacheType<CT>;
  launch_dependents();     // a dependent launched early waits for this grid before reading its output
  grid_dependency_wait();  // this grid may itself have been launched early
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  const int blocks_of_rows = (p.rows + kRows - 1) / kRows;
  const int h = blockIdx.y / blocks_of_rows, row0 = (blockIdx.y - h * blocks_of_rows) * kRows;
  const int b = blockIdx.z;
  const int nrows = min(kRows, p.rows - row0);
  const uint32_t rank = p.splits > 1 ? cta_rank_in_cluster() : 0u;
  const uint32_t wring = smem_addr(smem) + warp * (G::kStages * G::kStageBytes);

  // Keys [0, L), of which the last `drafts` are the new tokens.
  int L = p.seqlens[b];
  int drafts = p.draft_lens ? p.draft_lens[b] : p.n;
  const int64_t cap = static_cast<int64_t>(p.max_pages) * p.block_size;
  if (L < 0 || L > cap || drafts < 0 || drafts > p.n) {
    if (tid == 0 && rank == 0) set_status(p.status, NVB200_STATUS_BAD_SLOT);
    L = L < 0 ? 0 : static_cast<int>(min(static_cast<int64_t>(L), cap));
    drafts = max(0, min(drafts, p.n));
  }
  const int ctx = L - drafts;                          // negative: the first drafted tokens are not in the cache
  const bool masked = p.mask != nullptr || p.causal;
  const int open = masked ? max(ctx, 0) : L;           // every row sees the keys below this
  RowView rv;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = row0 + g + 8 * i, qi = r / p.group;
    rv.qi[i] = r < p.rows && qi < drafts ? qi : -1;
    rv.mrow[i] = p.mask ? p.mask + b * p.mask_batch_stride + (rv.qi[i] < 0 ? 0 : rv.qi[i]) * p.mask_row_stride : nullptr;
  }
  const bool any_row = row0 / p.group < drafts;  // else all rows of this CTA are padding
  // This CTA's share [js, je) of the keys, whole tiles.
  constexpr int kGrain = G::kTile;
  const int per = any_row ? ((L + p.splits - 1) / p.splits + kGrain - 1) / kGrain * kGrain : 0;
  const int js = static_cast<int>(min(static_cast<int64_t>(L), static_cast<int64_t>(rank) * per));
  const int je = any_row ? min(L - js, per) + js : js;
  const int ntiles = (je - js + G::kTile - 1) / G::kTile;
  const int my_tiles = warp < ntiles ? (ntiles - warp + kWarps - 1) / kWarps : 0;

  const int32_t *bt = p.block_table ? p.block_table + b * p.bt_stride : nullptr;
  auto key_of = [&](int i) { return js + (warp + i * kWarps) * G::kTile + (lane & (G::kTile - 1)); };
  auto block_of = [&](int j) {  // block of key j, -1 past the share
    if (j >= je) return -1;
    return bt ? __ldg(bt + page_of(p, j)) : b;
  };
  int next_blk = my_tiles > 0 ? block_of(key_of(0)) : -1;
  // Copies this warp's i-th tile into ring stage `stage`; the block number of the tile after it is fetched meanwhile.
  auto issue = [&](int i, int stage) {
    const int j = key_of(i);
    const int blk = next_blk;
    if (i + 1 < my_tiles) next_blk = block_of(key_of(i + 1));
    int64_t off = -1;  // element offset of key j's row for head h; -1 = not read (zero-filled)
    int in = 0;
    if (j < je) {
      in = j - page_of(p, j) * p.block_size;
      if (blk >= 0 && blk < p.num_blocks)
        off = blk * p.blk_stride + in * p.tok_stride + h * p.head_stride;
      else
        set_status(p.status, NVB200_STATUS_BAD_SLOT);
    }
    const uint32_t live = __ballot_sync(0xffffffffu, off >= 0 && lane < G::kTile);
    const uint32_t dst = wring + stage * G::kStageBytes;
    if (lane == 0) st_shared_u32(dst + 2 * G::kKvBytes + G::kScaleBytes, live);
    constexpr int RPI = 32 / G::kChunks;  // rows per warp-wide copy
    const int c = lane % G::kChunks;
#pragma unroll
    for (int r0 = 0; r0 < G::kTile; r0 += RPI) {
      const int row = r0 + lane / G::kChunks;
      const long long o = __shfl_sync(0xffffffffu, static_cast<long long>(off), row);
      const bool ok = o >= 0;
      const int64_t src = (ok ? o : 0) * C::kBytes + c * 16;
      const uint32_t to = dst + row * G::kRowBytes + G::chunk(row, c) * 16;
      cp_async16(to, p.k_cache + (ok ? src : 0), ok ? 16u : 0u);
      cp_async16(to + G::kKvBytes, p.v_cache + (ok ? src : 0), ok ? 16u : 0u);
    }
    if constexpr (C::kQuant) {
      if (lane < G::kTile) {
        const bool ok = off >= 0;
        const int64_t si = ok ? (static_cast<int64_t>(blk) * p.hkv + h) * p.block_size + in : 0;
        cp_async4(dst + 2 * G::kKvBytes + lane * 4, p.k_scale + si, ok ? 4u : 0u);
        cp_async4(dst + 2 * G::kKvBytes + (G::kTile + lane) * 4, p.v_scale + si, ok ? 4u : 0u);
      }
    }
  };
#pragma unroll
  for (int s = 0; s < G::kStages - 1; ++s) {
    if (s < my_tiles) issue(s, s);
    cp_async_commit();
  }

  // Query fragments. 16-bit caches: the instruction's own k order, bits as stored. 8-bit caches: k order as in
  // fold_tile, the row brought to fp16 by a power of two that puts its largest element in [2^13, 2^14) (bf16's range
  // does not fit fp16; elements below 2^-27 of the largest lose bits, fewer than the fp32 sum would). rs: what the
  // scores are multiplied by.
  uint32_t qa[D / 16][4];
  float rs[2] = {p.scale_log2, p.scale_log2};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = row0 + g + 8 * i, qi = r / p.group;
    const uint16_t *row = r < p.rows ? static_cast<const uint16_t *>(p.q) + b * p.q_batch_stride +
                                           qi * p.q_token_stride +
                                           static_cast<int64_t>(h * p.group + r - qi * p.group) * p.q_head_stride
                                     : nullptr;
    if constexpr (!C::kQuant) {
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        uint32_t lo = 0, hi = 0;
        if (row) {
          const int d = 16 * ks + 2 * t;
          lo = static_cast<uint32_t>(__ldg(row + d)) | static_cast<uint32_t>(__ldg(row + d + 1)) << 16;
          hi = static_cast<uint32_t>(__ldg(row + d + 8)) | static_cast<uint32_t>(__ldg(row + d + 9)) << 16;
        }
        qa[ks][i] = lo, qa[ks][2 + i] = hi;
      }
    } else {
      float x[D / 16][4];
      uint32_t am = 0;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint16_t u = row ? __ldg(row + 16 * ks + 4 * t + e) : uint16_t{0};
          x[ks][e] = p.q_is_f16 ? __half2float(__ushort_as_half(u)) : __uint_as_float(static_cast<uint32_t>(u) << 16);
          am = max(am, __float_as_uint(x[ks][e]) & 0x7FFFFFFFu);
        }
      }
      am = max(am, __shfl_xor_sync(0xffffffffu, am, 1));
      am = max(am, __shfl_xor_sync(0xffffffffu, am, 2));
      // 2^(13 - e), e the exponent of the largest element; rows of zeros, tiny or not finite: 1 (nothing to gain).
      const int ex = static_cast<int>(am >> 23);
      const bool norm = ex >= 20 && ex < 255;
      const float up = norm ? __uint_as_float(static_cast<uint32_t>(127 + 13 + 127 - ex) << 23) : 1.f;
      if (norm) rs[i] *= __uint_as_float(static_cast<uint32_t>(ex - 13) << 23);
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        qa[ks][i] = pack_f16x2(x[ks][0] * up, x[ks][1] * up);
        qa[ks][2 + i] = pack_f16x2(x[ks][2] * up, x[ks][3] * up);
      }
    }
  }
  RowState<D> st;
#pragma unroll
  for (int i = 0; i < 2; ++i) st.m[i] = st.M[i] = -INFINITY, st.l[i] = 0.f;
#pragma unroll
  for (int n = 0; n < D / 8; ++n) st.o[n][0] = st.o[n][1] = st.o[n][2] = st.o[n][3] = 0.f;
  bool dirty = false;  // an infinity or NaN was taken out of a V tile

  for (int i = 0; i < my_tiles; ++i) {
    if (i + G::kStages - 1 < my_tiles) issue(i + G::kStages - 1, (i + G::kStages - 1) % G::kStages);
    cp_async_commit();
    cp_async_wait<G::kStages - 1>();  // this lane's copies of tile i have landed
    __syncwarp();                     // ... and every other lane's
    const uint32_t kt = wring + (i % G::kStages) * G::kStageBytes;
    const int j0 = js + (warp + i * kWarps) * G::kTile;
    // 0 * inf is NaN in the matrix instruction, so where a row may not see a key of this tile, V must be finite. (Of the
    // 8-bit types e4m3 has a NaN, which the quantiser never writes; a NaN scale meets selected weights only.)
    if constexpr (CT != kI8) {
      if (j0 + G::kTile > open && (p.mask ? drafts > 0 : drafts > 1)) dirty |= clean_v_tile<CT, D>(kt, lane);
    }
    fold_tile<CT, D>(st, kt, qa, rs, rv, p, lane, j0, ctx, open);
  }
  cp_async_wait<0>();
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    st.l[i] += __shfl_xor_sync(0xffffffffu, st.l[i], 1);
    st.l[i] += __shfl_xor_sync(0xffffffffu, st.l[i], 2);
    if constexpr (!C::kQuant) st.M[i] = st.m[i];
  }
  __syncthreads();  // every warp is done with its ring: the records below reuse it
  if (p.splits > 1) cluster_arrive();

  float *rec = reinterpret_cast<float *>(smem);  // [kWarps][kRows][kStride]
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    float *w = rec + (warp * kRows + g + 8 * i) * G::kStride;
    if constexpr (!C::kQuant) {
#pragma unroll
      for (int n = 0; n < D / 8; ++n)
        *reinterpret_cast<float2 *>(w + 8 * n + 2 * t) = make_float2(st.o[n][2 * i], st.o[n][2 * i + 1]);
    } else {
#pragma unroll
      for (int c = 0; c < D / 16; ++c)
        *reinterpret_cast<float4 *>(w + 16 * c + 4 * t) =
            make_float4(st.o[2 * c][2 * i], st.o[2 * c + 1][2 * i], st.o[2 * c][2 * i + 1], st.o[2 * c + 1][2 * i + 1]);
    }
    if (t == 0) w[D] = st.m[i], w[D + 1] = st.l[i], w[D + 2] = st.M[i], w[D + 3] = dirty ? 1.f : 0.f;
  }
  __syncthreads();

  // Merges `count` records, `stride` floats apart, of one row at column d: unnormalised output, m, l, M, flag.
  struct Merged { float o, m, l, M, flag; };
  auto merge = [&](const float *r, int count, int stride, int d) {
    Merged x{0.f, -INFINITY, 0.f, -INFINITY, 0.f};
    for (int k = 0; k < count; ++k) {
      x.m = fmaxf(x.m, r[k * stride + D]);
      x.M = fmaxf(x.M, r[k * stride + D + 2]);
    }
    const float mu = x.m == -INFINITY ? 0.f : x.m, Mu = x.M == -INFINITY ? 0.f : x.M;
    for (int k = 0; k < count; ++k) {
      const float *w = r + k * stride;
      x.o = fmaf(exp2f(w[D + 2] - Mu), w[d], x.o);
      x.l = fmaf(exp2f(w[D] - mu), w[D + 1], x.l);
      x.flag = fmaxf(x.flag, w[D + 3]);
    }
    return x;
  };
  auto write = [&](int r, int d, const Merged &x) {  // r: row within the CTA
    const int row = row0 + r, qi = row / p.group, gq = row - qi * p.group;
    float y = 0.f;
    if (qi < drafts) {
      // l > 0 wherever a key was seen; NaN (a NaN score) is passed on.
      if (x.l != 0.f) y = x.o / x.l * (C::kQuant ? exp2f(x.M - x.m) : 1.f);
      if (CT != kI8 && x.flag != 0.f) y = add_nonfinite<CT>(p, bt, b, h, qi, d, ctx, L, drafts, y);
    }
    const int64_t idx = ((static_cast<int64_t>(b) * p.n + qi) * p.hq + h * p.group + gq) * D + d;
    if (C::kQuant ? p.q_is_f16 : CT == kF16) static_cast<__half *>(p.out)[idx] = __float2half_rn(y);
    else static_cast<__nv_bfloat16 *>(p.out)[idx] = __float2bfloat16_rn(y);
  };

  if (p.splits == 1) {
    for (int e = tid; e < nrows * D; e += kThreads) {
      const int r = e / D, d = e - r * D;
      write(r, d, merge(rec + r * G::kStride, kWarps, kRows * G::kStride, d));
    }
    return;
  }
  // Row r of the cluster is finished by CTA r mod splits: every CTA sends its merged record there (the first barrier: the
  // receiver's ring is no longer in use; the second: every record has arrived).
  float *part = rec + kWarps * kRows * G::kStride;  // [rows of this CTA][splits][kStride]
  cluster_wait();
  for (int e = tid; e < nrows * D; e += kThreads) {
    const int r = e / D, d = e - r * D;
    const Merged x = merge(rec + r * G::kStride, kWarps, kRows * G::kStride, d);
    const uint32_t to = map_shared_to(
        smem_addr(part + ((r / p.splits) * p.splits + static_cast<int>(rank)) * G::kStride), r % p.splits);
    st_cluster_f32(to + d * 4, x.o);
    if (d == 0) {
      st_cluster_f32(to + D * 4, x.m), st_cluster_f32(to + (D + 1) * 4, x.l);
      st_cluster_f32(to + (D + 2) * 4, x.M), st_cluster_f32(to + (D + 3) * 4, x.flag);
    }
  }
  cluster_arrive();
  cluster_wait();
  for (int e = tid; e < nrows * D; e += kThreads) {
    const int r = e / D, d = e - r * D;
    if (r % p.splits == static_cast<int>(rank))
      write(r, d, merge(part + (r / p.splits) * p.splits * G::kStride, p.splits, G::kStride, d));
  }
}

// ---------------------------------------------------------------------------------------------------------------
// Host side.

// CTAs of a cluster sharing the keys of one (sequence, KV head, row block): enough to give every SM two, at most 8, and
// each at least four tiles per warp of the longest sequence.
int choose_splits(int64_t units, int64_t max_keys, int tile) {
  const int64_t want = (2 * static_cast<int64_t>(sm_count()) + units - 1) / units;
  const int64_t most = std::max<int64_t>(1, max_keys / (kWarps * tile * 2));
  int64_t s = std::min<int64_t>(std::min(want, most), kMaxSplits);
  int pow2 = 1;
  while (pow2 * 2 <= s) pow2 *= 2;
  return pow2;
}

template <int CT, int D> int launch_cache_attention(CacheAttnParams &p, int batch, int num_splits, cudaStream_t s) {
  using G = Geometry<CT, D>;
  static std::atomic<uint64_t> ready{0};  // bit: device whose shared-memory limit is set
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return NVB200_ERR_CUDA;
  if (!(ready.load(std::memory_order_acquire) >> dev & 1)) {
    if (cudaFuncSetAttribute(cache_attention_kernel<CT, D>, cudaFuncAttributeMaxDynamicSharedMemorySize, G::kSmem) !=
        cudaSuccess) {
      cudaGetLastError();
      return NVB200_ERR_CUDA;
    }
    ready.fetch_or(uint64_t{1} << dev, std::memory_order_release);
  }
  const int64_t row_blocks = (p.rows + kRows - 1) / kRows;
  const int64_t y = row_blocks * p.hkv;
  if (y > 65535 || batch > 65535) return NVB200_ERR_UNSUPPORTED;
  p.splits = num_splits > 0 ? num_splits
                            : choose_splits(y * batch, static_cast<int64_t>(p.max_pages) * p.block_size, G::kTile);
  return launch_ex(cache_attention_kernel<CT, D>, dim3(p.splits, static_cast<unsigned>(y), batch), dim3(kThreads),
                   G::kSmem, s, p.splits, false, p);
}

template <int CT> int launch_dim(CacheAttnParams &p, int d, int batch, int num_splits, cudaStream_t s) {
  return d == 64 ? launch_cache_attention<CT, 64>(p, batch, num_splits, s)
                 : launch_cache_attention<CT, 128>(p, batch, num_splits, s);
}

}  // namespace
}  // namespace nvb200

using namespace nvb200;

extern "C" int nvb200_cache_attention(const nvb200_cache_attention_args *a, nvb200_stream_t stream) {
  if (!a || a->batch < 0 || a->queries_per_seq < 0 || a->num_q_heads <= 0 || a->num_kv_heads <= 0 ||
      a->num_q_heads % a->num_kv_heads != 0 || a->head_dim <= 0 || a->block_size <= 0 || a->max_blocks_per_seq < 0 ||
      a->num_blocks < 0 || a->num_splits < 0 || a->num_splits > kMaxSplits || (a->causal != 0 && a->causal != 1))
    return NVB200_ERR_ARG;
  if (a->dtype != NVB200_BF16 && a->dtype != NVB200_F16) return NVB200_ERR_ARG;
  int ct;
  if (a->cache_dtype == NVB200_E4M3) ct = kE4M3;
  else if (a->cache_dtype == NVB200_I8) ct = kI8;
  else if (a->cache_dtype == a->dtype) ct = a->dtype == NVB200_F16 ? kF16 : kBf16;
  else return NVB200_ERR_ARG;
  if (!std::isfinite(a->softmax_scale)) return NVB200_ERR_ARG;
  if (a->batch == 0 || a->queries_per_seq == 0) return NVB200_OK;
  const bool quant = ct == kE4M3 || ct == kI8;
  if (!a->out || !a->q || !a->k_cache || !a->v_cache || !a->seqlens || (quant && (!a->k_scale || !a->v_scale)))
    return NVB200_ERR_ARG;
  if (!a->block_table && a->num_blocks < a->batch) return NVB200_ERR_ARG;
  if (a->head_dim != 64 && a->head_dim != 128) return NVB200_ERR_UNSUPPORTED;
  const int64_t rows = static_cast<int64_t>(a->queries_per_seq) * (a->num_q_heads / a->num_kv_heads);
  if (a->queries_per_seq > 4096 || rows > 65536) return NVB200_ERR_UNSUPPORTED;
  const int64_t eb = quant ? 1 : 2;
  if (!aligned16(a->k_cache) || !aligned16(a->v_cache) || (a->cache_block_stride * eb) % 16 != 0 ||
      (a->cache_token_stride * eb) % 16 != 0 || (a->cache_head_stride * eb) % 16 != 0)
    return NVB200_ERR_UNSUPPORTED;
  const int64_t cap = static_cast<int64_t>(a->max_blocks_per_seq) * a->block_size;
  if (cap > (int64_t{1} << 31) - 65536) return NVB200_ERR_UNSUPPORTED;  // key indices are 32-bit
  if (int rc = check_device()) return rc;
  CacheAttnParams p{};
  p.q = a->q, p.q_batch_stride = a->q_batch_stride, p.q_token_stride = a->q_token_stride;
  p.q_head_stride = a->q_head_stride;
  p.k_cache = static_cast<const uint8_t *>(a->k_cache), p.v_cache = static_cast<const uint8_t *>(a->v_cache);
  p.blk_stride = a->cache_block_stride, p.tok_stride = a->cache_token_stride, p.head_stride = a->cache_head_stride;
  p.num_blocks = a->num_blocks, p.k_scale = a->k_scale, p.v_scale = a->v_scale;
  p.block_table = a->block_table, p.bt_stride = a->block_table_stride;
  p.max_pages = a->block_table ? a->max_blocks_per_seq : 1;
  p.seqlens = a->seqlens, p.draft_lens = a->draft_lens;
  p.mask = a->tree_mask, p.mask_batch_stride = a->mask_batch_stride, p.mask_row_stride = a->mask_row_stride;
  p.out = a->out, p.n = a->queries_per_seq, p.hq = a->num_q_heads, p.hkv = a->num_kv_heads;
  p.group = a->num_q_heads / a->num_kv_heads, p.block_size = a->block_size;
  p.bs_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (a->block_size == (1 << i)) p.bs_shift = i;
  p.rows = static_cast<int>(rows), p.causal = a->causal;
  p.q_is_f16 = a->dtype == NVB200_F16;
  p.scale_log2 = a->softmax_scale * 1.4426950408889634f;
  p.status = a->status;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (rows > kRows) {
    const int rc = launch_cache_attention_wide(p, ct, a->head_dim, a->batch, a->num_splits, s);
    if (rc != NVB200_ERR_UNSUPPORTED) return rc;
  }
  switch (ct) {
    case kBf16: return launch_dim<kBf16>(p, a->head_dim, a->batch, a->num_splits, s);
    case kF16: return launch_dim<kF16>(p, a->head_dim, a->batch, a->num_splits, s);
    case kE4M3: return launch_dim<kE4M3>(p, a->head_dim, a->batch, a->num_splits, s);
    default: return launch_dim<kI8>(p, a->head_dim, a->batch, a->num_splits, s);
  }
}
