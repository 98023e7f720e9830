// Attention of a few new tokens per sequence over the paged KV cache: single decode tokens, causal chains, and trees of
// drafted tokens (each drafted token sees the context, and of the drafted tokens those its mask row names: its
// ancestors), over 16-bit caches or the 8-bit ones of kv_quant.cu. The reference verifies linear drafts only, through
// flash_attn_with_kvcache (nanovllm/layers/attention.py:84-91); masks and 8-bit caches have no counterpart there.
//
// Mathematics, per query row (token i, query head h) over its visible keys j:
//   s_j = scale * ks_j * (q . k_j),  p_j = 2^(s_j log2 e - m),  out = (sum_j p_j vs_j v_j) / (sum_j p_j)
// with k_j, v_j the stored codes and ks_j, vs_j their row scales (1 for 16-bit caches); one pass over the keys with the
// running maximum m and sum l. Masked keys are selected away (p = 0 by selection, never by adding -inf), so no value of
// a key that a row does not see, infinities and NaN included, reaches it; a row that sees no key gives zeros. A weight below
// fp32's normal range, 2^-126 of the row's largest, is zero, whatever its value's scale.
//
// 8-bit caches run on fp16 matrix instructions: e4m3 and int8 codes are exact in fp16 (one conversion per two codes), and
// the query row is brought to fp16 by an exact power of two, so the only roundings are those of p and the output.
// The weights p_j vs_j carry the row scales, whose range fp16 does not have; they are held relative to M, the running
// maximum of s_j log2 e + (binary exponent of vs_j) + 1. fp16 weights (8-bit and fp16 caches) are held 2^kWeightUp times as
// large, the largest in (2^13, 2^14]: fp16's smallest step, 2^-24, is then 2^-37 of it or less, where weights of at most 1
// would vanish below 2^-25, and with them what thousands of keys beside one that takes almost the whole softmax add up to.
// The sums l carry the same factor. bf16 weights have fp32's range and stay at most 1.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "cache_attention.cuh"

namespace nvb200 {
namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr float kWeightUp = 14.f;
constexpr int kMinTiles = 16;  // of a CTA in the even-share form, where there are too few for all

NVB200_DEVICE void cp_async16(uint32_t dst, const void *src, uint32_t src_bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
}
NVB200_DEVICE void cp_async4(uint32_t dst, const void *src, uint32_t src_bytes) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(src_bytes) : "memory");
}
NVB200_DEVICE void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> NVB200_DEVICE void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

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

// (a, b) * (x, y) and (a, b) + (x, y), each lane rounded as the scalar operation, in one instruction.
NVB200_DEVICE void mul2(float &a, float &b, float x, float y) {
  asm("{\n .reg .b64 p, q;\n mov.b64 p, {%0, %1};\n mov.b64 q, {%2, %3};\n mul.rn.f32x2 p, p, q;\n mov.b64 {%0, %1}, p;\n}"
      : "+f"(a), "+f"(b)
      : "f"(x), "f"(y));
}
NVB200_DEVICE void add2(float &a, float &b, float x, float y) {
  asm("{\n .reg .b64 p, q;\n mov.b64 p, {%0, %1};\n mov.b64 q, {%2, %3};\n add.rn.f32x2 p, p, q;\n mov.b64 {%0, %1}, p;\n}"
      : "+f"(a), "+f"(b)
      : "f"(x), "f"(y));
}

// Transposes an 8 x 8 matrix of 16-bit elements held two to a lane.
NVB200_DEVICE uint32_t movmatrix_trans(uint32_t a) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(a));
  return r;
}

// The same for the byte pairs (0, 2) and (1, 3).
template <int CT> NVB200_DEVICE void codes_to_f16_even_odd(uint32_t w, uint32_t &even, uint32_t &odd) {
  codes_to_f16<CT>(__byte_perm(w, 0u, 0x3120), even, odd);
}

// Shared-memory geometry. A warp streams tiles of kTile keys: kTile K rows, kTile V rows, for 8-bit caches their 2 x kTile
// scales, and one word of flags (bit r: key r exists and its page is valid).
template <int CT, int D, int NT> struct Geometry {
  static constexpr int kRows = 8 * NT;  // query rows of a unit
  static constexpr int kRowBytes = D * CacheType<CT>::kBytes;  // 64, 128 or 256
  static constexpr int kChunks = kRowBytes / 16;
  static constexpr int kTile = kRowBytes >= 256 ? 16 : 32;
  static constexpr int kStages = kRowBytes == 64 ? 3 : 2;
  static constexpr int kKvBytes = kTile * kRowBytes;
  static constexpr int kScaleBytes = CacheType<CT>::kQuant ? 2 * kTile * 4 : 0;
  static constexpr int kStageBytes = 2 * kKvBytes + kScaleBytes + 128;  // a multiple of 128
  static constexpr int kStride = D + 4;  // floats per record: o[D], m, l, M, flag
  // Physical 16-byte chunk of logical chunk c of row r: the 8 rows of an 8 x 16-byte matrix at one logical chunk fall
  // in distinct bank groups (two 64-byte rows share a 128-byte line, so their swizzle steps every second row).
  static NVB200_DEVICE int chunk(int r, int c) { return kRowBytes == 64 ? c ^ ((r >> 1) & 3) : c ^ (r & 7); }
};

// What the two forms of the kernel lay out differently. The warps' records of their partial results lie, in the cluster
// form, where a CTA has one segment, in the warps' own rings; in the even-share form, where the next segment's tiles are
// landing there already, beside them. The saving lets three CTAs of the cluster form share an SM for at most 8 rows (256
// sequences of 300 keys, e4m3: 60 -> 49 us; six warps a CTA in the same memory: 56 us). At head_dim 64 both forms fit three
// times with 16 rows too (32 x 16 drafts, group 4, 2048 keys, bf16: 57 -> 48 us); at 128 their registers do not.
template <int CT, int D, int NT, bool CLUSTER> struct Form {
  using G = Geometry<CT, D, NT>;
  static constexpr int kWarpRing = G::kStages * G::kStageBytes;
  static constexpr int kRing = kWarps * kWarpRing;
  static constexpr int kRecord = G::kRows * G::kStride * 4;
  static constexpr int kRecords = CLUSTER ? 0 : kRing;                     // where the records lie
  static constexpr int kRecordStep = (CLUSTER ? kWarpRing : kRecord) / 4;  // floats from one warp's to the next
  static_assert(!CLUSTER || kRecord <= kWarpRing, "a warp's record takes its ring's place");
  // Cluster form: the records that a CTA receives, splits * ceil(kRows / splits) rows.
  static constexpr int kReceived = kRing;
  static constexpr int kRowsAt = kReceived + (CLUSTER ? (kMaxSplits + G::kRows - 1) * G::kStride * 4 : kWarps * kRecord);
  static constexpr int kSmem = kRowsAt + G::kRows * 16;  // merged m, l, M, flag per row
  static constexpr int kCtasPerSm = (NT == 1 || D == 64) && 228 * 1024 / (kSmem + 1024) >= 3 ? 3 : 2;
  static_assert(kCtasPerSm * (kSmem + 1024) <= 228 * 1024, "shared memory of an SM");
};

// One warp's softmax state. The products are S^T = K Q^T and O^T = V^T P^T: the keys (and the output's columns) fill the
// instruction's 16 rows and the query rows its 8 columns, so that 8 query rows cost half of what 16 do; a decode step has
// 1 to 8 per KV head. Lane 4 g + t has, of query-row tile n: rows 8 n + 2 t and 8 n + 2 t + 1 (index e) of the maxima and
// sums (l: the lane's share), and o[c][n][.] = columns (g, g + 8) of 16-column tile c by those two rows.
template <int D, int NT> struct RowState {
  float m[NT][2], l[NT][2], M[NT][2], o[D / 16][NT][4];
  NVB200_DEVICE void reset() {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      m[n][0] = m[n][1] = M[n][0] = M[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.f;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) o[c][n][0] = o[c][n][1] = o[c][n][2] = o[c][n][3] = 0.f;
    }
  }
};

// Query fragments (second operand of K Q^T) and what the scores of rows 8 n + 2 t + e are multiplied by.
template <int D, int NT> struct QueryFrags {
  uint32_t b[D / 16][NT][2];
  float rs[NT][2];
};

// Replaces every infinity and NaN of the V tile's rows from `first` on by zero; true if there were any (in any lane).
template <int CT, int D, int NT> NVB200_DEVICE bool clean_v_tile(uint32_t kt, int first, int lane) {
  using G = Geometry<CT, D, NT>;
  uint32_t found = 0;
  for (int o = first * G::kRowBytes + lane * 16; o < G::kKvBytes; o += 512) {
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

// Folds one tile. kt: the stage's base address. see[n][e]: which of the tile's keys that row sees, where `edge`; elsewhere
// every row sees every key.
template <int CT, int D, int NT>
NVB200_DEVICE void fold_tile(RowState<D, NT> &st, uint32_t kt, const QueryFrags<D, NT> &q, int lane, bool edge,
                             const uint32_t (&see)[NT][2]) {
  using G = Geometry<CT, D, NT>;
  using C = CacheType<CT>;
  constexpr int KB = G::kTile / 16;  // 16-key blocks
  const int g = lane >> 2, mq = lane >> 3, rr = lane & 7;
  float s[KB][NT][4];
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
    for (int n = 0; n < NT; ++n) s[kb][n][0] = s[kb][n][1] = s[kb][n][2] = s[kb][n][3] = 0.f;
  }
  if constexpr (!C::kQuant) {
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks) {
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const int key = kb * 16 + (mq & 1) * 8 + rr;
        uint32_t a[4];
        ldsm_x4(kt + key * G::kRowBytes + G::chunk(key, 2 * ks + (mq >> 1)) * 16, a);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_ct<CT>(s[kb][n], a, q.b[ks][n][0], q.b[ks][n][1]);
      }
    }
  } else {
    // A matrix is 8 keys x 16 codes: one k-step of 16, of which lane (g, t) gets key g's codes 4 t .. 4 t + 3. The
    // instruction's k order (2t, 2t + 1 | 2t + 8, 2t + 9) stands for those four; the query fragments are laid out alike.
#pragma unroll
    for (int k2 = 0; k2 < D / 32; ++k2) {
      uint32_t w[KB][4];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const int key = kb * 16 + (mq & 1) * 8 + rr;
        ldsm_x4(kt + key * G::kRowBytes + G::chunk(key, 2 * k2 + (mq >> 1)) * 16, w[kb]);
      }
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          uint32_t a[4];
          codes_to_f16<CT>(w[kb][2 * i], a[0], a[2]);
          codes_to_f16<CT>(w[kb][2 * i + 1], a[1], a[3]);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_ct<CT>(s[kb][n], a, q.b[2 * k2 + i][n][0], q.b[2 * k2 + i][n][1]);
        }
      }
    }
  }
  // Scores of keys 16 kb + g + 8 i by rows (n, e): s[kb][n][2 i + e].
  float vs[KB][2], ve[KB][2];  // row scale of V and its exponent bound (above its log2), for this lane's keys
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float ks = 1.f;
      const int key = 16 * kb + 8 * i + g;
      if constexpr (C::kQuant) {
        const uint32_t sc = kt + 2 * G::kKvBytes + key * 4;
        ks = __uint_as_float(ld_shared_u32(sc));
        const uint32_t v = ld_shared_u32(sc + G::kTile * 4);
        vs[kb][i] = __uint_as_float(v);
        ve[kb][i] = static_cast<float>(static_cast<int>(v >> 23 & 0xFFu) - 126);
      }
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        float &x0 = s[kb][n][2 * i], &x1 = s[kb][n][2 * i + 1];
        mul2(x0, x1, q.rs[n][0], q.rs[n][1]);
        if constexpr (C::kQuant) mul2(x0, x1, ks, ks);
      }
    }
  }
  bool bad = false;  // a row scale of V is not finite, and a row may not see its key
  if (edge) {
    bool odd = false;
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if constexpr (C::kQuant) odd |= !(vs[kb][i] <= 3.402823466e38f);
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int e = 0; e < 2; ++e)
            if (!((see[n][e] >> (16 * kb + 8 * i + g)) & 1u)) s[kb][n][2 * i + e] = -INFINITY;
        }
      }
    }
    bad = __any_sync(0xffffffffu, odd);
  }
  uint32_t pb[KB][NT][2];  // weights as the second operand of V^T P^T
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    float up[2], cw[2], ao[2];  // up: what turns a score into its weight's exponent
#pragma unroll
    for (int e = 0; e < 2; ++e) {
      float mt = st.m[n][e], Mt = st.M[n][e];
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        mt = fmaxf(mt, fmaxf(s[kb][n][e], s[kb][n][2 + e]));
        if constexpr (C::kQuant) Mt = fmaxf(Mt, fmaxf(s[kb][n][e] + ve[kb][0], s[kb][n][2 + e] + ve[kb][1]));
      }
#pragma unroll
      for (int o = 4; o < 32; o <<= 1) {
        mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, o));
        if constexpr (C::kQuant) Mt = fmaxf(Mt, __shfl_xor_sync(0xffffffffu, Mt, o));
      }
      const float mu = mt == -INFINITY ? 0.f : mt;  // no key seen yet: any finite reference
      up[e] = (C::kBf16Mma ? 0.f : kWeightUp) - mu;
      const float al = ex2_approx_ftz(st.m[n][e] - mu);
      ao[e] = al, cw[e] = 1.f;
      if constexpr (C::kQuant) {
        const float Mu = Mt == -INFINITY ? 0.f : Mt;
        ao[e] = ex2_approx_ftz(st.M[n][e] - Mu);
        cw[e] = ex2_approx_ftz(mu - Mu);
        st.M[n][e] = Mt;
      }
      st.m[n][e] = mt;
      st.l[n][e] *= al;
    }
    float w[KB][2][2];
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float &w0 = w[kb][i][0], &w1 = w[kb][i][1];
        w0 = s[kb][n][2 * i], w1 = s[kb][n][2 * i + 1];
        add2(w0, w1, up[0], up[1]);
        w0 = ex2_approx_ftz(w0), w1 = ex2_approx_ftz(w1);
        add2(st.l[n][0], st.l[n][1], w0, w1);
        if constexpr (C::kQuant) {
          mul2(w0, w1, vs[kb][i], vs[kb][i]);
          mul2(w0, w1, cw[0], cw[1]);
        }
      }
    }
    if (C::kQuant && bad) {
#pragma unroll
      for (int k = 0; k < KB * 4; ++k)
        if (s[k / 4][n][k % 4] == -INFINITY) w[k / 4][k % 4 / 2][k % 2] = 0.f;
    }
#pragma unroll
    for (int kb = 0; kb < KB; ++kb) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        pb[kb][n][i] = movmatrix_trans(C::kBf16Mma ? pack_bf16x2(w[kb][i][0], w[kb][i][1]) : pack_f16x2(w[kb][i][0], w[kb][i][1]));
    }
    if (__any_sync(0xffffffffu, ao[0] != 1.f || ao[1] != 1.f)) {
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        mul2(st.o[c][n][0], st.o[c][n][1], ao[0], ao[1]);
        mul2(st.o[c][n][2], st.o[c][n][3], ao[0], ao[1]);
      }
    }
  }
  const uint32_t vt = kt + G::kKvBytes;
#pragma unroll
  for (int kb = 0; kb < KB; ++kb) {
    if constexpr (!C::kQuant) {
      const int key = kb * 16 + (mq >> 1) * 8 + rr;
#pragma unroll
      for (int c = 0; c < D / 16; ++c) {
        uint32_t a[4];
        ldsm_x4_trans(vt + key * G::kRowBytes + G::chunk(key, 2 * c + (mq & 1)) * 16, a);
#pragma unroll
        for (int n = 0; n < NT; ++n) mma_ct<CT>(st.o[c][n], a, pb[kb][n][0], pb[kb][n][1]);
      }
    } else {
      // A 16-bit unit is two codes of neighbouring columns: of a 16-column tile the even columns are the instruction's rows
      // 0-7, the odd ones 8-15.
      const int key = kb * 16 + (mq & 1) * 8 + rr;
#pragma unroll
      for (int c2 = 0; c2 < D / 32; ++c2) {
        uint32_t w[4];
        ldsm_x4_trans(vt + key * G::kRowBytes + G::chunk(key, 2 * c2 + (mq >> 1)) * 16, w);
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          uint32_t a[4];
          codes_to_f16_even_odd<CT>(w[2 * i], a[0], a[1]);
          codes_to_f16_even_odd<CT>(w[2 * i + 1], a[2], a[3]);
#pragma unroll
          for (int n = 0; n < NT; ++n) mma_ct<CT>(st.o[2 * c2 + i][n], a, pb[kb][n][0], pb[kb][n][1]);
        }
      }
    }
  }
  __syncwarp();  // every lane is done with this stage before it is refilled
}

// CLUSTER: the CTAs of a cluster split one unit's keys evenly and merge through distributed shared memory (grid: splits,
// units of a sequence, batch). Else: even shares of the whole batch (cache_attention.cuh).
template <int CT, int D, int NT, bool CLUSTER>
__global__ void __launch_bounds__(kThreads, Form<CT, D, NT, CLUSTER>::kCtasPerSm)
    cache_attention_kernel(const __grid_constant__ CacheAttnParams p) {
  using G = Geometry<CT, D, NT>;
  using F = Form<CT, D, NT, CLUSTER>;
  using C = CacheType<CT>;
  launch_dependents();     // a dependent launched early waits for this grid before reading its output
  grid_dependency_wait();  // this grid may itself have been launched early
  extern __shared__ __align__(128) uint8_t smem[];
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, t = lane & 3;
  const uint32_t wring = smem_addr(smem) + warp * F::kWarpRing;
  float *rec = reinterpret_cast<float *>(smem + F::kRecords);  // kRecordStep apart, [kRows][kStride] each
  float4 *row_s = reinterpret_cast<float4 *>(smem + F::kRowsAt);  // [kRows]

  // The unit's query rows as the lanes take them (row g of each row tile), from row0 of KV head h.
  uint32_t wq[NT][D / 16][2];
  auto load_q = [&](int b, int h, int row0) {
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      const int r = row0 + 8 * n + g, qi = r / p.group;
      const uint16_t *row = r < p.rows ? static_cast<const uint16_t *>(p.q) + b * p.q_batch_stride +
                                             qi * p.q_token_stride +
                                             static_cast<int64_t>(h * p.group + r - qi * p.group) * p.q_head_stride
                                       : nullptr;
      // Lane t's elements: 16-bit caches 16 ks + 2 t, + 1, + 8, + 9; 8-bit caches 16 ks + 4 t .. + 3.
      uint32_t(&w)[D / 16][2] = wq[n];
      const bool pairs = (reinterpret_cast<uintptr_t>(row) & 7) == 0;
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) {
        const int d0 = 16 * ks + (C::kQuant ? 4 * t : 2 * t), d1 = C::kQuant ? d0 + 2 : d0 + 8;
        w[ks][0] = w[ks][1] = 0u;
        if (row && pairs) {
          w[ks][0] = __ldg(reinterpret_cast<const uint32_t *>(row + d0));
          w[ks][1] = __ldg(reinterpret_cast<const uint32_t *>(row + d1));
        } else if (row) {
          w[ks][0] = static_cast<uint32_t>(__ldg(row + d0)) | static_cast<uint32_t>(__ldg(row + d0 + 1)) << 16;
          w[ks][1] = static_cast<uint32_t>(__ldg(row + d1)) | static_cast<uint32_t>(__ldg(row + d1 + 1)) << 16;
        }
      }
    }
  };

  Segment seg;
  int u1, T = 0, ctas = 0;
  if constexpr (CLUSTER) {
    const int row_blocks = (p.rows + G::kRows - 1) / G::kRows;
    const int b = p.first_batch + blockIdx.z, rank = p.splits > 1 ? static_cast<int>(cta_rank_in_cluster()) : 0;
    const int h = blockIdx.y / row_blocks, block = blockIdx.y - h * row_blocks;
    // The queries' loads and the block table's first lines do not wait for the length, nor behind the keys' loads.
    load_q(b, h, block * G::kRows);
    if (p.block_table && 32 * lane < p.max_pages)
      asm volatile("prefetch.global.L1 [%0];" ::"l"(p.block_table + b * p.bt_stride + 32 * lane));
    seg.b = b;
    seg.s = seq_info(p, b, G::kTile, G::kRows, tid == 0 && rank == 0 && blockIdx.y == 0);
    const int tiles = block < seg.s.blocks ? seg.s.tiles : 0;  // else only padding rows
    seg.s.blocks = row_blocks;
    seg.unit = blockIdx.y;
    const int per = (tiles + p.splits - 1) / p.splits;
    seg.t0 = min(tiles, rank * per);
    seg.n = min(per, tiles - seg.t0);
    seg.u = seg.t0, seg.unit_u = 0, u1 = seg.u + seg.n;
  } else {
    T = total_work(p, G::kTile, G::kRows);
    ctas = active_ctas(T, gridDim.x, kMinTiles);
    zero_uncovered_rows(p, D, G::kTile, G::kRows, blockIdx.x, gridDim.x, tid, kThreads);
    seg.n = 0;
    const bool work = T > 0 && static_cast<int>(blockIdx.x) < ctas;
    if (work) {
      u1 = range_start(blockIdx.x + 1, T, ctas);
      seg = find_segment(p, range_start(blockIdx.x, T, ctas), u1, G::kTile, G::kRows);
    }
    if (tid == 0) write_cut(p, blockIdx.x, seg, T, ctas);
    if (!work) return;
  }
  const bool masked = p.mask != nullptr || (p.causal && p.n > 1);  // (one token of a chain sees every key)

  // The warp's issue cursor: it takes every kWarps-th tile of each segment, and runs ahead of the tiles being folded, past the
  // segment's end.
  Segment is = seg;
  int ik = warp, next_blk = -1;
  auto key_of = [&]() { return (is.t0 + ik) * G::kTile + (lane & (G::kTile - 1)); };
  auto fetch_block = [&]() {  // block of this lane's key of the next tile, one tile ahead of its use
    while (is.n > 0 && ik >= is.n) {
      if constexpr (CLUSTER) is.n = 0;
      else next_segment(is, p, u1, G::kTile, G::kRows);
      ik = warp;
    }
    next_blk = -1;
    if (is.n > 0) {
      const int j = key_of();
      if (j < is.s.L) next_blk = p.block_table ? __ldg(p.block_table + is.b * p.bt_stride + page_of(p, j)) : is.b;
    }
  };
  auto issue = [&](int stage) {
    if (is.n == 0) return;
    const int j = key_of(), blk = next_blk, h = is.unit / is.s.blocks;
    int64_t off = -1;  // element offset of key j's row for head h; -1 = not read (zero-filled)
    int in = 0;
    if (j < is.s.L) {
      in = j - page_of(p, j) * p.block_size;
      if (blk >= 0 && blk < p.num_blocks)
        off = blk * p.blk_stride + in * p.tok_stride + h * p.head_stride;
      else
        set_status(p.status, NVB200_STATUS_BAD_SLOT);
    }
    ik += kWarps;
    fetch_block();
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
      const int64_t src = ok ? o * C::kBytes + c * 16 : 0;
      const uint32_t to = dst + row * G::kRowBytes + G::chunk(row, c) * 16;
      cp_async16(to, p.k_cache + src, ok ? 16u : 0u);
      cp_async16(to + G::kKvBytes, p.v_cache + src, ok ? 16u : 0u);
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
  fetch_block();
#pragma unroll
  for (int s = 0; s < G::kStages - 1; ++s) {
    issue(s);
    cp_async_commit();
  }

  // Merges `count` records, `stride` floats apart, of the rows [0, rows): first, a thread per row, each record's m becomes
  // what its o is multiplied by and row_s gets the row's m, l, M, flag; then anybody sums four columns with row4().
  auto merge_rows = [&](float *r, int rows, int row_stride, int count, int stride) {
    if (tid < rows) {
      float *w = r + tid * row_stride + D;
      float m = -INFINITY, M = -INFINITY, l = 0.f, flag = 0.f;
      for (int k = 0; k < count; ++k) m = fmaxf(m, w[k * stride]), M = fmaxf(M, w[k * stride + 2]);
      const float mu = m == -INFINITY ? 0.f : m, Mu = M == -INFINITY ? 0.f : M;
      for (int k = 0; k < count; ++k) {
        float4 *x = reinterpret_cast<float4 *>(w + k * stride);
        const float4 y = *x;
        l = fmaf(exp2f(y.x - mu), y.y, l), flag = fmaxf(flag, y.w);
        x->x = exp2f(y.z - Mu);
      }
      row_s[tid] = make_float4(m, l, M, flag);
    }
    __syncthreads();
  };
  auto row4 = [&](const float *row, int d, int count, int stride) {
    float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
    for (int k = 0; k < count; ++k) {
      const float f = row[k * stride + D];
      const float4 o = *reinterpret_cast<const float4 *>(row + k * stride + d);
      y.x = fmaf(f, o.x, y.x), y.y = fmaf(f, o.y, y.y), y.z = fmaf(f, o.z, y.z), y.w = fmaf(f, o.w, y.w);
    }
    return y;
  };

  int stage = 0;  // of the tile to fold next
  do {
    bool dirty = false;  // an infinity or NaN was taken out of a V tile of this segment
    const int b = seg.b, h = seg.unit / seg.s.blocks, row0 = (seg.unit - h * seg.s.blocks) * G::kRows;
    const int L = seg.s.L, drafts = seg.s.drafts, ctx = L - drafts;  // ctx < 0: the first new tokens are not in the cache
    const int open = masked ? max(ctx, 0) : L;  // every row sees the keys below this
    // Query fragments (row g of each row tile). 16-bit caches: the instruction's own k order, bits as stored. 8-bit caches: k
    // order as in fold_tile, the row brought to fp16 by a power of two that puts its largest element in [2^13, 2^14)
    // (bf16's range does not fit fp16; elements below 2^-27 of the largest lose bits, fewer than the fp32 sum would). rs:
    // what the scores of rows 2 t and 2 t + 1 are multiplied by.
    QueryFrags<D, NT> q;
    if constexpr (!CLUSTER) load_q(b, h, row0);
#pragma unroll
    for (int n = 0; n < NT; ++n) {
      uint32_t(&w)[D / 16][2] = wq[n];
      float f = p.scale_log2;
      if constexpr (C::kQuant) {
        uint32_t am = 0;  // largest magnitude, as 16-bit patterns (they order like the values)
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
#pragma unroll
          for (int i = 0; i < 2; ++i) am = max(am, max(w[ks][i] & 0x7FFFu, (w[ks][i] >> 16) & 0x7FFFu));
        }
        am = max(am, __shfl_xor_sync(0xffffffffu, am, 1));
        am = max(am, __shfl_xor_sync(0xffffffffu, am, 2));
        const float a = p.q_is_f16 ? __half2float(__ushort_as_half(static_cast<unsigned short>(am))) : __uint_as_float(am << 16);
        // 2^(13 - exponent); rows of zeros, tiny or not finite: 1 (nothing to gain).
        const int ex = static_cast<int>(__float_as_uint(a) >> 23);
        const bool norm = ex >= 20 && ex < 255;
        const float up = norm ? __uint_as_float(static_cast<uint32_t>(127 + 13 + 127 - ex) << 23) : 1.f;
        if (norm) f *= __uint_as_float(static_cast<uint32_t>(ex - 13) << 23);
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float2 x = make_float2(bf16_lo(w[ks][i]), bf16_hi(w[ks][i]));
            if (p.q_is_f16) x = __half22float2(*reinterpret_cast<const __half2 *>(&w[ks][i]));
            w[ks][i] = pack_f16x2(x.x * up, x.y * up);
          }
        }
      }
#pragma unroll
      for (int ks = 0; ks < D / 16; ++ks) q.b[ks][n][0] = w[ks][0], q.b[ks][n][1] = w[ks][1];
      q.rs[n][0] = __shfl_sync(0xffffffffu, f, 8 * t), q.rs[n][1] = __shfl_sync(0xffffffffu, f, 8 * t + 4);
    }
    RowState<D, NT> st;
    st.reset();

    for (int k = warp; k < seg.n; k += kWarps) {
      int ahead = stage + G::kStages - 1;
      if (ahead >= G::kStages) ahead -= G::kStages;
      issue(ahead);
      cp_async_commit();
      cp_async_wait<G::kStages - 1>();  // this lane's copies of the tile have landed
      __syncwarp();                     // ... and every other lane's
      const uint32_t kt = wring + stage * G::kStageBytes;
      if (++stage == G::kStages) stage = 0;
      const int j0 = (seg.t0 + k) * G::kTile;
      const uint32_t live = ld_shared_u32(kt + 2 * G::kKvBytes + G::kScaleBytes);
      constexpr uint32_t kAll = G::kTile == 32 ? 0xFFFFFFFFu : (1u << (G::kTile & 31)) - 1u;
      const bool edge = live != kAll || j0 + G::kTile > open;
      uint32_t see[NT][2];
      if (edge && (!masked || j0 + G::kTile <= open)) {
        // Rows of padding tokens included: they are written as zeros whatever they sum.
#pragma unroll
        for (int n = 0; n < NT; ++n) see[n][0] = see[n][1] = live;
      } else if (edge) {
        // Keys below `open` are seen, then new token rel0 + k at key k.
        const int rel0 = j0 - ctx;
        const uint32_t before = open > j0 ? (open - j0 >= 32 ? 0xFFFFFFFFu : (1u << (open - j0)) - 1u) : 0u;
        int last_qi = -1;
        uint32_t word = 0;
#pragma unroll
        for (int n = 0; n < NT; ++n) {
#pragma unroll
          for (int r = 0; r < 8; ++r) {  // the warp reads a token's mask row together, one byte a lane
            const int qi = (row0 + 8 * n + r) / p.group;
            if (qi != last_qi) {
              last_qi = qi;
              word = 0;
              if (qi < drafts && row0 + 8 * n + r < p.rows) {
                if (p.mask) {
                  const int x = rel0 + lane;
                  const bool is = x >= 0 && x < drafts &&
                                  __ldg(p.mask + b * p.mask_batch_stride + qi * p.mask_row_stride + x) != 0;
                  word = __ballot_sync(0xffffffffu, is) | before;
                } else {
                  const int c = qi - rel0 + 1;  // keys 0 .. c - 1 of the tile
                  word = (c >= 32 ? 0xFFFFFFFFu : (c <= 0 ? 0u : (1u << c) - 1u)) | before;
                }
              }
            }
            if (r == 2 * t) see[n][0] = word & live;
            if (r == 2 * t + 1) see[n][1] = word & live;
          }
        }
        // 0 * inf is NaN in the matrix instruction, so where a row may not see a key of this tile, V must be finite. (Of the
        // 8-bit types e4m3 has a NaN, which the quantiser never writes; a NaN scale meets selected weights only.)
        if constexpr (CT != kI8) {
          if (j0 + G::kTile > open && (p.mask ? drafts > 0 : drafts > 1)) dirty |= clean_v_tile<CT, D, NT>(kt, max(0, open - j0), lane);
        }
      }
      fold_tile<CT, D, NT>(st, kt, q, lane, edge, see);
    }

    // The warp's record: o, m, l, M, flag per row.
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
#pragma unroll
        for (int o = 4; o < 32; o <<= 1) st.l[n][e] += __shfl_xor_sync(0xffffffffu, st.l[n][e], o);
        if constexpr (!C::kQuant) st.M[n][e] = st.m[n][e];
      }
    }
#pragma unroll
    for (int n = 0; n < NT; ++n) {
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        float *w = rec + warp * F::kRecordStep + (8 * n + 2 * t + e) * G::kStride;
#pragma unroll
        for (int c = 0; c < D / 16; ++c) {
          if constexpr (C::kQuant) {
            *reinterpret_cast<float2 *>(w + 16 * c + 2 * g) = make_float2(st.o[c][n][e], st.o[c][n][2 + e]);
          } else {
            w[16 * c + g] = st.o[c][n][e], w[16 * c + 8 + g] = st.o[c][n][2 + e];
          }
        }
        if (g == 0) *reinterpret_cast<float4 *>(w + D) = make_float4(st.m[n][e], st.l[n][e], st.M[n][e], dirty ? 1.f : 0.f);
      }
    }
    __syncthreads();

    const int32_t *bt = p.block_table ? p.block_table + b * p.bt_stride : nullptr;
    const int nrows = min(G::kRows, p.rows - row0);
    constexpr int kPer = D / 4;  // threads per row
    auto write = [&](int r, int d, const float4 &o, const float4 &x) {  // r: row within the unit; x: its m, l, M, flag
      const int row = row0 + r, qi = row / p.group, gq = row - qi * p.group;
      float y[4] = {o.x, o.y, o.z, o.w};
      // l > 0 wherever a key was seen; NaN (a NaN score) is passed on.
      const float f = x.y == 0.f ? 0.f : (C::kQuant ? exp2f(x.z - x.x) : 1.f) / x.y;
#pragma unroll
      for (int k = 0; k < 4; ++k) y[k] = qi < drafts && x.y != 0.f ? y[k] * f : 0.f;
      if (CT != kI8 && x.w != 0.f && qi < drafts) {
        const Columns<4> more = nonfinite_sum<CT, 4>(p, bt, b, h, qi, d, ctx, drafts);
#pragma unroll
        for (int k = 0; k < 4; ++k) y[k] += more.v[k];
      }
      const bool f16 = C::kQuant ? p.q_is_f16 : CT == kF16;
      const uint32_t lo = f16 ? pack_f16x2(y[0], y[1]) : pack_bf16x2(y[0], y[1]);
      const uint32_t hi = f16 ? pack_f16x2(y[2], y[3]) : pack_bf16x2(y[2], y[3]);
      uint16_t *to = static_cast<uint16_t *>(p.out) + ((static_cast<int64_t>(b) * p.n + qi) * p.hq + h * p.group + gq) * D + d;
      if ((reinterpret_cast<uintptr_t>(p.out) & 7) == 0) {
        *reinterpret_cast<uint2 *>(to) = make_uint2(lo, hi);
      } else {
        to[0] = static_cast<uint16_t>(lo), to[1] = static_cast<uint16_t>(lo >> 16);
        to[2] = static_cast<uint16_t>(hi), to[3] = static_cast<uint16_t>(hi >> 16);
      }
    };
    merge_rows(rec, nrows, G::kStride, kWarps, F::kRecordStep);

    if constexpr (CLUSTER) {
      if (p.splits == 1) {
        for (int e = tid; e < nrows * kPer; e += kThreads) {
          const int r = e / kPer, d = e % kPer * 4;
          write(r, d, row4(rec + r * G::kStride, d, kWarps, F::kRecordStep), row_s[r]);
        }
        return;
      }
      // Row r is finished by CTA r mod splits: every CTA sends its merged record there (the first barrier: every CTA of the
      // cluster has started; the second: every record has arrived).
      const int rank = static_cast<int>(cta_rank_in_cluster());
      float *part = reinterpret_cast<float *>(smem + F::kReceived);  // [rows finished here][splits][kStride]
      cluster_arrive();
      cluster_wait();
      for (int e = tid; e < nrows * kPer; e += kThreads) {
        const int r = e / kPer, d = e % kPer * 4;
        const float4 o = row4(rec + r * G::kStride, d, kWarps, F::kRecordStep);
        const uint32_t to = map_shared_to(smem_addr(part + ((r / p.splits) * p.splits + rank) * G::kStride), r % p.splits);
        st_cluster_v4(to + d * 4, o);
        if (d == 0) st_cluster_v4(to + D * 4, row_s[r]);
      }
      cluster_arrive();
      cluster_wait();
      const int mine = nrows > rank ? (nrows - rank + p.splits - 1) / p.splits : 0;  // rows rank, rank + splits, ...
      merge_rows(part, mine, p.splits * G::kStride, p.splits, G::kStride);
      for (int e = tid; e < mine * kPer; e += kThreads) {
        const int i = e / kPer, d = e % kPer * 4;
        write(i * p.splits + rank, d, row4(part + i * p.splits * G::kStride, d, p.splits, G::kStride), row_s[i]);
      }
      return;
    } else {
      const bool whole = seg.n == seg.s.tiles;
      float *out = p.records + static_cast<int64_t>(record_slot(blockIdx.x, seg.unit_u, T, ctas)) * G::kRows * G::kStride;
      for (int e = tid; e < nrows * kPer; e += kThreads) {
        const int r = e / kPer, d = e % kPer * 4;
        const float4 o = row4(rec + r * G::kStride, d, kWarps, F::kRecordStep);
        if (whole) {
          write(r, d, o, row_s[r]);
        } else {
          *reinterpret_cast<float4 *>(out + r * G::kStride + d) = o;
          if (d == 0) *reinterpret_cast<float4 *>(out + r * G::kStride + D) = row_s[r];
        }
      }
      next_segment(seg, p, u1, G::kTile, G::kRows);
      __syncthreads();  // the records have been read
    }
  } while (seg.n > 0);
  cp_async_wait<0>();
}

// ---------------------------------------------------------------------------------------------------------------
// Host side.

template <typename Kernel> int allow_smem(Kernel kernel, int bytes, std::atomic<uint64_t> &ready) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return NVB200_ERR_CUDA;
  if (ready.load(std::memory_order_acquire) >> dev & 1) return NVB200_OK;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess) {
    cudaGetLastError();
    return NVB200_ERR_CUDA;
  }
  ready.fetch_or(uint64_t{1} << dev, std::memory_order_release);
  return NVB200_OK;
}

// CTAs per cluster, a power of two: as many as the longest possible sequence feeds with a tile per warp, while the clusters
// fit on the GPU at once (one sequence of 611 keys: 4 CTAs 8.0 us, 8 CTAs 7.0 us); 1 for up to four tiles a warp, which take
// no longer than the start and the barriers of a cluster (42 x 4 heads of 59 keys in tables of 256: 6.2 against 8.3 us).
int cluster_splits(const CacheAttnParams &p, int64_t units, int cta_keys, int ctas_per_sm) {
  const int64_t max_keys = static_cast<int64_t>(p.max_pages) * p.block_size;
  if (max_keys < 4 * cta_keys) return 1;
  int s = 1;
  while (s < kMaxSplits && 2 * s * units <= static_cast<int64_t>(ctas_per_sm) * sm_count() && s * cta_keys <= max_keys)
    s *= 2;
  return s;
}

struct NarrowShape {
  int64_t units;  // of a sequence
  int tile, rows, ctas_per_sm;  // (of the even-share form)
};
template <int CT, int D, int NT> NarrowShape shape_of(const CacheAttnParams &p) {
  using G = Geometry<CT, D, NT>;
  return {static_cast<int64_t>(p.hkv) * ((p.rows + G::kRows - 1) / G::kRows), G::kTile, G::kRows,
          Form<CT, D, NT, false>::kCtasPerSm};
}

// The one place that picks a kernel: f(cache type, head_dim, row tiles of 8) as integral constants. More than 16 rows are
// blocks of 16 (a form with 32 rows a warp, its queries in shared memory, took 92 us on 64 rows of 32 x 2048 keys where this took 73: it has
// half the warps, and the code is bound by dependent issue).
template <int I> using Int = std::integral_constant<int, I>;
template <typename F> auto with_kernel(const CacheAttnParams &p, int ct, int d, F &&f) {
  auto rows = [&](auto CT, auto D) {
    if (p.rows <= 8) return f(CT, D, Int<1>{});
    return f(CT, D, Int<2>{});
  };
  auto dim = [&](auto CT) { return d == 64 ? rows(CT, Int<64>{}) : rows(CT, Int<128>{}); };
  switch (ct) {
    case kBf16: return dim(Int<kBf16>{});
    case kF16: return dim(Int<kF16>{});
    case kE4M3: return dim(Int<kE4M3>{});
    default: return dim(Int<kI8>{});
  }
}
NarrowShape narrow_shape(const CacheAttnParams &p, int ct, int d) {
  return with_kernel(p, ct, d, [&](auto CT, auto D, auto NT) { return shape_of<CT(), D(), NT()>(p); });
}

int64_t total_tiles(const CacheAttnParams &p, const NarrowShape &n) {
  const int64_t tiles = (static_cast<int64_t>(p.max_pages) * p.block_size + n.tile - 1) / n.tile;
  const int64_t units = n.units * p.batch;
  return tiles > 0 && units > INT64_MAX / tiles ? INT64_MAX : units * tiles;
}

// CTAs of the even-share form; 0: the call takes the cluster form, one launch instead of two, whose CTAs of one sequence are
// even but whose sequences may not be. That costs at most one sequence's keys, so it stays where the block tables address
// few (32 sequences of 1024 keys: 15.8 us; even shares 22.3), where the units fill several waves, and for one sequence, unless
// it has too few CTAs in its clusters (24 sequences of up to 32768 keys: 268 us; even shares 200). The host knows the tables'
// width, not the lengths: short sequences in wide tables take even shares too (the 32 x 1024 above in tables of 4096 keys
// 22.2 us, 16.3 with num_splits = 1).
constexpr int kFewKeys = 2048;
constexpr int64_t kMaxUnits = 65535;  // of a sequence, in the cluster form's grid
int narrow_grid(const CacheAttnParams &p, const NarrowShape &n, int num_splits) {
  if (num_splits > 0) return 0;
  const int64_t units = n.units * p.batch, slots = static_cast<int64_t>(n.ctas_per_sm) * sm_count();
  const int64_t tiles = total_tiles(p, n);
  if (tiles > INT32_MAX) return 0;  // tiles are counted in 32 bits
  if (static_cast<int64_t>(p.max_pages) * p.block_size <= kFewKeys || units >= 4 * slots) return 0;
  if (p.batch == 1 && units * kMaxSplits >= slots / 2) return 0;
  return static_cast<int>(std::max<int64_t>(1, std::min(slots, std::max(units, tiles / kMinTiles))));
}

template <int CT, int D, int NT> int launch_narrow(CacheAttnParams &p, int num_splits, void *workspace, cudaStream_t s) {
  using G = Geometry<CT, D, NT>;
  using Share = Form<CT, D, NT, false>;
  using Cluster = Form<CT, D, NT, true>;
  const NarrowShape n = shape_of<CT, D, NT>(p);
  const int grid = workspace ? narrow_grid(p, n, num_splits) : 0;
  if (grid > 0) {
    place_workspace(p, workspace, grid);
    static std::atomic<uint64_t> ready{0};  // bit: device whose shared-memory limit is set
    if (int rc = allow_smem(cache_attention_kernel<CT, D, NT, false>, Share::kSmem, ready)) return rc;
    if (int rc = launch_ex(cache_attention_kernel<CT, D, NT, false>, dim3(grid), dim3(kThreads), Share::kSmem, s, 1,
                           false, p))
      return rc;
    return launch_cache_attention_merge(p, CT, D, G::kRows, grid, s);
  }
  static std::atomic<uint64_t> ready{0};
  if (int rc = allow_smem(cache_attention_kernel<CT, D, NT, true>, Cluster::kSmem, ready)) return rc;
  if (n.units > kMaxUnits) return NVB200_ERR_UNSUPPORTED;
  p.splits = num_splits > 0 ? num_splits
                            : cluster_splits(p, n.units * p.batch, kWarps * G::kTile, Cluster::kCtasPerSm);
  constexpr int kMaxBatch = 65535;  // of a grid
  for (int64_t b = 0; b < p.batch; b += kMaxBatch) {
    p.first_batch = static_cast<int>(b);
    const dim3 grid(p.splits, static_cast<unsigned>(n.units), static_cast<unsigned>(std::min<int64_t>(kMaxBatch, p.batch - b)));
    if (int rc = launch_ex(cache_attention_kernel<CT, D, NT, true>, grid, dim3(kThreads), Cluster::kSmem, s, p.splits, false, p))
      return rc;
  }
  return NVB200_OK;
}

// Whether a call takes the wide kernel (128 rows a CTA on the 5th-generation tensor cores) rather than blocks of 16 rows of
// this one: above 32 (16-bit) or 64 rows (8-bit) where the tables address many keys, above twice that elsewhere. Measured on
// B200, head_dim 128, group 4, this kernel / the wide one, us, for ragged batches of (sequences x keys):
//   16-bit cache, 40 and 48 rows: 32 x 2048  74 /  68, 80 / 74
//   16-bit cache, 64 rows:  32 x 2048  78 /  77, 32 x 4096 182 / 109, 8 x 16384 144 /  94
//   16-bit cache, 128 rows: 32 x 2048 151 /  94, 32 x 4096 225 / 118, 8 x 16384 271 / 110
//   8-bit cache,  64 rows:  32 x 2048  70 / 129, 32 x 4096 133 / 183, 8 x 16384 105 / 144
//   8-bit cache,  72, 96 and 112 rows: 32 x 2048 82 / 123, 98 / 153, 112 / 137
//   8-bit cache,  128 rows: 32 x 2048 120 / 147, 32 x 4096 241 / 223, 8 x 16384 213 / 148
//   8-bit cache,  256 rows: 4 x 2048   61 /  46, 8 x 16384 351 / 227
// (8-bit tiles pass through shared memory twice there; long tables let its roles run undisturbed). The rule stands at measured
// row counts, not at the crossings: up to 8 % is lost at 40 to 64 rows of 16-bit caches in short tables, and in long tables the
// 8-bit lines cross somewhere between 64 and 128 rows. head_dim 64 has the same rule (32 x 2048: 16-bit 64 rows 51 / 58, 8-bit
// 72 rows 54 / 100, 128 rows 85 / 112).
bool prefers_wide(const CacheAttnParams &p, int ct) {
  const bool many_keys = static_cast<int64_t>(p.max_pages) * p.block_size > kFewKeys;
  const int few_rows = ct == kE4M3 || ct == kI8 ? 64 : 32;
  return p.rows > (many_keys ? few_rows : 2 * few_rows);
}

// Checks a call and fills `p` (all but the workspace) and *ct; *launch = false where there is nothing to do.
int prepare_attention(const nvb200_cache_attention_args *a, CacheAttnParams &p, int *ct, bool *launch) {
  *launch = false;
  if (!a || a->batch < 0 || a->queries_per_seq < 0 || a->num_q_heads <= 0 || a->num_kv_heads <= 0 ||
      a->num_q_heads % a->num_kv_heads != 0 || a->head_dim <= 0 || a->block_size <= 0 || a->max_blocks_per_seq < 0 ||
      a->num_blocks < 0 || a->num_splits < 0 || a->num_splits > kMaxSplits || (a->causal != 0 && a->causal != 1))
    return NVB200_ERR_ARG;
  if (a->dtype != NVB200_BF16 && a->dtype != NVB200_F16) return NVB200_ERR_ARG;
  if (a->cache_dtype == NVB200_E4M3) *ct = kE4M3;
  else if (a->cache_dtype == NVB200_I8) *ct = kI8;
  else if (a->cache_dtype == a->dtype) *ct = a->dtype == NVB200_F16 ? kF16 : kBf16;
  else return NVB200_ERR_ARG;
  if (!std::isfinite(a->softmax_scale)) return NVB200_ERR_ARG;
  if (a->batch == 0 || a->queries_per_seq == 0) return NVB200_OK;
  const bool quant = *ct == kE4M3 || *ct == kI8;
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
  p = CacheAttnParams{};
  p.q = a->q, p.q_batch_stride = a->q_batch_stride, p.q_token_stride = a->q_token_stride;
  p.q_head_stride = a->q_head_stride;
  p.k_cache = static_cast<const uint8_t *>(a->k_cache), p.v_cache = static_cast<const uint8_t *>(a->v_cache);
  p.blk_stride = a->cache_block_stride, p.tok_stride = a->cache_token_stride, p.head_stride = a->cache_head_stride;
  p.num_blocks = a->num_blocks, p.k_scale = quant ? a->k_scale : nullptr, p.v_scale = quant ? a->v_scale : nullptr;
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
  p.status = a->status, p.batch = a->batch;
  *launch = true;
  return NVB200_OK;
}

}  // namespace
}  // namespace nvb200

using namespace nvb200;

extern "C" int64_t nvb200_cache_attention_workspace_size(const nvb200_cache_attention_args *a) {
  CacheAttnParams p;
  int ct = 0;
  bool launch = false;
  if (prepare_attention(a, p, &ct, &launch) != NVB200_OK) return -1;
  if (!launch) return 0;
  if (prefers_wide(p, ct) && a->num_splits == 0 && wide_takes(p)) return wide_workspace_bytes(p, ct, a->head_dim);
  const NarrowShape n = narrow_shape(p, ct, a->head_dim);
  const int grid = narrow_grid(p, n, a->num_splits);
  return grid == 0 && n.units > kMaxUnits ? -1 : even_share_bytes(grid, n.rows, a->head_dim);
}

extern "C" int nvb200_cache_attention(const nvb200_cache_attention_args *a, void *workspace, int64_t workspace_bytes,
                                      nvb200_stream_t stream) {
  CacheAttnParams p;
  int ct = 0;
  bool launch = false;
  if (int rc = prepare_attention(a, p, &ct, &launch)) return rc;
  if (!launch) return NVB200_OK;
  if (workspace_bytes < 0 || !aligned16(workspace)) return NVB200_ERR_ARG;
  const int64_t need = nvb200_cache_attention_workspace_size(a);
  if (need < 0) return NVB200_ERR_UNSUPPORTED;
  if (int rc = check_device()) return rc;
  if (workspace && workspace_bytes < need) return NVB200_ERR_ARG;
  if (need == 0) workspace = nullptr;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (prefers_wide(p, ct) && a->num_splits == 0 && workspace && wide_takes(p)) {
    const int rc = launch_cache_attention_wide(p, ct, a->head_dim, workspace, s);
    if (rc != NVB200_ERR_UNSUPPORTED) return rc;
    workspace = nullptr;  // sized for the other kernel: the cluster form needs none
  }
  return with_kernel(p, ct, a->head_dim, [&](auto CT, auto D, auto NT) {
    return launch_narrow<CT(), D(), NT()>(p, a->num_splits, workspace, s);
  });
}
