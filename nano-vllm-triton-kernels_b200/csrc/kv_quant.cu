// The 8-bit paged KV cache: rows quantised as they are written (plainly, or behind the fused q/k RMSNorm + RoPE), and
// read back. Codes (e4m3 or int8) lie in [blocks, block_size, Hkv, D] like the 16-bit cache, one fp32 scale per token
// and KV head in [blocks, Hkv, block_size]: the tokens of one head are contiguous there, because the attention that
// reads the cache takes one head's scales for a run of tokens (16 keys: 64 bytes instead of 16 separate sectors), and
// the writes, 4 bytes per row either way, are merged in the L2. kv_quant_math.cuh has the quantiser.
//
// All three are HBM-bound: every row is read once and written once, and a row's maximum is taken from registers, so
// nothing is read a second time. A group of 4 to 32 lanes, the power of two of D / 16 or the next above it (lanes past
// D / 16 hold nothing), holds a row, 8 elements of each half a lane: 16-byte loads of 16-bit inputs, 8-byte stores of codes, and the maximum by shuffles within the group.
#include <algorithm>
#include <type_traits>

#include "common.cuh"
#include "kv_quant_math.cuh"
#include "qknr_math.cuh"

namespace nvb200 {
namespace {

constexpr int kQuantThreads = 256;

// Division of 32-bit numbers by a divisor that the host knows (Granlund and Montgomery, "Division by invariant integers
// using multiplication", 1994, figure 4.1).
struct Divider {
  uint32_t d, m;
  uint8_t s1, s2;
  void set(uint32_t divisor) {
    int l = 0;
    while ((uint64_t{1} << l) < divisor) ++l;
    d = divisor;
    m = static_cast<uint32_t>((((uint64_t{1} << l) - divisor) << 32) / divisor + 1);
    s1 = l > 0, s2 = l > 0 ? l - 1 : 0;
  }
  NVB200_DEVICE uint32_t quotient(uint32_t n) const {
    const uint32_t t = __umulhi(m, n);
    return (t + ((n - t) >> s1)) >> s2;
  }
};

struct QuantCache {
  uint8_t *k;
  uint8_t *v;
  float *k_scale;
  float *v_scale;
  int64_t num_slots;
  int block_size;
  int hkv;
  int d;
  Divider by_block, by_hkv;  // by block_size, by hkv
  int32_t *status;
};

// Index in the scale arrays of head h of slot s.
NVB200_DEVICE int64_t scale_index(const QuantCache &c, int64_t slot, int h) {
  const uint32_t blk = c.by_block.quotient(static_cast<uint32_t>(slot));  // num_slots < 2^32
  const uint32_t in = static_cast<uint32_t>(slot) - blk * static_cast<uint32_t>(c.block_size);
  return (static_cast<int64_t>(blk) * c.hkv + h) * c.block_size + in;
}

struct StoreQuantArgs {
  const char *key;
  const char *value;
  int64_t key_stride;  // elements between tokens
  int64_t value_stride;
  const void *slots;
  int slot64;
  uint32_t rows;  // tokens * hkv
  QuantCache c;
};

NVB200_DEVICE int64_t load_slot(const void *slots, int slot64, int64_t t) {
  return slot64 ? static_cast<int64_t>(__ldg(static_cast<const long long *>(slots) + t))
                : static_cast<int64_t>(__ldg(static_cast<const int *>(slots) + t));
}

// What a lane holds of a row: elements [8 j, 8 j + 8) and [D / 2 + 8 j, D / 2 + 8 j + 8), as they were loaded.
template <typename T> struct Piece {
  static constexpr int kWords = sizeof(T) / 2;  // 16-byte words of 8 elements
  uint4 w[2 * kWords];
  NVB200_DEVICE void clear() {
#pragma unroll
    for (int i = 0; i < 2 * kWords; ++i) w[i] = make_uint4(0, 0, 0, 0);
  }
  NVB200_DEVICE void load(const T *p, int half) {  // p + 8 j; 16-byte aligned, as is half * sizeof(T)
#pragma unroll
    for (int i = 0; i < kWords; ++i) {
      w[i] = __ldg(reinterpret_cast<const uint4 *>(p) + i);
      w[kWords + i] = __ldg(reinterpret_cast<const uint4 *>(p + half) + i);
    }
  }
  NVB200_DEVICE void values(int h, float (&f)[8]) const {
    if constexpr (std::is_same<T, float>::value) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const uint4 u = w[2 * h + i];
        f[4 * i] = __uint_as_float(u.x), f[4 * i + 1] = __uint_as_float(u.y);
        f[4 * i + 2] = __uint_as_float(u.z), f[4 * i + 3] = __uint_as_float(u.w);
      }
    } else if constexpr (std::is_same<T, __half>::value) {
      const uint32_t x[4] = {w[h].x, w[h].y, w[h].z, w[h].w};
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float2 y = __half22float2(*reinterpret_cast<const __half2 *>(&x[i]));
        f[2 * i] = y.x, f[2 * i + 1] = y.y;
      }
    } else {
      unpack8(w[h], f);
    }
  }
  // The largest magnitude's bits, in the element's own type (infinities and NaNs are above every finite value).
  NVB200_DEVICE uint32_t amax() const {
    uint32_t m = 0;
    constexpr uint32_t kAbs = std::is_same<T, float>::value ? 0x7FFFFFFFu : 0x7FFF7FFFu;
#pragma unroll
    for (int i = 0; i < 2 * kWords; ++i) {
      const uint32_t x[4] = {w[i].x & kAbs, w[i].y & kAbs, w[i].z & kAbs, w[i].w & kAbs};
#pragma unroll
      for (int e = 0; e < 4; ++e) m = std::is_same<T, float>::value ? max(m, x[e]) : __vmaxu2(m, x[e]);
    }
    return std::is_same<T, float>::value ? m : max(m & 0xFFFFu, m >> 16);
  }
};

// Bits of a non-negative value of type T as those of the fp32 value.
template <typename T> NVB200_DEVICE uint32_t bits32(uint32_t b) {
  if constexpr (std::is_same<T, float>::value) return b;
  else if constexpr (std::is_same<T, __half>::value)
    return __float_as_uint(__half2float(__ushort_as_half(static_cast<unsigned short>(b))));
  else return b << 16;
}

// The largest of ka and of va over a group of LPR lanes, as fp32 bits: one shuffle for both where they have 16 bits.
template <typename T, int LPR> NVB200_DEVICE void group_amax(uint32_t &ka, uint32_t &va) {
  if constexpr (std::is_same<T, float>::value) {
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) {
      ka = max(ka, __shfl_xor_sync(0xffffffffu, ka, o));
      va = max(va, __shfl_xor_sync(0xffffffffu, va, o));
    }
  } else {
    uint32_t m = ka | va << 16;
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) m = __vmaxu2(m, __shfl_xor_sync(0xffffffffu, m, o));
    ka = bits32<T>(m & 0xFFFFu), va = bits32<T>(m >> 16);
  }
}

NVB200_DEVICE uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }
// Row u (token u / hkv, head u % hkv) is held by a group of LPR lanes; lanes at or past D / 16 hold nothing. All loads are
// in flight at once; the values do not wait for the slot (a token without one has its row read for nothing).
template <typename T, int FMT, int LPR>
__global__ void __launch_bounds__(kQuantThreads) store_quant_kernel(const __grid_constant__ StoreQuantArgs a) {
  const int j = threadIdx.x % LPR, half = a.c.d / 2;
  const bool on = 8 * j < half;
  const uint32_t u = blockIdx.x * (kQuantThreads / LPR) + threadIdx.x / LPR;
  const uint32_t t = a.c.by_hkv.quotient(u), h = u - t * a.c.hkv;
  Piece<T> k, v;
  k.clear(), v.clear();
  int64_t slot = -1;
  if (u < a.rows) {
    slot = load_slot(a.slots, a.slot64, t);
    if (on) {
      k.load(reinterpret_cast<const T *>(a.key) + t * a.key_stride + static_cast<int64_t>(h) * a.c.d + 8 * j, half);
      v.load(reinterpret_cast<const T *>(a.value) + t * a.value_stride + static_cast<int64_t>(h) * a.c.d + 8 * j, half);
    }
  }
  uint32_t ka = k.amax(), va = v.amax();
  group_amax<T, LPR>(ka, va);
  if (slot < 0 || slot >= a.c.num_slots) {
    if (slot != -1 && j == 0) set_status(a.c.status, NVB200_STATUS_BAD_SLOT);
    return;
  }
  const RowScale ks = row_scale<FMT>(ka), vs = row_scale<FMT>(va);
  if (on) {
    const int64_t off = (slot * a.c.hkv + h) * a.c.d + 8 * j;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      float x[8];
      k.values(i, x);
      *reinterpret_cast<uint2 *>(a.c.k + off + i * half) = quantise8<FMT>(x, ks);
      v.values(i, x);
      *reinterpret_cast<uint2 *>(a.c.v + off + i * half) = quantise8<FMT>(x, vs);
    }
  }
  if (j == 0) {
    const int64_t si = scale_index(a.c, slot, h);
    a.c.k_scale[si] = ks.scale;
    a.c.v_scale[si] = vs.scale;
  }
}

// Rows that the vector kernel does not take (D not a multiple of 16 or above 512, addresses not 16-byte aligned): one
// warp per row, one element per access, the row read twice (the second time from the L1).
template <typename T, int FMT>
__global__ void __launch_bounds__(kQuantThreads) store_quant_any_kernel(const __grid_constant__ StoreQuantArgs a) {
  const int lane = threadIdx.x & 31;
  for (uint64_t u = static_cast<uint64_t>(blockIdx.x) * (kQuantThreads / 32) + threadIdx.x / 32;
       u < 2ull * a.rows; u += static_cast<uint64_t>(gridDim.x) * (kQuantThreads / 32)) {
    const bool is_v = u >= a.rows;
    const uint32_t w = static_cast<uint32_t>(is_v ? u - a.rows : u);
    const uint32_t t = w / static_cast<uint32_t>(a.c.hkv), h = w - t * a.c.hkv;
    const int64_t slot = load_slot(a.slots, a.slot64, t);
    if (slot < 0 || slot >= a.c.num_slots) {
      if (slot != -1 && lane == 0) set_status(a.c.status, NVB200_STATUS_BAD_SLOT);
      continue;
    }
    const T *x = (is_v ? reinterpret_cast<const T *>(a.value) + t * a.value_stride
                       : reinterpret_cast<const T *>(a.key) + t * a.key_stride) +
                 static_cast<int64_t>(h) * a.c.d;
    uint32_t am = 0;
    for (int i = lane; i < a.c.d; i += 32) am = max(am, abs_bits(Elem<T>::to_f(x[i])));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) am = max(am, __shfl_xor_sync(0xffffffffu, am, o));
    const RowScale s = row_scale<FMT>(am);
    uint8_t *out = (is_v ? a.c.v : a.c.k) + (slot * a.c.hkv + h) * a.c.d;
    for (int i = lane; i < a.c.d; i += 32) out[i] = quantise1<FMT>(Elem<T>::to_f(x[i]), s);
    if (lane == 0) (is_v ? a.c.v_scale : a.c.k_scale)[scale_index(a.c, slot, h)] = s.scale;
  }
}

int grid_for(int64_t units, int64_t per_cta, int per_sm) {
  return static_cast<int>(std::max<int64_t>(
      1, std::min<int64_t>((units + per_cta - 1) / per_cta, static_cast<int64_t>(sm_count()) * per_sm)));
}

// f(lanes that hold a row of D elements, 16 a lane)
template <typename F> int with_lanes(int d, F &&f) {
  if (d <= 64) return f(std::integral_constant<int, 4>{});
  if (d <= 128) return f(std::integral_constant<int, 8>{});
  return d <= 256 ? f(std::integral_constant<int, 16>{}) : f(std::integral_constant<int, 32>{});
}
bool fits_lanes(int d) { return d % 16 == 0 && d <= 512; }

template <typename T, int FMT> int launch_store_quant(const StoreQuantArgs &a, bool vec, cudaStream_t s) {
  if (!vec) {
    store_quant_any_kernel<T, FMT><<<grid_for(2ll * a.rows, kQuantThreads / 32, 8), kQuantThreads, 0, s>>>(a);
    return launch_status();
  }
  return with_lanes(a.c.d, [&](auto lanes) {
    constexpr uint32_t kGroups = kQuantThreads / lanes();
    store_quant_kernel<T, FMT, lanes()><<<(a.rows + kGroups - 1) / kGroups, kQuantThreads, 0, s>>>(a);
    return launch_status();
  });
}

template <typename T> int launch_store_fmt(const StoreQuantArgs &a, int fmt, bool vec, cudaStream_t s) {
  return fmt == kCacheE4M3 ? launch_store_quant<T, kCacheE4M3>(a, vec, s) : launch_store_quant<T, kCacheI8>(a, vec, s);
}

// ---------------------------------------------------------------------------------------------------------------
// Fused q/k RMSNorm + RoPE with the quantising write. A unit is one head of one token: Hq query heads, Hkv key heads
// and Hkv value heads. D / 16 lanes hold a unit, lane j the elements [8 j, 8 j + 8) and [D/2 + 8 j, D/2 + 8 j + 8), so a
// lane has both ends of its rotation pairs. The norm and rotation are the fused op's (qknr_math.cuh: same operations in
// the same order, so q_out, k_out and the bf16 rows that are quantised have the same bits as there).

struct QknrQuantArgs {
  const __nv_bfloat16 *q, *k, *v;
  int64_t q_stride, k_stride, v_stride;
  const int64_t *positions;
  const int32_t *slots;
  const __nv_bfloat16 *q_w, *k_w;
  const float *cos_sin;
  int64_t cs_stride, num_positions;
  __nv_bfloat16 *q_out, *k_out;
  uint32_t units;         // groups of R heads
  Divider by_parts;       // by a token's groups
  int hq, heads;          // heads = hq + 2 hkv
  float eps;
  QuantCache c;
};

template <int D, int FMT, int R>
__global__ void __launch_bounds__(kQuantThreads) qknr_quant_kernel(const __grid_constant__ QknrQuantArgs a) {
  constexpr int HALF = D / 2, LPH = D / 16;
  const int j = threadIdx.x % LPH;
  const uint32_t u = blockIdx.x * (kQuantThreads / LPH) + threadIdx.x / LPH;
  const bool live = u < a.units;
  const uint32_t t = live ? a.by_parts.quotient(u) : 0;
  const int head0 = live ? static_cast<int>(u - t * a.by_parts.d) * R : a.heads;
  uint4 xa[R], xb[R];
#pragma unroll
  for (int i = 0; i < R; ++i) {
    xa[i] = xb[i] = make_uint4(0, 0, 0, 0);
    const int head = head0 + i;
    if (head < a.heads) {
      const __nv_bfloat16 *x = head < a.hq ? a.q + t * a.q_stride + static_cast<int64_t>(head) * D
                               : head < a.hq + a.c.hkv
                                   ? a.k + t * a.k_stride + static_cast<int64_t>(head - a.hq) * D
                                   : a.v + t * a.v_stride + static_cast<int64_t>(head - a.hq - a.c.hkv) * D;
      xa[i] = __ldg(reinterpret_cast<const uint4 *>(x + 8 * j));
      xb[i] = __ldg(reinterpret_cast<const uint4 *>(x + HALF + 8 * j));
    }
  }
  const bool rotates = head0 < a.hq + a.c.hkv;  // a head of this lane's that is q or k
  int64_t slot = -1, pos = 0;
  if (live) {
    if (head0 + R > a.hq) slot = __ldg(a.slots + t);
    if (rotates) pos = __ldg(a.positions + t);
  }
  if (slot < -1 || slot >= a.c.num_slots) {
    if (j == 0) set_status(a.c.status, NVB200_STATUS_BAD_SLOT);
    slot = -1;
  }
  if (pos < 0 || pos >= a.num_positions) {
    if (j == 0) set_status(a.c.status, NVB200_STATUS_BAD_POSITION);
    pos = 0;
  }
  float c[8] = {}, sn[8] = {};
  if (rotates) {
    const float *cs = a.cos_sin + pos * a.cs_stride;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const float4 cc = __ldg(reinterpret_cast<const float4 *>(cs + 8 * j) + i);
      const float4 s4 = __ldg(reinterpret_cast<const float4 *>(cs + HALF + 8 * j) + i);
      c[4 * i] = cc.x, c[4 * i + 1] = cc.y, c[4 * i + 2] = cc.z, c[4 * i + 3] = cc.w;
      sn[4 * i] = s4.x, sn[4 * i + 1] = s4.y, sn[4 * i + 2] = s4.z, sn[4 * i + 3] = s4.w;
    }
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int head = head0 + i;
    const bool is_q = head < a.hq, is_v = head >= a.hq + a.c.hkv;
    const int h = is_q ? head : (is_v ? head - a.hq - a.c.hkv : head - a.hq);
    float x1[8], x2[8];
    unpack8(xa[i], x1);
    unpack8(xb[i], x2);
    float ss = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(x1[e], x1[e], ss);
#pragma unroll
    for (int e = 0; e < 8; ++e) ss = fmaf(x2[e], x2[e], ss);
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (!is_v) {
      uint32_t w1[4], w2[4];
      load_w8((is_q ? a.q_w : a.k_w) + 8 * j, w1);
      load_w8((is_q ? a.q_w : a.k_w) + HALF + 8 * j, w2);
      const float rstd = rsqrtf(ss / static_cast<float>(D) + a.eps);
      float y1[8], y2[8];
      norm_rope8(x1, x2, rstd, w1, w2, c, sn, y1, y2);
      xa[i] = pack8(y1), xb[i] = pack8(y2);
      __nv_bfloat16 *o = is_q ? a.q_out + (static_cast<int64_t>(t) * a.hq + h) * D
                              : (a.k_out ? a.k_out + (static_cast<int64_t>(t) * a.c.hkv + h) * D : nullptr);
      if (o) {
        *reinterpret_cast<uint4 *>(o + 8 * j) = xa[i];
        *reinterpret_cast<uint4 *>(o + HALF + 8 * j) = xb[i];
      }
    }
    // A warp's groups may hold heads of different kinds; the shuffles below need all of its lanes.
    if (__all_sync(0xffffffffu, is_q)) continue;
    const Piece<__nv_bfloat16> piece{{xa[i], xb[i]}};
    uint32_t am = piece.amax();
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) am = max(am, __shfl_xor_sync(0xffffffffu, am, o));
    if (is_q || slot < 0 || head >= a.heads) continue;
    const RowScale rs = row_scale<FMT>(bits32<__nv_bfloat16>(am));
    piece.values(0, x1);
    piece.values(1, x2);
    uint8_t *row = (is_v ? a.c.v : a.c.k) + (slot * a.c.hkv + h) * D;
    *reinterpret_cast<uint2 *>(row + 8 * j) = quantise8<FMT>(x1, rs);
    *reinterpret_cast<uint2 *>(row + HALF + 8 * j) = quantise8<FMT>(x2, rs);
    if (j == 0) (is_v ? a.c.v_scale : a.c.k_scale)[scale_index(a.c, slot, h)] = rs.scale;
  }
}

// R heads a group: 2 once that still fills the GPU (8192 tokens of 32 + 8 + 8 heads: 1 head 47 us, 2 40 us, 4 45 us, which
// leaves room for fewer warps).
template <int D, int FMT> int launch_qknr_dim(QknrQuantArgs &a, int64_t tokens, cudaStream_t s) {
  constexpr int64_t kGroups = kQuantThreads / (D / 16);
  auto launch = [&](auto kernel, int r) {
    a.by_parts.set(static_cast<uint32_t>((a.heads + r - 1) / r));
    a.units = static_cast<uint32_t>(tokens * a.by_parts.d);
    kernel<<<static_cast<unsigned>((a.units + kGroups - 1) / kGroups), kQuantThreads, 0, s>>>(a);
    return launch_status();
  };
  if (tokens * a.heads > 8 * kGroups * sm_count()) return launch(qknr_quant_kernel<D, FMT, 2>, 2);
  return launch(qknr_quant_kernel<D, FMT, 1>, 1);
}

template <int FMT> int launch_qknr_quant(QknrQuantArgs &a, int64_t tokens, cudaStream_t s) {
  switch (a.c.d) {
    case 64: return launch_qknr_dim<64, FMT>(a, tokens, s);
    case 128: return launch_qknr_dim<128, FMT>(a, tokens, s);
    case 256: return launch_qknr_dim<256, FMT>(a, tokens, s);
  }
  return NVB200_ERR_UNSUPPORTED;
}

// ---------------------------------------------------------------------------------------------------------------
// Read-back: packed row t of [total, Hkv, D] is token t - cu[b] of the sequence b with cu[b] <= t < cu[b + 1], found
// through the block table; value = code * scale in fp32, rounded once to the output type.

struct LoadQuantArgs {
  void *key;
  void *value;
  const int32_t *table;
  int64_t table_stride;
  const int32_t *cu;  // [batch + 1]
  int batch;
  int max_pages;
  int64_t num_blocks;
  int64_t total;
  int run;        // tokens a warp takes, at most 32
  int zero_rest;  // rows outside every sequence: 1 = zeros, 0 = left as they are
  QuantCache c;
};

template <typename T> NVB200_DEVICE void store8(T *p, const float (&f)[8]);
template <> NVB200_DEVICE void store8<__nv_bfloat16>(__nv_bfloat16 *p, const float (&f)[8]) {
  *reinterpret_cast<uint4 *>(p) = pack8(f);
}
template <> NVB200_DEVICE void store8<__half>(__half *p, const float (&f)[8]) {
  uint4 u;
  uint32_t *w = &u.x;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __half2 h = __floats2half2_rn(f[2 * i], f[2 * i + 1]);
    w[i] = *reinterpret_cast<const uint32_t *>(&h);
  }
  *reinterpret_cast<uint4 *>(p) = u;
}
template <> NVB200_DEVICE void store8<float>(float *p, const float (&f)[8]) {
  *reinterpret_cast<float4 *>(p) = make_float4(f[0], f[1], f[2], f[3]);
  *(reinterpret_cast<float4 *>(p) + 1) = make_float4(f[4], f[5], f[6], f[7]);
}

// The slot of packed row t: -1 = outside every sequence, -2 = its page cannot be followed (reported).
NVB200_DEVICE int64_t slot_of_row(const LoadQuantArgs &a, int64_t t) {
  // The last b with cu[b] <= t (cu does not fall; empty sequences share a boundary, and the last of them is taken).
  int lo = 0, hi = a.batch;  // cu[lo] <= t < cu[hi], once both ends are checked
  if (t < __ldg(a.cu) || t >= __ldg(a.cu + a.batch)) return -1;
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(a.cu + mid) <= t) lo = mid;
    else hi = mid;
  }
  const int64_t pos = t - __ldg(a.cu + lo);
  const int64_t page = pos / a.c.block_size;
  if (page >= a.max_pages) return -2;
  const int64_t blk = __ldg(a.table + lo * a.table_stride + page);
  if (blk < 0 || blk >= a.num_blocks) return -2;
  return blk * a.c.block_size + (pos - page * a.c.block_size);
}

// A warp takes a.run consecutive packed tokens at a time: lane i looks up the slot of token i (one search per token, not one
// per head), then the warp copies their rows, the LPR lanes of a group one head's row at a time, U rows in flight.
template <typename T, int FMT, int LPR>
__global__ void __launch_bounds__(kQuantThreads) load_quant_kernel(const __grid_constant__ LoadQuantArgs a) {
  constexpr int RPW = 32 / LPR, U = 2;
  const int lane = threadIdx.x & 31, j = lane % LPR, grp = lane / LPR, half = a.c.d / 2;
  const bool on = 8 * j < half;
  const int64_t t0 = (static_cast<int64_t>(blockIdx.x) * (kQuantThreads / 32) + threadIdx.x / 32) * a.run;
  if (t0 >= a.total) return;
  const int n = static_cast<int>(min(static_cast<int64_t>(a.run), a.total - t0)), rows = n * a.c.hkv;
  int64_t mine = -1;
  if (lane < n) {
    mine = slot_of_row(a, t0 + lane);
    if (mine == -2) set_status(a.c.status, NVB200_STATUS_BAD_SLOT);
  }
  for (int r0 = 0; r0 < rows; r0 += RPW * U) {
    uint2 kw[U][2], vw[U][2];
    float ks[U], vs[U];
    int64_t slot[U];
#pragma unroll
    for (int x = 0; x < U; ++x) {
      const int r = min(r0 + x * RPW + grp, rows - 1);
      const int i = static_cast<int>(a.c.by_hkv.quotient(r)), h = r - i * a.c.hkv;
      slot[x] = __shfl_sync(0xffffffffu, mine, i);
      kw[x][0] = kw[x][1] = vw[x][0] = vw[x][1] = make_uint2(0, 0);
      ks[x] = vs[x] = 0.f;
      if (on && slot[x] >= 0) {
        const int64_t src = (slot[x] * a.c.hkv + h) * a.c.d + 8 * j;
        const int64_t si = scale_index(a.c, slot[x], h);
        kw[x][0] = __ldg(reinterpret_cast<const uint2 *>(a.c.k + src));
        kw[x][1] = __ldg(reinterpret_cast<const uint2 *>(a.c.k + src + half));
        vw[x][0] = __ldg(reinterpret_cast<const uint2 *>(a.c.v + src));
        vw[x][1] = __ldg(reinterpret_cast<const uint2 *>(a.c.v + src + half));
        ks[x] = __ldg(a.c.k_scale + si), vs[x] = __ldg(a.c.v_scale + si);
      }
    }
#pragma unroll
    for (int x = 0; x < U; ++x) {
      const int r = r0 + x * RPW + grp;
      if (r >= rows || !on || (slot[x] == -1 && !a.zero_rest)) continue;
      const int64_t dst = (t0 * a.c.hkv + r) * a.c.d + 8 * j;
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float k[8], v[8];
        code_values8<FMT>(kw[x][i], k);
        code_values8<FMT>(vw[x][i], v);
#pragma unroll
        for (int e = 0; e < 8; ++e) k[e] *= ks[x], v[e] *= vs[x];
        store8(static_cast<T *>(a.key) + dst + i * half, k);
        store8(static_cast<T *>(a.value) + dst + i * half, v);
      }
    }
  }
}

// D not a multiple of 16 or above 512, or an address that is not 16-byte aligned: one warp per row of one tensor.
template <typename T, int FMT>
__global__ void __launch_bounds__(kQuantThreads) load_quant_any_kernel(const __grid_constant__ LoadQuantArgs a) {
  const int lane = threadIdx.x & 31;
  const int64_t rows = a.total * a.c.hkv;
  for (int64_t u = static_cast<int64_t>(blockIdx.x) * (kQuantThreads / 32) + threadIdx.x / 32; u < 2 * rows;
       u += static_cast<int64_t>(gridDim.x) * (kQuantThreads / 32)) {
    const bool is_v = u >= rows;
    const int64_t w = is_v ? u - rows : u;
    const int64_t t = w / a.c.hkv;
    const int h = static_cast<int>(w - t * a.c.hkv);
    const int64_t slot = slot_of_row(a, t);
    if (slot == -2 && lane == 0) set_status(a.c.status, NVB200_STATUS_BAD_SLOT);
    if (slot == -1 && !a.zero_rest) continue;
    T *out = static_cast<T *>(is_v ? a.value : a.key) + w * a.c.d;
    const uint8_t *in = (is_v ? a.c.v : a.c.k) + (slot < 0 ? 0 : (slot * a.c.hkv + h) * a.c.d);
    const float s = slot < 0 ? 0.f : (is_v ? a.c.v_scale : a.c.k_scale)[scale_index(a.c, slot, h)];
    for (int i = lane; i < a.c.d; i += 32)
      out[i] = Elem<T>::from_f(slot < 0 ? 0.f : code_value<FMT>(in[i]) * s);
  }
}

template <typename T, int FMT> int launch_load_quant(LoadQuantArgs &a, bool vec, cudaStream_t s) {
  if (!vec) {
    load_quant_any_kernel<T, FMT>
        <<<grid_for(2 * a.total * a.c.hkv, kQuantThreads / 32, 8), kQuantThreads, 0, s>>>(a);
    return launch_status();
  }
  // Tokens a warp: 2 share a search's latency; more leave the last warps behind (176k tokens of 8 heads: 2 99 us, 4 103 us, 8 110 us; fewer heads leave lanes without a row).
  const int64_t warps = static_cast<int64_t>(sm_count()) * 64;
  a.run = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(2, a.total / warps)));
  const int64_t per_cta = static_cast<int64_t>(a.run) * (kQuantThreads / 32);
  const unsigned grid = static_cast<unsigned>((a.total + per_cta - 1) / per_cta);
  return with_lanes(a.c.d, [&](auto lanes) {
    load_quant_kernel<T, FMT, lanes()><<<grid, kQuantThreads, 0, s>>>(a);
    return launch_status();
  });
}

template <typename T> int launch_load_fmt(LoadQuantArgs &a, int fmt, bool vec, cudaStream_t s) {
  return fmt == kCacheE4M3 ? launch_load_quant<T, kCacheE4M3>(a, vec, s) : launch_load_quant<T, kCacheI8>(a, vec, s);
}

// ---------------------------------------------------------------------------------------------------------------
// Host side.

// Checks the cache part of a call and fills `c`; *fmt gets the format.
int prepare_cache(const nvb200_quant_cache *q, int32_t *status, QuantCache &c, int *fmt) {
  if (q->dtype == NVB200_E4M3) *fmt = kCacheE4M3;
  else if (q->dtype == NVB200_I8) *fmt = kCacheI8;
  else return NVB200_ERR_ARG;
  if (q->num_blocks < 0 || q->block_size <= 0 || q->num_kv_heads <= 0 || q->head_dim <= 0) return NVB200_ERR_ARG;
  if (q->head_dim > (1 << 20) || q->num_kv_heads > (1 << 20)) return NVB200_ERR_ARG;
  // Slots are divided as 32-bit numbers.
  if (q->num_blocks > (int64_t{1} << 32) / q->block_size - 1) return NVB200_ERR_UNSUPPORTED;
  c.k = static_cast<uint8_t *>(q->k_cache), c.v = static_cast<uint8_t *>(q->v_cache);
  c.k_scale = q->k_scale, c.v_scale = q->v_scale;
  c.num_slots = q->num_blocks * q->block_size;
  c.block_size = q->block_size, c.hkv = q->num_kv_heads, c.d = q->head_dim;
  c.by_block.set(static_cast<uint32_t>(q->block_size)), c.by_hkv.set(static_cast<uint32_t>(q->num_kv_heads));
  c.status = status;
  return NVB200_OK;
}

bool has_pointers(const QuantCache &c) { return c.k && c.v && c.k_scale && c.v_scale; }
bool multiple16(int64_t bytes) { return (bytes & 15) == 0; }

}  // namespace
}  // namespace nvb200

using namespace nvb200;

extern "C" int nvb200_store_kvcache_quant(const void *key, int64_t key_token_stride, const void *value,
                                          int64_t value_token_stride, const void *slot_mapping, int slot_bytes,
                                          int64_t num_tokens, int dtype, const nvb200_quant_cache *cache,
                                          int32_t *status, nvb200_stream_t stream) {
  if (!cache || num_tokens < 0) return NVB200_ERR_ARG;
  if (dtype != NVB200_BF16 && dtype != NVB200_F16 && dtype != NVB200_F32) return NVB200_ERR_ARG;
  if (slot_bytes != 4 && slot_bytes != 8) return NVB200_ERR_ARG;
  StoreQuantArgs a{};
  int fmt = 0;
  if (int rc = prepare_cache(cache, status, a.c, &fmt)) return rc;
  if (num_tokens == 0) return NVB200_OK;
  if (!key || !value || !slot_mapping || !has_pointers(a.c)) return NVB200_ERR_ARG;
  if (num_tokens > (int64_t{1} << 31) / a.c.hkv) return NVB200_ERR_UNSUPPORTED;
  if (int rc = check_device()) return rc;
  const int64_t es = dtype == NVB200_F32 ? 4 : 2;
  a.key = static_cast<const char *>(key), a.value = static_cast<const char *>(value);
  a.key_stride = key_token_stride, a.value_stride = value_token_stride;
  a.slots = slot_mapping, a.slot64 = slot_bytes == 8;
  a.rows = static_cast<uint32_t>(num_tokens * a.c.hkv);
  const bool vec = fits_lanes(a.c.d) && aligned16(key) && aligned16(value) &&
                   multiple16(key_token_stride * es) && multiple16(value_token_stride * es) && aligned16(a.c.k) &&
                   aligned16(a.c.v);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == NVB200_BF16) return launch_store_fmt<__nv_bfloat16>(a, fmt, vec, s);
  if (dtype == NVB200_F16) return launch_store_fmt<__half>(a, fmt, vec, s);
  return launch_store_fmt<float>(a, fmt, vec, s);
}

extern "C" int nvb200_qk_norm_rope_kv_quant(const nvb200_qk_norm_rope_kv_args *q, const nvb200_quant_cache *cache,
                                            nvb200_stream_t stream) {
  if (!q || !cache) return NVB200_ERR_ARG;
  if (q->num_tokens < 0 || q->num_q_heads <= 0 || q->num_kv_heads <= 0 || q->num_q_heads % q->num_kv_heads != 0 ||
      q->head_dim <= 0 || q->head_dim % 2 != 0 || q->num_positions <= 0 || q->cos_sin_stride < 0)
    return NVB200_ERR_ARG;
  if (cache->num_kv_heads != q->num_kv_heads || cache->head_dim != q->head_dim) return NVB200_ERR_ARG;
  QknrQuantArgs a{};
  int fmt = 0;
  if (int rc = prepare_cache(cache, q->status, a.c, &fmt)) return rc;
  if (q->num_tokens == 0) return NVB200_OK;
  if (!q->q || !q->k || !q->v || !q->q_out || !q->positions || !q->slot_mapping || !q->q_weight || !q->k_weight ||
      !q->cos_sin || !has_pointers(a.c))
    return NVB200_ERR_ARG;
  const int D = q->head_dim;
  if (D != 64 && D != 128 && D != 256) return NVB200_ERR_UNSUPPORTED;
  const int64_t heads = static_cast<int64_t>(q->num_q_heads) + 2 * static_cast<int64_t>(q->num_kv_heads);
  if (heads > (1 << 20) || q->num_tokens > (int64_t{1} << 31) / heads) return NVB200_ERR_UNSUPPORTED;
  const void *aligned[] = {q->q, q->k, q->v, q->q_out, q->k_out, q->q_weight, q->k_weight, q->cos_sin, a.c.k, a.c.v};
  for (const void *p : aligned)
    if (!aligned16(p)) return NVB200_ERR_UNSUPPORTED;
  if (!multiple16(2 * q->q_token_stride) || !multiple16(2 * q->k_token_stride) || !multiple16(2 * q->v_token_stride) ||
      !multiple16(4 * q->cos_sin_stride))
    return NVB200_ERR_UNSUPPORTED;
  if (int rc = check_device()) return rc;
  using B = __nv_bfloat16;
  a.q = static_cast<const B *>(q->q), a.k = static_cast<const B *>(q->k), a.v = static_cast<const B *>(q->v);
  a.q_stride = q->q_token_stride, a.k_stride = q->k_token_stride, a.v_stride = q->v_token_stride;
  a.positions = q->positions, a.slots = q->slot_mapping;
  a.q_w = static_cast<const B *>(q->q_weight), a.k_w = static_cast<const B *>(q->k_weight);
  a.cos_sin = q->cos_sin, a.cs_stride = q->cos_sin_stride, a.num_positions = q->num_positions;
  a.q_out = static_cast<B *>(q->q_out), a.k_out = static_cast<B *>(q->k_out);
  a.hq = q->num_q_heads, a.heads = static_cast<int>(heads);
  a.eps = q->eps;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return fmt == kCacheE4M3 ? launch_qknr_quant<kCacheE4M3>(a, q->num_tokens, s)
                           : launch_qknr_quant<kCacheI8>(a, q->num_tokens, s);
}

extern "C" int nvb200_load_kvcache_quant(void *key, void *value, const nvb200_quant_cache *cache,
                                         const int32_t *block_table, int64_t block_table_stride,
                                         int32_t max_blocks_per_seq, const int32_t *cu_seqlens, int32_t batch,
                                         int64_t total_tokens, int dtype, int zero_rest, int32_t *status,
                                         nvb200_stream_t stream) {
  if (!cache || batch < 0 || total_tokens < 0 || max_blocks_per_seq < 0 || (zero_rest != 0 && zero_rest != 1))
    return NVB200_ERR_ARG;
  if (dtype != NVB200_BF16 && dtype != NVB200_F16 && dtype != NVB200_F32) return NVB200_ERR_ARG;
  LoadQuantArgs a{};
  int fmt = 0;
  if (int rc = prepare_cache(cache, status, a.c, &fmt)) return rc;
  if (total_tokens == 0) return NVB200_OK;
  if (!key || !value || !cu_seqlens || !has_pointers(a.c) || (batch > 0 && !block_table)) return NVB200_ERR_ARG;
  if (total_tokens > (int64_t{1} << 31) / a.c.hkv) return NVB200_ERR_UNSUPPORTED;
  if (int rc = check_device()) return rc;
  a.key = key, a.value = value, a.table = block_table, a.table_stride = block_table_stride, a.cu = cu_seqlens;
  a.batch = batch, a.max_pages = max_blocks_per_seq, a.num_blocks = cache->num_blocks, a.total = total_tokens;
  a.zero_rest = zero_rest;
  const bool vec = fits_lanes(a.c.d) && aligned16(key) && aligned16(value) && aligned16(a.c.k) &&
                   aligned16(a.c.v);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == NVB200_BF16) return launch_load_fmt<__nv_bfloat16>(a, fmt, vec, s);
  if (dtype == NVB200_F16) return launch_load_fmt<__half>(a, fmt, vec, s);
  return launch_load_fmt<float>(a, fmt, vec, s);
}
