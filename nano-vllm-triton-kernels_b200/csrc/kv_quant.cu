// The 8-bit paged KV cache: rows quantised as they are written (plainly, or behind the fused q/k RMSNorm + RoPE), and
// read back. Codes (e4m3 or int8) lie in [blocks, block_size, Hkv, D] like the 16-bit cache, one fp32 scale per token
// and KV head in [blocks, Hkv, block_size]: the tokens of one head are contiguous there, because the attention that
// reads the cache takes one head's scales for a run of tokens (16 keys: 64 bytes instead of 16 separate sectors), and
// the writes, 4 bytes per row either way, are merged in the L2. kv_quant_math.cuh has the quantiser.
//
// All three are HBM-bound: every row is read once and written once, and a row's maximum is taken from registers, so
// nothing is read a second time. A group of D / 8 lanes (a power of two of them) holds a row, 8 elements a lane: 16-byte
// loads of 16-bit inputs, 8-byte stores of codes, and the maximum by shuffles within the group.
#include <algorithm>

#include "common.cuh"
#include "kv_quant_math.cuh"
#include "qknr_math.cuh"

namespace nvb200 {
namespace {

constexpr int kQuantThreads = 256;

struct QuantCache {
  uint8_t *k;
  uint8_t *v;
  float *k_scale;
  float *v_scale;
  int64_t num_slots;
  int block_size;
  int hkv;
  int d;
  int32_t *status;
};

// Index in the scale arrays of head h of slot s.
NVB200_DEVICE int64_t scale_index(const QuantCache &c, int64_t slot, int h) {
  const uint32_t blk = static_cast<uint32_t>(slot) / static_cast<uint32_t>(c.block_size);  // num_slots < 2^32
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

// Eight consecutive elements as fp32. p is 16-byte aligned.
template <typename T> NVB200_DEVICE void load8(const T *p, float (&f)[8]);
template <> NVB200_DEVICE void load8<__nv_bfloat16>(const __nv_bfloat16 *p, float (&f)[8]) {
  unpack8(__ldg(reinterpret_cast<const uint4 *>(p)), f);
}
template <> NVB200_DEVICE void load8<__half>(const __half *p, float (&f)[8]) {
  const uint4 u = __ldg(reinterpret_cast<const uint4 *>(p));
  const uint32_t w[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
    f[2 * i] = x.x, f[2 * i + 1] = x.y;
  }
}
template <> NVB200_DEVICE void load8<float>(const float *p, float (&f)[8]) {
  const float4 a = __ldg(reinterpret_cast<const float4 *>(p)), b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
  f[0] = a.x, f[1] = a.y, f[2] = a.z, f[3] = a.w, f[4] = b.x, f[5] = b.y, f[6] = b.z, f[7] = b.w;
}

NVB200_DEVICE uint32_t abs_bits(float x) { return __float_as_uint(x) & 0x7FFFFFFFu; }
NVB200_DEVICE uint32_t amax8(const float (&f)[8]) {
  uint32_t a = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) a = max(a, abs_bits(f[i]));
  return a;
}

// Row u (token u / hkv, head u % hkv) is held by a group of LPR lanes; lanes at or past D / 8 hold nothing.
template <typename T, int FMT, int LPR>
__global__ void __launch_bounds__(kQuantThreads) store_quant_kernel(const __grid_constant__ StoreQuantArgs a) {
  const int j = threadIdx.x % LPR;
  const bool on = 8 * j < a.c.d;
  const uint32_t step = gridDim.x * (kQuantThreads / LPR);
  const uint32_t first = blockIdx.x * (kQuantThreads / LPR) + threadIdx.x / LPR;
  // Every lane of a warp runs the same number of rounds: the shuffles below are over whole warps.
  for (uint32_t base = first - threadIdx.x % 32 / LPR; base < a.rows; base += step) {
    const uint32_t u = base + threadIdx.x % 32 / LPR;
    int64_t slot = -1;
    uint32_t t = 0, h = 0;
    if (u < a.rows) {
      t = u / static_cast<uint32_t>(a.c.hkv), h = u - t * a.c.hkv;
      slot = load_slot(a.slots, a.slot64, t);
      if (slot < -1 || slot >= a.c.num_slots) {
        if (j == 0) set_status(a.c.status, NVB200_STATUS_BAD_SLOT);
        slot = -1;
      }
    }
    float k[8] = {}, v[8] = {};
    if (slot >= 0 && on) {
      load8(reinterpret_cast<const T *>(a.key) + t * a.key_stride + static_cast<int64_t>(h) * a.c.d + 8 * j, k);
      load8(reinterpret_cast<const T *>(a.value) + t * a.value_stride + static_cast<int64_t>(h) * a.c.d + 8 * j, v);
    }
    uint32_t ka = amax8(k), va = amax8(v);
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) {
      ka = max(ka, __shfl_xor_sync(0xffffffffu, ka, o));
      va = max(va, __shfl_xor_sync(0xffffffffu, va, o));
    }
    if (slot < 0) continue;
    const RowScale ks = row_scale<FMT>(ka), vs = row_scale<FMT>(va);
    if (on) {
      const int64_t off = (slot * a.c.hkv + h) * a.c.d + 8 * j;
      *reinterpret_cast<uint2 *>(a.c.k + off) = quantise8<FMT>(k, ks);
      *reinterpret_cast<uint2 *>(a.c.v + off) = quantise8<FMT>(v, vs);
    }
    if (j == 0) {
      const int64_t si = scale_index(a.c, slot, h);
      a.c.k_scale[si] = ks.scale;
      a.c.v_scale[si] = vs.scale;
    }
  }
}

// Rows that the vector kernel does not take (D not a multiple of 8 or above 256, addresses not 16-byte aligned): one
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

template <typename T, int FMT> int launch_store_quant(const StoreQuantArgs &a, bool vec, cudaStream_t s) {
  if (!vec) {
    store_quant_any_kernel<T, FMT><<<grid_for(2ll * a.rows, kQuantThreads / 32, 8), kQuantThreads, 0, s>>>(a);
    return launch_status();
  }
  const int lanes = a.c.d / 8;
  const int lpr = lanes <= 8 ? 8 : (lanes <= 16 ? 16 : 32);
  const int grid = grid_for(a.rows, kQuantThreads / lpr, 8);
  if (lpr == 8) store_quant_kernel<T, FMT, 8><<<grid, kQuantThreads, 0, s>>>(a);
  else if (lpr == 16) store_quant_kernel<T, FMT, 16><<<grid, kQuantThreads, 0, s>>>(a);
  else store_quant_kernel<T, FMT, 32><<<grid, kQuantThreads, 0, s>>>(a);
  return launch_status();
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
  uint32_t units;  // tokens * heads
  int hq, heads;   // heads = hq + 2 hkv
  float eps;
  QuantCache c;
};

template <int D, int FMT>
__global__ void __launch_bounds__(kQuantThreads) qknr_quant_kernel(const __grid_constant__ QknrQuantArgs a) {
  constexpr int HALF = D / 2, LPH = D / 16;
  const int j = threadIdx.x % LPH, in_warp = threadIdx.x % 32 / LPH;
  const uint32_t step = gridDim.x * (kQuantThreads / LPH);
  for (uint32_t base = blockIdx.x * (kQuantThreads / LPH) + threadIdx.x / 32 * (32 / LPH); base < a.units; base += step) {
    const uint32_t u = base + in_warp;
    const bool live = u < a.units;
    const uint32_t t = live ? u / static_cast<uint32_t>(a.heads) : 0;
    const int head = live ? static_cast<int>(u - t * a.heads) : 0;
    const bool is_q = head < a.hq, is_v = head >= a.hq + a.c.hkv;
    const int h = is_q ? head : (is_v ? head - a.hq - a.c.hkv : head - a.hq);
    const __nv_bfloat16 *x = (is_q ? a.q + t * a.q_stride : (is_v ? a.v + t * a.v_stride : a.k + t * a.k_stride)) +
                             static_cast<int64_t>(h) * D;
    uint4 xa = make_uint4(0, 0, 0, 0), xb = xa;
    int64_t slot = -1;
    if (live) {
      xa = __ldg(reinterpret_cast<const uint4 *>(x + 8 * j));
      xb = __ldg(reinterpret_cast<const uint4 *>(x + HALF + 8 * j));
      if (!is_q) slot = __ldg(a.slots + t);
    }
    if (slot < -1 || slot >= a.c.num_slots) {
      if (j == 0) set_status(a.c.status, NVB200_STATUS_BAD_SLOT);
      slot = -1;
    }
    float x1[8], x2[8];
    unpack8(xa, x1);
    unpack8(xb, x2);
    float ss = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(x1[i], x1[i], ss);
#pragma unroll
    for (int i = 0; i < 8; ++i) ss = fmaf(x2[i], x2[i], ss);
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (live && !is_v) {
      int64_t pos = __ldg(a.positions + t);
      if (pos < 0 || pos >= a.num_positions) {
        if (j == 0) set_status(a.c.status, NVB200_STATUS_BAD_POSITION);
        pos = 0;
      }
      const float *cs = a.cos_sin + pos * a.cs_stride;
      float c[8], sn[8];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const float4 cc = __ldg(reinterpret_cast<const float4 *>(cs + 8 * j) + i);
        const float4 s4 = __ldg(reinterpret_cast<const float4 *>(cs + HALF + 8 * j) + i);
        c[4 * i] = cc.x, c[4 * i + 1] = cc.y, c[4 * i + 2] = cc.z, c[4 * i + 3] = cc.w;
        sn[4 * i] = s4.x, sn[4 * i + 1] = s4.y, sn[4 * i + 2] = s4.z, sn[4 * i + 3] = s4.w;
      }
      uint32_t w1[4], w2[4];
      load_w8((is_q ? a.q_w : a.k_w) + 8 * j, w1);
      load_w8((is_q ? a.q_w : a.k_w) + HALF + 8 * j, w2);
      const float rstd = rsqrtf(ss / static_cast<float>(D) + a.eps);
      float y1[8], y2[8];
      norm_rope8(x1, x2, rstd, w1, w2, c, sn, y1, y2);
      xa = pack8(y1), xb = pack8(y2);
      __nv_bfloat16 *o = is_q ? a.q_out + (static_cast<int64_t>(t) * a.hq + h) * D
                              : (a.k_out ? a.k_out + (static_cast<int64_t>(t) * a.c.hkv + h) * D : nullptr);
      if (o) {
        *reinterpret_cast<uint4 *>(o + 8 * j) = xa;
        *reinterpret_cast<uint4 *>(o + HALF + 8 * j) = xb;
      }
    }
    unpack8(xa, x1);
    unpack8(xb, x2);
    uint32_t am = max(amax8(x1), amax8(x2));
#pragma unroll
    for (int o = LPH / 2; o > 0; o >>= 1) am = max(am, __shfl_xor_sync(0xffffffffu, am, o));
    if (slot < 0) continue;
    const RowScale rs = row_scale<FMT>(am);
    uint8_t *row = (is_v ? a.c.v : a.c.k) + (slot * a.c.hkv + h) * D;
    *reinterpret_cast<uint2 *>(row + 8 * j) = quantise8<FMT>(x1, rs);
    *reinterpret_cast<uint2 *>(row + HALF + 8 * j) = quantise8<FMT>(x2, rs);
    if (j == 0) (is_v ? a.c.v_scale : a.c.k_scale)[scale_index(a.c, slot, h)] = rs.scale;
  }
}

template <int FMT> int launch_qknr_quant(const QknrQuantArgs &a, cudaStream_t s) {
  const int lph = a.c.d / 16;
  const int grid = grid_for(a.units, kQuantThreads / lph, 8);
  switch (a.c.d) {
    case 64: qknr_quant_kernel<64, FMT><<<grid, kQuantThreads, 0, s>>>(a); break;
    case 128: qknr_quant_kernel<128, FMT><<<grid, kQuantThreads, 0, s>>>(a); break;
    case 256: qknr_quant_kernel<256, FMT><<<grid, kQuantThreads, 0, s>>>(a); break;
    default: return NVB200_ERR_UNSUPPORTED;
  }
  return launch_status();
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

// A warp takes 32 consecutive packed rows at a time: each lane looks up one row's slot (one search per token, not one
// per head), then the warp copies the 32 tokens, the LPR lanes of a group one head's row at a time.
template <typename T, int FMT, int LPR>
__global__ void __launch_bounds__(kQuantThreads) load_quant_kernel(const __grid_constant__ LoadQuantArgs a) {
  constexpr int RPW = 32 / LPR;
  const int lane = threadIdx.x & 31, j = lane % LPR, grp = lane / LPR;
  const bool vec_on = 8 * j < a.c.d;
  const int64_t warps = static_cast<int64_t>(gridDim.x) * (kQuantThreads / 32);
  const int rows_in_token = a.c.hkv;
  for (int64_t t0 = (static_cast<int64_t>(blockIdx.x) * (kQuantThreads / 32) + threadIdx.x / 32) * 8; t0 < a.total;
       t0 += warps * 8) {
    const int n = static_cast<int>(min(static_cast<int64_t>(8), a.total - t0));
    int64_t mine = -1;
    if (lane < n) {
      mine = slot_of_row(a, t0 + lane);
      if (mine == -2) set_status(a.c.status, NVB200_STATUS_BAD_SLOT);
    }
    for (int r = grp; r < n * rows_in_token + grp; r += RPW) {  // every group the same number of rounds
      const int rr = min(r, n * rows_in_token - 1);
      const int i = rr / rows_in_token, h = rr - i * rows_in_token;
      const int64_t slot = __shfl_sync(0xffffffffu, mine, i);
      if (r >= n * rows_in_token || !vec_on) continue;
      const int64_t dst = ((t0 + i) * a.c.hkv + h) * a.c.d + 8 * j;
      float k[8] = {}, v[8] = {};
      if (slot >= 0) {
        const int64_t src = (slot * a.c.hkv + h) * a.c.d + 8 * j;
        const uint2 kw = __ldg(reinterpret_cast<const uint2 *>(a.c.k + src));
        const uint2 vw = __ldg(reinterpret_cast<const uint2 *>(a.c.v + src));
        const int64_t si = scale_index(a.c, slot, h);
        const float ks = __ldg(a.c.k_scale + si), vs = __ldg(a.c.v_scale + si);
        code_values8<FMT>(kw, k);
        code_values8<FMT>(vw, v);
#pragma unroll
        for (int e = 0; e < 8; ++e) k[e] *= ks, v[e] *= vs;
      } else if (slot == -1 && !a.zero_rest) {
        continue;
      }
      store8(static_cast<T *>(a.key) + dst, k);
      store8(static_cast<T *>(a.value) + dst, v);
    }
  }
}

// D not a multiple of 8 or above 256, or an address that is not 16-byte aligned: one warp per row of one tensor.
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

template <typename T, int FMT> int launch_load_quant(const LoadQuantArgs &a, bool vec, cudaStream_t s) {
  if (!vec) {
    load_quant_any_kernel<T, FMT>
        <<<grid_for(2 * a.total * a.c.hkv, kQuantThreads / 32, 8), kQuantThreads, 0, s>>>(a);
    return launch_status();
  }
  const int lanes = a.c.d / 8;
  const int lpr = lanes <= 8 ? 8 : (lanes <= 16 ? 16 : 32);
  const int grid = grid_for(a.total, 8 * (kQuantThreads / 32), 8);
  if (lpr == 8) load_quant_kernel<T, FMT, 8><<<grid, kQuantThreads, 0, s>>>(a);
  else if (lpr == 16) load_quant_kernel<T, FMT, 16><<<grid, kQuantThreads, 0, s>>>(a);
  else load_quant_kernel<T, FMT, 32><<<grid, kQuantThreads, 0, s>>>(a);
  return launch_status();
}

template <typename T> int launch_load_fmt(const LoadQuantArgs &a, int fmt, bool vec, cudaStream_t s) {
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
  const bool vec = a.c.d % 8 == 0 && a.c.d <= 256 && aligned16(key) && aligned16(value) &&
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
  a.units = static_cast<uint32_t>(q->num_tokens * heads), a.hq = q->num_q_heads, a.heads = static_cast<int>(heads);
  a.eps = q->eps;
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  return fmt == kCacheE4M3 ? launch_qknr_quant<kCacheE4M3>(a, s) : launch_qknr_quant<kCacheI8>(a, s);
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
  const bool vec = a.c.d % 8 == 0 && a.c.d <= 256 && aligned16(key) && aligned16(value) && aligned16(a.c.k) &&
                   aligned16(a.c.v);
  cudaStream_t s = reinterpret_cast<cudaStream_t>(stream);
  if (dtype == NVB200_BF16) return launch_load_fmt<__nv_bfloat16>(a, fmt, vec, s);
  if (dtype == NVB200_F16) return launch_load_fmt<__half>(a, fmt, vec, s);
  return launch_load_fmt<float>(a, fmt, vec, s);
}
