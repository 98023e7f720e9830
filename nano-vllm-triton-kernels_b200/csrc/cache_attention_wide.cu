// The wide form of nvb200_cache_attention (cache_attention.cu has the mathematics): up to 128 query rows of one KV head
// per CTA, on the 5th-generation tensor cores. For trees and chains whose tokens x group fill more than the 16 rows of
// the warp-level kernel, which would read and convert the keys once per 16 rows.
//
// A CTA takes 128 rows (token i, head of the group) of one (sequence, KV head) and a run of its keys, in tiles of 64:
//   * warp 4, the producer: K and V tiles by TMA from the paged cache (one box per page run), into a ring;
//   * 8-bit caches: warps 6 to 9 convert the landed codes to fp16 operand tiles (exact), and bring the row scales;
//   * warp 5, one lane: S = Q K^T (128 x 64, fp32, one of two TMEM buffers), later O += P V (128 x D, fp32, TMEM), with
//     P read from TMEM, where it overwrites its S;
//   * warps 0-3, one thread per row: the running softmax. The maximum that weights refer to moves only when a row exceeds
//     it by 2^8, so O is rarely rescaled; the sums are fp32. fp16 weights are held 2^kWeightUp times as large (why: see
//     cache_attention.cu), at most 2^14.
// 16-bit caches: two CTAs share an SM (113 KB of shared memory and 256 TMEM columns each), the one computes while the other
// waits; 8-bit caches: one, with deeper rings. The grid is what the GPU holds at once, and each CTA takes an even share of the batch's tiles (cache_attention.cuh); the
// roles walk the CTA's segments independently, so the loads of a segment start while the one before is finished.
// Waits are bounded; a CTA that gives up sets NVB200_STATUS_WAIT_TIMEOUT and lets its copies land.
#include <algorithm>
#include <atomic>
#include <cmath>

#include "cache_attention.cuh"
#include "tcgen05.cuh"

namespace nvb200 {
namespace {

constexpr int kTileKeys = 64;
constexpr int kTileRows = 128;
constexpr int kTmemCols = 256;  // S: 2 x 64, O: up to 128
constexpr int kColO = 128;
constexpr int kPrefetch = 5;  // tiles ahead of the one being loaded that are brought into the L2
constexpr float kWeightUp = 6.f;
constexpr int kMinTiles = 4;  // of a CTA, where there are too few for all

template <int CT, int D> struct Wide {
  static constexpr bool kQuant = CacheType<CT>::kQuant;
  static constexpr int kThreads = kQuant ? 320 : 192;
  // CTAs per SM. 16-bit caches: two, of 113 KB of shared memory each (228 KB, 1 KB of it reserved per CTA), so that nothing
  // that holds TMEM fits beside two and a CTA never waits for TMEM that another kernel's CTA holds. 8-bit caches: one with
  // deep rings; at two per SM the four converting warps beside the softmax leave too few registers, and spilled ones go to
  // the L2 (the L1 is all shared memory here).
  static constexpr int kCtas = kQuant ? 1 : 2;
  static constexpr int kSmem = kQuant ? 227 * 1024 : 113 * 1024;
  static constexpr int kConvWarps = 4;  // one per scheduler
  static constexpr int kQBytes = kTileRows * D * 2;
  static constexpr int kOpBytes = kTileKeys * D * 2;  // a K or V operand tile
  static constexpr int kRawBytes = kTileKeys * D;     // the same as codes
  // Ring depths: K and V operand tiles, pairs of raw tiles, slots of per-key information.
  static constexpr int NK = kQuant ? 2 : (D == 128 ? 2 : 4);
  static constexpr int NV = kQuant ? 2 : (D == 128 ? 3 : 4);
  static constexpr int NR = kQuant ? 6 : 0;
  static constexpr int kSlots = 8;  // >= NK + 3: a slot is rewritten only after its tile's softmax
  static constexpr int kOffK = kQBytes;
  static constexpr int kOffV = kOffK + NK * kOpBytes;
  static constexpr int kOffRaw = kOffV + NV * kOpBytes;
  static constexpr int kOffRawScale = kOffRaw + NR * 2 * kRawBytes;          // [NR][2][64] fp32: K scales, V scales
  // [kSlots] of [3][64] fp32 (K scales, V scales, log2 bounds), 2 x largest and 2 x smallest bound
  static constexpr int kOffScale = kOffRawScale + NR * 2 * kTileKeys * 4;
  static constexpr int kSlotBytes = kQuant ? 3 * kTileKeys * 4 + 16 : 0;
  static constexpr int kOffHdr = kOffScale + kSlots * kSlotBytes;
  static_assert(kOffHdr + 1024 <= kSmem, "a CTA's shared memory");
};

struct WideMaps {
  CUtensorMap k, v;
};

struct WideParams {
  CacheAttnParams a;
  int box_rows;  // tokens per TMA box: gcd(block_size, 64), 8 to 64
  float sign;    // of softmax_scale; scale_log2 is its magnitude here
};

NVB200_DEVICE void tma_load_4d(uint32_t dst, const CUtensorMap *map, int c0, int c1, int c2, int c3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}

// Brings a box into the L2.
NVB200_DEVICE void tma_prefetch_4d(const CUtensorMap *map, int c0, int c1, int c2, int c3) {
  asm volatile("cp.async.bulk.prefetch.tensor.4d.L2.global.tile [%0, {%1, %2, %3, %4}];" ::"l"(map), "r"(c0), "r"(c1),
               "r"(c2), "r"(c3)
               : "memory");
}

// D[tmem] (+)= A[tmem] B[shared], 16-bit operands.
NVB200_DEVICE void tc_mma_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 64 consecutive fp32 columns of this thread's TMEM lane.
NVB200_DEVICE void tmem_ld64(uint32_t taddr, float (&v)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31]), "=f"(v[32]), "=f"(v[33]), "=f"(v[34]), "=f"(v[35]), "=f"(v[36]), "=f"(v[37]), "=f"(v[38]), "=f"(v[39]), "=f"(v[40]), "=f"(v[41]), "=f"(v[42]), "=f"(v[43]), "=f"(v[44]), "=f"(v[45]), "=f"(v[46]), "=f"(v[47]), "=f"(v[48]), "=f"(v[49]), "=f"(v[50]), "=f"(v[51]), "=f"(v[52]), "=f"(v[53]), "=f"(v[54]), "=f"(v[55]), "=f"(v[56]), "=f"(v[57]), "=f"(v[58]), "=f"(v[59]), "=f"(v[60]), "=f"(v[61]), "=f"(v[62]), "=f"(v[63])
      : "r"(taddr)
      : "memory");
}

// 16 or 32 consecutive 32-bit columns of this thread's TMEM lane (tmem_st_wait before another thread may rely on them).
NVB200_DEVICE void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15};" ::"r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(taddr)
               : "memory");
}
NVB200_DEVICE void tmem_st32(uint32_t taddr, const float (&v)[32]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};" ::"f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]), "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]), "f"(v[16]), "f"(v[17]), "f"(v[18]), "f"(v[19]), "f"(v[20]), "f"(v[21]), "f"(v[22]), "f"(v[23]), "f"(v[24]), "f"(v[25]), "f"(v[26]), "f"(v[27]), "f"(v[28]), "f"(v[29]), "f"(v[30]), "f"(v[31]), "r"(taddr)
               : "memory");
}
NVB200_DEVICE void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// max(a, b, c) as one instruction; a NaN operand is ignored, as by fmaxf.
NVB200_DEVICE float fmax3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// (a, b) *= (c, d) in one packed instruction, each lane rounded as the scalar product.
NVB200_DEVICE void mul2(float &a, float &b, float c, float d) {
  const float2 r = f32x2_unpack(f32x2_mul(f32x2_pack(a, b), f32x2_pack(c, d)));
  a = r.x, b = r.y;
}

// Swizzled position of 16-byte chunk c (0-7) of 128-byte row r in a tile of such rows.
NVB200_DEVICE uint32_t swz128(int r, int c) { return static_cast<uint32_t>(r * 128 + ((c ^ (r & 7)) << 4)); }

template <int CT, int D>
__global__ void __launch_bounds__(Wide<CT, D>::kThreads, Wide<CT, D>::kCtas)
    cache_attention_wide_kernel(const __grid_constant__ WideParams wp, const __grid_constant__ WideMaps maps) {
  using W = Wide<CT, D>;
  using C = CacheType<CT>;
  launch_dependents();     // a dependent launched early waits for this grid before reading its output
  grid_dependency_wait();  // this grid may itself have been launched early
  extern __shared__ __align__(1024) uint8_t smem[];
  const CacheAttnParams &p = wp.a;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const uint32_t base = smem_addr(smem);
  const int T = total_work(p, kTileKeys, kTileRows);  // by every warp
  const int G = active_ctas(T, gridDim.x, kMinTiles);
  zero_uncovered_rows(p, D, kTileKeys, kTileRows, blockIdx.x, gridDim.x, tid, W::kThreads);
  const bool work = T > 0 && static_cast<int>(blockIdx.x) < G;
  const int u0 = work ? range_start(blockIdx.x, T, G) : 0, u1 = work ? range_start(blockIdx.x + 1, T, G) : 0;
  Segment seg;
  seg.n = 0;
  if (work) seg = find_segment(p, u0, u1, kTileKeys, kTileRows);
  if (tid == 0) write_cut(p, blockIdx.x, seg, T, G);
  if (!work) return;
  auto next = [&]() { next_segment(seg, p, u1, kTileKeys, kTileRows); };

  const uint32_t hdr = base + W::kOffHdr;
  const uint32_t b_kfull = hdr, b_kempty = hdr + 32, b_vfull = hdr + 64, b_vempty = hdr + 96;  // up to 4 each
  const uint32_t b_sfull = hdr + 128, b_pready = hdr + 144, b_q = hdr + 168;
  const uint32_t b_pv = hdr + 184;  // 2, like b_sfull and b_pready by tile parity: the softmax may be two P V ahead of one
  const uint32_t b_rfull = hdr + 200, b_rempty = hdr + 264;              // up to 8 each
  const uint32_t live_slot = hdr + 328, raw_live = hdr + 392;            // 64-bit words: up to 8 each
  uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(smem + W::kOffHdr + 456);
  const uint32_t failed = hdr + 460;  // flag
  // Word q % 4 holds q + 1 once segment q of the CTA's had an infinity or NaN taken out of V. V of a tile is converted once
  // the P V two tiles before it is done, so at most two segments ahead of the one that the softmax finishes.
  const uint32_t dirty = hdr + 464;
  auto dirty_word = [&](int q) { return dirty + 4 * (q & 3); };

  if (tid == 0) {
    for (int i = 0; i < W::NK; ++i) mbar_init(b_kfull + 8 * i, W::kQuant ? W::kConvWarps : 1), mbar_init(b_kempty + 8 * i, 1);
    for (int i = 0; i < W::NV; ++i) mbar_init(b_vfull + 8 * i, W::kQuant ? W::kConvWarps : 1), mbar_init(b_vempty + 8 * i, 1);
    for (int i = 0; i < 2; ++i) mbar_init(b_sfull + 8 * i, 2), mbar_init(b_pready + 8 * i, 4), mbar_init(b_pv + 8 * i, 2);
    mbar_init(b_q, 4);
    for (int i = 0; i < W::NR; ++i) mbar_init(b_rfull + 8 * i, 1), mbar_init(b_rempty + 8 * i, W::kConvWarps);
    st_shared_u32(failed, 0u);
    for (int i = 0; i < 4; ++i) st_shared_u32(dirty + 4 * i, 0u);
    fence_mbar_init();
  }
  if (warp == 5) tmem_alloc(smem_addr(tmem_slot), kTmemCols);
  if (warp == 4 && lane < 2) prefetch_tmap(lane ? &maps.v : &maps.k);
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;

  auto give_up = [&]() {
    set_status(p.status, NVB200_STATUS_WAIT_TIMEOUT);
    st_shared_u32(failed, 1u);
  };
  // One lane polls: a warp-wide poll is 32 requests to the barrier, and the warps that wait would slow those that work.
  auto wait1 = [&](uint32_t bar, uint32_t parity) {
    return mbar_try_wait(bar, parity) || (ld_shared_u32(failed) == 0u && mbar_wait_bounded(bar, parity));
  };
  auto wait = [&](uint32_t bar, uint32_t parity) {
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    int ok = 1;
    if (lane == 0) ok = wait1(bar, parity) ? 1 : 0;
    return __shfl_sync(0xffffffffu, ok, 0) != 0;  // and orders the lanes behind lane 0's acquire
  };
  auto arrive = [&](uint32_t bar) {
    __syncwarp();
    if (lane == 0) mbar_arrive(bar);
  };

  const bool masked = p.mask != nullptr || p.causal;
  // Of the current segment: first tile's first key, end of its keys; keys before the new tokens; every row sees the keys
  // below `open`; whether a row may not see a key that others see (V must then be finite: see nonfinite_sum).
  auto first_key = [&]() { return seg.t0 * kTileKeys; };
  auto end_key = [&]() { return min(static_cast<int64_t>(seg.s.L), static_cast<int64_t>(seg.t0 + seg.n) * kTileKeys); };
  auto context = [&]() { return seg.s.L - seg.s.drafts; };
  auto open_below = [&]() { return masked ? max(context(), 0) : seg.s.L; };
  auto hides_keys = [&]() { return p.mask ? seg.s.drafts > 0 : (p.causal && seg.s.drafts > 1); };
  auto table_of = [&]() { return p.block_table ? p.block_table + seg.b * p.bt_stride : nullptr; };

  if (warp == 4) {
    // ---------------------------------------------------------------- producer: lane r has box r of every tile
    const int R = wp.box_rows, boxes = kTileKeys / R;
    const uint32_t row_bytes = D * C::kBytes;
    int i = 0;  // tile of the CTA
    bool go = true;
    for (; seg.n > 0 && go; next()) {
    const int32_t *bt = table_of();
    const int b = seg.b, h = seg.unit / seg.s.blocks, js = first_key(), je = static_cast<int>(end_key());
    auto block_at = [&](int t) {
      const int j = js + t * kTileKeys + lane * R;
      return lane < boxes && j < je ? (bt ? __ldg(bt + page_of(p, j)) : b) : -1;
    };
    auto prefetch = [&](int t, int block) {
      if (block < 0 || block >= p.num_blocks) return;
      const int j = js + t * kTileKeys + lane * R, tok = j - page_of(p, j) * p.block_size;
#pragma unroll
      for (int u = 0; u < (W::kQuant ? 1 : D / 64); ++u) {
        tma_prefetch_4d(&maps.k, 64 * u, tok, h, block);
        tma_prefetch_4d(&maps.v, 64 * u, tok, h, block);
      }
    };
    int blk = block_at(0), far = -1;
    for (int t = 0; t < seg.n; ++t, ++i) {
      const int j = js + t * kTileKeys + lane * R;
      const bool mine = lane < boxes && j < je;
      const bool ok = mine && blk >= 0 && blk < p.num_blocks;
      if (mine && !ok) set_status(p.status, NVB200_STATUS_BAD_SLOT);
      const int here = blk, page = mine ? page_of(p, j) : 0;
      const int tok = j - page * p.block_size;
      if (t + 1 < seg.n) blk = block_at(t + 1);
      // The ring holds two or three tiles, less than HBM's latency wants: tiles further ahead start their way into the L2.
      if (t == 0) {
        for (int a = 1; a <= kPrefetch; ++a) prefetch(a, a < seg.n ? block_at(a) : -1);
      } else {
        prefetch(t + kPrefetch, far);
      }
      far = t + 1 + kPrefetch < seg.n ? block_at(t + 1 + kPrefetch) : -1;
      // Bit k: key k of the tile exists and its page can be followed.
      unsigned long long bits = 0;
      if (ok) {
        const int n = min(R, je - j);
        bits = (n >= 64 ? ~0ull : (1ull << n) - 1ull) << (lane * R & 63);
      }
      const uint32_t lo = __reduce_or_sync(0xffffffffu, static_cast<uint32_t>(bits));
      const uint32_t hi = __reduce_or_sync(0xffffffffu, static_cast<uint32_t>(bits >> 32));
      const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, ok)) * R * row_bytes;
      if constexpr (W::kQuant) {
        const int st = i % W::NR;
        go = wait(b_rempty + 8 * st, ((i / W::NR) & 1) ^ 1);
        if (!go) break;
        if (lane == 0) {
          st_shared_u32(raw_live + 8 * st, lo), st_shared_u32(raw_live + 8 * st + 4, hi);
          mbar_arrive_expect_tx(b_rfull + 8 * st, 2 * (bytes + bytes / D * 4));
        }
        __syncwarp();
        if (ok) {
          const uint32_t dst = base + W::kOffRaw + st * 2 * W::kRawBytes + lane * R * row_bytes;
          tma_load_4d(dst, &maps.k, 0, tok, h, here, b_rfull + 8 * st);
          tma_load_4d(dst + W::kRawBytes, &maps.v, 0, tok, h, here, b_rfull + 8 * st);
          const int64_t si = (static_cast<int64_t>(here) * p.hkv + h) * p.block_size + tok;
          const uint32_t sc = base + W::kOffRawScale + st * 2 * kTileKeys * 4 + lane * R * 4;
          bulk_g2s(sc, p.k_scale + si, R * 4, b_rfull + 8 * st);
          bulk_g2s(sc + kTileKeys * 4, p.v_scale + si, R * 4, b_rfull + 8 * st);
        }
      } else {
        const int sk = i % W::NK, sv = i % W::NV, slot = i % W::kSlots;
        go = wait(b_kempty + 8 * sk, ((i / W::NK) & 1) ^ 1);
        if (!go) break;
        if (lane == 0) {
          st_shared_u32(live_slot + 8 * slot, lo), st_shared_u32(live_slot + 8 * slot + 4, hi);
          mbar_arrive_expect_tx(b_kfull + 8 * sk, bytes);
        }
        __syncwarp();
        if (ok) {
#pragma unroll
          for (int u = 0; u < D / 64; ++u)
            tma_load_4d(base + W::kOffK + sk * W::kOpBytes + u * kTileKeys * 128 + lane * R * 128, &maps.k, 64 * u, tok,
                        h, here, b_kfull + 8 * sk);
        }
        go = wait(b_vempty + 8 * sv, ((i / W::NV) & 1) ^ 1);
        if (!go) {
          if (lane == 0) mbar_wait_bounded(b_kfull + 8 * sk, (i / W::NK) & 1);  // its K tile lands
          break;
        }
        if (lane == 0) mbar_arrive_expect_tx(b_vfull + 8 * sv, bytes);
        __syncwarp();
        if (ok) {
#pragma unroll
          for (int u = 0; u < D / 64; ++u)
            tma_load_4d(base + W::kOffV + sv * W::kOpBytes + u * kTileKeys * 128 + lane * R * 128, &maps.v, 64 * u, tok,
                        h, here, b_vfull + 8 * sv);
        }
      }
    }
    }
    const int issued = i;
    if (!go) {
      // Gave up: let the copies in flight land before the shared memory is released.
      if (lane == 0) {
        give_up();
        if constexpr (W::kQuant) {
          for (int i = max(0, issued - W::NR); i < issued; ++i) mbar_wait_bounded(b_rfull + 8 * (i % W::NR), (i / W::NR) & 1);
        } else {
          for (int i = max(0, issued - W::NK); i < issued; ++i) mbar_wait_bounded(b_kfull + 8 * (i % W::NK), (i / W::NK) & 1);
          for (int i = max(0, issued - W::NV); i < issued; ++i) mbar_wait_bounded(b_vfull + 8 * (i % W::NV), (i / W::NV) & 1);
        }
      }
      __syncwarp();
    }
  } else if (warp == 5) {
    // ---------------------------------------------------------------- MMA issuer
    // The whole warp runs the loop and one lane issues: inside a divergent branch the compiler would move every operand
    // of every instruction to a uniform register one by one.
    constexpr uint32_t fmt = C::kBf16Mma ? 1u : 0u;
    constexpr uint32_t idesc = (1u << 4) | (fmt << 7) | (fmt << 10) | (static_cast<uint32_t>(kTileRows >> 4) << 24);
    constexpr uint32_t idesc_s = idesc | (static_cast<uint32_t>(kTileKeys >> 3) << 17);
    constexpr uint32_t idesc_o = idesc | (1u << 16) | (static_cast<uint32_t>(D >> 3) << 17);  // V: columns contiguous
    const uint32_t td = __shfl_sync(0xffffffffu, tmem, 0);
    const uint64_t ad = smem_desc(base, 16, 1024, 2);
    auto qk = [&](int i) {
      const int st = i % W::NK;
      if (!wait(b_kfull + 8 * st, (i / W::NK) & 1)) return false;
      tc_fence_after();
      const uint64_t bd = smem_desc(base + W::kOffK + st * W::kOpBytes, 16, 1024, 2);
      const uint32_t d = td + (i & 1) * kTileKeys;
      if (lane == 0) {
#pragma unroll
        for (int k = 0; k < D / 16; ++k)
          tc_mma<false>(d, ad + (k / 4) * (kTileRows * 128 >> 4) + (k % 4) * 2,
                        bd + (k / 4) * (kTileKeys * 128 >> 4) + (k % 4) * 2, idesc_s, k > 0 ? 1u : 0u);
        tc_commit(b_kempty + 8 * st);
        tc_commit(b_sfull + 8 * (i & 1));
        mbar_arrive(b_sfull + 8 * (i & 1));  // orders the tile's per-key information, seen through b_kfull, for the softmax
      }
      __syncwarp();
      return true;
    };
    bool ok = true;
    int i = 0;  // tile of the CTA
    for (int q = 0; seg.n > 0 && ok; next(), ++q) {
      // The segment's query rows are in place, which also says that the softmax is done with O of the segment before.
      ok = wait(b_q, q & 1) && qk(i);
      for (int t = 0; t < seg.n && ok; ++t, ++i) {
        // S of the next tile before this tile's P V: the softmax has it while P V runs. Its buffer's P was consumed by
        // the P V of tile i - 1, issued before it.
        if (t + 1 < seg.n) ok = qk(i + 1);
        const int st = i % W::NV;
        ok = ok && wait(b_pready + 8 * (i & 1), (i >> 1) & 1) && wait(b_vfull + 8 * st, (i / W::NV) & 1);
        if (!ok) break;
        tc_fence_after();
        const uint64_t bd = smem_desc(base + W::kOffV + st * W::kOpBytes, kTileKeys * 128, 1024, 2);
        const uint32_t pa = td + (i & 1) * kTileKeys;
        if (lane == 0) {
#pragma unroll
          for (int k = 0; k < kTileKeys / 16; ++k)
            tc_mma_ts(td + kColO, pa + k * 8, bd + k * (16 * 128 >> 4), idesc_o, (t > 0 || k > 0) ? 1u : 0u);
          tc_commit(b_vempty + 8 * st);
          tc_commit(b_pv + 8 * (i & 1));
          mbar_arrive(b_pv + 8 * (i & 1));  // orders the marks of V's infinities (dirty_word), seen through b_vfull and b_pready
        }
        __syncwarp();
      }
    }
    if (!ok && lane == 0) give_up();
    __syncwarp();
  } else if (warp >= 6) {
    // ---------------------------------------------------------------- converters (8-bit caches)
    if constexpr (W::kQuant) {
      const int ct = tid - 192;  // 0 .. 127; below 64 also the key whose scales this thread brings
      constexpr int kChunks = D / 16;            // 16-byte chunks of a raw row
      constexpr int kRowsPer = 128 / kChunks;    // rows that the 128 threads cover at a time
      const int r8 = (ct & 7) | (ct >> 3) / kChunks * 8, ch = (ct >> 3) % kChunks;
      // Converts a raw tile to an operand tile; rows whose bit of `live` is clear become zeros, and from row `finite` on
      // e4m3's NaN codes too (q: the segment).
      auto convert = [&](int src, int dst, unsigned long long live, int finite, int q) {
        uint4 u[kTileKeys / kRowsPer];  // all loads before the first store
#pragma unroll
        for (int k = 0; k < kTileKeys / kRowsPer; ++k) {
          const int r = k * kRowsPer + r8;
          const int pc = D == 128 ? ch ^ (r & 7) : ch ^ ((r >> 1) & 3);  // TMA's 128- or 64-byte swizzle
          u[k] = *reinterpret_cast<const uint4 *>(smem + src + r * D + pc * 16);
        }
#pragma unroll
        for (int k = 0; k < kTileKeys / kRowsPer; ++k) {
          const int r = k * kRowsPer + r8;
          if (!((live >> r) & 1ull)) u[k] = make_uint4(0u, 0u, 0u, 0u);
          uint32_t *w = &u[k].x;
          if (CT == kE4M3 && r >= finite) {
            uint32_t found = 0;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
              const uint32_t bad = nonfinite_bits<CT>(w[e]);
              w[e] &= ~bad, found |= bad;
            }
            if (found) st_shared_u32(dirty_word(q), q + 1);
          }
          uint4 x, y;
          codes_to_f16<CT>(w[0], x.x, x.y), codes_to_f16<CT>(w[1], x.z, x.w);
          codes_to_f16<CT>(w[2], y.x, y.y), codes_to_f16<CT>(w[3], y.z, y.w);
          uint8_t *to = smem + dst + (ch / 4) * (kTileKeys * 128);
          *reinterpret_cast<uint4 *>(to + swz128(r, 2 * (ch % 4))) = x;
          *reinterpret_cast<uint4 *>(to + swz128(r, 2 * (ch % 4) + 1)) = y;
        }
        fence_proxy_async_smem();
      };
      auto live_of = [&](int st) {
        return static_cast<unsigned long long>(ld_shared_u32(raw_live + 8 * st + 4)) << 32 | ld_shared_u32(raw_live + 8 * st);
      };
      auto convert_k = [&](int i) {
        const int st = i % W::NR, slot = i % W::kSlots, sk = i % W::NK;
        if (!wait(b_rfull + 8 * st, (i / W::NR) & 1) || !wait(b_kempty + 8 * sk, ((i / W::NK) & 1) ^ 1)) return false;
        const unsigned long long live = live_of(st);
        convert(W::kOffRaw + st * 2 * W::kRawBytes, W::kOffK + sk * W::kOpBytes, live, kTileKeys, 0);
        if (ct < kTileKeys) {
          // The key's scales; zeros where it is none (its slot of the raw tile was not loaded).
          const bool is = (live >> ct) & 1ull;
          const float *rsc = reinterpret_cast<const float *>(smem + W::kOffRawScale + st * 2 * kTileKeys * 4);
          const float ks = is ? rsc[ct] : 0.f, vs = is ? rsc[kTileKeys + ct] : 0.f;
          float *sc = reinterpret_cast<float *>(smem + W::kOffScale + slot * W::kSlotBytes);
          sc[ct] = ks, sc[kTileKeys + ct] = vs;
          // Above log2 of the V scale: its exponent + 1, and the largest and smallest of the warp's keys. Rows of zeros (and
          // of less than e4m3 holds of fp32's smallest) have the smallest scale and no say.
          const int ve = static_cast<int>(__float_as_uint(vs) >> 23 & 0xFFu) - 126;
          sc[2 * kTileKeys + ct] = static_cast<float>(ve);
          const int hi = __reduce_max_sync(0xffffffffu, ve), lo = __reduce_min_sync(0xffffffffu, ve <= -125 ? 1 << 10 : ve);
          if (lane == 0)
            sc[3 * kTileKeys + (warp - 6)] = static_cast<float>(hi), sc[3 * kTileKeys + 2 + (warp - 6)] = static_cast<float>(lo);
          if (ct == 0) {
            st_shared_u32(live_slot + 8 * slot, static_cast<uint32_t>(live));
            st_shared_u32(live_slot + 8 * slot + 4, static_cast<uint32_t>(live >> 32));
          }
        }
        arrive(b_kfull + 8 * sk);
        return true;
      };
      // K of the next tile goes before V of this one: its product is wanted first, and V's buffer is only free once P V of
      // the tile before is done.
      bool ok = convert_k(0);
      const int total = u1 - u0;
      int i = 0;
      for (int q = 0; seg.n > 0 && ok; next(), ++q) {
        const bool hides = hides_keys();
        for (int t = 0; t < seg.n; ++t, ++i) {
          if (i + 1 < total) ok = convert_k(i + 1);
          const int st = i % W::NR, sv = i % W::NV;
          ok = ok && wait(b_vempty + 8 * sv, ((i / W::NV) & 1) ^ 1);
          if (!ok) break;
          convert(W::kOffRaw + st * 2 * W::kRawBytes + W::kRawBytes, W::kOffV + sv * W::kOpBytes, live_of(st),
                  hides ? open_below() - (first_key() + t * kTileKeys) : kTileKeys, q);
          arrive(b_vfull + 8 * sv);
          arrive(b_rempty + 8 * st);
        }
      }
      if (!ok) give_up();
    }
  } else {
    // ---------------------------------------------------------------- softmax: thread = row
    bool ok = true;
    int i = 0;  // tile of the CTA
    for (int q = 0; seg.n > 0 && ok; next(), ++q) {
    const int b = seg.b, h = seg.unit / seg.s.blocks, row0 = (seg.unit - h * seg.s.blocks) * kTileRows;
    const int nrows = min(kTileRows, p.rows - row0), drafts = seg.s.drafts, ctx = context();
    const int js = first_key(), je = static_cast<int>(end_key()), open = open_below();
    const bool hides = hides_keys();
    const int32_t *bt = table_of();
    float m = -INFINITY, l = 0.f, M = -INFINITY;
    const int r = row0 + tid, qi_raw = r / p.group;
    const int qi = tid < nrows && qi_raw < drafts ? qi_raw : -1;
    const bool warp_live = __any_sync(0xffffffffu, qi >= 0);
    // The query row into shared memory (128-byte swizzled rows, two sub-tiles of 64 elements at head_dim 128). 8-bit
    // caches: brought to fp16 by an exact power of two (see cache_attention.cu), which the scores give back.
    float rs = p.scale_log2;
    {
      const uint16_t *row = static_cast<const uint16_t *>(p.q) + b * p.q_batch_stride + qi_raw * p.q_token_stride +
                            static_cast<int64_t>(h * p.group + r - qi_raw * p.group) * p.q_head_stride;
      const bool aligned = (reinterpret_cast<uintptr_t>(row) & 15) == 0;
      uint4 u[D / 8];  // the whole row: its loads are in flight together
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        u[c] = make_uint4(0u, 0u, 0u, 0u);
        if (qi >= 0 && aligned) u[c] = __ldg(reinterpret_cast<const uint4 *>(row) + c);
      }
      if (qi >= 0 && !aligned) {
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          uint32_t *w = &u[c].x;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[e] = static_cast<uint32_t>(__ldg(row + 8 * c + 2 * e)) |
                   static_cast<uint32_t>(__ldg(row + 8 * c + 2 * e + 1)) << 16;
        }
      }
      const uint32_t flip = wp.sign < 0.f ? 0x80008000u : 0u;
      float up = 1.f;
      if constexpr (W::kQuant) {
        uint32_t am = 0;  // largest magnitude, as 16-bit patterns (they order like the values)
#pragma unroll
        for (int c = 0; c < D / 8; ++c) {
          const uint32_t w[4] = {u[c].x, u[c].y, u[c].z, u[c].w};
#pragma unroll
          for (int e = 0; e < 4; ++e) am = max(am, max(w[e] & 0x7FFFu, (w[e] >> 16) & 0x7FFFu));
        }
        const float a = p.q_is_f16 ? __half2float(__ushort_as_half(static_cast<unsigned short>(am)))
                                   : __uint_as_float(am << 16);
        const int ex = static_cast<int>(__float_as_uint(a) >> 23);
        if (ex >= 20 && ex < 255) {
          up = __uint_as_float(static_cast<uint32_t>(127 + 13 + 127 - ex) << 23);
          rs = fmaxf(rs * __uint_as_float(static_cast<uint32_t>(ex - 13) << 23), 1.17549435e-38f);  // never 0: rs * -inf
        }
      }
#pragma unroll
      for (int c = 0; c < D / 8; ++c) {
        uint32_t *w = &u[c].x;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          w[e] ^= flip;
          if constexpr (W::kQuant) {
            float x, y;
            if (p.q_is_f16) {
              const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[e]));
              x = f.x, y = f.y;
            } else {
              x = bf16_lo(w[e]), y = bf16_hi(w[e]);
            }
            w[e] = pack_f16x2(x * up, y * up);
          }
        }
        st_shared_v4(base + (c / 8) * (kTileRows * 128) + swz128(tid, c % 8), u[c]);
      }
      fence_proxy_async_smem();
      arrive(b_q);
    }
    // Bit k: this row sees new token rel0 + k (tokens outside [0, n): 0). Warp-wide: the warp reads the mask rows of its
    // tokens one after another, 64 bytes at a time, so that all of a row's bytes come with two loads.
    const int q_lo = __reduce_min_sync(0xffffffffu, qi < 0 ? INT32_MAX : qi), q_hi = __reduce_max_sync(0xffffffffu, qi);
    auto gather = [&](int rel0) {
      unsigned long long mine = 0;
      for (int q0 = q_lo; q0 <= q_hi; q0 += 4) {
        uint32_t lo[4], hi[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint8_t *mr = p.mask + b * p.mask_batch_stride + (q0 + k) * p.mask_row_stride + rel0;
          const int x = rel0 + lane;
          lo[k] = q0 + k <= q_hi && x >= 0 && x < p.n ? __ldg(mr + lane) : 0u;
          hi[k] = q0 + k <= q_hi && x + 32 >= 0 && x + 32 < p.n ? __ldg(mr + lane + 32) : 0u;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t l32 = __ballot_sync(0xffffffffu, lo[k] != 0), h32 = __ballot_sync(0xffffffffu, hi[k] != 0);
          if (qi == q0 + k) mine = static_cast<unsigned long long>(h32) << 32 | l32;
        }
      }
      return mine;
    };
    // Up to 64 new tokens: the row's whole mask, fetched here, while the first tiles are on their way.
    const unsigned long long mask64 = p.mask && p.n <= 64 && je > open ? gather(0) : 0ull;
    const uint32_t lanes = static_cast<uint32_t>(warp) << 21;  // TMEM lane 32 * warp
    float vhi = -INFINITY, vlo = INFINITY;  // over the segment's tiles so far: largest and smallest bound of a V scale
    for (int t = 0; t < seg.n; ++t, ++i) {
      const uint32_t s_addr = tmem + lanes + (i & 1) * kTileKeys;
      const int slot = i % W::kSlots, j0 = js + t * kTileKeys;
      ok = wait(b_sfull + 8 * (i & 1), (i >> 1) & 1);
      if (!ok) break;
      tc_fence_after();
      const uint32_t lo = ld_shared_u32(live_slot + 8 * slot), hi = ld_shared_u32(live_slot + 8 * slot + 4);
      const bool full = (lo & hi) == 0xFFFFFFFFu;
      const bool edge = !full || j0 + kTileKeys > open;
      if constexpr (!W::kQuant) {
        // Rows of V that are no keys become zeros, and infinities and NaN too where a row may not see them.
        if (!full || (hides && j0 + kTileKeys > open)) {
          const int sv = i % W::NV;
          ok = wait(b_vfull + 8 * sv, (i / W::NV) & 1);
          if (!ok) break;
          const int finite = hides ? open - j0 : kTileKeys;  // rows from here on hold new tokens
          for (int c = tid; c < W::kOpBytes / 16; c += kTileRows) {
            const int row = (c >> 3) & (kTileKeys - 1);
            const uint32_t at = base + W::kOffV + sv * W::kOpBytes + c * 16;
            uint4 u = ld_shared_v4(at);
            uint32_t *w = &u.x, change = 0;
            if (!((row < 32 ? lo >> row : hi >> (row - 32)) & 1u)) {
              u = make_uint4(0u, 0u, 0u, 0u), change = 1;
            } else if (row >= finite) {
#pragma unroll
              for (int e = 0; e < 4; ++e) {
                const uint32_t bad = nonfinite_bits<CT>(w[e]);
                w[e] &= ~bad, change |= bad;
              }
              if (change) st_shared_u32(dirty_word(q), q + 1);
            }
            if (change) st_shared_v4(at, u);
          }
          fence_proxy_async_smem();
        }
      }
      if (warp_live) {
        const float4 *sc = reinterpret_cast<const float4 *>(smem + W::kOffScale + slot * W::kSlotBytes);
        uint32_t see_lo = 0xFFFFFFFFu, see_hi = 0xFFFFFFFFu;
        if (edge) {
          unsigned long long see = ~0ull;
          if (j0 + kTileKeys > open) {
            // Keys below `open` are seen, then new token rel0 + k at key k.
            const int rel0 = j0 - ctx;
            if (p.mask) {
              if (p.n > 64) see = gather(rel0);
              else if (rel0 >= 64 || rel0 <= -64) see = 0ull;
              else see = rel0 >= 0 ? mask64 >> rel0 : mask64 << -rel0;
            } else if (p.causal) {
              const int k = qi - rel0 + 1;  // keys 0 .. k - 1 of the tile
              see = k >= 64 ? ~0ull : (k <= 0 ? 0ull : (1ull << k) - 1ull);
            }
            const int before = open - j0;
            if (before > 0) see |= (1ull << before) - 1ull;
          }
          if (qi < 0) see = 0ull;
          see_lo = lo & static_cast<uint32_t>(see), see_hi = hi & static_cast<uint32_t>(see >> 32);
        }
        // Scores of columns c0 .. c0 + CW before the row's factor rs > 0. 8-bit caches read S twice, 32 columns at a
        // time (for the maximum, then for the weights; a third time where row scales lie far apart): a tile's 64 scores beside
        // three numbers per key do not fit the registers of a thread, and what is spilled goes to the L2, the L1 being all
        // shared memory here.
        constexpr int CW = W::kQuant ? 32 : 64;
        float x[CW];
        auto scores = [&](int c0) {
          if constexpr (CW == 32) tmem_ld32(s_addr + c0, x);
          else tmem_ld64(s_addr, x);
          if constexpr (W::kQuant) {
#pragma unroll
            for (int c = 0; c < CW; c += 4) {
              const float4 k4 = sc[c0 / 4 + c / 4];
              mul2(x[c], x[c + 1], k4.x, k4.y);
              mul2(x[c + 2], x[c + 3], k4.z, k4.w);
            }
          }
          if (edge) {
#pragma unroll
            for (int c = 0; c < CW; ++c) {
              const uint32_t see = CW == 64 ? (c < 32 ? see_lo : see_hi) : (c0 ? see_hi : see_lo);
              if (!((see >> (c & 31)) & 1u)) x[c] = -INFINITY;
            }
          }
        };
        float top = -INFINITY;
#pragma unroll 1
        for (int c0 = 0; c0 < kTileKeys; c0 += CW) {
          scores(c0);
          float mx = fmax3(top, x[0], x[1]), mx1 = fmaxf(x[2], x[3]);
#pragma unroll
          for (int c = 4; c < CW; c += 4) mx = fmax3(mx, x[c], x[c + 1]), mx1 = fmax3(mx1, x[c + 2], x[c + 3]);
          top = fmaxf(mx, mx1);
        }
        top *= rs;  // the tile's largest score
        const float mt = fmaxf(m, top);
        // The weights' reference M. While the row scales of V stay within 2^8 of each other it is the running maximum plus
        // the bound of the largest one: no weight exceeds it, and fp16 holds the smallest ones' weights to 2^-23 of them. Once
        // they do not, and in tiles with keys that a row may not see (and must not notice), it is the row's own maximum of
        // score + bound.
        float Mt = M;
        if constexpr (W::kQuant) {
          if (!edge) {
            const float4 bound = sc[3 * kTileKeys / 4];  // largest (two), smallest (two)
            vhi = fmax3(vhi, bound.x, bound.y), vlo = fminf(vlo, fminf(bound.z, bound.w));
          }
          if (!edge && vhi - vlo <= 8.f) {
            Mt = mt + vhi;
          } else if (edge || __any_sync(0xffffffffu, mt + vhi > M + 8.f || M == -INFINITY)) {
#pragma unroll 1
            for (int c0 = 0; c0 < kTileKeys; c0 += CW) {
              scores(c0);
#pragma unroll
              for (int c = 0; c < CW; c += 4) {
                const float4 e4 = sc[(2 * kTileKeys + c0 + c) / 4];
                Mt = fmax3(Mt, fmaf(x[c], rs, e4.x), fmaf(x[c + 1], rs, e4.y));
                Mt = fmax3(Mt, fmaf(x[c + 2], rs, e4.z), fmaf(x[c + 3], rs, e4.w));
              }
            }
          }
        }
        // The references move only when they are exceeded by 8 (a factor 256), or are not set yet.
        const bool move = mt > m + 8.f || m == -INFINITY || (W::kQuant && (Mt > M + 8.f || M == -INFINITY));
        if (__any_sync(0xffffffffu, move)) {
          const float mn = move ? mt : m, Mn = move ? Mt : M;
          const float al = mn == -INFINITY ? 1.f : ex2_approx_ftz(m - mn);
          const float ao = W::kQuant ? (Mn == -INFINITY ? 1.f : ex2_approx_ftz(M - Mn)) : al;
          m = mn, M = Mn;
          l *= al;
          if (t > 0) {
            ok = wait(b_pv + 8 * ((i - 1) & 1), ((i - 1) >> 1) & 1);  // P V of the tile before is done: O is at rest
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int c = 0; c < D; c += 32) {
              float t[32];
              tmem_ld32(tmem + lanes + kColO + c, t);
#pragma unroll
              for (int e = 0; e < 32; ++e) t[e] *= ao;
              tmem_st32(tmem + lanes + kColO + c, t);
            }
          }
        }
        const float mu = m == -INFINITY ? 0.f : m;
        const float up = (C::kBf16Mma ? 0.f : kWeightUp) - mu;
        const float cw = W::kQuant ? ex2_approx_ftz(mu - (M == -INFINITY ? 0.f : M)) : 1.f;
        uint64_t sum0 = 0, sum1 = 0;  // pairs of fp32
#pragma unroll 1
        for (int c0 = 0; c0 < kTileKeys; c0 += CW) {
          if constexpr (W::kQuant) scores(c0);
#pragma unroll
          for (int h0 = 0; h0 < CW; h0 += 32) {
            uint32_t pk[16];
#pragma unroll
            for (int c = 0; c < 32; c += 4) {
              float w[4];
#pragma unroll
              for (int e = 0; e < 4; ++e) w[e] = ex2_approx_ftz(fmaf(x[h0 + c + e], rs, up));
              sum0 = f32x2_add(sum0, f32x2_pack(w[0], w[1])), sum1 = f32x2_add(sum1, f32x2_pack(w[2], w[3]));
              if constexpr (W::kQuant) {
                const float4 v4 = sc[(kTileKeys + c0) / 4 + c / 4];
                mul2(w[0], w[1], v4.x, v4.y), mul2(w[0], w[1], cw, cw);
                mul2(w[2], w[3], v4.z, v4.w), mul2(w[2], w[3], cw, cw);
              }
              pk[c / 2] = C::kBf16Mma ? pack_bf16x2(w[0], w[1]) : pack_f16x2(w[0], w[1]);
              pk[c / 2 + 1] = C::kBf16Mma ? pack_bf16x2(w[2], w[3]) : pack_f16x2(w[2], w[3]);
            }
            if (W::kQuant && edge) {  // 0 times a NaN row scale
              const uint32_t see = c0 ? see_hi : see_lo;
#pragma unroll
              for (int c = 0; c < 16; ++c)
                pk[c] &= ((see >> (2 * c)) & 1u ? 0xFFFFu : 0u) | ((see >> (2 * c + 1)) & 1u ? 0xFFFF0000u : 0u);
            }
            tmem_st16(s_addr + (c0 + h0) / 2, pk);  // over scores that have been read
          }
        }
        const float2 sum = f32x2_unpack(f32x2_add(sum0, sum1));
        l += sum.x + sum.y;
        tmem_st_wait();
      }
      tc_fence_before();
      arrive(b_pready + 8 * (i & 1));
    }
    if (ok) ok = wait(b_pv + 8 * ((i - 1) & 1), ((i - 1) >> 1) & 1);
    if (!ok) break;
    tc_fence_after();

    if constexpr (!W::kQuant) M = m;
    const bool whole = seg.n == seg.s.tiles;
    const bool flagged = ld_shared_u32(dirty_word(q)) == static_cast<uint32_t>(q + 1);
    const int gq = r - qi_raw * p.group;
    const float f = l == 0.f ? 0.f : (W::kQuant ? exp2f(M - m) : 1.f) / l;
    float *rec = p.records + (static_cast<int64_t>(record_slot(blockIdx.x, seg.unit_u, T, G)) * kTileRows + tid) * (D + 4);
    const int64_t row = ((static_cast<int64_t>(b) * p.n + qi_raw) * p.hq + h * p.group + gq) * D;
#pragma unroll
    for (int c = 0; c < D; c += 32) {
      float t[32];
      tmem_ld32(tmem + lanes + kColO + c, t);
      if (tid < nrows && whole) {
#pragma unroll
        for (int e = 0; e < 32; e += 8) {
          float y[8];
#pragma unroll
          for (int k = 0; k < 8; ++k) y[k] = qi < 0 ? 0.f : t[e + k] * f;
          if (CT != kI8 && flagged && qi >= 0) {
            const Columns<8> more = nonfinite_sum<CT, 8>(p, bt, b, h, qi, c + e, ctx, drafts);
#pragma unroll
            for (int k = 0; k < 8; ++k) y[k] += more.v[k];
          }
          uint4 u;
          if (W::kQuant ? p.q_is_f16 : CT == kF16)
            u = make_uint4(pack_f16x2(y[0], y[1]), pack_f16x2(y[2], y[3]), pack_f16x2(y[4], y[5]), pack_f16x2(y[6], y[7]));
          else
            u = pack8(y);
          *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(p.out) + row + c + e) = u;
        }
      } else if (tid < nrows) {
#pragma unroll
        for (int e = 0; e < 32; e += 4)
          *reinterpret_cast<float4 *>(rec + c + e) = make_float4(t[e], t[e + 1], t[e + 2], t[e + 3]);
      }
    }
    if (tid < nrows && !whole) *reinterpret_cast<float4 *>(rec + D) = make_float4(m, l, M, flagged ? 1.f : 0.f);
    tc_fence_before();
    }
    if (!ok) give_up();
  }
  tc_fence_before();
  __syncthreads();  // every MMA, copy and read of this CTA is done
  if (warp == 5) tmem_dealloc(tmem, kTmemCols);
}

// ---------------------------------------------------------------------------------------------------------------
// Host side.

// 4-D map of a cache: {D, token of the block, head, block}, boxes of `box_rows` tokens of one head.
bool make_cache_map(CUtensorMap *map, const void *base, const CacheAttnParams &p, int ct, int D, int box_rows) {
  auto fn = encode_fn();
  if (fn == nullptr) return false;
  const bool quant = ct == kE4M3 || ct == kI8;
  const int64_t eb = quant ? 1 : 2;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(D), static_cast<cuuint64_t>(p.block_size),
                              static_cast<cuuint64_t>(p.hkv), static_cast<cuuint64_t>(p.num_blocks)};
  const int64_t st[3] = {p.tok_stride * eb, p.head_stride * eb, p.blk_stride * eb};
  for (int64_t s : st)
    if (s <= 0 || s >= (int64_t{1} << 40)) return false;
  const cuuint64_t strides[3] = {static_cast<cuuint64_t>(st[0]), static_cast<cuuint64_t>(st[1]),
                                 static_cast<cuuint64_t>(st[2])};
  const cuuint32_t box[4] = {static_cast<cuuint32_t>(quant ? D : 64), static_cast<cuuint32_t>(box_rows), 1, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUtensorMapDataType type = quant ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                         : (ct == kBf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16);
  return fn(map, type, 4, const_cast<void *>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            quant && D == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int64_t wide_units(const CacheAttnParams &p) {
  return static_cast<int64_t>(p.batch) * p.hkv * ((p.rows + kTileRows - 1) / kTileRows);
}

// CTAs: as many as run at once, fewer where the longest possible sequences could not feed them.
int wide_grid(const CacheAttnParams &p, int ct) {
  const int64_t units = wide_units(p), slots = (ct == kE4M3 || ct == kI8 ? 1 : 2) * sm_count();
  const int64_t tiles = (static_cast<int64_t>(p.max_pages) * p.block_size + kTileKeys - 1) / kTileKeys;
  return static_cast<int>(std::max<int64_t>(1, std::min(slots, std::max(units, units * tiles / kMinTiles))));
}

template <int CT, int D> int launch_wide(const WideParams &wp, const WideMaps &maps, cudaStream_t s) {
  static std::atomic<uint64_t> ready{0};  // bit: device whose shared-memory limit is set
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return NVB200_ERR_CUDA;
  if (!(ready.load(std::memory_order_acquire) >> dev & 1)) {
    if (cudaFuncSetAttribute(cache_attention_wide_kernel<CT, D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                             Wide<CT, D>::kSmem) != cudaSuccess) {
      cudaGetLastError();
      return NVB200_ERR_CUDA;
    }
    ready.fetch_or(uint64_t{1} << dev, std::memory_order_release);
  }
  const int grid = wide_grid(wp.a, CT);
  if (int rc = launch_ex(cache_attention_wide_kernel<CT, D>, dim3(grid), dim3(Wide<CT, D>::kThreads), Wide<CT, D>::kSmem, s, 1,
                         false, wp, maps))
    return rc;
  return launch_cache_attention_merge(wp.a, CT, D, kTileRows, grid, s);
}

}  // namespace

bool wide_takes(const CacheAttnParams &p) {
  // Boxes are runs of tokens of one page: 8 rows is the swizzle's period. A zero scale would make masked scores 0 * -inf.
  if (p.block_size % 8 != 0 || p.num_blocks > INT32_MAX || !aligned16(p.out) || !(std::fabs(p.scale_log2) > 1e-30f))
    return false;
  // Row scales (NULL for 16-bit caches) come by bulk copies: whole runs of 8 tokens, so their bases decide the alignment.
  if (!aligned16(p.k_scale) || !aligned16(p.v_scale)) return false;
  // Tiles are counted in 32 bits.
  const int64_t tiles = (static_cast<int64_t>(p.max_pages) * p.block_size + kTileKeys - 1) / kTileKeys;
  return wide_units(p) <= INT32_MAX / std::max<int64_t>(tiles, 1);
}

int64_t wide_workspace_bytes(const CacheAttnParams &p, int ct, int head_dim) {
  return even_share_bytes(wide_grid(p, ct), kTileRows, head_dim);
}

int launch_cache_attention_wide(const CacheAttnParams &p, int ct, int head_dim, void *workspace, cudaStream_t stream) {
  WideParams wp{p, 64, p.scale_log2 < 0.f ? -1.f : 1.f};
  place_workspace(wp.a, workspace, wide_grid(p, ct));
  while (p.block_size % wp.box_rows != 0) wp.box_rows /= 2;
  wp.a.scale_log2 = std::fabs(p.scale_log2);
  WideMaps maps;
  if (!make_cache_map(&maps.k, p.k_cache, p, ct, head_dim, wp.box_rows) ||
      !make_cache_map(&maps.v, p.v_cache, p, ct, head_dim, wp.box_rows))
    return NVB200_ERR_UNSUPPORTED;
  switch (ct) {
    case kBf16: return head_dim == 64 ? launch_wide<kBf16, 64>(wp, maps, stream) : launch_wide<kBf16, 128>(wp, maps, stream);
    case kF16: return head_dim == 64 ? launch_wide<kF16, 64>(wp, maps, stream) : launch_wide<kF16, 128>(wp, maps, stream);
    case kE4M3: return head_dim == 64 ? launch_wide<kE4M3, 64>(wp, maps, stream) : launch_wide<kE4M3, 128>(wp, maps, stream);
    default: return head_dim == 64 ? launch_wide<kI8, 64>(wp, maps, stream) : launch_wide<kI8, 128>(wp, maps, stream);
  }
}

}  // namespace nvb200
