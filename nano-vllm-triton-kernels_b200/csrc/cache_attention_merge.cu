// Second step of the even-share forms of nvb200_cache_attention: block (c - 1, .) merges the records of the unit that the start
// of CTA c's range is the first to cut, in the order of the CTAs (so results do not depend on timing). Launched to start
// while the first kernel finishes. A record: per row o[D] unnormalised, m, l, M, flag (see cache_attention.cu for m, l, M).
//
// Latency is all of it (a few hundred records of a few KB): the first kernel leaves the plan, one 48-byte line per block, and
// a thread has the records of four CTAs in flight.
#include "cache_attention.cuh"

namespace nvb200 {
namespace {

constexpr int kMergeThreads = 256;

template <int CT, int D>
__global__ void __launch_bounds__(kMergeThreads)
    cache_attention_merge_kernel(const __grid_constant__ CacheAttnParams p, int block_rows) {
  using C = CacheType<CT>;
  constexpr int kPer = D / 4;                        // threads per row
  constexpr int kBlockRows = kMergeThreads / kPer;   // rows of a block
  const int c = blockIdx.x + 1;
  const int r = blockIdx.y * kBlockRows + threadIdx.x / kPer, d = threadIdx.x % kPer * 4;
  grid_dependency_wait();  // every block: none ends before the first kernel has
  CutInfo x;
  {
    const uint4 *from = reinterpret_cast<const uint4 *>(p.cuts + c);
    uint4 *to = reinterpret_cast<uint4 *>(&x);
    to[0] = __ldcg(from), to[1] = __ldcg(from + 1), to[2] = __ldcg(from + 2);
  }
  if (x.parts == 0) return;
  const int h = x.unit / x.blocks, row0 = (x.unit - h * x.blocks) * block_rows;
  if (r >= min(block_rows, p.rows - row0)) return;
  const int64_t rec_floats = static_cast<int64_t>(block_rows) * (D + 4);
  const float *row = p.records + r * (D + 4);
  float m = -INFINITY, M = -INFINITY, l = 0.f, flag = 0.f, y[4] = {};
  for (int k0 = 0; k0 < x.parts; k0 += 4) {
    float4 s[4], o[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      s[i] = make_float4(-INFINITY, 0.f, -INFINITY, 0.f), o[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (k0 + i < x.parts) {
        const float *w = row + record_slot(c - 1 + k0 + i, x.unit_u, x.T, x.G) * rec_floats;
        s[i] = __ldcg(reinterpret_cast<const float4 *>(w + D)), o[i] = __ldcg(reinterpret_cast<const float4 *>(w + d));
      }
    }
    float mx = m, Mx = M;
#pragma unroll
    for (int i = 0; i < 4; ++i) mx = fmaxf(mx, s[i].x), Mx = fmaxf(Mx, s[i].z);
    const float mu = mx == -INFINITY ? 0.f : mx, Mu = Mx == -INFINITY ? 0.f : Mx;
    const float al = exp2f(m - mu), ao = exp2f(M - Mu);
    l *= al, y[0] *= ao, y[1] *= ao, y[2] *= ao, y[3] *= ao;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float a = exp2f(s[i].z - Mu);
      l = fmaf(exp2f(s[i].x - mu), s[i].y, l), flag = fmaxf(flag, s[i].w);
      y[0] = fmaf(a, o[i].x, y[0]), y[1] = fmaf(a, o[i].y, y[1]), y[2] = fmaf(a, o[i].z, y[2]), y[3] = fmaf(a, o[i].w, y[3]);
    }
    m = mx, M = Mx;
  }
  const int row_all = row0 + r, qi = row_all / p.group, gq = row_all - qi * p.group;
  const float f = l == 0.f ? 0.f : (C::kQuant ? exp2f(M - m) : 1.f) / l;
  Columns<4> more{};
  if (CT != kI8 && flag != 0.f && qi < x.drafts)
    more = nonfinite_sum<CT, 4>(p, p.block_table ? p.block_table + x.b * p.bt_stride : nullptr, x.b, h, qi, d, x.L - x.drafts,
                                x.drafts);
  uint16_t out[4];
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const float v = (qi < x.drafts ? y[k] * f : 0.f) + more.v[k];
    out[k] = (C::kQuant ? p.q_is_f16 : CT == kF16) ? __half_as_ushort(__float2half_rn(v))
                                                   : __bfloat16_as_ushort(__float2bfloat16_rn(v));
  }
  uint16_t *to = static_cast<uint16_t *>(p.out) + ((static_cast<int64_t>(x.b) * p.n + qi) * p.hq + h * p.group + gq) * D + d;
#pragma unroll
  for (int k = 0; k < 4; ++k) to[k] = out[k];
}

template <int CT, int D> int launch_merge(const CacheAttnParams &p, int block_rows, int grid, cudaStream_t s) {
  const int rows = block_rows < p.rows ? block_rows : p.rows, per = kMergeThreads / (D / 4);
  return launch_ex(cache_attention_merge_kernel<CT, D>, dim3(grid - 1, (rows + per - 1) / per), dim3(kMergeThreads), 0, s, 1,
                   true, p, block_rows);
}

}  // namespace

int launch_cache_attention_merge(const CacheAttnParams &p, int ct, int head_dim, int block_rows, int grid, cudaStream_t s) {
  if (grid <= 1) return NVB200_OK;  // one CTA cuts nothing
#define NVB200_MERGE(CT) \
  (head_dim == 64 ? launch_merge<CT, 64>(p, block_rows, grid, s) : launch_merge<CT, 128>(p, block_rows, grid, s))
  switch (ct) {
    case kBf16: return NVB200_MERGE(kBf16);
    case kF16: return NVB200_MERGE(kF16);
    case kE4M3: return NVB200_MERGE(kE4M3);
    default: return NVB200_MERGE(kI8);
  }
#undef NVB200_MERGE
}

}  // namespace nvb200
