// Second step of the even-share forms of nvb200_cache_attention: block c - 1 looks at the end between the ranges of CTAs
// c - 1 and c, and if it is the first that cuts its unit, merges the unit's records, in the order of the CTAs (so results do
// not depend on timing). Launched to start while the first kernel finishes: the plan needs the lengths only.
// A record: per row o[D] unnormalised, m, l, M, flag (see cache_attention.cu for m, l, M).
#include "cache_attention.cuh"

namespace nvb200 {
namespace {

constexpr int kMergeThreads = 256;
constexpr int kMergeRows = 16;  // of a block

template <int CT, int D>
__global__ void __launch_bounds__(kMergeThreads)
    cache_attention_merge_kernel(const __grid_constant__ CacheAttnParams p, int tile_keys, int block_rows, int min_tiles,
                                 int grid) {
  using C = CacheType<CT>;
  const int T = total_work(p, tile_keys, block_rows), G = active_ctas(T, grid, min_tiles);
  const int c = blockIdx.x + 1;
  const bool there = T > 0 && c < G;
  const int at = there ? range_start(c, T, G) : 0;
  Segment g;
  if (there) g = find_segment(p, at, at + 1, tile_keys, block_rows);
  grid_dependency_wait();  // the records are complete; no block ends before the first kernel has
  if (!there || g.t0 == 0 || range_start(c - 1, T, G) > g.unit_u) return;  // no cut, or not the unit's first
  const int last = range_owner(g.unit_u + g.s.tiles - 1, T, G);
  const int h = g.unit / g.s.blocks, row0 = (g.unit - h * g.s.blocks) * block_rows;
  const int nrows = min(block_rows, p.rows - row0);
  const int64_t rec_floats = static_cast<int64_t>(block_rows) * (D + 4);
  constexpr int kPer = D / 4;  // threads per row
  for (int e = threadIdx.x; e < kMergeRows * kPer; e += kMergeThreads) {
    const int r = blockIdx.y * kMergeRows + e / kPer, d = e % kPer * 4;
    if (r >= nrows) break;
    const float *row = p.records + r * (D + 4);
    float mx = -INFINITY, Mx = -INFINITY;
    for (int k = c - 1; k <= last; ++k) {
      const float4 x = __ldcg(reinterpret_cast<const float4 *>(row + record_slot(k, g.unit_u, T, G) * rec_floats + D));
      mx = fmaxf(mx, x.x), Mx = fmaxf(Mx, x.z);
    }
    const float mu = mx == -INFINITY ? 0.f : mx, Mu = Mx == -INFINITY ? 0.f : Mx;
    float l = 0.f, flag = 0.f, y[4] = {};
    for (int k = c - 1; k <= last; ++k) {
      const float *w = row + record_slot(k, g.unit_u, T, G) * rec_floats;
      const float4 x = __ldcg(reinterpret_cast<const float4 *>(w + D)), o = __ldcg(reinterpret_cast<const float4 *>(w + d));
      const float ao = exp2f(x.z - Mu);
      l = fmaf(exp2f(x.x - mu), x.y, l), flag = fmaxf(flag, x.w);
      y[0] = fmaf(ao, o.x, y[0]), y[1] = fmaf(ao, o.y, y[1]), y[2] = fmaf(ao, o.z, y[2]), y[3] = fmaf(ao, o.w, y[3]);
    }
    const int row_all = row0 + r, qi = row_all / p.group, gq = row_all - qi * p.group;
    const float f = l == 0.f ? 0.f : (C::kQuant ? exp2f(Mx - mx) : 1.f) / l;
    uint16_t out[4];
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      float v = qi < g.s.drafts ? y[k] * f : 0.f;
      if (CT != kI8 && flag != 0.f && qi < g.s.drafts)
        v = add_nonfinite<CT>(p, p.block_table ? p.block_table + g.b * p.bt_stride : nullptr, g.b, h, qi, d + k,
                              g.s.L - g.s.drafts, g.s.L, g.s.drafts, v);
      out[k] = (C::kQuant ? p.q_is_f16 : CT == kF16) ? __half_as_ushort(__float2half_rn(v))
                                                     : __bfloat16_as_ushort(__float2bfloat16_rn(v));
    }
    uint16_t *to = static_cast<uint16_t *>(p.out) + ((static_cast<int64_t>(g.b) * p.n + qi) * p.hq + h * p.group + gq) * D + d;
#pragma unroll
    for (int k = 0; k < 4; ++k) to[k] = out[k];
  }
}

template <int CT, int D>
int launch_merge(const CacheAttnParams &p, int tile_keys, int block_rows, int min_tiles, int grid, cudaStream_t s) {
  const int rows = block_rows < p.rows ? block_rows : p.rows;
  return launch_ex(cache_attention_merge_kernel<CT, D>, dim3(grid - 1, (rows + kMergeRows - 1) / kMergeRows),
                   dim3(kMergeThreads), 0, s, 1, true, p, tile_keys, block_rows, min_tiles, grid);
}

}  // namespace

int launch_cache_attention_merge(const CacheAttnParams &p, int ct, int head_dim, int tile_keys, int block_rows,
                                 int min_tiles, int grid, cudaStream_t s) {
  if (grid <= 1) return NVB200_OK;  // one CTA cuts nothing
#define NVB200_MERGE(CT)                                                                                  \
  (head_dim == 64 ? launch_merge<CT, 64>(p, tile_keys, block_rows, min_tiles, grid, s)                    \
                  : launch_merge<CT, 128>(p, tile_keys, block_rows, min_tiles, grid, s))
  switch (ct) {
    case kBf16: return NVB200_MERGE(kBf16);
    case kF16: return NVB200_MERGE(kF16);
    case kE4M3: return NVB200_MERGE(kE4M3);
    default: return NVB200_MERGE(kI8);
  }
#undef NVB200_MERGE
}

}  // namespace nvb200
