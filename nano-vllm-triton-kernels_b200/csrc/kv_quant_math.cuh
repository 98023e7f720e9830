// The row quantiser of the 8-bit KV cache, shared by the kernels that write one (kv_quant.cu).
//
// A row is one token of one KV head; a = max|x| over it.
//   e4m3: scale = 2^E with E the smallest integer >= -126 for which a <= 448 * 2^E; code = x * 2^-E rounded to e4m3.
//     A power of two, because the scaling is then exact: each code is ONE rounding of its element (half a step of
//     2^-4 relative at most), and e4m3 being a floating format, up to one binade of unused headroom costs no precision.
//   int8: scale = d / 127 with d = max(a, 127 * 2^-126); code = 127 x / d rounded half to even, as in exact arithmetic.
//   A row that holds an infinity or NaN gets scale NaN and codes 0, so it reads back as NaN throughout.
#pragma once

#include "common.cuh"

namespace nvb200 {
namespace {

enum { kCacheE4M3 = 0, kCacheI8 = 1 };

// Two fp32 values (|x| <= 448 here) to e4m3, lo in the low byte, round to nearest even.
NVB200_DEVICE uint32_t pack_e4m3x2(float lo, float hi) {
  uint16_t r;
  asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
  return r;
}

struct RowScale {
  float scale;  // what is stored (NaN for a row that is not finite)
  float mul;    // e4m3: 2^-E. int8: 127 (times 2^-8 for rows above 2^100, so that 127 x stays finite)
  float den;    // int8: d, times the same factor
  float quot;   // int8: 127 / d rounded (at most 2^126: finite)
  bool finite;
};

// amax_bits: the fp32 bits of max|x| (compared as integers, so infinities and NaNs win over every finite value).
template <int FMT> NVB200_DEVICE RowScale row_scale(uint32_t amax_bits) {
  RowScale r;
  r.finite = amax_bits < 0x7F800000u;
  if constexpr (FMT == kCacheE4M3) {
    // a = 1.f * 2^e; 448 = 1.75 * 2^8, so E = e - 8, or e - 7 when the fraction is above .75.
    int E = static_cast<int>(amax_bits >> 23) - 127 - 8 + ((amax_bits & 0x7FFFFFu) > 0x600000u ? 1 : 0);
    E = E < -126 ? -126 : E;
    r.scale = __uint_as_float(static_cast<uint32_t>(E + 127) << 23);
    r.mul = __uint_as_float(static_cast<uint32_t>(127 - E) << 23);
    r.den = r.quot = 1.f;
  } else {
    const float d = fmaxf(__uint_as_float(amax_bits), 127.f * 1.17549435e-38f);
    r.scale = __fdiv_rn(d, 127.f);
    const float h = d > 1.2676506e30f ? 0.00390625f : 1.f;  // 2^100, 2^-8
    r.mul = 127.f * h;
    r.den = d * h;
    r.quot = __fdiv_rn(127.f, d);
  }
  if (!r.finite) r.scale = __uint_as_float(0x7FC00000u);
  return r;
}

// int8: the code of exact arithmetic, in the low byte. p: 127 x / d to within an eighth. The code's magnitude is n = floor(|p|)
// or n + 1, by the sign of 127 |x| - (n + 1/2) d: the product is taken as hi + lo, exactly, and next to the middle the
// difference of hi and (n + 1/2) d is one fp32 number (its unit is 2^-25 of d or more), so the sum's sign is the true one.
NVB200_DEVICE uint32_t exact_code(float x, float p, const RowScale &r) {
  const float ax = fabsf(x), n = floorf(fabsf(p));
  const float hi = __fmul_rn(ax, r.mul), lo = __fmaf_rn(ax, r.mul, -hi);
  const float side = __fadd_rn(__fmaf_rn(-(n + 0.5f), r.den, hi), lo);
  const int k = static_cast<int>(n);
  const int code = side > 0.f || (side == 0.f && (k & 1)) ? k + 1 : k;
  return static_cast<uint32_t>(x < 0.f ? -code : code);
}
// Sums of this and a number of magnitude below 2^22 are rounded at the unit, half to even, and have it in the low bits.
constexpr float kCodeMagic = 12582912.f;  // 1.5 * 2^23
// A product x * (127 / d) as near as this to the middle between two codes says nothing of the code: its own rounding and the
// quotient's move a value of at most 127 by less than 3 * 127 * 2^-24.
constexpr float kCodeNear = 127.f * 2.384185791015625e-7f;  // 127 * 2^-22

// Eight elements to eight codes, element 0 in the lowest byte.
template <int FMT> NVB200_DEVICE uint2 quantise8(const float (&x)[8], const RowScale &r) {
  uint2 out;
  if (!r.finite) return make_uint2(0u, 0u);
  if constexpr (FMT == kCacheE4M3) {
    out.x = pack_e4m3x2(x[0] * r.mul, x[1] * r.mul) | pack_e4m3x2(x[2] * r.mul, x[3] * r.mul) << 16;
    out.y = pack_e4m3x2(x[4] * r.mul, x[5] * r.mul) | pack_e4m3x2(x[6] * r.mul, x[7] * r.mul) << 16;
  } else {
    // x times the row's 127 / d, rounded, where no product lies near the middle between two codes; else the exact codes.
    uint32_t c[8];
    float off = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const float p = __fmul_rn(x[i], r.quot), m = __fadd_rn(p, kCodeMagic);
      off = fmaxf(off, fabsf(__fsub_rn(p, __fsub_rn(m, kCodeMagic))));
      c[i] = __float_as_uint(m);
    }
    if (off > 0.5f - kCodeNear) {
#pragma unroll
      for (int i = 0; i < 8; ++i) c[i] = exact_code(x[i], __fmul_rn(x[i], r.quot), r);
    }
    out.x = __byte_perm(__byte_perm(c[0], c[1], 0x0040), __byte_perm(c[2], c[3], 0x0040), 0x5410);
    out.y = __byte_perm(__byte_perm(c[4], c[5], 0x0040), __byte_perm(c[6], c[7], 0x0040), 0x5410);
  }
  return out;
}

// One element (the kernels for rows that no wider access fits).
template <int FMT> NVB200_DEVICE uint8_t quantise1(float x, const RowScale &r) {
  if (!r.finite) return 0;
  if constexpr (FMT == kCacheE4M3)
    return static_cast<uint8_t>(pack_e4m3x2(x * r.mul, 0.f) & 0xFFu);
  else
    return static_cast<uint8_t>(exact_code(x, __fmul_rn(x, r.quot), r) & 0xFFu);
}

// Two e4m3 codes (low byte first) as two fp16 values: exact, every e4m3 value is an fp16 value.
NVB200_DEVICE uint32_t e4m3x2_to_f16x2(uint16_t w) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(w));
  return r;
}

// One code as fp32 (exact).
template <int FMT> NVB200_DEVICE float code_value(uint8_t c) {
  if constexpr (FMT == kCacheE4M3) {
    const uint32_t h = e4m3x2_to_f16x2(c);
    return __half2float(__ushort_as_half(static_cast<unsigned short>(h & 0xFFFFu)));
  } else {
    return static_cast<float>(static_cast<int8_t>(c));
  }
}

// Eight codes as fp32.
template <int FMT> NVB200_DEVICE void code_values8(const uint2 &w, float (&f)[8]) {
  const uint32_t u[2] = {w.x, w.y};
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    if constexpr (FMT == kCacheE4M3) {
#pragma unroll
      for (int k = 0; k < 2; ++k) {
        const uint32_t h = e4m3x2_to_f16x2(static_cast<uint16_t>(u[i] >> (16 * k)));
        f[4 * i + 2 * k] = __half2float(__ushort_as_half(static_cast<unsigned short>(h & 0xFFFFu)));
        f[4 * i + 2 * k + 1] = __half2float(__ushort_as_half(static_cast<unsigned short>(h >> 16)));
      }
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) f[4 * i + k] = static_cast<float>(static_cast<int8_t>(u[i] >> (8 * k)));
    }
  }
}

}  // namespace
}  // namespace nvb200
