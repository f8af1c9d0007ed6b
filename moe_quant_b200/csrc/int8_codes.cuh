// 8-bit codes of rows of numbers: scale = max|x| / 127, code = round_half_even(127 x / max|x|).
#pragma once

#include <math_constants.h>

#include "common.cuh"

namespace mq {

// code = round_half_even(127 x / top).  x * (127 / top) is formed and rounded to an integer in one fused step, by adding 1.5 * 2^23; the
// one rounding in front, that of 127 / top, moves it by at most 127 * 2^-24 = 7.6e-6 of a code.  Where the fraction lies that near to the
// middle m of two codes, the sign of 2 m top - 254 x decides.  It comes out exactly: 254 x is a pair of fp32 numbers (one, for 16-bit
// types), and 2 m top, a product of 8 and 24 bits, agrees with it in its first 15 bits at least, so that the fused difference
// has no more than 24.
// Among 16-bit values exact ties are common (half of all rows of bf16 have some in every 256 values, where the largest is even), and
// nothing else comes near a middle: with significands of b bits, 127 x / top keeps a relative distance of 2^-(2b-3) / 1.02 or more, 2^-19.03
// for fp16.  So x * (127 / top), which is off by 3 * 2^-24 of its leading bit at most, is rounded to twenty bits first: ties then are
// ties, nothing else is (8 + 3 < 32 / 1.02 in units of 2^-24), and the sum with 1.5 * 2^23 rounds them to even.  No branch.
constexpr float TO_INTEGER = 12582912.0f;
constexpr float NEAR_MIDDLE = 0.49999f;

template <typename T>
struct alignas(8 * sizeof(T)) Eight { T v[8]; };

// the eight values as fp32, from whole words (taken one by one, halves of words cost several instructions each)
__device__ __forceinline__ void to_floats(const Eight<float>& a, float (&x)[8]) {
#pragma unroll
  for (int j = 0; j < 8; ++j) x[j] = a.v[j];
}
__device__ __forceinline__ void to_floats(const Eight<__nv_bfloat16>& a, float (&x)[8]) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(a.v);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    x[2 * j] = __uint_as_float(w[j] << 16);
    x[2 * j + 1] = __uint_as_float(w[j] & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void to_floats(const Eight<__half>& a, float (&x)[8]) {
  const __half2* w = reinterpret_cast<const __half2*>(a.v);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 f = __half22float2(w[j]);
    x[2 * j] = f.x;
    x[2 * j + 1] = f.y;
  }
}

__device__ __forceinline__ float max3_abs_nan(float a, float b, float c) {   // NaN if one is
  float v;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(v) : "f"(a), "f"(b), "f"(c));
  return v;
}

// the largest |x| as bits, NaN above infinity above all numbers
__device__ __forceinline__ uint32_t largest_bits(const Eight<float>& a) {
  const float m = max3_abs_nan(max3_abs_nan(a.v[0], a.v[1], a.v[2]), max3_abs_nan(a.v[3], a.v[4], a.v[5]), max3_abs_nan(a.v[6], a.v[7], 0.0f));
  return __float_as_uint(m) & 0x7FFFFFFFu;
}
template <typename T, typename T2>
__device__ __forceinline__ uint32_t largest_bits_16(const Eight<T>& a) {
  const T2* p = reinterpret_cast<const T2*>(a.v);
  const T2 m = __hmax2_nan(__hmax2_nan(__habs2(p[0]), __habs2(p[1])), __hmax2_nan(__habs2(p[2]), __habs2(p[3])));
  return __float_as_uint(to_float(__hmax_nan(m.x, m.y))) & 0x7FFFFFFFu;
}
__device__ __forceinline__ uint32_t largest_bits(const Eight<__nv_bfloat16>& a) { return largest_bits_16<__nv_bfloat16, __nv_bfloat162>(a); }
__device__ __forceinline__ uint32_t largest_bits(const Eight<__half>& a) { return largest_bits_16<__half, __half2>(a); }

// the code of x, given the integer r next to x * inv and `off` = x * inv - r, which is nearly 1/2 or -1/2
__device__ __forceinline__ float decide(float x, float top, float r, float off) {
  const float step = off < 0.0f ? -1.0f : 1.0f;       // the other candidate is r + step
  const float p = 254.0f * x, p_low = __fmaf_rn(254.0f, x, -p);
  // beyond the middle in the direction of `step`?
  const float e = (p_low - __fmaf_rn(2.0f * r + step, top, -p)) * step;
  const bool odd = (__float_as_uint(r + TO_INTEGER) & 1u) != 0;
  return e > 0.0f || (e == 0.0f && odd) ? r + step : r;
}

__device__ __forceinline__ uint2 low_bytes(const float (&r)[8]) {
  uint32_t b[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) b[j] = __float_as_uint(r[j]);
  return make_uint2(__byte_perm(__byte_perm(b[0], b[1], 0x0040), __byte_perm(b[2], b[3], 0x0040), 0x5410),
                    __byte_perm(__byte_perm(b[4], b[5], 0x0040), __byte_perm(b[6], b[7], 0x0040), 0x5410));
}

// The codes of eight values, four to a word, where one lies next to a middle, is no number, or the row is lifted.  Out of line: sixteen copies of it in a
// kernel would not fit the instruction cache beside the rest.
template <typename T>
__device__ __noinline__ uint2 careful_codes(Eight<T> a, float top, float inv, float lift) {
  if (inv == 0.0f) return make_uint2(0, 0);   // an infinity or a NaN in the row, and here
  float r[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const float x = to_float(a.v[j]) * lift, n = __fmaf_rn(x, inv, TO_INTEGER) - TO_INTEGER, off = __fmaf_rn(x, inv, -n);
    r[j] = (fabsf(off) > NEAR_MIDDLE ? decide(x, top, n, off) : n) + TO_INTEGER;
  }
  return low_bytes(r);
}

// What a row's largest |x| (as bits) makes of it.  A row with an infinity or a NaN has the scale NaN and codes of zero.
struct RowCodes {
  float scale, top, inv;     // inv is zero where all codes are
  float careful_from;        // distance from an integer from which careful_codes decides
  float lift;                // 2^60 or 2^-60 for rows whose 127 / top or 254 top would overflow (exact in the row's own type; fp16 never needs it)
  __device__ __forceinline__ explicit RowCodes(uint32_t bits) {
    const bool whole = bits < 0x7F800000u;
    top = __uint_as_float(bits);
    scale = whole ? top / 127.0f : CUDART_NAN_F;
    const bool some = whole && top > 0.0f;
    lift = top < 0x1p-100f ? 0x1p60f : top > 0x1p100f ? 0x1p-60f : 1.0f;
    top *= lift;
    inv = some ? 127.0f / top : 0.0f;
    careful_from = !whole || lift != 1.0f ? -1.0f : NEAR_MIDDLE;
  }
  template <typename T>
  __device__ __forceinline__ uint2 of(const Eight<T>& a) const {
    float r[8], x[8];
    to_floats(a, x);
    if constexpr (sizeof(T) == 2) {
      if (careful_from < 0.0f) return careful_codes(a, top, inv, lift);
#pragma unroll
      for (int j = 0; j < 8; ++j)
        r[j] = __uint_as_float((__float_as_uint(x[j] * inv) + 8u) & ~15u) + TO_INTEGER;
    } else {
      float off[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        r[j] = __fmaf_rn(x[j], inv, TO_INTEGER);
        off[j] = __fmaf_rn(x[j], inv, TO_INTEGER - r[j]);
      }
      const float far = max3_abs_nan(max3_abs_nan(off[0], off[1], off[2]), max3_abs_nan(off[3], off[4], off[5]), max3_abs_nan(off[6], off[7], 0.0f));
      if (!(far <= careful_from)) return careful_codes(a, top, inv, lift);
    }
    return low_bytes(r);
  }
};

// Eight values from k on of a row of K; zeros behind its end.  VEC: K is a multiple of 8 and rows start on boundaries of eight values.
template <bool VEC, typename S>
__device__ __forceinline__ Eight<S> eight_of(const S* row, int k, int K) {
  Eight<S> a;
  if (VEC) {
    if (k < K) a = *reinterpret_cast<const Eight<S>*>(row + k);
    else a = Eight<S>{};
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) a.v[j] = k + j < K ? row[k + j] : from_float<S>(0.0f);
  }
  return a;
}

}  // namespace mq
