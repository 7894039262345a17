// Pages of 16 tokens that carry their own scale (TSB200_KV_FP8_PAGE): 16 * d e4m3 codes (K [16][d], V [d][16]) and, behind them, 16 bytes
// whose first four are the scale of the page and head, a power of two 2^e with kPageExpMin <= e <= kPageExpMax.
#pragma once
#include "common.cuh"

namespace tsb {

// The range keeps 2^(e_K) q K and the quotients of two pages' V scales far inside fp32: values below 448 * 2^-40 lose bits, values above
// 448 * 2^40 saturate.
constexpr int kPageExpMin = -40, kPageExpMax = 40;
__host__ __device__ constexpr int page_record_bytes(int d) { return 16 * d + 16; }

// Smallest e with amax <= 448 * 2^e (448 = 1.75 * 2^8), clamped.  amax >= 0; zero and subnormal numbers end at the lower end.
__device__ __forceinline__ int page_exponent(float amax) {
  const int e = (int)((__float_as_uint(amax) + 0x1fffffu) >> 23) - 127 - 8;     // one more where the fraction is above 1.75
  return min(max(e, kPageExpMin), kPageExpMax);
}
__device__ __forceinline__ float exp2_int(int e) { return __uint_as_float((unsigned)(e + 127) << 23); }
// Exponent of a stored scale (a page that was never written holds zero).
__device__ __forceinline__ int scale_exponent(float s) { return min(max((int)(__float_as_uint(s) >> 23) - 127, kPageExpMin), kPageExpMax); }

}  // namespace tsb
