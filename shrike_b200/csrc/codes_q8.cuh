// The codes of 8-bit cache rows: the nearest integer to 127 x / a, of two equally near ones the even, in 32-bit arithmetic.
// Every step is one rounding of its own (no contraction), so that a host compiler gives the same codes as the kernels.
#pragma once
#include <math.h>

#ifdef __CUDACC__
#define SHRIKE_CODES __host__ __device__ __forceinline__
#else
#define SHRIKE_CODES inline
#endif

namespace cacheq8 {

SHRIKE_CODES float rounded_product(float a, float b) {
#ifdef __CUDA_ARCH__
  return __fmul_rn(a, b);
#else
  return a * b;
#endif
}
SHRIKE_CODES float rounded_sum(float a, float b) {
#ifdef __CUDA_ARCH__
  return __fadd_rn(a, b);
#else
  return a + b;
#endif
}

// The code of x in a row of largest magnitude a (2^-100 ... 2^100), `inv` = 127 / a rounded.  The first guess q is off by one at
// most, next to a border between two codes; the distance d = 127 x - q a tells, by 2 |d| against a, and it is formed exactly:
//   127 x = h + l and q a = p + e, products and what their rounding left out;
//   h - p is exact: for q = 0 there is nothing to subtract, for |q| > 1 the two lie within a factor of two of one another, and for
//     |q| = 1 they do too, or h lies just below a / 2 in the binade of a / 2, whose steps hold the difference (where a / 2 is a
//     power of two, 127 / a is exact and no guess of one lies below the border);
//   l - e is exact: both are multiples of x's last place, and neither is larger than 2^8 of them;
//   near a border 2 |h - p| - a is exact (within a factor of two again), so the last addition has the right sign, and gives zero
//     on the border alone; far from one it is far larger than l - e.
SHRIKE_CODES int code_of(float x, float a, float inv) {
  const float q = rintf(rounded_product(x, inv));
  const float h = rounded_product(127.f, x), l = fmaf(127.f, x, -h);
  const float p = rounded_product(q, a), e = fmaf(q, a, -p);
  const float d = rounded_sum(h, -p), rest = rounded_sum(l, -e);
  const float over = rounded_sum(rounded_sum(2.f * fabsf(d), -a), 2.f * (d > 0.f ? rest : -rest));
  const int code = static_cast<int>(q);
  return over > 0.f || (over == 0.f && (code & 1)) ? code + (d > 0.f ? 1 : -1) : code;
}

}  // namespace cacheq8
