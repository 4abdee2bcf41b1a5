// What the two files of attention over 8-bit pages share: their arguments, and how weights and codes are formed.
#pragma once
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stddef.h>

// The arguments, packed by the caller: a call with thirty arguments costs the host more to make
// than to launch.
struct ShrikeAttentionQ8 {
  const void* q;
  const void* k_codes;
  const float* k_scales;
  const void* v_codes;
  const float* v_scales;
  const int* block_table;
  const int* q_start;
  const int* ctx_len;
  const int* seq_of_token;
  void* out;
  float* scratch;   // of the few-rows form, or of split portions
  int* arrivals;
  int* status;
  cudaStream_t stream;
  int max_blocks, dtype, num_tokens, num_seqs, num_heads, num_kv_heads, page_size, num_pages, window;
  int has_single, has_portions, max_q_len;   // has_single: of the portions' kernel, entries of one token are left out
  int others;                                // longer entries belong to another kernel
  int splits, cluster, tiles;
  float scale;
};
// As the caller packs them: fourteen addresses, sixteen 32-bit integers and a 32-bit number side by side.
static_assert(offsetof(ShrikeAttentionQ8, max_blocks) == 14 * 8 && offsetof(ShrikeAttentionQ8, scale) == 14 * 8 + 16 * 4, "packed");

#ifdef __CUDACC__
namespace q8 {

constexpr float LOG2E = 1.4426950408889634f;
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ unsigned pack_half(float lo, float hi) {
  const __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const unsigned*>(&h);
}
// Two codes, biased by 128 in bytes 0, 1 (or 2, 3) of `biased`, as float16: byte b under 0x64 is 1024 + b.
template <int SELECT> __device__ __forceinline__ unsigned codes_to_half(unsigned biased) {
  const unsigned raw = __byte_perm(biased, 0x64646464u, SELECT), offset = 0x64806480u;   // 1152 twice
  const __half2 h = __hsub2(*reinterpret_cast<const __half2*>(&raw), *reinterpret_cast<const __half2*>(&offset));
  return *reinterpret_cast<const unsigned*>(&h);
}
// F's range: sums of 2^(z - m) stay within float32 for any count of keys, and weights of 2^-19 of the largest above its least.
// The largest scale that a store leaves is below 2^122: a weight is then below 2^15 if the base does not lag, and where a step's
// largest scale is above F's range it does not.
constexpr int LEAST_EXPONENT = -93, MOST_EXPONENT = 107, SCALE_BITS = 8;
constexpr float BASE_LAG = 6.0f;   // float16's largest power of two is 2^15: 2^9 times 2^6
// A magnitude's bits (which order as the magnitudes do), 0 for infinities and NaN.
__device__ __forceinline__ unsigned finite_bits(float x) {
  const unsigned bits = __float_as_uint(x) & 0x7fffffffu;
  return bits < 0x7f800000u ? bits : 0u;
}
// x 2^d for d <= 0, also where 2^d is below float32's range: a sum under the least exponent F (a row whose values were all zeros
// so far) becomes one under a large one, 2^200 smaller.  Outputs need not go that far: they are nothing beside the values that F
// rose for.
__device__ __forceinline__ float scale_sum(float x, float d) { return x * fast_exp2(fmaxf(d, -126.f)) * fast_exp2(fminf(d + 126.f, 0.f)); }

// 2^e for e in [-126, 127].
__device__ __forceinline__ float power_of_two(int e) { return __int_as_float((e + 127) << 23); }

}  // namespace q8
#endif
