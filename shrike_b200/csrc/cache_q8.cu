// Keys and values in 8 bits: written into their pages, with and without the rotation in front, and read back.
//
// A row x of a head's D elements is kept as codes c_i = round(127 x_i / a) (half to even), a = max |x_i|, and one float32
// scale s = a / 127 (rounded once): x_i is about c_i s.  A row of zeros has scale 0; a row that holds an infinity or a NaN has
// scale NaN and codes 0, so that whatever reads it gets NaN and nothing else.  Pages: codes int8 [pages, page size, kv heads,
// D], scales float32 [pages, kv heads, page size]: the attention reads the scales of one head, and a page's lie together.
#include "cache_q8_call.cuh"
#include "codes_q8.cuh"
#include "common.cuh"

namespace cacheq8 {

// `code_of` for bfloat16 elements, in fewer steps.  With X and A the eight-bit significands of x and a, and x smaller by 2^s, 127 x / a lies at
// least 1 / (510 2^s) from a border it does not lie on, and the product below is off by 2^-23 of up to 127 / 2^s: it decides
// rightly.  127 x / a lies on a border where 254 X is an odd multiple of A: where A is 254 (the product is exact then, and
// rounds to the even code) or x = a / 2.
__device__ __forceinline__ int code_of_bf16(float x, float a, float inv) {
  const int code = __float2int_rn(__fmul_rn(x, inv));
  return fabsf(x) * 2.f == a ? (x > 0.f ? 64 : -64) : code;
}

// What a row's codes are formed with: rows of very small or very large elements are scaled by a power of two first, so that
// neither 127 / a nor the products leave float32's range (elements that lose bits by it lie far below half a step).
struct RowScale {
  float a, inv, lift, scale;
  bool good;
};
__device__ __forceinline__ RowScale row_scale(float a) {
  RowScale r;
  r.good = a > 0.f && a < INFINITY;   // false for NaN too
  r.scale = r.good ? __fdiv_rn(a, 127.f) : a == 0.f ? 0.f : __int_as_float(0x7fffffff);
  r.lift = a < 1e-30f ? 0x1p100f : a > 1e30f ? 0x1p-100f : 1.f;
  r.a = __fmul_rn(a, r.lift);
  r.inv = __fdiv_rn(127.f, r.a);
  return r;
}
template <typename T> __device__ __forceinline__ unsigned pack_codes(const float (&x)[4], const RowScale& r) {
  if (!r.good) return 0u;
  int code[4];
#pragma unroll
  for (int e = 0; e < 4; ++e)
    code[e] = sizeof(T) == 2 ? code_of_bf16(x[e] * r.lift, r.a, r.inv) : code_of(x[e] * r.lift, r.a, r.inv);
  const unsigned lo = __byte_perm(code[0], code[1], 0x0040), hi = __byte_perm(code[2], code[3], 0x0040);
  return __byte_perm(lo, hi, 0x5410);
}
// The larger magnitude, NaN if either is NaN (fmaxf would drop it).
__device__ __forceinline__ float largest(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}

// Eight elements with 16-byte stores.
__device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
  reinterpret_cast<float4*>(p)[0] = make_float4(x[0], x[1], x[2], x[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(x[4], x[5], x[6], x[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&x)[8]) {
  unsigned w[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 two = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
    w[i] = *reinterpret_cast<const unsigned*>(&two);
  }
  *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}

struct Pages {
  signed char* codes;
  float* scales;
};

// ---- store of rows as they are
// LANES threads a row (a head of a token's keys or values), four elements each a turn (two turns above 128 elements), 8, 16 or
// 32 lanes by the head size, so that few are idle; a block is 256 threads.  Bound by the latency of a dependent chain (slot and
// row, the maximum over the lanes, codes): 2,048 tokens of 4 heads of 128 in bfloat16, 6.3 MB in and out, take 5 us.
template <typename T, int LANES>
__global__ void __launch_bounds__(256)
kv_write_q8_kernel(const T* __restrict__ k_new, const T* __restrict__ v_new, long long k_stride, long long v_stride, const Pages keys,
                   const Pages values, const int* __restrict__ slots, unsigned rows, unsigned kv_heads, int dim, unsigned page_size,
                   unsigned num_slots, int aligned) {
  constexpr int TURNS = LANES == 32 ? 2 : 1;   // heads of up to 256 elements
  let_dependents_start();
  wait_for_previous();
  const unsigned row = blockIdx.x * (256 / LANES) + threadIdx.x / LANES;
  const int lane = threadIdx.x % LANES;
  // rows in the order token, keys | values, head; a row behind the last takes part in the shuffles with nothing
  const unsigned at = row < rows ? row : rows - 1;
  const unsigned token = at / (2 * kv_heads), within = at - token * 2 * kv_heads;
  const bool is_value = within >= kv_heads;
  const unsigned head = is_value ? within - kv_heads : within;
  const int slot = slots[token];
  const T* src = (is_value ? v_new + token * v_stride : k_new + token * k_stride) + head * static_cast<unsigned>(dim);
  float x[TURNS][4], a = 0.f;
#pragma unroll
  for (int i = 0; i < TURNS; ++i) {
    const int first = (lane + i * LANES) * 4;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[i][e] = 0.f;
    if (first < dim) {
      if (aligned) {
        load4<T>(src + first, x[i]);
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) x[i][e] = to_float(src[first + e]);
      }
    }
#pragma unroll
    for (int e = 0; e < 4; ++e) a = largest(a, fabsf(x[i][e]));
  }
#pragma unroll
  for (int offset = LANES / 2; offset > 0; offset >>= 1) a = largest(a, __shfl_xor_sync(0xffffffffu, a, offset));
  if (row >= rows || static_cast<unsigned>(slot) >= num_slots) return;   // a negative one is none of the pool's either
  const RowScale r = row_scale(a);
  const Pages& to = is_value ? values : keys;
  signed char* dst = to.codes + (static_cast<size_t>(slot) * kv_heads + head) * dim;
#pragma unroll
  for (int i = 0; i < TURNS; ++i) {
    const int first = (lane + i * LANES) * 4;
    if (first < dim) *reinterpret_cast<unsigned*>(dst + first) = pack_codes<T>(x[i], r);
  }
  if (lane == 0) {
    const unsigned page = static_cast<unsigned>(slot) / page_size;
    to.scales[(static_cast<size_t>(page) * kv_heads + head) * page_size + (slot - page * page_size)] = r.scale;
  }
}

// ---- bias, rotation and store of a fused q/k/v projection
// As rope_kv_write_kernel (its formulas, its order of operations: queries get the same bits), with keys and values into 8-bit
// pages.  A warp owns a head at a time, since a row's largest magnitude is needed before its first code; a block is one
// token (a slice of its heads where tokens are few) and forms the token's angles once.  Its accesses are an element a lane wide,
// queries included: 28 heads of 128 over 4 kv heads in bfloat16 take 2.2 us for a token, 10.6 for 512 and 21.6 for 2,048 (55 MB:
// 8.3 at the measured bandwidth), where the store into bfloat16 pages takes 1.3, 4.9 and 10.7.
template <typename T>
__global__ void __launch_bounds__(256)
rope_kv_write_q8_kernel(const float* __restrict__ qkv, const float* __restrict__ bias, const int* __restrict__ positions,
                        const float* __restrict__ inv_freq, T* __restrict__ q_out, const Pages keys, const Pages values,
                        const int* __restrict__ slots, int num_heads, int num_kv_heads, int head_dim, int page_size,
                        long long num_slots, int partials, long long partial_stride) {
  constexpr int TURNS = 4;   // heads of up to 256 elements: 128 pairs
  let_dependents_start();
  // Before the wait: what no kernel writes (the step's positions and slots, the frequencies).
  const int token = blockIdx.x, half = head_dim / 2;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = blockDim.x >> 5;
  const int q_width = num_heads * head_dim, kv_width = num_kv_heads * head_dim, all_heads = num_heads + 2 * num_kv_heads;
  long long slot = slots[token];
  if (slot < 0 || slot >= num_slots) slot = -1;  // never store outside the pool
  __shared__ float2 angle[128];
  if (inv_freq != nullptr) {
    const float pos = static_cast<float>(positions[token]);
    for (int j = threadIdx.x; j < half; j += blockDim.x) {
      float s, c;
      sincosf(__fmul_rn(pos, inv_freq[j]), &s, &c);
      angle[j] = make_float2(s, c);
    }
  }
  __syncthreads();
  wait_for_previous();
  const float* row = qkv + static_cast<size_t>(token) * (q_width + 2 * kv_width);
  for (int head = blockIdx.y * warps + warp; head < all_heads; head += gridDim.y * warps) {   // the same for a whole warp
    const bool is_q = head < num_heads, is_v = head >= num_heads + num_kv_heads;
    float lo[TURNS], hi[TURNS], a = 0.f;
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
      const int j = lane + 32 * i;
      lo[i] = hi[i] = 0.f;
      if (j < half) {
        const int at = head * head_dim + j;
        float x = sum_partials(row + at, partial_stride, partials), y = sum_partials(row + at + half, partial_stride, partials);
        if (bias != nullptr) {
          x = __fadd_rn(x, bias[at]);
          y = __fadd_rn(y, bias[at + half]);
        }
        lo[i] = x;
        hi[i] = y;
        if (inv_freq != nullptr && !is_v) {
          const float s = angle[j].x, c = angle[j].y;
          lo[i] = __fsub_rn(__fmul_rn(x, c), __fmul_rn(y, s));
          hi[i] = __fadd_rn(__fmul_rn(y, c), __fmul_rn(x, s));
        }
      }
      a = largest(a, largest(fabsf(lo[i]), fabsf(hi[i])));
    }
    if (is_q) {
      T* dst = q_out + static_cast<size_t>(token) * q_width + head * head_dim;
#pragma unroll
      for (int i = 0; i < TURNS; ++i) {
        const int j = lane + 32 * i;
        if (j < half) {
          dst[j] = from_float<T>(lo[i]);
          dst[j + half] = from_float<T>(hi[i]);
        }
      }
      continue;
    }
    if (slot < 0) continue;
#pragma unroll
    for (int offset = 16; offset > 0; offset >>= 1) a = largest(a, __shfl_xor_sync(0xffffffffu, a, offset));
    const RowScale r = row_scale(a);
    const Pages& to = is_v ? values : keys;
    const int kv_head = head - num_heads - (is_v ? num_kv_heads : 0);
    signed char* dst = to.codes + (slot * num_kv_heads + kv_head) * head_dim;
#pragma unroll
    for (int i = 0; i < TURNS; ++i) {
      const int j = lane + 32 * i;
      if (j < half) {
        dst[j] = r.good ? static_cast<signed char>(code_of(lo[i] * r.lift, r.a, r.inv)) : static_cast<signed char>(0);
        dst[j + half] = r.good ? static_cast<signed char>(code_of(hi[i] * r.lift, r.a, r.inv)) : static_cast<signed char>(0);
      }
    }
    if (lane == 0) to.scales[(slot / page_size * num_kv_heads + kv_head) * page_size + slot % page_size] = r.scale;
  }
}

// ---- reading back
// A thread takes 16 codes of a key and the 16 of its value: two 16-byte loads that do not wait for one another, two to four
// 16-byte stores each.  Bound by memory: 32,768 tokens of 8 heads of 128 to bfloat16, 204 MB, take 34.5 us, 5.9 TB/s.
template <typename T> __device__ __forceinline__ void read_chunk(const Pages& from, long long row, long long scale_at, int within, T* out) {
  uint4 words = make_uint4(0u, 0u, 0u, 0u);
  float scale = 0.f;
  if (row >= 0) {
    words = __ldg(reinterpret_cast<const uint4*>(from.codes + row + within));
    scale = __ldg(from.scales + scale_at);
  }
  const unsigned w[4] = {words.x, words.y, words.z, words.w};
#pragma unroll
  for (int i = 0; i < 4; i += 2) {
    float x[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = __fmul_rn(static_cast<float>(static_cast<signed char>(w[i + e / 4] >> (8 * (e % 4)))), scale);
    store8(out + 4 * i, x);
  }
}
template <typename T>
__global__ void __launch_bounds__(256)
kv_read_q8_kernel(const Pages keys, const Pages values, const int* __restrict__ slots, T* __restrict__ k_out, T* __restrict__ v_out,
                  long long chunks, unsigned per_row, int kv_heads, int dim, int page_size, long long num_slots) {
  let_dependents_start();
  wait_for_previous();
  const long long i = static_cast<long long>(blockIdx.x) * blockDim.x + threadIdx.x;
  if (i >= chunks) return;
  long long token;
  unsigned chunk;
  if (chunks <= 0xffffffffll) {   // a 32-bit division wherever it will do
    token = static_cast<unsigned>(i) / per_row;
    chunk = static_cast<unsigned>(i) - static_cast<unsigned>(token) * per_row;
  } else {
    token = i / per_row;
    chunk = static_cast<unsigned>(i - token * per_row);
  }
  const int per_head = dim / 16, head = static_cast<int>(chunk) / per_head, within = (static_cast<int>(chunk) - head * per_head) * 16;
  const int slot = slots[token];
  long long row = -1, scale_at = 0;
  if (slot >= 0 && slot < num_slots) {
    const int page = slot / page_size;
    row = (static_cast<long long>(slot) * kv_heads + head) * dim;
    scale_at = (static_cast<long long>(page) * kv_heads + head) * page_size + (slot - page * page_size);
  }
  read_chunk(keys, row, scale_at, within, k_out + i * 16);
  read_chunk(values, row, scale_at, within, v_out + i * 16);
}

static bool good_pages(const void* codes, const void* scales) {
  return codes != nullptr && scales != nullptr && reinterpret_cast<uintptr_t>(codes) % 16 == 0;
}

}  // namespace cacheq8

using namespace cacheq8;

// Stores n rows of kv_heads * dim elements of `dtype`.  Rows whose slot is not one of the pool's are left out; the others' slots
// have to differ from one another.
SHRIKE_API int shrike_kv_write_q8(const ShrikeCacheQ8* call) {
  const auto [k_new, v_new, k_codes, v_codes, k_scale_at, v_scale_at, slot_at, stream_at, k_stride, v_stride, dtype, n, kv_heads, dim, pages, page_size] = *call;
  float *const k_scales = static_cast<float*>(k_scale_at), *const v_scales = static_cast<float*>(v_scale_at);
  const int* const slots = static_cast<const int*>(slot_at);
  const cudaStream_t stream = static_cast<cudaStream_t>(stream_at);
  const long long num_slots = static_cast<long long>(pages) * page_size;
  if (n <= 0) return SHRIKE_OK;
  if (kv_heads <= 0 || dim <= 0 || dim % 16 || dim > 256 || page_size <= 0 || !good_pages(k_codes, k_scales) ||
      !good_pages(v_codes, v_scales) || (dtype != SHRIKE_F32 && dtype != SHRIKE_BF16))
    return SHRIKE_BAD_ARGUMENT;
  const Pages keys{static_cast<signed char*>(k_codes), k_scales}, values{static_cast<signed char*>(v_codes), v_scales};
  const int element = dtype == SHRIKE_F32 ? 4 : 2;
  const int aligned = (reinterpret_cast<uintptr_t>(k_new) | reinterpret_cast<uintptr_t>(v_new)) % (4 * element) == 0 &&
                      k_stride % 4 == 0 && v_stride % 4 == 0;
  const long long rows = 2ll * n * kv_heads;
  const int lanes = dim <= 32 ? 8 : dim <= 64 ? 16 : 32;
  const long long blocks = (rows * lanes + 255) / 256;
  if (rows > 0x7fffffff || num_slots > 0x7fffffff) return SHRIKE_BAD_ARGUMENT;
#define SHRIKE_WRITE_Q8(T, LANES)                                                                                              \
  launch_dependent(kv_write_q8_kernel<T, LANES>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream,                    \
                   static_cast<const T*>(k_new), static_cast<const T*>(v_new), k_stride, v_stride, keys, values, slots, static_cast<unsigned>(rows), \
                   static_cast<unsigned>(kv_heads), dim, static_cast<unsigned>(page_size), static_cast<unsigned>(num_slots), aligned)
  cudaError_t err;
  if (dtype == SHRIKE_F32) err = lanes == 8 ? SHRIKE_WRITE_Q8(float, 8) : lanes == 16 ? SHRIKE_WRITE_Q8(float, 16) : SHRIKE_WRITE_Q8(float, 32);
  else err = lanes == 8 ? SHRIKE_WRITE_Q8(__nv_bfloat16, 8) : lanes == 16 ? SHRIKE_WRITE_Q8(__nv_bfloat16, 16) : SHRIKE_WRITE_Q8(__nv_bfloat16, 32);
#undef SHRIKE_WRITE_Q8
  return err == cudaSuccess ? shrike_launch_status() : static_cast<int>(err);
}

// As shrike_rope_kv_write, into 8-bit pages.
SHRIKE_API int shrike_rope_kv_write_q8(const float* qkv, const float* bias, const int* positions, const float* inv_freq, void* q_out,
                                       void* k_codes, float* k_scales, void* v_codes, float* v_scales, const int* slots, int dtype,
                                       int n, int num_heads, int num_kv_heads, int head_dim, int page_size, long long num_slots,
                                       int partials, long long partial_stride, cudaStream_t stream) {
  if (n <= 0) return SHRIKE_OK;
  if (partials < 1 || head_dim <= 0 || head_dim % 16 || head_dim > 256 || num_heads <= 0 || num_kv_heads <= 0 || page_size <= 0 ||
      !good_pages(k_codes, k_scales) || !good_pages(v_codes, v_scales))
    return SHRIKE_BAD_ARGUMENT;
  const Pages keys{static_cast<signed char*>(k_codes), k_scales}, values{static_cast<signed char*>(v_codes), v_scales};
  const int all_heads = num_heads + 2 * num_kv_heads;
  const int threads = n >= 256 ? 256 : 64;
  const int slices = n >= 256 ? 1 : (all_heads + 1) / 2;
  if (slices > 65535) return SHRIKE_BAD_ARGUMENT;
#define SHRIKE_ROPE_Q8(T)                                                                                                          \
  launch_dependent(rope_kv_write_q8_kernel<T>, dim3(n, slices), dim3(threads), 0, stream, qkv, bias, positions, inv_freq,          \
                   static_cast<T*>(q_out), keys, values, slots, num_heads, num_kv_heads, head_dim, page_size, num_slots, partials, \
                   partial_stride)
  cudaError_t err;
  if (dtype == SHRIKE_F32) err = SHRIKE_ROPE_Q8(float);
  else if (dtype == SHRIKE_BF16) err = SHRIKE_ROPE_Q8(__nv_bfloat16);
  else return SHRIKE_BAD_ARGUMENT;
#undef SHRIKE_ROPE_Q8
  return err == cudaSuccess ? shrike_launch_status() : static_cast<int>(err);
}

// Reads n rows of kv_heads * dim elements of `dtype` back to k and v, 16-byte aligned and dense; rows whose slot is not one of
// the pool's become zeros.
SHRIKE_API int shrike_kv_read_q8(const ShrikeCacheQ8* call) {
  const auto [k_out, v_out, k_codes, v_codes, k_scale_at, v_scale_at, slot_at, stream_at, k_stride, v_stride, dtype, n, kv_heads, dim, pages, page_size] = *call;
  float *const k_scales = static_cast<float*>(k_scale_at), *const v_scales = static_cast<float*>(v_scale_at);
  const int* const slots = static_cast<const int*>(slot_at);
  const cudaStream_t stream = static_cast<cudaStream_t>(stream_at);
  const long long num_slots = static_cast<long long>(pages) * page_size;
  if (n <= 0) return SHRIKE_OK;
  if (kv_heads <= 0 || dim <= 0 || dim % 16 || page_size <= 0 || !good_pages(k_codes, k_scales) || !good_pages(v_codes, v_scales) ||
      (reinterpret_cast<uintptr_t>(k_out) | reinterpret_cast<uintptr_t>(v_out)) % 16)
    return SHRIKE_BAD_ARGUMENT;
  const Pages keys{static_cast<signed char*>(k_codes), k_scales}, values{static_cast<signed char*>(v_codes), v_scales};
  const unsigned per_row = static_cast<unsigned>(kv_heads) * static_cast<unsigned>(dim / 16);
  const long long chunks = static_cast<long long>(n) * per_row, blocks = (chunks + 255) / 256;
  if (blocks > 0x7fffffff || num_slots > 0x7fffffff) return SHRIKE_BAD_ARGUMENT;
  cudaError_t err;
  if (dtype == SHRIKE_F32)
    err = launch_dependent(kv_read_q8_kernel<float>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, keys, values, slots,
                           static_cast<float*>(k_out), static_cast<float*>(v_out), chunks, per_row, kv_heads, dim, page_size, num_slots);
  else if (dtype == SHRIKE_BF16)
    err = launch_dependent(kv_read_q8_kernel<__nv_bfloat16>, dim3(static_cast<unsigned>(blocks)), dim3(256), 0, stream, keys, values, slots,
                           static_cast<__nv_bfloat16*>(k_out), static_cast<__nv_bfloat16*>(v_out), chunks, per_row, kv_heads, dim,
                           page_size, num_slots);
  else
    return SHRIKE_BAD_ARGUMENT;
  return err == cudaSuccess ? shrike_launch_status() : static_cast<int>(err);
}
