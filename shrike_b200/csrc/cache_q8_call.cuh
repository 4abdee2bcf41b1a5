// The arguments of a store or a reading back of 8-bit pages, packed by the caller (a call with a dozen arguments costs more to make
// than the kernel takes for a token): rows k and v, `k_stride` / `v_stride` elements apart where they are stored, dense where they
// are read.  Host code without any CUDA call of its own.
#pragma once
#include <stddef.h>

struct ShrikeCacheQ8 {
  void *k, *v, *k_codes, *v_codes;
  void *k_scales, *v_scales;   // float32
  const void* slots;           // int32
  void* stream;                // cudaStream_t
  long long k_stride, v_stride;
  int dtype, n, kv_heads, dim, pages, page_size;
};
// As the caller packs them without the native module: eight addresses, two 64-bit and six 32-bit integers side by side.
static_assert(offsetof(ShrikeCacheQ8, k_stride) == 64 && offsetof(ShrikeCacheQ8, dtype) == 80 && sizeof(ShrikeCacheQ8) == 104, "packed");
