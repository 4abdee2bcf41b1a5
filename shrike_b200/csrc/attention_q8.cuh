// The arguments of attention over 8-bit pages, packed by the caller: a call with thirty arguments costs the host more to make
// than to launch.
#pragma once
#include <cuda_runtime.h>
#include <stddef.h>

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
