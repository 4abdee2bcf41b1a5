// Paged attention over keys and values in 8 bits, for any head size up to 256, any page size, queries in bfloat16 or float32.
//
// With codes c and scales s (keys: c^k_j, s^k_j; values: c^v_j, s^v_j) a row q of head h sees
//   z_j = scale s^k_j (q . c^k_j),   p_j = 2^(log2e z_j - m),   o = sum_j (p_j s^v_j) c^v_j / sum_j p_j
// Codes are integers up to 127: exact in float16.  Both products run on mma.sync m16n8k16 with float16 operands and 32-bit
// sums, and nothing but the queries and the weights is ever rounded:
//   queries   scaled by a power of two per row (largest magnitude in [2^14, 2^15)); bfloat16 queries are then exact, float32
//             ones are split in two float16 parts (22 bits) whose products are added in the accumulator.  A score leaves
//             float32's range, and its row is NaN, where keys are of 2^105 (4e31) and more: (q . c) s^k with q of 2^15
//   weights   w_j = p_j s^v_j.  The base m of the exponentials is a row's largest score (it may lag by up to 2^6) plus an
//             exponent F that puts the largest value scale the row has seen at 2^8 ... 2^9 (the sums and the outputs are all in
//             units of 2^m, so F costs nothing): float16 then keeps 11 bits of a weight down to 2^-22 of the largest possible
//             one (bfloat16 would keep 8 bits), and 22 bits in two parts for float32
// KEYS ARE THE M OF THE PRODUCTS, query rows the N: S^T = K Q^T and O^T = V^T P^T.  The heads that share a kv head lie side by
// side, token by token, as rows; eight of them make a product's N, so that the usual groups of up to eight heads waste nothing
// (rows as M would be padded to 16: twice the products, softmax work and registers), and wider tiles (`NT` times eight rows)
// share the conversion of the codes, which is what the kernel spends most of its instructions on.
// A warp takes 32 keys a step.  The keys' order inside a product is free as long as scores and values agree on it, and so is
// the order of a head's elements in q . c: both are chosen so that a lane's operands are consecutive bytes.  Element order: a
// lane reads 16 codes of a key with one load and they are its operands of four products.  Key order: row n of a group of eight
// is key n ^ ((n >> 1) & 1), and 16-byte chunks of a row are swizzled with it, so that neither the keys' nor the values' loads
// meet in a bank.  Four codes become two registers of float16 pairs by a byte permutation (1024 + code + 128, exact) and a
// subtraction; the weights go from the scores' layout to an operand's through movmatrix.
//
// Two forms.  Few rows (single tokens, and small portions, eight or sixteen rows a tile): the rows' keys are dealt to `splits` CTAs and to each CTA's four warps, each with its
// own ring of cp.async copies (no barrier in the loop); the warps' results meet in shared memory, those of up to eight CTAs in
// the shared memory of their cluster, and the clusters' in global memory, where the last CTA to arrive adds them up in order.
// Bound by memory at many keys (64 sequences of 4,096 keys, 40 heads of 128: 85 us, 5.0 TB/s, with warm caches, where with the
// products left out the copies alone take 71; 95 us, 4.5 TB/s, where every pass finds other data), and by the chain metadata,
// page, codes, products, merges at few (one sequence of 517 keys: 5.6 us).
// Metadata and pages are looked up while the kernel before still runs (that sequence: 6.1 us without).  Many rows (portions):
// four warps of 8 NT rows each share one ring of key tiles.
#include <cuda_fp16.h>

#include "attention_q8.cuh"
#include "common.cuh"

#ifndef SHRIKE_HEAD_DIM
#error "compile with -DSHRIKE_HEAD_DIM=<head size>"
#endif

namespace attnq8 {
using namespace q8;

constexpr int D = SHRIKE_HEAD_DIM;
static_assert(D % 16 == 0 && D >= 16 && D <= 256, "head sizes are multiples of 16 up to 256");
constexpr int WARPS = 4, THREADS = WARPS * 32;
constexpr int KEYS = 32;                 // keys of a step
constexpr int CHUNKS = D / 16;           // 16-byte chunks of a key's codes
constexpr int STEPS_K = D / 16;          // products along the head size, for 8 keys
constexpr int BLOCKS_V = (D + 31) / 32;  // runs of 32 elements of the output
constexpr bool WIDE = D % 64 == 0;       // keys are read 16 bytes a lane (else 4)
constexpr int TILE = KEYS * D;           // bytes of a step's key (or value) codes
constexpr int SCALES = 2 * KEYS * 4;     // of both kinds of a step's scales
constexpr int RING = 3 * TILE + 2 * SCALES;   // a warp's share of the few-rows form
constexpr int STEP_BYTES = 2 * TILE + SCALES;   // a step of the other form: keys, values, scales
constexpr int MAX_SPLITS = 64;

struct Args {
  const signed char* k_codes;
  const float* k_scales;
  const signed char* v_codes;
  const float* v_scales;
  const int* block_table;
  const int* q_start;
  const int* ctx_len;
  const void* q;
  void* out;
  int max_blocks, num_heads, num_kv_heads, page_size, num_pages, window;
  int page_shift;      // page_size is 2^page_shift, or -1
  int only;            // 1: entries of one token, 2: longer ones, 0: all
  float scale_log2;
  int splits, cluster; // CTAs that share a row tile's keys, and how many of them form a cluster
  float* scratch;      // [(entry, kv head, row tile)][cluster][rows][D + 2]: unnormalised rows, then each row's base and sum
  int* arrivals;       // [(entry, kv head, row tile)]: CTAs that have left their share; zero between launches
};

__device__ __forceinline__ unsigned smem_u32(const void* p) { return static_cast<unsigned>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void copy16(unsigned dst, const void* src, bool there) {   // zeros where there is nothing
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy4(unsigned dst, const void* src, bool there) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(there ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copies_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int LEFT> __device__ __forceinline__ void copies_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(LEFT) : "memory"); }

__device__ __forceinline__ void mma(float (&c)[4], const unsigned (&a)[4], unsigned b0, unsigned b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float low_half(unsigned v) { return __low2float(*reinterpret_cast<const __half2*>(&v)); }
__device__ __forceinline__ float high_half(unsigned v) { return __high2float(*reinterpret_cast<const __half2*>(&v)); }
// The key of column n of a group of eight columns.
__device__ __forceinline__ constexpr int key_of(int n) { return n ^ ((n >> 1) & 1); }
// What the 16-byte chunks of a row are exchanged by.
__device__ __forceinline__ int swizzle(int row) {
  if (D % 128 == 0) return (((((row ^ (row >> 1) ^ (row >> 2)) & 1) << 1) | ((row >> 1) & 1)) << 1);
  if (D == 64) return ((row >> 2) & 1) << 1;
  return 0;
}
__device__ __forceinline__ int chunk_at(int row, int chunk) { return row * D + ((chunk ^ swizzle(row)) << 4); }

__device__ __forceinline__ void cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ unsigned map_to_rank(unsigned address, int rank) {
  unsigned there;
  asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(address), "r"(rank));
  return there;
}
__device__ __forceinline__ float2 load_peer2(unsigned address) {
  float2 v;
  asm volatile("ld.shared::cluster.v2.f32 {%0, %1}, [%2];" : "=f"(v.x), "=f"(v.y) : "r"(address) : "memory");
  return v;
}
__device__ __forceinline__ float4 load_peer4(unsigned address) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(address) : "memory");
  return v;
}

// Where a lane's key lies: its row among all codes, its place among the scales, and whether it exists.  A key that does not
// has scales of zero and whatever codes the pool's first row holds: codes are finite whatever they are, so it counts as zeros.
struct Place {
  int row;
  bool there;
  long long scale;
};
// The page of a key, -1 if the key lies behind `last_key`: to be asked for a step before its place is formed, since the answer
// takes as long as a quarter of a step.  A context near 2^31, which no table holds, makes steps whose keys pass 32 bits: as
// unsigned numbers they lie behind every table.
__device__ __forceinline__ int page_of(const Args& args, const int* table, unsigned key, int last_key) {
  const unsigned block = args.page_shift >= 0 ? key >> args.page_shift : key / static_cast<unsigned>(args.page_size);
  return static_cast<int>(key) <= last_key && block < static_cast<unsigned>(args.max_blocks) ? table[block] : -1;
}
// The key's place, given its page; nowhere if that is not one of the pool's.
__device__ __forceinline__ Place place_of(const Args& args, int page, int kv_head, unsigned key) {
  Place at{0, false, 0};
  const int within = static_cast<int>(args.page_shift >= 0 ? key & (args.page_size - 1) : key % static_cast<unsigned>(args.page_size));
  if (page >= 0 && page < args.num_pages) {
    at.row = page * args.page_size + within;
    at.there = true;
    at.scale = (static_cast<long long>(page) * args.num_kv_heads + kv_head) * args.page_size + within;
  }
  return at;
}

// Brings the codes of 32 keys (or of their values) into shared memory; `COUNT` threads of which this is number `id` share the
// work, and each of their warps holds in lane l the row of key l (`Place::row`).
template <int COUNT>
__device__ __forceinline__ void load_codes(const signed char* codes, int row_bytes, int head_at, int row_of_lane, unsigned tile, int id) {
  if constexpr (COUNT % CHUNKS == 0) {
    // COUNT / CHUNKS keys a turn.  Where these are few, a turn's number and a thread's own key are different bits of the key's
    // number, and since a swizzle is made of exclusive ors, the thread's part of it is formed once.
    constexpr int AT_ONCE = COUNT / CHUNKS;
    const int chunk = id % CHUNKS, own = id / CHUNKS;
    const signed char* src = codes + (head_at + chunk * 16);
    const int own_at = own * D;
    const int own_chunk = chunk ^ swizzle(own);
#pragma unroll
    for (int k = 0; k < (KEYS + AT_ONCE - 1) / AT_ONCE; ++k) {
      const int row = __shfl_sync(0xffffffffu, row_of_lane, (k * AT_ONCE + own) & 31);
      if (AT_ONCE <= KEYS || own < KEYS)
        copy16(tile + (k * AT_ONCE * D + own_at + ((own_chunk ^ swizzle(k * AT_ONCE)) << 4)), src + static_cast<long long>(row) * row_bytes, true);
    }
  } else {
#pragma unroll
    for (int k = 0; k < (KEYS * CHUNKS + COUNT - 1) / COUNT; ++k) {
      const int idx = id + k * COUNT;
      const int key = idx / CHUNKS, chunk = idx - key * CHUNKS;
      const int row = __shfl_sync(0xffffffffu, row_of_lane, key & 31);
      if (KEYS * CHUNKS % COUNT == 0 || idx < KEYS * CHUNKS)
        copy16(tile + chunk_at(key, chunk), codes + (static_cast<long long>(row) * row_bytes + (head_at + chunk * 16)), true);
    }
  }
}
__device__ __forceinline__ void load_scales(const Args& args, const Place& place, unsigned scales, int id) {
  if (id < KEYS) {
    copy4(scales + id * 4, args.k_scales + place.scale, place.there);
    copy4(scales + KEYS * 4 + id * 4, args.v_scales + place.scale, place.there);
  }
}

template <typename T> struct Parts { static constexpr int COUNT = 1; };
template <> struct Parts<float> { static constexpr int COUNT = 2; };

// The 8x8 matrix of 16-bit elements whose row g a quad of lanes holds, transposed.
__device__ __forceinline__ unsigned transpose8(unsigned v) {
  unsigned d;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
  return d;
}

// A warp's rows, NT times eight of them: queries as operands, running bases, sums and outputs.  Lane 4 g + t holds query row g's
// operands (of each eight), and the scores, sums and outputs of rows 2 t and 2 t + 1.
template <typename T, int NT>
struct Rows {
  static constexpr int ROWS = 8 * NT;
  static constexpr int PARTS = Parts<T>::COUNT;
  static constexpr bool IN_SHARED = STEPS_K * PARTS * NT > 16;   // query operands in shared memory, else in registers
  static constexpr int SHARED_BYTES = IN_SHARED ? STEPS_K * PARTS * NT * 256 : 0;   // for one warp's rows
  uint2 q[IN_SHARED ? 1 : STEPS_K * PARTS * NT];
  float factor[NT][2];         // what q . c s^k is multiplied by to be a score
  int first[NT][2], last[NT][2];   // the keys a row sees
  float most[NT][2], base[NT][2], sum[NT][2];   // what is taken for the largest score, base m = most + F, sum of 2^(z - m)
  int exponent[NT][2];         // F
  float o[NT][BLOCKS_V * 2][4];

  __device__ __forceinline__ static int element_of(int step, int t) {   // a lane's first element of four in a product
    return WIDE ? 16 * (t + 4 * (step / 4)) + 4 * (step % 4) : 4 * (t + 4 * step);
  }
  // The element of the head that o[nt][2 b][0] belongs to; o[nt][2 b + m][c] is 2 m + (c >> 1) further.
  __device__ __forceinline__ static int out_element(int b, int g) { return WIDE ? 64 * (b / 2) + 8 * g + 4 * (b % 2) : 32 * b + 4 * g; }

  // Rows row0 ... of an entry whose tokens begin at `start`; `group` heads share kv head `kv_head`.
  __device__ __forceinline__ void begin(const Args& args, int row0, int rows, int start, int group, int kv_head, int pos0, uint2* shared, int lane) {
    const int g = lane >> 2, t = lane & 3;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      const int row = row0 + 8 * nt + g, token = row / group, head = kv_head * group + row - token * group;
      const bool there = row < rows;
      const T* src = static_cast<const T*>(args.q) + (there ? (static_cast<size_t>(start + token) * args.num_heads + head) * D : 0);
      float x[STEPS_K][4];
      unsigned top = 0u;   // the largest magnitude's bits, of finite elements
#pragma unroll
      for (int s = 0; s < STEPS_K; ++s) {
        x[s][0] = x[s][1] = x[s][2] = x[s][3] = 0.f;
        if (there) load4<T>(src + element_of(s, t), x[s]);
#pragma unroll
        for (int e = 0; e < 4; ++e) top = max(top, finite_bits(x[s][e]));
      }
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = max(static_cast<int>(top >> 23) - 127, -100);
      const float lift = args.scale_log2 < 0.f ? -power_of_two(14 - e) : power_of_two(14 - e);
#pragma unroll
      for (int s = 0; s < STEPS_K; ++s) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[s][i] *= lift;
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
          const uint2 b = make_uint2(pack_half(x[s][0], x[s][1]), pack_half(x[s][2], x[s][3]));
          if (IN_SHARED) shared[((s * PARTS + part) * NT + nt) * 32 + lane] = b;
          else q[IN_SHARED ? 0 : (s * PARTS + part) * NT + nt] = b;
          if (part + 1 < PARTS) {
            x[s][0] -= low_half(b.x);
            x[s][1] -= high_half(b.x);
            x[s][2] -= low_half(b.y);
            x[s][3] -= high_half(b.y);
          }
        }
      }
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const int mine = row0 + 8 * nt + 2 * t + c;
        // a scale of zero leaves all scores equal; a hidden key's -inf has to stay one
        factor[nt][c] = fmaxf(fabsf(args.scale_log2) * power_of_two(__shfl_sync(0xffffffffu, e, 4 * (2 * t + c)) - 14), 1e-38f);
        // a row that is not there sees what the last one sees: nobody reads it
        last[nt][c] = pos0 + min(mine, rows - 1) / group;
        first[nt][c] = first_visible_key(last[nt][c], args.window);
        most[nt][c] = base[nt][c] = -INFINITY;
        sum[nt][c] = 0.f;
        exponent[nt][c] = LEAST_EXPONENT;
      }
#pragma unroll
      for (int i = 0; i < BLOCKS_V * 2; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[nt][i][c] = 0.f;
    }
  }

  // Hides from two rows the keys that they do not see, and finds the largest value scale of the others.
  static __device__ __forceinline__ void hide(float (&s)[2][4], int key0, int g, const int (&first)[2], const int (&last)[2], const float (&v_scale)[4],
                                           unsigned (&top)[2]) {
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int key = key0 + 8 * j + key_of(g);
        if (key >= first[r] && key <= last[r]) top[r] = max(top[r], finite_bits(v_scale[j]));
        else s[j >> 1][2 * (j & 1) + r] = -INFINITY;
      }
  }

  using Weights = unsigned[NT][2][2][PARTS];   // [16 keys][eight of them]: operands of the second product

  // The weights of the 32 keys from `key0` on, whose codes lie in `k_tile` and whose scales in `scales` (the keys', the values').
  __device__ __forceinline__ void weigh(const unsigned char* k_tile, const float* scales, int key0, const uint2* shared, int lane, Weights& weights) {
    const int g = lane >> 2, t = lane & 3;
    const float* k_scales = scales;
    const float* v_scales = scales + KEYS;
    float s[NT][2][4];   // [16 keys]: c & 1 the row, c >> 1 the eight keys
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int c = 0; c < 4; ++c) s[nt][kk][c] = 0.f;
    // scores
#pragma unroll
    for (int i = 0; i < (WIDE ? D / 64 : STEPS_K); ++i) {
      constexpr int WORDS = WIDE ? 4 : 1;
      unsigned words[4][WORDS];   // of keys 8 j + key_of(g)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int key = 8 * j + key_of(g);
        if (WIDE) {
          const uint4 v = *reinterpret_cast<const uint4*>(k_tile + chunk_at(key, t + 4 * i));
          words[j][0] = v.x;
          words[j][WIDE ? 1 : 0] = WIDE ? v.y : v.x;
          words[j][WIDE ? 2 : 0] = WIDE ? v.z : v.x;
          words[j][WIDE ? 3 : 0] = WIDE ? v.w : v.x;
        } else {
          words[j][0] = *reinterpret_cast<const unsigned*>(k_tile + chunk_at(key, i) + 4 * t);
        }
      }
#pragma unroll
      for (int w = 0; w < WORDS; ++w) {
        uint2 b[PARTS][NT];
#pragma unroll
        for (int part = 0; part < PARTS; ++part)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            const int index = ((i * WORDS + w) * PARTS + part) * NT + nt;
            b[part][nt] = IN_SHARED ? shared[index * 32 + lane] : q[IN_SHARED ? 0 : index];
          }
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          const unsigned lo = words[2 * kk][w] ^ 0x80808080u, hi = words[2 * kk + 1][w] ^ 0x80808080u;
          const unsigned a[4] = {codes_to_half<0x4140>(lo), codes_to_half<0x4140>(hi), codes_to_half<0x4342>(lo), codes_to_half<0x4342>(hi)};
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int part = 0; part < PARTS; ++part) mma(s[nt][kk], a, b[part][nt].x, b[part][nt].y);
        }
      }
    }
    // this lane's keys: their scales
    float k_scale[4], v_scale[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      k_scale[j] = k_scales[8 * j + key_of(g)];
      v_scale[j] = v_scales[8 * j + key_of(g)];
    }
    bool inside = true;   // whether every row sees every key
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 2; ++r) inside = inside && key0 >= first[nt][r] && key0 + KEYS - 1 <= last[nt][r];
    const bool edge = __any_sync(0xffffffffu, !inside);
    // the largest of this lane's value scales (negative ones, infinities and NaN, none of which a store leaves but the last,
    // order above all finite bits)
    unsigned all_top = max(max(__float_as_uint(v_scale[0]), __float_as_uint(v_scale[1])), max(__float_as_uint(v_scale[2]), __float_as_uint(v_scale[3])));
    const bool odd_scale = all_top >= 0x7f800000u, careful = edge && __any_sync(0xffffffffu, odd_scale);
    if (odd_scale) {
      all_top = max(max(finite_bits(v_scale[0]), finite_bits(v_scale[1])), max(finite_bits(v_scale[2]), finite_bits(v_scale[3])));
      // A value that is no number makes the rows that see it none: by way of their sums, since its weight may be zero in 32 bits,
      // here or where shares are added up.
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (!(fabsf(v_scale[j]) < INFINITY)) {
          const int key = key0 + 8 * j + key_of(g);
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int r = 0; r < 2; ++r)
              if (key >= first[nt][r] && key <= last[nt][r]) sum[nt][r] = __int_as_float(0x7fffffff);
        }
    }
    if (edge) all_top = 0u;
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float largest[2] = {-INFINITY, -INFINITY};
      unsigned top[2] = {all_top, all_top};
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < 2; ++r) s[nt][j >> 1][2 * (j & 1) + r] *= k_scale[j];
      if (edge) hide(s[nt], key0, g, first[nt], last[nt], v_scale, top);
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < 2; ++r) largest[r] = fmaxf(largest[r], s[nt][j >> 1][2 * (j & 1) + r]);
      // the base moves only where a score or a value scale has outgrown it
      bool stays = true;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        largest[r] *= factor[nt][r];
        stays = stays && largest[r] <= most[nt][r] + BASE_LAG && static_cast<int>(top[r] >> 23) - 127 - SCALE_BITS <= exponent[nt][r];
      }
      if (__any_sync(0xffffffffu, !stays)) {
        float correction[2];
#pragma unroll
        for (int r = 0; r < 2; ++r) {
#pragma unroll
          for (int offset = 4; offset < 32; offset <<= 1) {
            largest[r] = fmaxf(largest[r], __shfl_xor_sync(0xffffffffu, largest[r], offset));
            top[r] = max(top[r], __shfl_xor_sync(0xffffffffu, top[r], offset));
          }
          exponent[nt][r] = max(exponent[nt][r], min(static_cast<int>(top[r] >> 23) - 127 - SCALE_BITS, MOST_EXPONENT));
          most[nt][r] = fmaxf(most[nt][r], largest[r]);
          const float next = most[nt][r] + static_cast<float>(exponent[nt][r]);
          const float down = fmaxf(base[nt][r], -1e30f) - fmaxf(next, -1e30f);   // 0 for a row that has seen no key yet
          correction[r] = fast_exp2(down);
          base[nt][r] = next;
          sum[nt][r] = scale_sum(sum[nt][r], down);
        }
#pragma unroll
        for (int i = 0; i < BLOCKS_V * 2; ++i)
#pragma unroll
          for (int c = 0; c < 4; ++c) o[nt][i][c] *= correction[c & 1];
      }
      float p[4][2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float from = base[nt][r] == -INFINITY ? 0.f : base[nt][r];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
          p[j][r] = fast_exp2(fmaf(s[nt][j >> 1][2 * (j & 1) + r], factor[nt][r], -from));
          sum[nt][r] += p[j][r];
        }
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        float x = p[j][0] * v_scale[j], y = p[j][1] * v_scale[j];
        if (careful) {   // a key that a row does not see has no part in it, not even a scale of NaN
          x = p[j][0] == 0.f ? 0.f : x;
          y = p[j][1] == 0.f ? 0.f : y;
        }
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
          const unsigned packed = pack_half(x, y);
          weights[nt][j >> 1][j & 1][part] = transpose8(packed);
          if (part + 1 < PARTS) {
            x -= low_half(packed);
            y -= high_half(packed);
          }
        }
      }
    }
  }

  // Adds the same keys' values, in `v_tile`.
  __device__ __forceinline__ void add(const unsigned char* v_tile, int lane, const Weights& weights) {
    const int g = lane >> 2, t = lane & 3;
    constexpr int RUN = WIDE ? 2 : 1;   // words a lane reads of a value row at a time
#pragma unroll
    for (int b = 0; b < BLOCKS_V; b += RUN) {
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        unsigned rows[4][RUN];
#pragma unroll
        for (int i = 0; i < 4; ++i) {   // keys 2 t, 2 t + 1 of the first eight, then of the second
          const int key = 16 * kk + 8 * (i >> 1) + key_of(2 * t + (i & 1));
          const int at = WIDE ? 4 * (b / 2) + (g >> 1) : 2 * b + (g >> 2);
          if (WIDE) {
            const uint2 v = *reinterpret_cast<const uint2*>(v_tile + chunk_at(key, at) + 8 * (g & 1));
            rows[i][0] = v.x ^ 0x80808080u;
            rows[i][RUN - 1] = WIDE ? v.y ^ 0x80808080u : v.x ^ 0x80808080u;
          } else {
            rows[i][0] = D % 32 == 0 || at < CHUNKS ? *reinterpret_cast<const unsigned*>(v_tile + chunk_at(key, at) + 4 * (g & 3)) : 0u;
            rows[i][0] ^= 0x80808080u;
          }
        }
#pragma unroll
        for (int w = 0; w < RUN; ++w)
#pragma unroll
          for (int m = 0; m < 2; ++m) {   // of a word's four elements the pair 2 m, 2 m + 1: rows g and g + 8 of the product
            const unsigned lo = __byte_perm(rows[0][w], rows[1][w], m == 0 ? 0x5140 : 0x7362), hi = __byte_perm(rows[2][w], rows[3][w], m == 0 ? 0x5140 : 0x7362);
            const unsigned a[4] = {codes_to_half<0x4140>(lo), codes_to_half<0x4342>(lo), codes_to_half<0x4140>(hi), codes_to_half<0x4342>(hi)};
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int part = 0; part < PARTS; ++part) mma(o[nt][2 * (b + w) + m], a, weights[nt][kk][0][part], weights[nt][kk][1][part]);
          }
      }
    }
  }

  // Sums of whole rows.
  __device__ __forceinline__ void finish() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
      for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int offset = 4; offset < 32; offset <<= 1) sum[nt][r] += __shfl_xor_sync(0xffffffffu, sum[nt][r], offset);
  }
  // Rows that others are added to: half of F leaves the base.  Bases of rows with equally large scores are then within 2^100 of one
  // another, whatever their values' sizes, and the sum of one whose values are all zeros is not lost beside another's.
  __device__ __forceinline__ void meet() {
#pragma unroll
    for (int nt = 0; nt < NT; ++nt) {
      float factor[2];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const int half = exponent[nt][r] / 2;
        factor[r] = power_of_two(half);
        base[nt][r] -= static_cast<float>(half);
        sum[nt][r] *= factor[r];
      }
#pragma unroll
      for (int i = 0; i < BLOCKS_V * 2; ++i)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[nt][i][c] *= factor[c & 1];
    }
  }
};

// Which entry this is, and whether it is this launch's.
__device__ __forceinline__ bool entry_of(const Args& args, int seq, int& start, int& q_len, int& context) {
  start = args.q_start[seq];
  q_len = args.q_start[seq + 1] - start;
  context = args.ctx_len[seq];
  return q_len > 0 && !(args.only == 1 && q_len > 1) && !(args.only == 2 && q_len == 1);
}

// A share of a row is its elements in units of 2^base, the sum of its exponentials likewise, and the base.  Adds one to others
// whose largest base is `base`.
__device__ __forceinline__ void add_share(float m, float l, const float4& v, float base, float& total, float (&acc)[4]) {
  const float weight = m == -INFINITY ? 0.f : fast_exp2(m - base);
  if (l != l) total = l;   // a score or a value that is no number: the row is none either, whatever the others hold
  if (weight == 0.f) return;
  total += l * weight;
  acc[0] += v.x * weight; acc[1] += v.y * weight; acc[2] += v.z * weight; acc[3] += v.w * weight;
}
__device__ __forceinline__ void leave_share(float* share, int rows, int row, int element, float base, float total, const float (&acc)[4]) {
  *reinterpret_cast<float4*>(share + row * D + element) = make_float4(acc[0], acc[1], acc[2], acc[3]);
  if (element == 0) *reinterpret_cast<float2*>(share + rows * D + 2 * row) = make_float2(base, total);
}
template <typename T>
__device__ __forceinline__ void store_row(const Args& args, int row, int start, int group, int kv_head, int element, float total, float (&acc)[4]) {
  const float inv = total == 0.f ? 0.f : 1.f / total;   // a row that sees nothing is zeros
#pragma unroll
  for (int e = 0; e < 4; ++e) acc[e] *= inv;
  const int token = row / group, head = kv_head * group + row - token * group;
  store4<T>(static_cast<T*>(args.out) + (static_cast<size_t>(start + token) * args.num_heads + head) * D + element, acc);
}

// Few rows: grid (splits, kv heads * row tiles, entries).
template <typename T, int NT>
__global__ void __launch_bounds__(THREADS, Parts<T>::COUNT * NT * D <= 128 ? 4 : 1)
split_keys_kernel(const Args args) {
  using R = Rows<T, NT>;
  constexpr int ROWS = R::ROWS;
  extern __shared__ __align__(128) unsigned char smem[];
  let_dependents_start();
  const int seq = blockIdx.z, split = blockIdx.x;
  const int kv_head = blockIdx.y % args.num_kv_heads, tile = blockIdx.y / args.num_kv_heads;
  const int group = args.num_heads / args.num_kv_heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  int start, q_len, context;   // metadata, and so is the block table: written before the step's kernels
  if (!entry_of(args, seq, start, q_len, context)) {
    wait_for_previous();
    return;
  }
  const int rows = q_len * group, row0 = tile * ROWS;
  if (row0 >= rows) {
    wait_for_previous();
    return;
  }
  const int pos0 = context - q_len;
  const int tile_rows = min(ROWS, rows - row0);
  const int last_key = pos0 + (row0 + tile_rows - 1) / group, first_key = first_visible_key(pos0 + row0 / group, args.window);
  const int step_lo = max(first_key, 0) / KEYS, steps = last_key < 0 ? 0 : last_key / KEYS + 1 - step_lo;
  const int per = (steps + args.splits - 1) / args.splits;
  const int mine_lo = step_lo + min(steps, split * per), mine_hi = step_lo + min(steps, (split + 1) * per);

  uint2* shared_q = reinterpret_cast<uint2*>(smem + WARPS * RING);
  // A warp's ring: three tiles that keys and values go through in turn (K0 V0 K1 V1 ...), so that each is asked for a whole step
  // before it is used, and two steps' scales.  Four warps' rings are 50 KB at a head size of 128: an SM holds four CTAs.  (One
  // tile more a warp left room for three: 96 us instead of 89 for 64 sequences of 4,096 keys, as it was then.)
  unsigned char* ring = smem + warp * RING;
  const float* scales = reinterpret_cast<const float*>(ring + 3 * TILE);
  const unsigned ring_at = smem_u32(ring), scales_at = ring_at + 3 * TILE;
  const int* table = args.block_table + static_cast<size_t>(seq) * args.max_blocks;
  const int row_bytes = args.num_kv_heads * D, head_at = kv_head * D;
  auto load_keys = [&](const Place& place, int tile, int slot) {
    load_codes<32>(args.k_codes, row_bytes, head_at, place.row, ring_at + tile, lane);
    load_scales(args, place, scales_at + slot * SCALES, lane);
  };
  R r;
  // this warp's steps: mine_lo + warp, + WARPS, ...
  const int begin = mine_lo + warp;
  auto page_at = [&](int step) { return page_of(args, table, static_cast<unsigned>(step) * KEYS + lane, step < mine_hi ? last_key : -1); };
  auto place_at = [&](int page, int step) { return place_of(args, page, kv_head, static_cast<unsigned>(step) * KEYS + lane); };
  int page = page_at(begin), next_page = page_at(begin + WARPS), ahead = page_at(begin + 2 * WARPS);
  wait_for_previous();   // the query and the newest keys come from the kernel before this one
  Place place = place_at(page, begin), next = place_at(next_page, begin + WARPS);
  if (begin < mine_hi) load_keys(place, 0, 0);
  copies_commit();
  if (begin < mine_hi) load_codes<32>(args.v_codes, row_bytes, head_at, place.row, ring_at + TILE, lane);
  copies_commit();
  if (begin + WARPS < mine_hi) load_keys(next, 2 * TILE, 1);
  copies_commit();
  place = place_at(ahead, begin + 2 * WARPS);
  ahead = page_at(begin + 3 * WARPS);
  r.begin(args, row0, rows, start, group, kv_head, pos0, shared_q, lane);   // all warps write the same operands
  __syncwarp();
  int k_now = 0, v_now = TILE, k_next = 2 * TILE, slot = 0;   // `next`: the place of the step after this one, `place`: of the one after that
  for (int step = begin; step < mine_hi; step += WARPS) {
    typename R::Weights weights;
    copies_wait<2>();   // outstanding: this step's values, the next step's keys
    __syncwarp();
    r.weigh(ring + k_now, scales + slot * 2 * KEYS, step * KEYS, shared_q, lane, weights);
    __syncwarp();
    if (step + WARPS < mine_hi) load_codes<32>(args.v_codes, row_bytes, head_at, next.row, ring_at + k_now, lane);
    copies_commit();
    copies_wait<2>();   // outstanding: the next step's keys and values
    __syncwarp();
    r.add(ring + v_now, lane, weights);
    __syncwarp();
    if (step + 2 * WARPS < mine_hi) load_keys(place, v_now, slot);
    copies_commit();
    next = place;
    place = place_at(ahead, step + 3 * WARPS);
    ahead = page_at(step + 4 * WARPS);
    const int used = k_now;
    k_now = k_next;
    k_next = v_now;
    v_now = used;
    slot ^= 1;
  }
  copies_wait<0>();
  r.finish();
  r.meet();
  __syncthreads();
  // the warps' rows meet: [warp][ROWS][D + 4] (four more, so that the stores of a quad fall into different banks), and
  // [warp][ROWS][base, sum]
  constexpr int ROW_FLOATS = D + 4;
  float* all_o = reinterpret_cast<float*>(smem);
  float* all_m = all_o + WARPS * ROWS * ROW_FLOATS;
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int row = warp * ROWS + 8 * nt + 2 * t + c;
#pragma unroll
      for (int b = 0; b < BLOCKS_V; ++b)
        if (D % 32 == 0 || R::out_element(b, g) < D)
          *reinterpret_cast<float4*>(all_o + row * ROW_FLOATS + R::out_element(b, g)) =
              make_float4(r.o[nt][2 * b][c], r.o[nt][2 * b][2 + c], r.o[nt][2 * b + 1][c], r.o[nt][2 * b + 1][2 + c]);
      if (g == 0) {
        all_m[2 * row] = r.base[nt][c];
        all_m[2 * row + 1] = r.sum[nt][c];
      }
    }
  __syncthreads();
  // What leaves this CTA: a share of the result, in shared memory for the cluster, in global memory beyond it, or the result.
  const size_t pair = (static_cast<size_t>(seq) * gridDim.y + blockIdx.y);
  constexpr int SHARE = ROWS * (D + 2);
  const int cluster = args.cluster, clusters = args.splits / cluster;
  float* merged = all_m + WARPS * ROWS * 2;   // [ROWS][D], then [ROWS][base, sum]: for the cluster's other CTAs
  float* share = clusters > 1 ? args.scratch + (pair * clusters + split / cluster) * SHARE : nullptr;
  for (int i = threadIdx.x; i < tile_rows * (D / 4); i += THREADS) {
    const int row = i / (D / 4), element = (i - row * (D / 4)) * 4;
    float base = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) base = fmaxf(base, all_m[(w * ROWS + row) * 2]);
    float total = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < WARPS; ++w)
      add_share(all_m[(w * ROWS + row) * 2], all_m[(w * ROWS + row) * 2 + 1],
                *reinterpret_cast<const float4*>(all_o + (w * ROWS + row) * ROW_FLOATS + element), base, total, acc);
    if (cluster > 1) leave_share(merged, ROWS, row, element, base, total, acc);
    else if (share != nullptr) leave_share(share, ROWS, row, element, base, total, acc);
    else store_row<T>(args, row0 + row, start, group, kv_head, element, total, acc);
  }
  if (cluster > 1) {
    const int rank = split % cluster;
    cluster_sync();
    const unsigned here = smem_u32(merged);
    for (int i = rank * THREADS + threadIdx.x; i < tile_rows * (D / 4); i += cluster * THREADS) {
      const int row = i / (D / 4), element = (i - row * (D / 4)) * 4;
      float2 ml[8];
      float4 v[8];
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (c < cluster) {
          const unsigned peer = map_to_rank(here, c);
          ml[c] = load_peer2(peer + (ROWS * D + 2 * row) * 4);
          v[c] = load_peer4(peer + (row * D + element) * 4);
        }
      float base = -INFINITY;
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (c < cluster) base = fmaxf(base, ml[c].x);
      float total = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (c < cluster) add_share(ml[c].x, ml[c].y, v[c], base, total, acc);
      if (share != nullptr) leave_share(share, ROWS, row, element, base, total, acc);
      else store_row<T>(args, row0 + row, start, group, kv_head, element, total, acc);
    }
    cluster_sync();   // nobody leaves while another CTA reads its shares
  }
  if (clusters == 1) return;
  __threadfence();
  __syncthreads();
  __shared__ int arrived;
  if (threadIdx.x == 0) arrived = atomicAdd(args.arrivals + pair, 1);
  __syncthreads();
  if (arrived != args.splits - 1) return;
  __threadfence();
  const float* shares = args.scratch + pair * clusters * SHARE;
  for (int i = threadIdx.x; i < tile_rows * (D / 4); i += THREADS) {
    const int row = i / (D / 4), element = (i - row * (D / 4)) * 4;
    float base = -INFINITY, total = 0.f, acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int first = 0; first < clusters; first += 8) {   // eight shares' loads at a time
      float2 ml[8];
      float4 v[8];
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const float* share_c = shares + static_cast<size_t>(min(first + c, clusters - 1)) * SHARE;
        ml[c] = __ldcg(reinterpret_cast<const float2*>(share_c + ROWS * D + 2 * row));
        v[c] = __ldcg(reinterpret_cast<const float4*>(share_c + row * D + element));
      }
      float next = base;
#pragma unroll
      for (int c = 0; c < 8; ++c) next = fmaxf(next, ml[c].x);
      const float down = base == -INFINITY ? 0.f : fast_exp2(base - next);
      total *= down;
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[e] *= down;
      base = next;
#pragma unroll
      for (int c = 0; c < 8; ++c)
        if (first + c < clusters) add_share(ml[c].x, ml[c].y, v[c], base, total, acc);
    }
    store_row<T>(args, row0 + row, start, group, kv_head, element, total, acc);
  }
  if (threadIdx.x == 0) args.arrivals[pair] = 0;
}

// Many rows: grid (row tiles of 4 * 8 NT, kv heads, entries); the CTA's warps share the key tiles.
template <typename T, int NT>
__global__ void __launch_bounds__(THREADS)
portion_rows_kernel(const Args args) {
  using R = Rows<T, NT>;
  constexpr int ROWS = R::ROWS;
  extern __shared__ __align__(128) unsigned char smem[];
  let_dependents_start();
  const int seq = blockIdx.z, kv_head = blockIdx.y;
  const int group = args.num_heads / args.num_kv_heads;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  int start, q_len, context;   // metadata, as above
  const bool mine = entry_of(args, seq, start, q_len, context);
  const int rows = q_len * group;
  const int tiles = (rows + WARPS * ROWS - 1) / (WARPS * ROWS);
  if (!mine || static_cast<int>(blockIdx.x) >= tiles) {
    wait_for_previous();
    return;
  }
  const int cta_row0 = (tiles - 1 - static_cast<int>(blockIdx.x)) * WARPS * ROWS;   // the longest first
  const int row0 = cta_row0 + warp * ROWS;
  const int pos0 = context - q_len;
  const int last_key = pos0 + (min(cta_row0 + WARPS * ROWS, rows) - 1) / group;
  const int first_key = first_visible_key(pos0 + cta_row0 / group, args.window);
  const int step_lo = max(first_key, 0) / KEYS, step_hi = last_key < 0 ? step_lo : last_key / KEYS + 1;
  // this warp's own part of that range
  const int my_last = row0 < rows ? pos0 + (min(row0 + ROWS, rows) - 1) / group : -1;
  const int my_first = first_visible_key(pos0 + row0 / group, args.window);

  uint2* shared_q = reinterpret_cast<uint2*>(smem + 2 * STEP_BYTES + warp * R::SHARED_BYTES);
  const unsigned ring_at = smem_u32(smem);
  const int* table = args.block_table + static_cast<size_t>(seq) * args.max_blocks;
  const int row_bytes = args.num_kv_heads * D, head_at = kv_head * D;
  auto load_step = [&](const Place& place, unsigned to) {
    load_codes<THREADS>(args.k_codes, row_bytes, head_at, place.row, to, threadIdx.x);
    load_codes<THREADS>(args.v_codes, row_bytes, head_at, place.row, to + TILE, threadIdx.x);
    load_scales(args, place, to + 2 * TILE, threadIdx.x);
  };
  R r;
  auto page_at = [&](int step) { return page_of(args, table, static_cast<unsigned>(step) * KEYS + lane, last_key); };
  auto place_at = [&](int page, int step) { return place_of(args, page, kv_head, static_cast<unsigned>(step) * KEYS + lane); };
  int page = page_at(step_lo), ahead = page_at(step_lo + 1);
  wait_for_previous();
  if (step_lo < step_hi) load_step(place_at(page, step_lo), ring_at);
  copies_commit();
  r.begin(args, row0, rows, start, group, kv_head, pos0, shared_q, lane);
  __syncwarp();
  int stage = 0;
  for (int step = step_lo; step < step_hi; ++step) {
    copies_wait<0>();
    __syncthreads();   // this step's copies of all threads have landed; everyone has left the stage that is loaded next
    if (step + 1 < step_hi) load_step(place_at(ahead, step + 1), ring_at + (stage ^ 1) * STEP_BYTES);
    copies_commit();
    ahead = page_at(step + 2);
    if (step * KEYS <= my_last && step * KEYS + KEYS > my_first) {
      typename R::Weights weights;
      const unsigned char* at = smem + stage * STEP_BYTES;
      r.weigh(at, reinterpret_cast<const float*>(at + 2 * TILE), step * KEYS, shared_q, lane, weights);
      r.add(at + TILE, lane, weights);
    }
    stage ^= 1;
  }
  copies_wait<0>();
  r.finish();
#pragma unroll
  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
    for (int c = 0; c < 2; ++c) {
      const int row = row0 + 8 * nt + 2 * t + c;
      if (row >= rows) continue;
#pragma unroll
      for (int b = 0; b < BLOCKS_V; ++b) {
        float v[4] = {r.o[nt][2 * b][c], r.o[nt][2 * b][2 + c], r.o[nt][2 * b + 1][c], r.o[nt][2 * b + 1][2 + c]};
        if (D % 32 == 0 || R::out_element(b, g) < D) store_row<T>(args, row, start, group, kv_head, R::out_element(b, g), r.sum[nt][c], v);
      }
    }
}

template <typename T, int NT> constexpr size_t split_keys_smem() {
  const size_t ring = static_cast<size_t>(WARPS) * RING + Rows<T, NT>::SHARED_BYTES;
  const size_t merge = (static_cast<size_t>(WARPS) * Rows<T, NT>::ROWS * (D + 6) + Rows<T, NT>::ROWS * (D + 2)) * 4;
  return ring > merge ? ring : merge;
}
template <typename T, int NT> constexpr size_t portion_rows_smem() { return 2 * static_cast<size_t>(STEP_BYTES) + WARPS * Rows<T, NT>::SHARED_BYTES; }

constexpr int PORTION_NT = 2;
// Row tiles of the few-rows form: eights, pairs of them for groups of more than eight heads.
static int few_rows(int group) { return group <= 8 ? 8 : 16; }

template <typename T, int NT>
static int resident() {
  static PerDevice raised;
  if (shrike_raise_smem(raised, split_keys_kernel<T, NT>, split_keys_smem<T, NT>()) != 0) return shrike_device().sm_count;
  int per_sm = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, split_keys_kernel<T, NT>, THREADS, split_keys_smem<T, NT>()) != cudaSuccess || per_sm < 1)
    per_sm = 1;
  return per_sm * shrike_device().sm_count;
}

template <typename T>
static int resident_many() {
  static PerDevice raised;
  if (shrike_raise_smem(raised, portion_rows_kernel<T, PORTION_NT>, portion_rows_smem<T, PORTION_NT>()) != 0) return shrike_device().sm_count;
  int per_sm = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, portion_rows_kernel<T, PORTION_NT>, THREADS, portion_rows_smem<T, PORTION_NT>()) != cudaSuccess ||
      per_sm < 1)
    per_sm = 1;
  return per_sm * shrike_device().sm_count;
}

template <typename T, int NT>
static int launch_few(const Args& args, int num_seqs, int tokens, cudaStream_t stream) {
  static PerDevice raised;
  const int rc = shrike_raise_smem(raised, split_keys_kernel<T, NT>, split_keys_smem<T, NT>());
  if (rc != 0) return rc;
  const long long tiles = (static_cast<long long>(tokens) * (args.num_heads / args.num_kv_heads) + 8 * NT - 1) / (8 * NT);
  if (tiles * args.num_kv_heads > 65535) return SHRIKE_BAD_ARGUMENT;
  const dim3 grid(args.splits, static_cast<unsigned>(tiles * args.num_kv_heads), num_seqs);
  if (args.cluster == 1)
    return static_cast<int>(launch_dependent(split_keys_kernel<T, NT>, grid, dim3(THREADS), split_keys_smem<T, NT>(), stream, args));
  return static_cast<int>(launch_dependent_clusters(split_keys_kernel<T, NT>, grid, dim3(THREADS), split_keys_smem<T, NT>(), stream,
                                                    static_cast<unsigned>(args.cluster), args));
}

template <typename T>
static int launch(const Args& base, int num_seqs, int max_q_len, int has_single, int has_portions, int others, cudaStream_t stream) {
  Args args = base;
  const int group = args.num_heads / args.num_kv_heads;
  if (has_single) {
    args.only = has_portions || others ? 1 : 0;
    const int tokens = args.only ? 1 : max_q_len;
    const int rc = few_rows(group) == 8 ? launch_few<T, 1>(args, num_seqs, tokens, stream) : launch_few<T, 2>(args, num_seqs, tokens, stream);
    if (rc != 0) return rc;
  }
  if (has_portions) {
    static PerDevice raised;
    const int rc = shrike_raise_smem(raised, portion_rows_kernel<T, PORTION_NT>, portion_rows_smem<T, PORTION_NT>());
    if (rc != 0) return rc;
    args.only = has_single ? 2 : 0;
    constexpr int ROWS = WARPS * Rows<T, PORTION_NT>::ROWS;
    const long long tiles = (static_cast<long long>(max_q_len) * group + ROWS - 1) / ROWS;
    if (tiles > 0x7fffffff) return SHRIKE_BAD_ARGUMENT;
    const cudaError_t err = launch_dependent(portion_rows_kernel<T, PORTION_NT>, dim3(static_cast<unsigned>(tiles), args.num_kv_heads, num_seqs),
                                             dim3(THREADS), portion_rows_smem<T, PORTION_NT>(), stream, args);
    if (err != cudaSuccess) return static_cast<int>(err);
  }
  return shrike_launch_status();
}

}  // namespace attnq8

// Query rows of a tile of the few-rows form, for groups of `group` heads a kv head.
SHRIKE_API int shrike_attention_q8_tile_rows(int group) { return attnq8::few_rows(group); }
// CTAs of the few-rows form that the device holds at once, for queries of `dtype`.
SHRIKE_API int shrike_attention_q8_resident_ctas(int dtype, int group) {
  using namespace attnq8;
  if (dtype == SHRIKE_F32) return few_rows(group) == 8 ? resident<float, 1>() : resident<float, 2>();
  return few_rows(group) == 8 ? resident<__nv_bfloat16, 1>() : resident<__nv_bfloat16, 2>();
}
// Floats of scratch for a row of a (entry, kv head, row tile) and split, and the most splits.
SHRIKE_API int shrike_attention_q8_row_floats() { return attnq8::D + 2; }
SHRIKE_API int shrike_attention_q8_max_splits() { return attnq8::MAX_SPLITS; }

// Query rows of a CTA of the form for many.
SHRIKE_API int shrike_attention_q8_portion_rows() { return attnq8::WARPS * 8 * attnq8::PORTION_NT; }
// CTAs of that form that the device holds at once, for queries of `dtype`.
SHRIKE_API int shrike_attention_q8_resident_portions(int dtype) {
  return dtype == SHRIKE_F32 ? attnq8::resident_many<float>() : attnq8::resident_many<__nv_bfloat16>();
}
// Whether a batch's single tokens should run on the form for many rows too, `ctas` CTAs with theirs over block tables of `keys`
// keys, instead of a launch of their own after it: while the CTAs find room beside one another, and while the keys, which that
// form does not split, are few or not many more than the `longest` portion's CTAs walk in any case (a single token of many keys
// beside a short portion would be walked for long by one CTA: 53 us for 1,000 keys, 28 heads of 128 in float32, which its own
// launch takes 12 for).  Measured, us, two launches and one (float32): 28
// heads of 128, 196 CTAs over 250 keys 24.7 and 21.9, 248 CTAs 27.3 and 28.2 (296 find room); 40 heads, 104 CTAs 22.8 and 21.5, 360
// CTAs 29.0 and 30.4; 6 heads of 32, a portion of 16 tokens and a single one over 64 keys 7.2 and 4.5, over 250 keys 13.3 and 9.7, one of 475 tokens and 20 single
// ones over 483 keys 25.0 and 20.3.
SHRIKE_API int shrike_attention_q8_one_launch(int dtype, long long ctas, long long keys, long long longest) {
  if (keys > 256 && 2 * keys > 3 * longest) return 0;
  return 4 * ctas <= 3ll * shrike_attention_q8_resident_portions(dtype) ? 1 : 0;
}

// q and out [tokens, heads * D] of `dtype`, 16-byte aligned; codes [pages, page_size, kv heads, D], 16-byte aligned, scales
// [pages, kv heads, page_size].  `has_single`: entries of one token (every entry, where has_portions is 0: then `max_q_len`
// tokens at most) run on the few-rows form with `splits` CTAs a row tile; `has_portions`: the longer ones (all of them where
// has_single is 0) on the other, or on another kernel where `others` is set.  splits > 1 needs `scratch` (row_floats() for every row of a tile of (entry, kv head, row tile) and split)
// and `arrivals` (an int a pair, zero before the first launch).
SHRIKE_API int shrike_paged_attention_q8(const ShrikeAttentionQ8* call) {
  const auto& [q, k_codes, k_scales, v_codes, v_scales, block_table, q_start, ctx_len, seq_of_token, out, scratch, arrivals, status, stream, max_blocks,
               dtype, num_tokens, num_seqs, num_heads, num_kv_heads, page_size, num_pages, window, has_single, has_portions, max_q_len, others, splits,
               cluster, tiles, scale] = *call;
  if (num_seqs <= 0) return SHRIKE_OK;
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || num_kv_heads > 65535 || max_blocks <= 0 || page_size <= 0 ||
      num_pages <= 0 || static_cast<long long>(num_pages) * page_size > 0x7fffffff ||
      static_cast<long long>(max_blocks) * page_size > 0x7fffffff - 4096 || max_q_len < 1 || num_seqs > 65535 || splits < 1 ||
      static_cast<long long>(max_q_len) * (num_heads / num_kv_heads) > 0x7fffffff - 4096 ||
      cluster < 1 || cluster > 8 || splits % cluster || splits > attnq8::MAX_SPLITS ||
      (splits > cluster && (scratch == nullptr || arrivals == nullptr)) ||
      (reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(k_codes) |
       reinterpret_cast<uintptr_t>(v_codes) | reinterpret_cast<uintptr_t>(scratch)) % 16)
    return SHRIKE_BAD_ARGUMENT;
  attnq8::Args args;
  args.k_codes = static_cast<const signed char*>(k_codes);
  args.k_scales = k_scales;
  args.v_codes = static_cast<const signed char*>(v_codes);
  args.v_scales = v_scales;
  args.block_table = block_table;
  args.q_start = q_start;
  args.ctx_len = ctx_len;
  args.q = q;
  args.out = out;
  args.max_blocks = max_blocks;
  args.num_heads = num_heads;
  args.num_kv_heads = num_kv_heads;
  args.page_size = page_size;
  args.num_pages = num_pages;
  args.window = window;
  args.page_shift = (page_size & (page_size - 1)) == 0 ? __builtin_ctz(page_size) : -1;
  args.only = 0;
  args.scale_log2 = scale * attnq8::LOG2E;
  args.splits = splits;
  args.cluster = cluster;
  args.scratch = scratch;
  args.arrivals = arrivals;
  if (dtype == SHRIKE_F32) return attnq8::launch<float>(args, num_seqs, max_q_len, has_single, has_portions, others, stream);
  if (dtype == SHRIKE_BF16) return attnq8::launch<__nv_bfloat16>(args, num_seqs, max_q_len, has_single, has_portions, others, stream);
  return SHRIKE_BAD_ARGUMENT;
}
