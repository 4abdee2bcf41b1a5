// Paged causal attention for portions (q_len > 1) over keys and values in 8 bits, queries in bfloat16, on the fifth-generation
// tensor cores.  The mathematics is that of attention_q8.cu: codes are exact in float16, queries are scaled by a power of two
// per row so that they are too, weights p s^v are rounded to float16 under a base that keeps the row's largest value scale at
// 2^8 ... 2^9, everything else is in 32 bits.
//
// One CTA owns two chains of up to 128 query rows.  The rows of a chain are 128 / group tokens of ALL the heads that share a kv
// head, token by token: a key tile is turned into float16 once for every head that reads it, a portion of a few dozen tokens
// fills the rows, and a chain's tokens lie close together, so that little is computed behind the causal border.  A chain walks
// the keys 64 at a time, as the kernel over bfloat16 pages does (attention_tcgen05.cu): scores by tcgen05.mma into tensor
// memory, softmax, weights back into tensor memory as the operand of the second product, outputs there.
//
// The way of the keys and values: TMA brings a tile's codes (one box a page, in the swizzle of their row length), eight warps
// turn them into float16 tiles in the 128-byte swizzle (four the keys', four the values'; two threads a key), and those are
// what the products read.  Eight codes take 10 instructions (a byte permutation and a subtraction a pair, an exclusive or for
// four).
// The softmax bounds it (with scores passed through untouched, 40 heads' 512 tokens over 8,192 keys took 60 % of the time), and
// what bounds the softmax is the latency of its instructions and how fast they are fetched.  So it has sixteen warps (with
// eight, a thread a row, a prompt of 2,048 tokens took 66 us where these took 58), a warp has sixteen rows and all 64 keys of a
// step, as fragments: the four lanes of a row agree on its base by shuffles, and only where one has to move (two warps a row,
// each with half of the keys, met at a barrier every step: 8 % of the time).  And the code is kept small, by loops that stay
// loops: with the tries of every wait unrolled and 64 codes converted in one piece the kernel was 128 KB instead of 60, a warp
// waited for its next instruction as long as for anything else, and the time was 154 us instead of 128 (as measured then).
//
// Roles: warp 0 brings key codes (and the queries), warp 3 value codes (and owns tensor memory), warps 1 and 2 issue the products
// of a chain each, warps 4..11 and 12..19 are the softmax and epilogue of a chain each (a warp reaches the 32 lanes of tensor memory
// that its number modulo 4 says: two share them, sixteen rows each), warps 20..23 convert keys, 24..27 values.
// Registers a thread: 72 at launch, 96 in the softmax warpgroups, 40 in the others (16 x 96 + 12 x 40 = 28 x 72).
// Barriers: raw_k / raw_v full[raw stage] (TMA) and free (converters, an arrival a warp); k_full / v_full[stage] (converters;
// v_full also says that the tile's scales lie in shared memory), k_free / v_free[stage] (commits of both chains); q_ready[chain]
// once the softmax warps have turned the queries into float16; the others as in attention_tcgen05.cu.
// Every wait is bounded (status word, CTA-wide abort flag); no TMA load uses multicast.
// Built once per head size; serves head sizes 64 and 128, page sizes 8, 16, 32, 64, and groups of up to 64 heads.
#include <cuda_fp16.h>

#include <algorithm>

#include "attention_q8.cuh"
#include "blackwell.cuh"

#ifndef SHRIKE_HEAD_DIM
#error "compile with -DSHRIKE_HEAD_DIM=<head size>"
#endif

#if SHRIKE_HEAD_DIM == 64 || SHRIKE_HEAD_DIM == 128

namespace tcq8 {
using namespace bw;
using namespace q8;

constexpr int D = SHRIKE_HEAD_DIM;
constexpr int BM = 128;                         // query rows of one chain
constexpr int HALVES = D / 64;                 // 64-element groups of the head size
constexpr int Q_HALF = BM * 128;               // bytes of one 64-element-wide sub-tile of a query tile
constexpr int Q_BYTES = 2 * Q_HALF;              // room for a query tile, and for 64 elements of 128 rows of 32-bit output
static_assert(HALVES * Q_HALF <= Q_BYTES && BM * 256 <= Q_BYTES, "the output's pieces leave by way of the query tile");
constexpr int KEYS = 64;                       // keys of a tile, and of a softmax step
constexpr int STAGES = 3, RAW_STAGES = 3;
constexpr int KV_HALF = KEYS * 128;            // bytes of one 64-element-wide sub-tile of a float16 key (or value) tile
constexpr int KV_TILE = HALVES * KV_HALF;
constexpr int RAW_TILE = KEYS * D;             // a tile's codes
constexpr int WARPS = 28, THREADS = WARPS * 32;
constexpr unsigned CHAIN_COLS = 256, P_COL = 64, O_COL = 128, TMEM_COLS = 512;   // as in attention_tcgen05.cu
constexpr int NOT_FINITE = 4096;   // above any exponent

enum : int { ERR_PRODUCER = 61, ERR_CONVERT = 62, ERR_MMA = 63, ERR_SOFTMAX = 64, ERR_DRAIN = 65, ERR_ALIGNMENT = 66 };

__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
__device__ __forceinline__ unsigned long long pair_of(float lo, float hi) {
  unsigned long long d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
  return d;
}
__device__ __forceinline__ void halves_of(unsigned long long v, float& lo, float& hi) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v));
}
__device__ __forceinline__ unsigned long long fma_pair(unsigned long long a, unsigned long long b, unsigned long long c) {
  unsigned long long d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ unsigned long long add_pair(unsigned long long a, unsigned long long b) {
  unsigned long long d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ unsigned long long mul_pair(unsigned long long a, unsigned long long b) {
  unsigned long long d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
// kind::f16 instruction descriptor: D float32, A and B float16, A K-major; B K-major or MN-major.
__device__ __forceinline__ unsigned half_descriptor(int m, int n, bool b_mn_major) {
  return (1u << 4) | ((b_mn_major ? 1u : 0u) << 16) | (static_cast<unsigned>(n >> 3) << 17) | (static_cast<unsigned>(m >> 4) << 24);
}
__device__ __forceinline__ void tma_load_3d(void* smem, const CUtensorMap* map, unsigned long long* bar, int x, int y, int z) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cta.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_u32(smem)), "l"(reinterpret_cast<unsigned long long>(map)), "r"(smem_u32(bar)), "r"(x), "r"(y), "r"(z)
      : "memory");
}
// D[tmem] (+)= A[tmem] * B[smem]: the A operand (weights, float16 packed two to a column, one row per lane) from tensor memory.
__device__ __forceinline__ void umma_a_in_tmem(unsigned leader, unsigned tmem_d, unsigned tmem_a, unsigned long long b, unsigned idesc,
                                               unsigned accumulate) {
  asm volatile(
      "{\n\t.reg .pred p, e;\n\tsetp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 e, %5, 0;\n\t"
      "@e tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
      ::"r"(tmem_d), "r"(tmem_a), "l"(b), "r"(idesc), "r"(accumulate), "r"(leader) : "memory");
}
template <int REGISTERS> __device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGISTERS)); }
template <int REGISTERS> __device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGISTERS)); }

// As mbar_wait, in less code (see above).
__device__ __forceinline__ bool wait_bar(unsigned long long* bar, unsigned parity, volatile int* abort, int* status, int who) {
  if (mbar_test_wait(bar, parity)) return true;
#pragma unroll 1
  for (unsigned tries = 0; tries < WAIT_LIMIT; ++tries) {
    if (mbar_try_wait(bar, parity)) return true;
    if (*abort) return false;
  }
  *abort = 1;
  if (status != nullptr && *status == 0) *status = who;
  return false;
}

struct Args {
  const float* k_scales;
  const float* v_scales;
  const int* block_table;
  const int* q_start;
  const int* ctx_len;
  __nv_bfloat16* out;
  int* status;
  int max_blocks, num_heads, num_kv_heads, page_size, page_shift, num_pages, window, skip_single;
  int group, tokens;   // heads of a kv head, tokens of a chain (128 / group)
  float scale_log2;
  int splits;          // CTAs that share a query tile's keys; > 1: results go to the scratch below
  float* partial_o;    // [splits][tokens][heads][D] unnormalised output rows
  float* partial_ml;   // [splits][tokens][heads][2] their base (log2 domain) and sum
  int num_tokens, num_seqs;
  const int* seq_of_token;   // [tokens], for the second kernel
};

// What a CTA with work index `work` owns: sequences in order, each with its query tiles of `rows` tokens, the last (longest to
// walk) first; sequences of one token own none when skip_single.  Every lane of the calling warp gets the answer; tile_start
// < 0: no such work.
struct Work {
  int seq, tile_start, start, q_len, context;
};
__device__ __forceinline__ Work find_work(const Args& args, int work, int rows) {
  const int lane = threadIdx.x & 31;
  int before = 0;
  for (int base = 0; base < args.num_seqs; base += 32) {
    const int s = base + lane;
    int tiles = 0, start = 0, q_len = 0, context = 0;
    if (s < args.num_seqs) {
      start = args.q_start[s];
      q_len = args.q_start[s + 1] - start;
      context = args.ctx_len[s];
      tiles = q_len <= 0 || (q_len == 1 && args.skip_single) ? 0 : (q_len + rows - 1) / rows;
    }
    int inclusive = tiles;
#pragma unroll
    for (int offset = 1; offset < 32; offset <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, inclusive, offset);
      if (lane >= offset) inclusive += other;
    }
    const int first = before + inclusive - tiles;            // work index of this sequence's first tile
    const unsigned owner = __ballot_sync(0xffffffffu, tiles > 0 && work >= first && work < first + tiles);
    if (owner != 0) {
      const int src = __ffs(owner) - 1;
      const int from = __shfl_sync(0xffffffffu, first, src), count = __shfl_sync(0xffffffffu, tiles, src);
      return Work{base + src, (count - 1 - (work - from)) * rows, __shfl_sync(0xffffffffu, start, src),
                  __shfl_sync(0xffffffffu, q_len, src), __shfl_sync(0xffffffffu, context, src)};
    }
    before += __shfl_sync(0xffffffffu, inclusive, 31);
  }
  return Work{-1, -1, 0, 0, 0};
}

struct Shared {
  float k_scale[STAGES][KEYS], v_scale[STAGES][KEYS];
  int4 v_top[STAGES];   // of each 32 keys the exponent of the largest value scale: x, y with NOT_FINITE added where one is no finite number; z, w
  unsigned long long q_full, q_ready[2], s_full[2], s_read[2], p_full[2][2], pv_done[2][2], pv_last[2], stagger;
  unsigned long long raw_k_full[RAW_STAGES], raw_k_free[RAW_STAGES], raw_v_full[RAW_STAGES], raw_v_free[RAW_STAGES];
  unsigned long long k_full[STAGES], k_free[STAGES], v_full[STAGES], v_free[STAGES];
  unsigned tmem_base;
  volatile int abort;
};
constexpr size_t SMEM = 2 * Q_BYTES + 2 * STAGES * KV_TILE + 2 * RAW_STAGES * RAW_TILE + sizeof(Shared);
static_assert(SMEM <= 232448, "more than an SM's shared memory");

// 16 lanes x 64 columns of 32-bit as the fragments of a matrix: r[4 j + 2 m + c] is row lane / 4 + 8 m, column 8 j + 2 (lane % 4) + c.
__device__ __forceinline__ void tmem_load_fragments(unsigned taddr, unsigned (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x8.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
        "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
        "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_store_fragments(unsigned taddr, const unsigned (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x256b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]),
        "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]),
        "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
// 16 lanes x 32 columns, two 16-bit elements in each: r[2 j + m] is row lane / 4 + 8 m, column 4 j + lane % 4.
__device__ __forceinline__ void tmem_store_pairs(unsigned taddr, const unsigned (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
      ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]),
        "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
// A warp's sixteen output rows.
__device__ __noinline__ void rescale_output_rows(unsigned tmem_o, float upper, float lower) {
  for (int c = 0; c < D; c += 64) {
    unsigned o[32];
    tmem_load_fragments(tmem_o + c, o);
    tmem_wait_load();
#pragma unroll
    for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * ((j & 2) ? lower : upper));
    tmem_store_fragments(tmem_o + c, o);
  }
}

// Which of two rows see a value that is no finite number among 16 keys of a step: bits 0 and 1.  `key`: the first of them, two side by
// side of every eight.  Rare, and out of the loop's code.
__device__ __noinline__ unsigned rows_of_no_number(const float* v_scale, int key, int first_0, int last_0, int first_1, int last_1) {
  unsigned rows = 0u;
#pragma unroll 1
  for (int i = 0; i < 16; ++i) {
    const int within = 8 * (i >> 1) + (i & 1), at = key + within;
    if (fabsf(v_scale[within]) < INFINITY) continue;
    rows |= (at >= first_0 && at <= last_0 ? 1u : 0u) | (at >= first_1 && at <= last_1 ? 2u : 0u);
  }
  return rows;
}

// A converting thread's share: 16-byte chunks first ... first + COUNT - 1 of its key's codes, and the float16 they become.
constexpr int RAW_CHUNKS = D / 16, MY_CHUNKS = RAW_CHUNKS / 2;
__device__ __forceinline__ void convert_chunk(const unsigned char* raw, unsigned char* tile, int row, int chunk) {
  // rows of 128 bytes in the 128-byte swizzle, rows of 64 bytes in the 64-byte one
  const uint4 codes = *reinterpret_cast<const uint4*>(raw + row * D + ((chunk ^ (D == 128 ? row & 7 : (row >> 1) & 3)) << 4));
  unsigned char* half = tile + (chunk / 4) * KV_HALF + row * 128;
  const unsigned w[4] = {codes.x ^ 0x80808080u, codes.y ^ 0x80808080u, codes.z ^ 0x80808080u, codes.w ^ 0x80808080u};
#pragma unroll
  for (int i = 0; i < 2; ++i)
    *reinterpret_cast<uint4*>(half + (((2 * (chunk % 4) + i) ^ (row & 7)) << 4)) =
        make_uint4(codes_to_half<0x4140>(w[2 * i]), codes_to_half<0x4342>(w[2 * i]), codes_to_half<0x4140>(w[2 * i + 1]), codes_to_half<0x4342>(w[2 * i + 1]));
}

__global__ void __launch_bounds__(THREADS, 1)
portions_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                const __grid_constant__ CUtensorMap map_v, const Args args) {
  extern __shared__ __align__(1024) unsigned char smem_raw[];
  const int kv_head = blockIdx.x, split = blockIdx.z;
  const Work own = find_work(args, blockIdx.y, 2 * args.tokens);           // metadata: written before the step's kernels
  const int seq = own.seq, tile_start = own.tile_start, start = own.start, q_len = own.q_len;
  if (tile_start < 0 || (smem_u32(smem_raw) & 1023u)) {
    if (tile_start >= 0 && threadIdx.x == 0 && args.status != nullptr) *args.status = ERR_ALIGNMENT;
    let_dependents_start();
    wait_for_previous();
    return;
  }
  unsigned char* q_tiles = smem_raw;                             // [2 chains][Q_BYTES]
  unsigned char* k_tiles = q_tiles + 2 * Q_BYTES;                // [STAGES][KV_TILE]
  unsigned char* v_tiles = k_tiles + STAGES * KV_TILE;           // [STAGES][KV_TILE]
  unsigned char* raw_k = v_tiles + STAGES * KV_TILE;             // [RAW_STAGES][RAW_TILE]
  unsigned char* raw_v = raw_k + RAW_STAGES * RAW_TILE;          // [RAW_STAGES][RAW_TILE]
  Shared* sh = reinterpret_cast<Shared*>(raw_v + RAW_STAGES * RAW_TILE);
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;

  const int pos0 = own.context - q_len;                         // position of the first new token
  // chain c owns tokens tile_start + c * tokens ...; tokens_1 <= 0: the later chain has none
  const int tokens_0 = min(args.tokens, q_len - tile_start), tokens_1 = min(args.tokens, q_len - tile_start - args.tokens);
  const int lo = first_visible_key(max(pos0 + tile_start, 0), args.window);   // first key any row sees
  const int hi_0 = pos0 + tile_start + tokens_0 - 1;            // last key chain 0 sees (below 0: none)
  const int hi_1 = tokens_1 > 0 ? hi_0 + tokens_1 : -1;
  const int hi = max(hi_0, hi_1);
  const int tile_hi = hi >= 0 ? hi / KEYS : -1;
  const int all_tiles = hi >= 0 ? tile_hi - lo / KEYS + 1 : 0;
  const int per = (all_tiles + args.splits - 1) / args.splits;
  // this CTA's share: tiles tile_lo ... last_tile (none: an empty split).  The later chain takes up to two tiles (its 128
  // tokens at most) that the earlier one does not, the last ones: nobody waits for a stage to be free that such a tile was in.
  const int tile_lo = lo / KEYS + split * per;
  const int last_tile = min(tile_hi, tile_lo + per - 1);
  const int steps_0 = hi_0 >= 0 ? max(0, min(last_tile, hi_0 / KEYS) - tile_lo + 1) : 0;
  const int steps_1 = hi_1 >= 0 ? max(0, min(last_tile, hi_1 / KEYS) - tile_lo + 1) : 0;
  const int num_tiles = max(steps_0, steps_1);

  if (warp == 3) tmem_alloc(&sh->tmem_base, TMEM_COLS);
  const unsigned users = (steps_0 > 0 ? 1u : 0u) + (steps_1 > 0 ? 1u : 0u);   // chains that read the key and value stages
  if (threadIdx.x == 0) {
    mbar_init(&sh->q_full, 1);
    for (int c = 0; c < 2; ++c) {
      mbar_init(&sh->q_ready[c], 8);
      mbar_init(&sh->s_full[c], 1);
      mbar_init(&sh->s_read[c], 8);
      for (int b = 0; b < 2; ++b) {
        mbar_init(&sh->p_full[c][b], 8);
        mbar_init(&sh->pv_done[c][b], 1);
      }
      mbar_init(&sh->pv_last[c], 1);
    }
    for (int s = 0; s < RAW_STAGES; ++s) {
      mbar_init(&sh->raw_k_full[s], 1);
      mbar_init(&sh->raw_v_full[s], 1);
      mbar_init(&sh->raw_k_free[s], 4);
      mbar_init(&sh->raw_v_free[s], 4);
    }
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&sh->k_full[s], 4);
      mbar_init(&sh->k_free[s], users > 0 ? users : 1u);
      mbar_init(&sh->v_full[s], 4);
      mbar_init(&sh->v_free[s], users > 0 ? users : 1u);
    }
    mbar_init(&sh->stagger, 1);
    sh->abort = 0;
    mbar_init_fence();
  }
  // The first page ids (metadata): the loaders' a chunk of 32 at a time (lane l: page l of the chunk, several tiles' worth), the
  // converting threads' their own key's.
  const int* table = args.block_table + static_cast<size_t>(seq) * args.max_blocks;
  auto page_of = [&](unsigned key) -> int {   // of a key that some row sees; -1 for one that none does, or that passes 32 bits
    const unsigned block = key >> args.page_shift;
    return static_cast<int>(key) <= hi && block < static_cast<unsigned>(args.max_blocks) ? table[block] : -1;
  };
  const int pages_per_tile = KEYS >> args.page_shift, tiles_per_chunk = 32 / pages_per_tile;
  auto load_chunk = [&](int chunk) -> int {
    return chunk * tiles_per_chunk < num_tiles ? page_of(static_cast<unsigned>(tile_lo) * KEYS + (static_cast<unsigned>(chunk * 32 + lane) << args.page_shift)) : -1;
  };
  auto load_page = [&](int i, int row) -> int { return i < num_tiles ? page_of(static_cast<unsigned>(tile_lo + i) * KEYS + row) : -1; };
  const bool scales = warp == 24 || warp == 25;   // the converting warps that bring the tiles' scales
  int chunk_pages = -1, next_pages = -1;          // chunks 0 and 1, or this thread's pages of tiles 0 and 1
  if (warp == 0 || warp == 3) {
    chunk_pages = load_chunk(0);
    next_pages = load_chunk(1);
  } else if (scales) {
    chunk_pages = load_page(0, threadIdx.x & 63);
    next_pages = load_page(1, threadIdx.x & 63);
  }
  fence_before_sync();
  __syncthreads();
  fence_after_sync();
  let_dependents_start();
  wait_for_previous();   // the query and the newest keys come from the kernel before this one

  if (warp < 4) {
    fewer_registers<40>();
    if (warp == 0 || warp == 3) {
      // Key (warp 0) and value codes (warp 3): lane 0 waits for the buffer and arms its barrier, then lane pg issues the box of
      // page pg of the tile.
      const bool for_keys = warp == 0;
      const int nowhere = args.num_pages * args.page_size;      // a row coordinate outside the cache: reads zeros
      if (for_keys && lane == 0 && num_tiles > 0) {
        mbar_expect_tx(&sh->q_full, 2 * HALVES * args.tokens * args.group * 128);
        for (int c = 0; c < 2; ++c)
          for (int h = 0; h < HALVES; ++h)
            tma_load_3d(q_tiles + c * Q_BYTES + h * Q_HALF, &map_q, &sh->q_full, h * 64, kv_head * args.group, start + tile_start + c * args.tokens);
      }
      unsigned char* const raw = for_keys ? raw_k : raw_v;
      unsigned long long* const full = for_keys ? sh->raw_k_full : sh->raw_v_full;
      unsigned long long* const free_again = for_keys ? sh->raw_k_free : sh->raw_v_free;
      const CUtensorMap* const map = for_keys ? &map_k : &map_v;
      int issued = 0, within = 0, chunk = 0;
#pragma unroll 1
      for (int i = 0; i < num_tiles; ++i) {
        const int s = i % RAW_STAGES;
        if (within == tiles_per_chunk) {
          within = 0;
          chunk_pages = next_pages;
          next_pages = load_chunk(++chunk + 1);
        }
        int page = __shfl_sync(0xffffffffu, chunk_pages, within * pages_per_tile + (lane & (pages_per_tile - 1)));
        ++within;
        if (page >= args.num_pages) page = -1;
        const int y = page < 0 ? nowhere : page << args.page_shift;
        int ok = 1;
        if (lane == 0) {
          ok = wait_bar(&free_again[s], ((i / RAW_STAGES) & 1) ^ 1, &sh->abort, args.status, ERR_PRODUCER) ? 1 : 0;
          if (ok) mbar_expect_tx(&full[s], RAW_TILE);
        }
        ok = __shfl_sync(0xffffffffu, ok, 0);
        if (!ok) break;
        if (lane < pages_per_tile) tma_load_2d(raw + s * RAW_TILE + ((lane << args.page_shift) * D), map, &full[s], kv_head * D, y);
        issued = i + 1;
      }
      if (lane == 0 && sh->abort) {   // copies may still be in flight: wait for the buffers armed last
        for (int i = max(0, issued - RAW_STAGES); i < issued; ++i) {
          bool landed = false;
#pragma unroll 1
          for (unsigned tries = 0; tries < WAIT_LIMIT && !landed; ++tries) landed = mbar_try_wait(&full[i % RAW_STAGES], (i / RAW_STAGES) & 1);
          if (!landed && args.status != nullptr) *args.status = ERR_DRAIN;
        }
        bool landed = !for_keys || num_tiles <= 0;
#pragma unroll 1
        for (unsigned tries = 0; tries < WAIT_LIMIT && !landed; ++tries) landed = mbar_try_wait(&sh->q_full, 0);
      }
    } else {
      // One issuing warp per chain, as in attention_tcgen05.cu: s_read(h) -> S(h + 1), p_full(h) -> PV(h).
      const int c = warp - 1;
      const int steps = c == 0 ? steps_0 : steps_1;
      if (steps > 0) {
        const unsigned leader = elect_one();
        auto wait_for = [&](unsigned long long* bar, unsigned parity) {
          return __all_sync(0xffffffffu, wait_bar(bar, parity, &sh->abort, args.status, ERR_MMA)) != 0;
        };
        const unsigned idesc_s = half_descriptor(BM, KEYS, false);
        const unsigned idesc_o = half_descriptor(BM, D, true);
        const unsigned tmem_chain = __shfl_sync(0xffffffffu, sh->tmem_base, 0) + c * CHAIN_COLS, tmem_o = tmem_chain + O_COL;
        const unsigned long long q_base = smem_descriptor(smem_u32(q_tiles + c * Q_BYTES));
        const unsigned long long k_desc0 = smem_descriptor(smem_u32(k_tiles));
        const unsigned long long v_desc0 = smem_descriptor(smem_u32(v_tiles), KV_HALF, 1024);
        bool ok = wait_for(&sh->q_ready[c], 0);
        auto issue_scores = [&](int h) {
          const int st = h % STAGES;
          ok = wait_for(&sh->k_full[st], (h / STAGES) & 1);
          if (!ok) return;
          fence_after_sync();
          const unsigned long long k_base = k_desc0 + static_cast<unsigned>((st * KV_TILE) >> 4);
#pragma unroll
          for (int kk = 0; kk < D / 16; ++kk)
            umma(leader, tmem_chain, q_base + (((kk / 4) * Q_HALF + (kk % 4) * 32) >> 4), k_base + (((kk / 4) * KV_HALF + (kk % 4) * 32) >> 4), idesc_s,
                 kk > 0 ? 1u : 0u);
          umma_commit(leader, &sh->s_full[c]);
          umma_commit(leader, &sh->k_free[st]);
        };
        // the later chain starts most of a step behind the earlier one, where that is not most of its time
        if (ok && c == 1 && steps_0 > 4) ok = wait_for(&sh->stagger, 0);
        if (ok) issue_scores(0);
#pragma unroll 1
        for (int h = 0; h < steps && ok; ++h) {
          if (h + 1 < steps) {
            ok = wait_for(&sh->s_read[c], h & 1);
            if (!ok) break;
            issue_scores(h + 1);
            if (!ok) break;
          }
          const int st = h % STAGES;
          ok = wait_for(&sh->v_full[st], (h / STAGES) & 1);
          if (ok) ok = wait_for(&sh->p_full[c][h & 1], (h >> 1) & 1);
          if (!ok) break;
          if (c == 0 && h == 0 && leader) mbar_arrive(&sh->stagger);   // on every path: the other issuer waits for it
          fence_after_sync();
          const unsigned long long v_base = v_desc0 + static_cast<unsigned>((st * KV_TILE) >> 4);
          const unsigned tmem_p = tmem_chain + P_COL + (h & 1) * 32;
#pragma unroll
          for (int kk = 0; kk < KEYS / 16; ++kk)
            umma_a_in_tmem(leader, tmem_o, tmem_p + kk * 8, v_base + ((kk * 16 * 128) >> 4), idesc_o, (h > 0 || kk > 0) ? 1u : 0u);
          umma_commit(leader, &sh->pv_done[c][h & 1]);
          if (h + 1 == steps) umma_commit(leader, &sh->pv_last[c]);
          umma_commit(leader, &sh->v_free[st]);
        }
      }
    }
  } else if (warp >= 20) {
    // ---- converters: two threads a key, each half of its codes
    fewer_registers<40>();
    const bool for_keys = warp < 24;
    const int row = threadIdx.x & 63, half = (threadIdx.x >> 6) & 1, first = half * MY_CHUNKS;
    const unsigned char* const raw = for_keys ? raw_k : raw_v;
    unsigned char* const tiles = for_keys ? k_tiles : v_tiles;
    unsigned long long* const raw_full = for_keys ? sh->raw_k_full : sh->raw_v_full;
    unsigned long long* const raw_free = for_keys ? sh->raw_k_free : sh->raw_v_free;
    unsigned long long* const full = for_keys ? sh->k_full : sh->v_full;
    unsigned long long* const free_again = for_keys ? sh->k_free : sh->v_free;
    auto scale_at = [&](int page, int i) -> long long {   // the place of this thread's key among the scales; -1: no such key
      if (page < 0 || page >= args.num_pages) return -1;
      return ((static_cast<long long>(page) * args.num_kv_heads + kv_head) << args.page_shift) + (((tile_lo + i) * KEYS + row) & (args.page_size - 1));
    };
    float k_scale = 0.f, v_scale = 0.f;
    int ahead = -1;   // this thread's page, two tiles ahead
    long long place = -1;
    if (scales) {
      place = scale_at(chunk_pages, 0);
      if (place >= 0) {
        k_scale = args.k_scales[place];
        v_scale = args.v_scales[place];
      }
      place = scale_at(next_pages, 1);
      ahead = load_page(2, row);
    }
#pragma unroll 1
    for (int i = 0; i < num_tiles; ++i) {
      const int st = i % STAGES, rs = i % RAW_STAGES;
      float next_k = 0.f, next_v = 0.f;
      if (scales) {
        if (place >= 0) {
          next_k = args.k_scales[place];
          next_v = args.v_scales[place];
        }
        place = scale_at(ahead, i + 2);
        ahead = load_page(i + 3, row);
      }
      bool ok = wait_bar(&raw_full[rs], (i / RAW_STAGES) & 1, &sh->abort, args.status, ERR_CONVERT);
      if (!__all_sync(0xffffffffu, ok)) break;
      ok = wait_bar(&free_again[st], ((i / STAGES) & 1) ^ 1, &sh->abort, args.status, ERR_CONVERT);
      if (!__all_sync(0xffffffffu, ok)) break;
      if (scales) {   // the softmax threads have read the scales of the tile that was here: its products are done
        sh->k_scale[st][row] = k_scale;
        sh->v_scale[st][row] = v_scale;
        const unsigned top = __reduce_max_sync(0xffffffffu, finite_bits(v_scale));
        const bool bad = __any_sync(0xffffffffu, !(fabsf(v_scale) < INFINITY));
        if (lane == 0) {
          int* tops = reinterpret_cast<int*>(&sh->v_top[st]) + (row >> 5);
          tops[0] = static_cast<int>(top >> 23) - 127 + (bad ? NOT_FINITE : 0);
          tops[2] = static_cast<int>(top >> 23) - 127;
        }
        k_scale = next_k;
        v_scale = next_v;
      }
#pragma unroll 1
      for (int c = 0; c < MY_CHUNKS; ++c) convert_chunk(raw + rs * RAW_TILE, tiles + st * KV_TILE, row, first + c);
      fence_async_shared();
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&raw_free[rs]);
        mbar_arrive(&full[st]);
      }
    }
  } else {
    // ---- softmax and epilogue: a warp has sixteen rows, four lanes a row, and a lane two rows
    more_registers<96>();
    const int chain = (warp - 4) >> 3, t = lane & 3;
    const int row0 = (warp & 3) * 32 + ((warp - 4) >> 2 & 1) * 16;   // this warp's first row, among the tensor memory lanes that it reaches
    const int my_steps = chain == 0 ? steps_0 : steps_1;
    const int chain_tokens = chain == 0 ? tokens_0 : tokens_1;
    // Row lane % 16 of the warp's is this lane's where queries come in and outputs leave.
    const int moved = row0 + (lane & 15), moved_token = chain * args.tokens + moved / args.group;
    const bool there = moved < args.tokens * args.group && tile_start + moved_token < q_len;
    // Between them it has rows lane / 4 and lane / 4 + 8.  A row that is not there (128 is no multiple of the group, or the
    // portion ends) has zeros for a query and sees what the chain's last token sees, so that it takes the same turns; nobody
    // reads it.
    int first[2], last[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      last[r] = pos0 + tile_start + chain * args.tokens + min((row0 + (lane >> 2) + 8 * r) / args.group, chain_tokens - 1);
      first[r] = first_visible_key(max(last[r], 0), args.window);
    }
    const int latest_first = max(first[0], first[1]), earliest_last = min(last[0], last[1]);
    const unsigned tmem_chain = sh->tmem_base + chain * CHAIN_COLS + (static_cast<unsigned>(row0) << 16), tmem_o = tmem_chain + O_COL;
    float most[2] = {-INFINITY, -INFINITY}, base[2] = {-INFINITY, -INFINITY}, row_sum[2] = {0.f, 0.f}, factor[2] = {0.f, 0.f};
    int exponent[2] = {LEAST_EXPONENT, LEAST_EXPONENT};
    bool ok = true;
    if (num_tiles > 0) {   // a chain without steps as well: its outputs leave by way of the tile that the queries land in
      ok = wait_bar(&sh->q_full, 0, &sh->abort, args.status, ERR_SOFTMAX);
      ok = __all_sync(0xffffffffu, ok);
      if (ok && my_steps > 0) {   // the query's row, half of it each of two lanes: scaled so that its largest element lies in [2^14, 2^15), then float16
        constexpr int MINE = HALVES * 4;   // 16-byte chunks of this thread
        unsigned char* q_row = q_tiles + chain * Q_BYTES + moved * 128;
        auto chunk_of = [&](int c) { return reinterpret_cast<uint4*>(q_row + (((lane >> 4) * MINE + c) / 8) * Q_HALF + (((((lane >> 4) * MINE + c) % 8) ^ (moved & 7)) << 4)); };
        uint4 x[MINE];
        unsigned top = 0u;   // the largest magnitude's upper sixteen bits
#pragma unroll
        for (int c = 0; c < MINE; ++c) {
          x[c] = *chunk_of(c);
          top = __vmaxu2(top, __vmaxu2(__vmaxu2(x[c].x & 0x7fff7fffu, x[c].y & 0x7fff7fffu), __vmaxu2(x[c].z & 0x7fff7fffu, x[c].w & 0x7fff7fffu)));
        }
        top = max(top & 0xffffu, top >> 16);
        if (top >= 0x7f80u) {   // an infinity or a NaN: of the finite elements, then
          top = 0u;
#pragma unroll
          for (int c = 0; c < MINE; ++c) {
            const unsigned w[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
#pragma unroll
            for (int i = 0; i < 4; ++i) top = max(top, max(finite_bits(__uint_as_float(w[i] << 16)), finite_bits(__uint_as_float(w[i] & 0xffff0000u))) >> 16);
          }
        }
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 16));
        const int e = min(max(static_cast<int>(top >> 7) - 127, -100), 126);
        const float lift = args.scale_log2 < 0.f ? -power_of_two(14 - e) : power_of_two(14 - e);
        const float own_factor = fmaxf(fabsf(args.scale_log2) * power_of_two(e - 14), 1e-38f);   // a hidden key's -inf has to stay one
#pragma unroll
        for (int r = 0; r < 2; ++r) factor[r] = __shfl_sync(0xffffffffu, own_factor, (lane >> 2) + 8 * r);
#pragma unroll
        for (int c = 0; c < MINE; ++c) {
          const unsigned w[4] = {x[c].x, x[c].y, x[c].z, x[c].w};
          unsigned h[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) h[i] = there ? pack_half(__uint_as_float(w[i] << 16) * lift, __uint_as_float(w[i] & 0xffff0000u) * lift) : 0u;   // whatever lay there
          *chunk_of(c) = make_uint4(h[0], h[1], h[2], h[3]);
        }
        fence_async_shared();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh->q_ready[chain]);
      }
    }
    unsigned phase = 0;   // of the stage
#pragma unroll 1
    for (int h = 0, st = 0; h < my_steps && ok; ++h, st = st + 1 == STAGES ? 0 : st + 1, phase ^= st == 0 ? 1u : 0u) {
      ok = wait_bar(&sh->v_full[st], phase, &sh->abort, args.status, ERR_SOFTMAX);   // the tile's scales
      if (ok) ok = wait_bar(&sh->s_full[chain], h & 1, &sh->abort, args.status, ERR_SOFTMAX);
      ok = __all_sync(0xffffffffu, ok);   // the warp stays together: the tensor-memory accesses below are warp-wide
      if (!ok) break;
      unsigned v[32];   // [4 j + 2 r + c]: row r, key 8 j + 2 t + c of the step
      const int key_base = (tile_lo + h) * KEYS;
      const bool edge = key_base < latest_first || key_base + KEYS - 1 > earliest_last;   // only steps at the edge of a row's range pay for masking
      fence_after_sync();
      tmem_load_fragments(tmem_chain, v);
      int top[2];
      const int2 tops = *reinterpret_cast<const int2*>(&sh->v_top[st]);
      const int tile_top = max(tops.x, tops.y);
      top[0] = top[1] = tile_top;
      float2 scale[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) scale[j] = *reinterpret_cast<const float2*>(sh->k_scale[st] + 8 * j + 2 * t);   // while the scores come
      tmem_wait_load();
      fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->s_read[chain]);    // the scores are in registers: their columns may take the next step
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        float x0, x1;
        halves_of(mul_pair(pair_of(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), pair_of(scale[i / 4].x, scale[i / 4].y)), x0, x1);
        v[i] = __float_as_uint(x0);
        v[i + 1] = __float_as_uint(x1);
      }
      const float* v_scale = sh->v_scale[st] + 2 * t;
      if (__builtin_expect(edge, 0)) {
        unsigned top_bits[2] = {0u, 0u};
#pragma unroll
        for (int i = 0; i < 32; ++i) {
          const int r = (i >> 1) & 1, within = 8 * (i / 4) + (i & 1), key = key_base + 2 * t + within;
          if (key < first[r] || key > last[r]) v[i] = 0xff800000u;   // -inf
          else top_bits[r] = max(top_bits[r], finite_bits(v_scale[within]));
        }
        top[0] = static_cast<int>(top_bits[0] >> 23) - 127;
        top[1] = static_cast<int>(top_bits[1] >> 23) - 127;
      }
      float step_max[2];
      bool moves = false;
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float part[2] = {-INFINITY, -INFINITY};
#pragma unroll
        for (int j = 0; j < 8; ++j) part[j & 1] = max3(part[j & 1], __uint_as_float(v[4 * j + 2 * r]), __uint_as_float(v[4 * j + 2 * r + 1]));
        step_max[r] = fmaxf(part[0], part[1]) * factor[r];
        top[r] -= SCALE_BITS;   // above MOST_EXPONENT the base never lags: the weights have no room for it
        moves = moves || step_max[r] > most[r] + BASE_LAG || top[r] > exponent[r] || most[r] == -INFINITY;
      }
      // The base follows the largest score lazily (2^6), and the largest value scale at once: the weights stay below 2^15.
      // The four lanes of a row have the same.
      bool rescales = false;
      float correction[2] = {1.0f, 1.0f};
      if (__builtin_expect(__any_sync(0xffffffffu, moves), 0)) {
        if (tile_top >= NOT_FINITE / 2 && !edge) top[0] = top[1] = max(sh->v_top[st].z, sh->v_top[st].w) - SCALE_BITS;
#pragma unroll
        for (int r = 0; r < 2; ++r) {
#pragma unroll
          for (int offset = 1; offset < 4; offset <<= 1) {
            step_max[r] = fmaxf(step_max[r], __shfl_xor_sync(0xffffffffu, step_max[r], offset));
            top[r] = max(top[r], __shfl_xor_sync(0xffffffffu, top[r], offset));
          }
          most[r] = fmaxf(most[r], step_max[r]);
          exponent[r] = max(exponent[r], min(top[r], MOST_EXPONENT));
          const float next = most[r] + static_cast<float>(exponent[r]);
          // a row that has seen no key yet has O = 0 and a sum of 0: nothing to rescale
          const float base_was = base[r];
          correction[r] = base_was == -INFINITY ? 1.0f : fast_exp2(base_was - next);
          base[r] = next;
          row_sum[r] = scale_sum(row_sum[r], fmaxf(base_was, -1e30f) - fmaxf(next, -1e30f));
        }
        rescales = h > 0 && __any_sync(0xffffffffu, correction[0] != 1.0f || correction[1] != 1.0f);
      }
      unsigned long long factor_pair[2], base_pair[2], sum_pair[4];
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const float from = base[r] == -INFINITY ? 0.f : -base[r];
        factor_pair[r] = pair_of(factor[r], factor[r]);
        base_pair[r] = pair_of(from, from);
        sum_pair[r] = sum_pair[2 + r] = pair_of(0.f, 0.f);
      }
      // one kind of instruction after the other over all elements: in the order of the elements each would wait for the one before
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        float x0, x1;
        halves_of(fma_pair(pair_of(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), factor_pair[(i >> 1) & 1], base_pair[(i >> 1) & 1]), x0, x1);
        v[i] = __float_as_uint(x0);
        v[i + 1] = __float_as_uint(x1);
      }
#pragma unroll
      for (int i = 0; i < 32; ++i) v[i] = __float_as_uint(fast_exp2(__uint_as_float(v[i])));
#pragma unroll
      for (int i = 0; i < 32; i += 2)
        sum_pair[(i >> 1) & 3] = add_pair(sum_pair[(i >> 1) & 3], pair_of(__uint_as_float(v[i]), __uint_as_float(v[i + 1])));
      unsigned weights[16];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float2 s = *reinterpret_cast<const float2*>(v_scale + 8 * j);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          float w0, w1;
          halves_of(mul_pair(pair_of(__uint_as_float(v[4 * j + 2 * r]), __uint_as_float(v[4 * j + 2 * r + 1])), pair_of(s.x, s.y)), w0, w1);
          weights[2 * j + r] = pack_half(w0, w1);
        }
      }
      if (__builtin_expect(tile_top >= NOT_FINITE / 2, 0)) {   // rare: a value that is no number
        // A key that a row does not see has no part in it, not even a scale of NaN.
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int key = key_base + 8 * (i / 2) + 2 * t;
          if (key < first[i & 1] || key > last[i & 1]) weights[i] &= 0xffff0000u;
          if (key + 1 < first[i & 1] || key + 1 > last[i & 1]) weights[i] &= 0x0000ffffu;
        }
        // The rows that see it are none either: by way of their sums, since its weight may be zero where splits are added up.
        const unsigned none = rows_of_no_number(v_scale, key_base + 2 * t, first[0], last[0], first[1], last[1]);
        if (none & 1u) row_sum[0] = __int_as_float(0x7fffffff);
        if (none & 2u) row_sum[1] = __int_as_float(0x7fffffff);
      }
      // P(h) goes where P(h - 2) was.  The product that read that was issued before the scores of step h, and a commit waits for
      // everything its thread has issued: s_full(h) says that it has been read.
      tmem_store_pairs(tmem_chain + P_COL + (h & 1) * 32, weights);   // keys 2 j and 2 j + 1 of the step in column j
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        float sum_lo, sum_hi;
        halves_of(add_pair(sum_pair[r], sum_pair[2 + r]), sum_lo, sum_hi);
        row_sum[r] += sum_lo + sum_hi;
      }
      if (__builtin_expect(rescales, 0)) {
        // O still takes the step before: wait for its PV, then rescale
        ok = wait_bar(&sh->pv_done[chain][(h - 1) & 1], ((h - 1) >> 1) & 1, &sh->abort, args.status, ERR_SOFTMAX);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        fence_after_sync();
        rescale_output_rows(tmem_o, correction[0], correction[1]);
      }
      tmem_wait_store();
      fence_before_sync();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh->p_full[chain][h & 1]);
    }
    if (ok && my_steps > 0) ok = wait_bar(&sh->pv_last[chain], 0, &sh->abort, args.status, ERR_SOFTMAX);
    ok = __all_sync(0xffffffffu, ok);
    fence_after_sync();
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
      for (int offset = 1; offset < 4; offset <<= 1) row_sum[r] += __shfl_xor_sync(0xffffffffu, row_sum[r], offset);
    // Outputs leave by way of the chain's query tile, which no product reads any more: 64 elements of the warp's rows a turn, so
    // that a store writes whole lines.
    const int token_head = there && ok ? (start + tile_start + moved_token) * args.num_heads + kv_head * args.group + moved % args.group : -1;
    const bool partial = args.splits > 1;
    bool nothing[2];
    float inv[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      nothing[r] = row_sum[r] == 0.f;   // a row that sees nothing is zeros
      inv[r] = nothing[r] ? 0.f : 1.0f / row_sum[r];
      const int at = __shfl_sync(0xffffffffu, token_head, (lane >> 2) + 8 * r);
      if (partial && at >= 0 && t == 0)
        *reinterpret_cast<float2*>(args.partial_ml + 2 * (static_cast<size_t>(split) * args.num_tokens * args.num_heads + at)) =
            make_float2(my_steps > 0 ? base[r] : -INFINITY, my_steps > 0 ? row_sum[r] : 0.f);
    }
    if (my_steps > 0 || !partial) {
      const int row_bytes = partial ? 256 : 128, lanes = row_bytes / 16, spread = partial ? 1 : 0;   // of 64 elements: lanes a row
      unsigned char* stage = q_tiles + chain * Q_BYTES;
#pragma unroll 1
      for (int turn = 0; turn < D / 64; ++turn) {
        unsigned o[32];
        if (my_steps > 0 && ok) {
          tmem_load_fragments(tmem_o + turn * 64, o);
          tmem_wait_load();
        } else {
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = 0u;
        }
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int row = row0 + (lane >> 2) + 8 * r;
          unsigned char* mine = stage + row * row_bytes;
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            if (partial) {
              *reinterpret_cast<uint2*>(mine + (((2 * j + (t >> 1)) ^ ((row & 7) << 1)) << 4) + 8 * (t & 1)) = make_uint2(o[4 * j + 2 * r], o[4 * j + 2 * r + 1]);
            } else {
              const float x = nothing[r] ? 0.f : __uint_as_float(o[4 * j + 2 * r]) * inv[r], y = nothing[r] ? 0.f : __uint_as_float(o[4 * j + 2 * r + 1]) * inv[r];
              *reinterpret_cast<__nv_bfloat162*>(mine + ((j ^ (row & 7)) << 4) + 4 * t) = __floats2bfloat162_rn(x, y);
            }
          }
        }
        __syncwarp();
        const int piece = lane & (lanes - 1), rows_at_once = 32 / lanes;
#pragma unroll 1
        for (int i = 0; i < 16 / rows_at_once; ++i) {
          const int within = i * rows_at_once + lane / lanes, from = row0 + within;
          const int at = __shfl_sync(0xffffffffu, token_head, within);
          const uint4 v = *reinterpret_cast<const uint4*>(stage + from * row_bytes + ((piece ^ ((from & 7) << spread)) << 4));
          if (at >= 0) {
            if (partial)
              *reinterpret_cast<uint4*>(args.partial_o + (static_cast<size_t>(split) * args.num_tokens * args.num_heads + at) * D + turn * 64 + piece * 4) = v;
            else
              *reinterpret_cast<uint4*>(args.out + static_cast<size_t>(at) * D + turn * 64 + piece * 8) = v;
          }
        }
        __syncwarp();   // the tile is written again in the next turn
      }
    }
  }
  fence_before_sync();
  __syncthreads();
  if (warp == 3) {
    fence_after_sync();
    tmem_free(sh->tmem_base, TMEM_COLS);
  }
}

// Adds up the splits of every query row of the portions: out = sum_s O_s 2^(base_s - M) / sum_s l_s 2^(base_s - M) with M the
// largest base.  One warp per (token, head), lanes over the splits first (bases and sums), then over the head size.  Tokens of
// one-token sequences belong to the other kernel and are left alone.
// The splits' rows are asked for four at a time, the first four before their weights are known.
__global__ void __launch_bounds__(256)
combine_portions_kernel(const Args args) {
  constexpr int VEC = D / 32, AT_ONCE = 4;
  let_dependents_start();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int token = blockIdx.y * 8 + warp, head = blockIdx.x;
  bool mine = token < args.num_tokens && token < args.q_start[args.num_seqs];   // rows behind the last sequence stay as they are
  if (mine) {
    const int seq = args.seq_of_token[token];
    mine = seq >= 0 && seq < args.num_seqs && !(args.skip_single && args.q_start[seq + 1] - args.q_start[seq] == 1);
  }
  wait_for_previous();
  if (!mine) return;
  const size_t token_head = static_cast<size_t>(token) * args.num_heads + head;
  const size_t slice = static_cast<size_t>(args.num_tokens) * args.num_heads;
  const float* rows = args.partial_o + token_head * D + lane * VEC;
  float v[AT_ONCE][VEC];
  auto load = [&](int first) {   // what a split that saw no key of this row left there is whatever it is
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i)
      if (first + i < args.splits) {
        const float* src = rows + (first + i) * slice * D;
        if constexpr (VEC == 4) {
          const float4 x = *reinterpret_cast<const float4*>(src);
          v[i][0] = x.x; v[i][1] = x.y; v[i][2] = x.z; v[i][3] = x.w;
        } else {
          const float2 x = *reinterpret_cast<const float2*>(src);
          v[i][0] = x.x; v[i][1] = x.y;
        }
      }
  };
  load(0);
  float2 ml = make_float2(-INFINITY, 0.f);            // lane s holds split s (at most 32 splits)
  if (lane < args.splits) ml = *reinterpret_cast<const float2*>(args.partial_ml + 2 * (lane * slice + token_head));
  const float m = ml.x, l = ml.y;
  float base = m;
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) base = fmaxf(base, __shfl_xor_sync(0xffffffffu, base, offset));
  const float weight = m == -INFINITY ? 0.f : fast_exp2(m - base);   // a split that saw no key of this row has base -inf
  float total = l != l ? l : m == -INFINITY ? 0.f : scale_sum(l, m - base);   // a score or a value that is no number makes the row none
#pragma unroll
  for (int offset = 16; offset > 0; offset >>= 1) total += __shfl_xor_sync(0xffffffffu, total, offset);
  float acc[VEC];
#pragma unroll
  for (int c = 0; c < VEC; ++c) acc[c] = 0.f;
  for (int first = 0; first < args.splits; first += AT_ONCE) {
    if (first > 0) load(first);
#pragma unroll
    for (int i = 0; i < AT_ONCE; ++i) {
      const float w = __shfl_sync(0xffffffffu, weight, (first + i) & 31);
      if (first + i < args.splits && w != 0.f)
#pragma unroll
        for (int c = 0; c < VEC; ++c) acc[c] += v[i][c] * w;
    }
  }
  const float inv = total == 0.f ? 0.f : 1.0f / total;
  unsigned packed[VEC / 2];
#pragma unroll
  for (int c = 0; c < VEC; c += 2) {
    const __nv_bfloat162 two = __floats2bfloat162_rn(acc[c] * inv, acc[c + 1] * inv);
    packed[c / 2] = *reinterpret_cast<const unsigned*>(&two);
  }
  __nv_bfloat16* dst = args.out + token_head * D + lane * VEC;
  if constexpr (VEC == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(packed[0], packed[VEC / 2 - 1]);
  else *reinterpret_cast<unsigned*>(dst) = packed[0];
}

// Tensor maps, kept by what they describe (host only).
struct Key {
  const void* base;
  long long rows;
  int a, b, c;
  bool operator==(const Key& o) const { return base == o.base && rows == o.rows && a == o.a && b == o.b && c == o.c; }
};
struct KeyHash {
  size_t operator()(const Key& k) const {
    size_t h = reinterpret_cast<size_t>(k.base);
    for (const long long v : {k.rows, static_cast<long long>(k.a), static_cast<long long>(k.b), static_cast<long long>(k.c)}) h = h * 1000003u ^ static_cast<size_t>(v);
    return h;
  }
};
template <typename Encode>
static int kept_map(const Key& key, CUtensorMap* out, Encode&& encode) {
  static std::mutex mutex;
  static std::unordered_map<Key, CUtensorMap, KeyHash> cache;
  EncodeTiled fn = encode_tiled();
  if (fn == nullptr) return SHRIKE_BAD_ARGUMENT;
  try {
    std::lock_guard<std::mutex> guard(mutex);
    const auto found = cache.find(key);
    if (found != cache.end()) {
      *out = found->second;
      return SHRIKE_OK;
    }
    const CUresult rc = encode(fn, out);
    if (rc != CUDA_SUCCESS) return 1000 + static_cast<int>(rc);
    if (cache.size() > 4096) cache.clear();
    cache.emplace(key, *out);
    return SHRIKE_OK;
  } catch (...) {   // out of memory for the table: the map itself is made
    return encode(fn, out) == CUDA_SUCCESS ? SHRIKE_OK : SHRIKE_BAD_ARGUMENT;
  }
}
// Codes [rows, cols bytes] as boxes of `box_rows` rows of D bytes, in the swizzle of that row length.
static int map_codes(const void* base, long long rows, int cols, int box_rows, CUtensorMap* out) {
  return kept_map(Key{base, rows, cols, box_rows, 1}, out, [&](EncodeTiled fn, CUtensorMap* map) {
    const cuuint64_t dims[2] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(rows)}, strides[1] = {static_cast<cuuint64_t>(cols)};
    const cuuint32_t box[2] = {D, static_cast<cuuint32_t>(box_rows)}, steps[2] = {1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
              D == 128 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_64B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  });
}
// Queries [tokens, heads, D] as boxes of `box_tokens` tokens, `group` heads and 64 elements in the 128-byte swizzle.
static int map_queries(const void* base, long long tokens, int heads, int group, int box_tokens, CUtensorMap* out) {
  return kept_map(Key{base, tokens, heads, group, 2}, out, [&](EncodeTiled fn, CUtensorMap* map) {
    const cuuint64_t dims[3] = {D, static_cast<cuuint64_t>(heads), static_cast<cuuint64_t>(tokens)};
    const cuuint64_t strides[2] = {D * 2, static_cast<cuuint64_t>(heads) * D * 2};
    const cuuint32_t box[3] = {64, static_cast<cuuint32_t>(group), static_cast<cuuint32_t>(box_tokens)}, steps[3] = {1, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  });
}

}  // namespace tcq8

// Tokens of a query tile for groups of `group` heads a kv head: what the caller counts the portions' tiles in; 0: not served.
SHRIKE_API int shrike_attention_q8_tc_tokens(int group) { return group >= 1 && group <= 64 ? 2 * (tcq8::BM / group) : 0; }

// The time of a batch whose portions make `tiles` query tiles over block tables of `keys` keys, in a key tile's time, and how
// many CTAs should share the keys of a query tile for it: the GPU holds one CTA per SM, so the time is that of the rounds of
// CTAs, each its key tiles and about CTA_START of their time for a CTA's start and end, and a split launch pays COMBINE more for
// the second kernel.  Measured (40 heads, 512 tokens over 8,192 keys, 88 CTAs' worth of query tiles): unsplit 164 us, two splits
// 170, three 127, four 145, five 131, six 148, eight 159; 12 heads, 475 tokens over 1,115 keys, 24 CTAs' worth: unsplit 28.5, two
// 22.0, four 18.0, six 17.2.
static long long portions_time(int tiles, int num_kv_heads, long long keys, int& splits) {
  constexpr long long CTA_START = 8, COMBINE = 4;
  const long long ctas = static_cast<long long>(num_kv_heads) * tiles, capacity = shrike_device().sm_count;
  const long long key_tiles = (keys + tcq8::KEYS - 1) / tcq8::KEYS;
  long long least = -1;
  for (int s = 1; s <= 32 && (s == 1 || key_tiles / s >= 2); ++s) {
    const long long rounds = (ctas * s + capacity - 1) / capacity;
    const long long time = rounds * ((key_tiles + s - 1) / s + CTA_START) + (s > 1 ? COMBINE : 0);
    if (least < 0 || time < least) {
      least = time;
      splits = s;
    }
  }
  return least;
}
SHRIKE_API int shrike_attention_q8_tc_time(int tiles, int num_kv_heads, long long keys) {
  int splits;
  return static_cast<int>(std::min(portions_time(tiles, num_kv_heads, keys, splits), 0x7fffffffll));
}
SHRIKE_API int shrike_attention_q8_tc_splits(int tiles, int num_kv_heads, long long keys) {
  int splits = 1;
  portions_time(tiles, num_kv_heads, keys, splits);
  return splits;
}
// Whether a batch's single tokens should be portions too (`all_tiles` query tiles then, `tiles` without them) instead of a launch
// of their own, which comes after the portions' and takes at least OWN_LAUNCH: a single token then wastes most of its CTA's rows,
// but the CTA runs beside the others where there are SMs left.  Measured, us, two launches and one: 28 heads, a portion of 64
// tokens beside 8 single tokens over 250 keys 18.0 and 12.1, over 1,000 keys 23.3 and 18.1; 40 heads, portions of up to 70 tokens
// beside 30 (288 CTAs) over 150 keys 19.0 and 20.2, one of 64 tokens beside 8 over 1,000 keys 26.4 and 27.4.
SHRIKE_API int shrike_attention_q8_tc_one_launch(int all_tiles, int tiles, int num_kv_heads, long long keys) {
  constexpr long long OWN_LAUNCH = 8;
  int splits;
  if (all_tiles > 65535) return 0;   // more than a launch takes
  return portions_time(all_tiles, num_kv_heads, keys, splits) <= portions_time(tiles, num_kv_heads, keys, splits) + OWN_LAUNCH ? 1 : 0;
}

// Portions (q_len > 1) of a batch; entries with q_len == 1 are skipped when skip_single.  `tiles`: the query tiles of
// shrike_attention_q8_tc_tokens(group) tokens that they make.  splits > 1 needs `scratch`, splits * num_tokens * num_heads *
// (D + 2) floats, and `seq_of_token`.
SHRIKE_API int shrike_paged_attention_q8_tc(const ShrikeAttentionQ8* call) {
  const auto& [q, k_codes, k_scales, v_codes, v_scales, block_table, q_start, ctx_len, seq_of_token, out, scratch, arrivals, status, stream, max_blocks,
               dtype, num_tokens, num_seqs, num_heads, num_kv_heads, page_size, num_pages, window, skip_single, has_portions, max_q_len, others, splits,
               cluster, tiles, scale] = *call;
  using namespace tcq8;
  if (num_seqs <= 0 || num_tokens <= 0 || tiles <= 0) return SHRIKE_OK;
  if (num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || num_heads / num_kv_heads > 64 || max_blocks <= 0 || num_pages <= 0 ||
      tiles > 65535 || static_cast<long long>(num_tokens) * num_heads > 0x7fffffff || (splits > 1 && num_tokens > 8 * 65535) || !(page_size == 8 || page_size == 16 || page_size == 32 || page_size == 64) || splits < 1 || splits > 32 ||
      static_cast<long long>(num_pages) * page_size > 0x7fffffff || static_cast<long long>(max_blocks) * page_size > 0x7fffffff - 4096 ||
      (splits > 1 && (scratch == nullptr || seq_of_token == nullptr)) ||
      (reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(k_codes) |
       reinterpret_cast<uintptr_t>(v_codes) | reinterpret_cast<uintptr_t>(scratch)) % 16)
    return SHRIKE_BAD_ARGUMENT;
  static PerDevice raised;
  const int raise_rc = shrike_raise_smem(raised, portions_kernel, SMEM);
  if (raise_rc != 0) return raise_rc;
  const int group = num_heads / num_kv_heads;
  CUtensorMap map_q, map_k, map_v;
  int rc = map_queries(q, num_tokens, num_heads, group, BM / group, &map_q);
  if (rc != SHRIKE_OK) return rc;
  rc = map_codes(k_codes, static_cast<long long>(num_pages) * page_size, num_kv_heads * D, page_size, &map_k);
  if (rc != SHRIKE_OK) return rc;
  rc = map_codes(v_codes, static_cast<long long>(num_pages) * page_size, num_kv_heads * D, page_size, &map_v);
  if (rc != SHRIKE_OK) return rc;
  Args args;
  args.k_scales = k_scales;
  args.v_scales = v_scales;
  args.block_table = block_table;
  args.q_start = q_start;
  args.ctx_len = ctx_len;
  args.out = static_cast<__nv_bfloat16*>(out);
  args.status = status;
  args.max_blocks = max_blocks;
  args.num_heads = num_heads;
  args.num_kv_heads = num_kv_heads;
  args.page_size = page_size;
  args.page_shift = __builtin_ctz(page_size);
  args.num_pages = num_pages;
  args.window = window;
  args.skip_single = skip_single;
  args.group = group;
  args.tokens = BM / group;
  args.scale_log2 = scale * LOG2E;
  args.splits = splits;
  args.num_tokens = num_tokens;
  args.num_seqs = num_seqs;
  args.seq_of_token = seq_of_token;
  args.partial_o = splits > 1 ? scratch : nullptr;   // rows first (16-byte stores), then the (base, sum) pairs
  args.partial_ml = splits > 1 ? scratch + static_cast<long long>(splits) * num_tokens * num_heads * D : nullptr;
  cudaError_t err = launch_dependent(portions_kernel, dim3(num_kv_heads, tiles, splits), dim3(THREADS), SMEM, stream, map_q, map_k, map_v, args);
  if (err != cudaSuccess) return static_cast<int>(err);
  if (splits > 1) {
    err = launch_dependent(combine_portions_kernel, dim3(num_heads, (num_tokens + 7) / 8), dim3(256), 0, stream, args);
    if (err != cudaSuccess) return static_cast<int>(err);
  }
  return shrike_launch_status();
}

#else  // other head sizes: the mma.sync kernel serves them

SHRIKE_API int shrike_attention_q8_tc_tokens(int) { return 0; }
SHRIKE_API int shrike_attention_q8_tc_time(int, int, long long) { return 0; }
SHRIKE_API int shrike_attention_q8_tc_splits(int, int, long long) { return 1; }
SHRIKE_API int shrike_attention_q8_tc_one_launch(int, int, int, long long) { return 0; }
SHRIKE_API int shrike_paged_attention_q8_tc(const ShrikeAttentionQ8*) { return SHRIKE_BAD_ARGUMENT; }

#endif
