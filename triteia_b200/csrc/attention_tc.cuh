// Attention of new tokens over a paged cache on the fifth-generation tensor cores: prompts, chunks and other calls of more than
// 16 rows for an average sequence, over caches of the inputs' type or e4m3 whose pages hold whole groups of 16 tokens.  Definition
// and masks as in attention.cuh.
//
// A CTA owns 256 rows (token, query head of the group) of one sequence and key head, as two tiles of 128, and walks the
// visible keys in tiles of 128.  While the tensor cores work on one tile, the other one's softmax runs:
//   scores   S = Q K^T   tcgen05.mma, both operands K-major in shared memory, S fp32 in tensor memory (128 columns a tile)
//   softmax  one thread per row: the row comes out of tensor memory into registers, no shuffle is needed; weights go back
//            as 16-bit numbers into the same columns
//   values   O += P V    A operand = the weights in tensor memory, B operand = V rows as they lie in memory (MN-major)
// so scores and weights never touch shared memory.  O stays in tensor memory; it is rescaled only when a row's maximum
// has grown by more than 2^8 since the last time (the weights are then at most 2^8 times what they would be, which fp32
// sums and fp16 or bf16 weights hold), so almost never after the first tiles.  Two row tiles in turn and the rare rescaling are
// known from published work on attention for this generation of tensor cores; roles, barriers and the e4m3 path are this file's.
//   warps 0-3, 4-7   softmax and epilogue of tile 0, 1 (TMEM lanes 32 * (warp % 4) ..)
//   warp 8           issues the MMAs (an elected lane), owns the tensor memory
//   warp 9           loads: one box per page and 64 sizes, a lane per page.  A page outside the cache, and boxes that no
//                    row sees, become boxes past the end of the cache, which TMA fills with zeros.
//   warps 10, 11     complete the third warpgroup, which hands registers to the other two; e4m3: exponents and factors; rows of
//                    the output that belong to no sequence, where they are to be zero
// Order of the MMAs: S0(0) S1(0), then for every key tile O0 += P0 V, S0(next), O1 += P1 V, S1(next): S(next) of a tile may
// overwrite its P because the pipe runs in order, and when S(next) is complete so is that tile's O.
//
// An e4m3 cache: the codes land in a ring of their own and four more warps (12-15) turn them into fp16 tiles, exactly: times
// 2^(e_j - E), E the largest exponent among their 128 tokens, but no less than 2^-15, the last factor that leaves every code a
// number of fp16.  What is left of the power enters per token, at the scores: the keys' as a factor, the values' as in
// attention.cuh, where 2^(t_j - m) with t_j = log2 weight + e_j meets the code of v_j.  A head of zeros has no part in E.
// Queries and weights are fp16 there whatever T is (queries scaled by a power of two per row).
//
// A call with few items over long keys gives each item to a cluster of 2, 4 or 8 CTAs, which walk a run of its key tiles each
// and join their states over distributed shared memory; the rule and its figures stand at the launch.
//
// Measured (32 heads of 128): a prompt of 8192 tokens over 32 key heads, fp16, 515 us = 1.07 PFLOP/s (600 to 615 us in a loop,
// where the power cap holds the clock at 1.64 GHz); five chunks of 20 to 700 tokens over 1020 to 6000, 8 key heads, bf16, 147 us in
// a graph and 153 as calls in a row; two chunks over 8362 and 12000 e4m3 tokens 308 and 311.  A key tile takes a CTA about 3400
// clocks, of which the MMAs need 2048 and the exponentials as many (16 a clock); the rest is the way of one tile from its scores to
// the next ones.  The prompt's 228 key tiles an SM are 395 us of that at 1.965 GHz and 473 at 1.64; the rest of its time, entry and
// exit of seven items an SM and the clock of a short run, is not told apart.  Calls of one to a few waves lose most to the last one.  Cutting them like the short calls (persistent CTAs, pieces joined) cost 8 us a piece and was
// slower (152 -> 190 us); so were clusters of two where they do not all run at once (chunks 144 -> 152, e4m3 300 -> 307).
// Moving a quarter or half of the exponentials to the multiply-add pipe changed the chunks by -2 and +1 %, the prompt by +1 and
// +6 %.
//
// Shared memory: 64 KB of queries and a ring of five 32 KB tiles (K0, V0, K1, ..) -- e4m3: three, and three of codes.
// 512 tensor memory columns: S and O of both tiles.
#pragma once

#include "attention.cuh"

namespace trb {

template <int D_, bool FP8_>
struct AttnTcCfg {
  static constexpr int D = D_;
  static constexpr bool FP8 = FP8_;
  static constexpr int HALVES = D / 64;                  // 128-byte swizzle atoms of a row
  static constexpr int TILE_BYTES = 128 * D * 2;         // 128 rows of queries, keys or values
  static constexpr int BUFS = FP8 ? 3 : 5;
  static constexpr int CODE_BYTES = 128 * D, CODE_BUFS = FP8 ? 3 : 0;
  static constexpr int Q_OFF = 0;
  static constexpr int KV_OFF = 2 * TILE_BYTES;
  static constexpr int CODE_OFF = KV_OFF + BUFS * TILE_BYTES;
  // e4m3, per key tile modulo 2: 2^E of the keys, E of the values, 2^-E, whether keys or values have rests; the values' rests
  // [128]; the powers that the keys' scores still need [128].
  static constexpr int EXP_OFF = CODE_OFF + CODE_BUFS * CODE_BYTES, EXP_FLOATS = 4 + 2 * 128;
  static constexpr int SCALE_OFF = EXP_OFF + (FP8 ? 2 * EXP_FLOATS * 4 : 0);      // fp16 [2][2][128]: factors of keys and values
  static constexpr int MAX_OFF = SCALE_OFF + (FP8 ? 2 * 2 * 128 * 2 : 0);         // int [2][2][2]: two warps' largest exponents
  static constexpr int BAR_OFF = MAX_OFF + (FP8 ? 32 : 0);
  static constexpr int NUM_BARS = 2 * BUFS + 1 + 4 * 2 + 2 * CODE_BUFS + 6;
  static constexpr int SMEM_BYTES = BAR_OFF + NUM_BARS * 8 + 16;
  static constexpr int SMEM_ALLOC = SMEM_BYTES + 1024;
  static constexpr int GROUPS = FP8 ? 4 : 3;             // warpgroups
  static constexpr int THREADS = GROUPS * 128;
  // Registers a thread: the softmax warps hold a row of 128 scores, the other warpgroups need few; together they stay
  // within what the launch has.
  static constexpr int LAUNCH_REGS = FP8 ? 128 : 168, SOFTMAX_REGS = FP8 ? 184 : 216, OTHER_REGS = 72;
  static_assert(2 * SOFTMAX_REGS + (GROUPS - 2) * OTHER_REGS <= GROUPS * LAUNCH_REGS, "the register split is covered by the launch");
  static constexpr uint32_t TMEM_COLS = 512;
  static constexpr uint32_t S_COL = 0, O_COL = 256;      // tile t: S_COL + 128 t, O_COL + 128 t
};
static_assert(AttnTcCfg<128, false>::SMEM_ALLOC <= 232448 && AttnTcCfg<128, true>::SMEM_ALLOC <= 232448, "shared memory of one CTA");

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(smem_u32(bar))
      : "memory");
}
// The issuing instructions below carry the elected lane as a predicate: the warp stays converged around them.
__device__ __forceinline__ void tc_commit_one(uint64_t* bar, uint32_t elected) {
  asm volatile(
      "{\n\t.reg .pred q;\n\tsetp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)), "r"(elected)
      : "memory");
}
// D[128, N] (+)= A[128, 16] B[16, N]; A and B in shared memory.
__device__ __forceinline__ void tc_mma_f16_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate,
                                              uint32_t elected) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d_tmem),
      "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(elected)
      : "memory");
}
// The same with A in tensor memory: 8 columns of two 16-bit numbers per row.
__device__ __forceinline__ void tc_mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate,
                                              uint32_t elected) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\tsetp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate), "r"(elected)
      : "memory");
}
// Waits for the warp's loads from tensor memory; the registers pass through, so that no use of them moves before it.
__device__ __forceinline__ void tc_wait_ld32(uint32_t (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(v[0]), "+r"(v[1]), "+r"(v[2]), "+r"(v[3]), "+r"(v[4]), "+r"(v[5]), "+r"(v[6]), "+r"(v[7]), "+r"(v[8]), "+r"(v[9]),
                 "+r"(v[10]), "+r"(v[11]), "+r"(v[12]), "+r"(v[13]), "+r"(v[14]), "+r"(v[15]), "+r"(v[16]), "+r"(v[17]), "+r"(v[18]),
                 "+r"(v[19]), "+r"(v[20]), "+r"(v[21]), "+r"(v[22]), "+r"(v[23]), "+r"(v[24]), "+r"(v[25]), "+r"(v[26]), "+r"(v[27]),
                 "+r"(v[28]), "+r"(v[29]), "+r"(v[30]), "+r"(v[31])::"memory");
}
__device__ __forceinline__ void tc_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(v[0]),
      "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]),
      "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tc_st32(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,"
      "%31,%32};" ::"r"(taddr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
      "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]),
      "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]),
      "r"(v[31])
      : "memory");
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// SPLIT: the 2, 4 or 8 CTAs of a cluster share an item, each with a run of its key tiles.  At the end CTA r finishes the rows of
// 8 / split softmax warps: the others send it those rows' outputs, maxima and sums, through distributed shared memory into its
// idle ring.
template <class T, class Cfg, bool SPLIT>
__global__ void __launch_bounds__(Cfg::THREADS, 1)
attn_tc_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v, const AttnArgs a, int tiles_bound,
               int box, int split) {
  using TM = typename AttnMma<T, Cfg::FP8>::type;
  constexpr int D = Cfg::D, BUFS = Cfg::BUFS, CODE_BUFS = Cfg::CODE_BUFS;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(smem + Cfg::BAR_OFF);   // a tile of keys or values has landed
  uint64_t* empty_bar = full_bar + BUFS;                                   // its MMAs have retired
  uint64_t* q_bar = empty_bar + BUFS;                                      // the queries are in shared memory
  uint64_t* s_bar = q_bar + 1;                                             // [2] scores complete
  uint64_t* p_bar = s_bar + 2;                                             // [2][2] weights of the first and the last 64 keys stored
  uint64_t* o_bar = p_bar + 4;                                             // [2] output complete
  uint64_t* code_full = o_bar + 2;                                         // e4m3: codes have landed,
  uint64_t* code_empty = code_full + CODE_BUFS;                            // have been read,
  uint64_t* exp_bar = code_empty + CODE_BUFS;                              // [2] the exponents of a key tile are there
  uint64_t* fac_bar = exp_bar + 2;                                         // [2] its factors are there,
  uint64_t* fac_free = fac_bar + 2;                                        // [2] both have been read
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(fac_free + 2);
  volatile int* dead = reinterpret_cast<volatile int*>(tmem_slot + 1);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

  // Late tiles of a causal prompt see the most keys: they go first.
  const int item = SPLIT ? blockIdx.x / split : blockIdx.x, rank = SPLIT ? blockIdx.x % split : 0;
  const int kvh = item % a.kv_heads;
  AttnTile t;
  if (!attn_find_tile<256>(a, tiles_bound - 1 - item / a.kv_heads, t)) {
    if (a.clear) attn_clear_rest<T, D>(a, tid, Cfg::THREADS);
    return;
  }
  int lo, hi;
  attn_key_range(a, t, lo, hi);
  // Key tiles [kt0, kt0 + n[i]) of this CTA concern the rows of tile i.
  const int all = hi > lo ? (hi + 127) / 128 - lo / 128 : 0;
  const int k0 = SPLIT ? (int)((long long)all * rank / split) : 0, k1 = SPLIT ? (int)((long long)all * (rank + 1) / split) : all;
  const int kt0 = lo / 128 + k0;
  const int base_pos = t.length - t.new_tokens;
  int n[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int rows = min(128, t.rows - 128 * i);
    int h = hi;
    if (a.causal && rows > 0) h = min(hi, base_pos + (t.row0 + 128 * i + rows - 1) / a.group + 1);
    // The same in every lane, which the reduction tells the compiler: loop counters and the MMAs' operands stay in uniform
    // registers.
    n[i] = __reduce_max_sync(0xffffffffu, rows > 0 && h > lo ? max(0, min((h + 127) / 128 - lo / 128, k1) - k0) : 0);
  }
  const int n_all = max(n[0], n[1]);

  if (tid == 0) {
    for (int i = 0; i < BUFS; ++i) {
      mbar_init(&full_bar[i], Cfg::FP8 ? 4 : 1);
      mbar_init(&empty_bar[i], 1);
    }
    for (int i = 0; i < CODE_BUFS; ++i) {
      mbar_init(&code_full[i], 1);
      mbar_init(&code_empty[i], 4);
    }
    mbar_init(q_bar, 8);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&exp_bar[i], 2);
      mbar_init(&fac_bar[i], 2);
      mbar_init(&fac_free[i], 4 + 8);
      mbar_init(&s_bar[i], 1);
      mbar_init(&p_bar[2 * i], 4);
      mbar_init(&p_bar[2 * i + 1], 4);
      mbar_init(&o_bar[i], 1);
    }
    *dead = 0;
    fence_mbar_init();
  }
  if (warp == 8) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(Cfg::TMEM_COLS)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = __reduce_max_sync(0xffffffffu, *tmem_slot);
  const uint32_t smem_base = smem_u32(smem);
  const int* table = a.page_table + t.seq * a.table_stride;

  if (warp >= 8 && warp < 12) {
   asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::OTHER_REGS));
   if (warp == 9) {
    // ------------------------------ loads ------------------------------
    const int boxes = 128 / box;                      // at most 8
    const bool mine = lane < boxes;
    if (lane == 0) {
      prefetch_tmap(&tm_k);
      prefetch_tmap(&tm_v);
    }
    int buf = 0;
    uint32_t phase = 0;
    for (int i = 0; i < n_all; ++i) {
      const int j = (kt0 + i) * 128 + lane * box;
      int page = -1, place = 0;
      if (mine && j < hi && j + box > lo) {
        const int p = a.page_shift >= 0 ? j >> a.page_shift : j / a.page_size;
        page = table[p];
        place = j - p * a.page_size;
      }
      if (page < 0 || page >= a.num_pages) page = (int)a.num_pages;     // past the end: zeros
#pragma unroll
      for (int kv = 0; kv < 2; ++kv) {
        if constexpr (Cfg::FP8) {
          mbar_wait(&code_empty[buf], phase ^ 1, dead);
          if (lane == 0) mbar_arrive_expect_tx(&code_full[buf], Cfg::CODE_BYTES);
          __syncwarp();
          const uint32_t dst = smem_base + Cfg::CODE_OFF + buf * Cfg::CODE_BYTES + lane * box * D;
          if (mine) tma_load_4d(dst, kv ? &tm_v : &tm_k, 0, kvh, place, page, &code_full[buf]);
          if (++buf == CODE_BUFS) { buf = 0; phase ^= 1; }
        } else {
          mbar_wait(&empty_bar[buf], phase ^ 1, dead);
          if (lane == 0) mbar_arrive_expect_tx(&full_bar[buf], Cfg::TILE_BYTES);
          __syncwarp();
          if (mine) {
            const uint32_t dst = smem_base + Cfg::KV_OFF + buf * Cfg::TILE_BYTES + lane * box * 128;
#pragma unroll
            for (int h = 0; h < Cfg::HALVES; ++h) tma_load_4d(dst + h * 16384, kv ? &tm_v : &tm_k, h * 64, kvh, place, page, &full_bar[buf]);
          }
          if (++buf == BUFS) { buf = 0; phase ^= 1; }
        }
      }
    }
   } else if (warp == 8) {
    // ------------------------------ MMAs ------------------------------
    constexpr uint32_t fmt = std::is_same<TM, __nv_bfloat16>::value ? 1u : 0u;
    constexpr uint32_t idesc_s = (1u << 4) | (fmt << 7) | (fmt << 10) | ((128u >> 3) << 17) | ((128u >> 4) << 24);
    constexpr uint32_t idesc_o = (1u << 4) | (fmt << 7) | (fmt << 10) | (1u << 16) | (((uint32_t)D >> 3) << 17) | ((128u >> 4) << 24);
    auto scores = [&](int tile, int buf) {            // S[tile] = Q[tile] K^T
      const uint64_t qd = tc_smem_desc(smem_base + Cfg::Q_OFF + tile * Cfg::TILE_BYTES);
      const uint64_t kd = tc_smem_desc(smem_base + Cfg::KV_OFF + buf * Cfg::TILE_BYTES);
      const uint32_t one = elect_one();
#pragma unroll
      for (int k = 0; k < D / 16; ++k) {              // 32 bytes along a row; the next 64 sizes are 16 KB further
        const uint64_t step = (uint64_t)((k >> 2) * (16384 >> 4) + (k & 3) * 2);
        tc_mma_f16_ss(tmem + Cfg::S_COL + tile * 128, qd + step, kd + step, idesc_s, k > 0, one);
      }
      tc_commit_one(&s_bar[tile], one);
      __syncwarp();
    };
    // O[tile] += P[tile] V, 64 keys as soon as their weights are there.
    auto outputs = [&](int tile, int buf, int i) {
      const uint32_t v = smem_base + Cfg::KV_OFF + buf * Cfg::TILE_BYTES;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        mbar_wait(&p_bar[2 * tile + h], i & 1, dead);
        tc_fence_after();
        const uint32_t one = elect_one();
#pragma unroll
        for (int k = 4 * h; k < 4 * h + 4; ++k)       // 16 tokens = 16 rows of 128 bytes
          tc_mma_f16_ts(tmem + Cfg::O_COL + tile * 128, tmem + Cfg::S_COL + tile * 128 + k * 8, tc_smem_desc_mn(v + k * 2048, 16384, 1024),
                        idesc_o, i > 0 || k > 0, one);
        if (h == 1 && i + 1 == n[tile]) tc_commit_one(&o_bar[tile], one);
        __syncwarp();
      }
    };
    auto release = [&](int buf) {
      tc_commit_one(&empty_bar[buf], elect_one());
      __syncwarp();
    };
    // Items of the ring: K of key tile i is number 2i, V number 2i + 1.
    auto landed = [&](int x) { mbar_wait(&full_bar[x % BUFS], (x / BUFS) & 1, dead); };
    if (n_all > 0) {
      mbar_wait(q_bar, 0, dead);
      landed(0);
      tc_fence_after();
      for (int i = 0; i < 2; ++i)
        if (n[i] > 0) scores(i, 0);
      release(0);
    }
    for (int i = 0; i < n_all; ++i) {
      const int vbuf = (2 * i + 1) % BUFS, kbuf = (2 * i + 2) % BUFS;
      landed(2 * i + 1);
      // Values of tokens that no row sees may be anything, and 0 * NaN is NaN: they become zeros (of an e4m3 cache they
      // are zeros already).
      const int j0 = (kt0 + i) * 128, from = max(0, lo - j0), to = min(128, hi - j0);
      if (!Cfg::FP8 && (from > 0 || to < 128)) {
        const uint32_t v = smem_base + Cfg::KV_OFF + vbuf * Cfg::TILE_BYTES;
        for (int x = lane; x < 128 * 8 * Cfg::HALVES; x += 32) {      // 16 bytes each
          const int r = (x >> 3) & 127;
          if (r < from || r >= to) asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(v + x * 16), "r"(0) : "memory");
        }
        fence_proxy_async();
        __syncwarp();
      }
      const bool more = i + 1 < n_all;
      for (int tile = 0; tile < 2; ++tile) {
        if (i < n[tile]) outputs(tile, vbuf, i);
        if (more && tile == 0) landed(2 * i + 2);
        if (i + 1 < n[tile]) scores(tile, kbuf);
      }
      release(vbuf);
      if (more) release(kbuf);
    }
   } else if (Cfg::FP8) {
    // ------------------------------ e4m3: exponents and factors (warps 10, 11) ------------------------------
    // A lane has two tokens of a key tile.  Page numbers are asked for two tiles ahead and exponents one, so that neither load
    // is waited for.
    const int first = (warp - 10) * 32 + lane;
    int page[2], place[2], kb[2], vb[2];              // of the next tile but one; of the next tile (-1: not there)
    long long code_at[2];                             // the next tile's codes
    auto ask_pages = [&](int i) {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int j = (kt0 + i) * 128 + first + 64 * x;
        page[x] = -1;
        place[x] = 0;
        if (i < n_all && j >= lo && j < hi) {
          const int p = a.page_shift >= 0 ? j >> a.page_shift : j / a.page_size;
          page[x] = table[p];
          place[x] = j - p * a.page_size;
        }
      }
    };
    auto ask_exps = [&]() {
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        kb[x] = vb[x] = -1;
        code_at[x] = 0;
        if (page[x] >= 0 && page[x] < a.num_pages) {
          const long long at = (long long)page[x] * a.e_page + (long long)place[x] * a.e_tok + (long long)kvh * a.e_head;
          kb[x] = a.key_exp[at];
          vb[x] = a.value_exp[at];
          code_at[x] = (long long)page[x] * a.c_page + (long long)place[x] * a.c_tok + (long long)kvh * a.c_head;
        }
      }
    };
    int2* maxima = reinterpret_cast<int2*>(smem + Cfg::MAX_OFF);
    ask_pages(0);
    ask_exps();
    ask_pages(1);
    for (int i = 0; i < n_all; ++i) {
      const int s = i & 1;
      // The slot is free once the converting warps have its factors and every softmax that uses the tile its exponents.
      mbar_wait(&fac_free[s], ((i >> 1) & 1) ^ 1, dead);
      // A head of zeros (byte 127) takes the tile's exponent, whatever it is, and has no part in it.
      if (__any_sync(0xffffffffu, kb[0] == 127 || kb[1] == 127 || vb[0] == 127 || vb[1] == 127)) {
        // In line: these warps have given registers away, which a function would not know.  And small, for the loops around it
        // (two chunks over 12000 tokens in a graph: 310 us, with all loads of a head in flight 318).  Where every head has the
        // byte 127 (largest magnitudes of 224 to 448) chunks take 3 % longer, where all value heads are zeros 46 %.
#pragma unroll 1
        for (int x = 0; x < 4; ++x) {                 // keys and values of two tokens; real ones end at their first codes
          const int byte = x == 0 ? kb[0] : x == 1 ? kb[1] : x == 2 ? vb[0] : vb[1];
          bool zeros = byte == 127;
          const uint4* codes = reinterpret_cast<const uint4*>(static_cast<const uint8_t*>(x < 2 ? a.key_cache : a.value_cache) +
                                                              (x & 1 ? code_at[1] : code_at[0]));
#pragma unroll 1
          for (int y = 0; zeros && y < D / 16; ++y) zeros = attn_zero_codes(codes[y]);
          if (zeros) {
            if (x == 0) kb[0] = -1;
            else if (x == 1) kb[1] = -1;
            else if (x == 2) vb[0] = -1;
            else vb[1] = -1;
          }
        }
      }
      const int2 most = make_int2(__reduce_max_sync(0xffffffffu, max(kb[0], kb[1])), __reduce_max_sync(0xffffffffu, max(vb[0], vb[1])));
      if (lane == 0) maxima[2 * s + (warp - 10)] = most;
      named_bar_sync(1, 64);
      const int2 m0 = maxima[2 * s], m1 = maxima[2 * s + 1];
      int ek = max(m0.x, m1.x), ev = max(m0.y, m1.y);
      if (ek < 0) ek = 127;                           // no token of the tile is there, or all of its keys are zeros
      if (ev < 0) ev = 127 + kZeroValueExp;           // the same of its values
      float* e = reinterpret_cast<float*>(smem + Cfg::EXP_OFF) + s * Cfg::EXP_FLOATS;
      __half* scales = reinterpret_cast<__half*>(smem + Cfg::SCALE_OFF) + s * 256;
      bool any = false;
#pragma unroll
      for (int x = 0; x < 2; ++x) {
        const int tok = first + 64 * x;
        const int kd = min(ek - kb[x], 15), vd = min(ev - vb[x], 15);
        const float rest = vb[x] >= 0 ? (float)(vb[x] + vd - ev) : 0.f;
        const int k_up = kb[x] >= 0 ? kb[x] + kd : ek;
        scales[tok] = __float2half_rn(pow2_of_byte(127 - kd));
        scales[128 + tok] = __float2half_rn(pow2_of_byte(127 - vd));
        e[4 + tok] = rest;
        e[132 + tok] = pow2_of_byte(k_up);
        any |= rest != 0.f || k_up != ek;
      }
      any = __any_sync(0xffffffffu, any);
      if (lane == 0) reinterpret_cast<uint16_t*>(e + 3)[warp - 10] = any ? 1 : 0;      // two halves, read as one number
      if (tid == 320) {
        e[0] = pow2_of_byte(ek);
        e[1] = (float)(ev - 127);
        e[2] = pow2_of_byte(254 - ev);
      }
      __syncwarp();
      if (lane == 0) {
        mbar_arrive(&fac_bar[s]);
        mbar_arrive(&exp_bar[s]);
      }
      ask_exps();
      ask_pages(i + 2);
    }
   }
   if (warp >= 10 && a.clear) attn_clear_rest<T, D>(a, tid - 320, 64);      // these warps have the least to do
   if constexpr (SPLIT) {
     __syncwarp();
     cluster_sync_all();
     cluster_sync_all();
   }
  } else if (warp >= 12) {
    // ------------------------------ e4m3: codes -> fp16 tiles ------------------------------
    if constexpr (Cfg::FP8) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Cfg::OTHER_REGS));
      const int ct = tid - 384;                       // 0 .. 127
      constexpr int CH = D / 16;                      // 16-byte pieces of a token's codes
      constexpr int PASSES = 128 * CH / 128;
      const int ch = ct % CH, r0 = ct / CH;
      int buf = 0, cbuf = 0;
      uint32_t phase = 0, cphase = 0;
      for (int i = 0; i < n_all; ++i) {
        const int j0 = (kt0 + i) * 128;
        mbar_wait(&fac_bar[i & 1], (i >> 1) & 1, dead);
        const __half* scales = reinterpret_cast<const __half*>(smem + Cfg::SCALE_OFF) + (i & 1) * 256;
#pragma unroll 1
        for (int kv = 0; kv < 2; ++kv) {
          mbar_wait(&code_full[cbuf], cphase, dead);
          uint4 w[PASSES];
          __half2 f[PASSES];
#pragma unroll
          for (int x = 0; x < PASSES; ++x) f[x] = __half2half2(scales[kv * 128 + r0 + x * (128 / CH)]);
          const uint32_t src = smem_base + Cfg::CODE_OFF + cbuf * Cfg::CODE_BYTES + ct * 16;
#pragma unroll
          for (int x = 0; x < PASSES; ++x) {
            w[x] = lds128(src + x * 2048);
            const int j = j0 + r0 + x * (128 / CH);
            if (j < lo || j >= hi) w[x] = make_uint4(0, 0, 0, 0);        // tokens that no row sees: anything may lie there
          }
          fence_proxy_async();                        // TMA writes the buffer through another proxy than these reads
          __syncwarp();
          if (lane == 0) mbar_arrive(&code_empty[cbuf]);
          if (++cbuf == CODE_BUFS) { cbuf = 0; cphase ^= 1; }
          mbar_wait(&empty_bar[buf], phase ^ 1, dead);
          const uint32_t dst = smem_base + Cfg::KV_OFF + buf * Cfg::TILE_BYTES;
#pragma unroll
          for (int x = 0; x < PASSES; ++x) {
            const int r = r0 + x * (128 / CH);
            auto times = [&](uint32_t h) {
              const __half2 y = __hmul2(*reinterpret_cast<const __half2*>(&h), f[x]);
              return *reinterpret_cast<const uint32_t*>(&y);
            };
            const uint32_t c4[4] = {w[x].x, w[x].y, w[x].z, w[x].w};
            // Sizes 16 ch .. + 15: two 16-byte pieces of the fp16 row.  Lanes of the second half of a row store them the
            // other way round, so that a row's lanes meet all eight bank groups.
#pragma unroll
            for (int y = 0; y < 2; ++y) {
              const int z = y ^ (CH == 8 ? (ch >> 2) : 0);
              const int piece = 2 * ch + z;
              const uint32_t lo4 = z ? c4[2] : c4[0], hi4 = z ? c4[3] : c4[1];
              const uint32_t at = dst + (piece >> 3) * 16384 + r * 128 + (((piece & 7) ^ (r & 7)) << 4);
              asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(times(e4m3x2_to_half2(lo4))),
                           "r"(times(e4m3x2_hi_to_half2(lo4))), "r"(times(e4m3x2_to_half2(hi4))), "r"(times(e4m3x2_hi_to_half2(hi4)))
                           : "memory");
            }
          }
          fence_proxy_async();
          __syncwarp();
          if (lane == 0) mbar_arrive(&full_bar[buf]);
          if (++buf == BUFS) { buf = 0; phase ^= 1; }
        }
        if (lane == 0) mbar_arrive(&fac_free[i & 1]);
      }
      if constexpr (SPLIT) {
        __syncwarp();
        cluster_sync_all();
        cluster_sync_all();
      }
    }
  } else {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Cfg::SOFTMAX_REGS));
    // ------------------------------ softmax: a thread per row ------------------------------
    const int tile = warp >> 2, quarter = warp & 3;
    const int row = quarter * 32 + lane;              // of the tile
    const int trow = tile * 128 + row;                // of the work item
    const bool on = trow < t.rows;
    const int rq = t.row0 + (on ? trow : 0);
    const int qi = rq / a.group, head = kvh * a.group + (rq - qi * a.group);
    const uint32_t qtile = smem_base + Cfg::Q_OFF + tile * Cfg::TILE_BYTES;
    // A negative scale turns the sign of the queries, so that the largest score is the largest product.
    float c = fmaxf(fabsf(a.scale_log2), 1e-35f);     // a scale of zero: masked scores stay -inf
    {
      const T* qp = static_cast<const T*>(a.query) + (long long)(t.q0 + qi) * a.q_tok + (long long)head * a.q_head;
      const uint32_t flip = a.scale_log2 < 0.f ? 0x80008000u : 0u;
      // The whole row on its way before the first store, which no load may pass.
      uint4 w[D / 8];
#pragma unroll
      for (int x = 0; x < D / 8; ++x) w[x] = on ? *reinterpret_cast<const uint4*>(qp + x * 8) : make_uint4(0, 0, 0, 0);
      if constexpr (!std::is_same<T, TM>::value) {    // bf16 as fp16: see AttnMma
        float top = 0.f;
#pragma unroll
        for (int x = 0; x < D / 8; ++x) {
          const uint32_t word[4] = {w[x].x, w[x].y, w[x].z, w[x].w};
#pragma unroll
          for (int y = 0; y < 4; ++y) {
            const float2 v = two_of(word[y], T());
            top = fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y)));
          }
        }
        const int k = attn_row_shift(top);
        const float up = __uint_as_float((uint32_t)k << 23);
        c *= __uint_as_float((uint32_t)(254 - k) << 23);
        auto scaled = [&](uint32_t word) { return word_of(mul2(two_of(word, T()), make_float2(up, up)), TM()); };
#pragma unroll
        for (int x = 0; x < D / 8; ++x) w[x] = make_uint4(scaled(w[x].x), scaled(w[x].y), scaled(w[x].z), scaled(w[x].w));
      }
#pragma unroll
      for (int x = 0; x < D / 8; ++x) {
        const uint32_t at = qtile + (x >> 3) * 16384 + row * 128 + (((x & 7) ^ (row & 7)) << 4);
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(w[x].x ^ flip), "r"(w[x].y ^ flip), "r"(w[x].z ^ flip),
                     "r"(w[x].w ^ flip)
                     : "memory");
      }
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) mbar_arrive(q_bar);
    }
    const int pos = base_pos + qi;
    const int row_hi = a.causal ? min(hi, pos + 1) : hi;
    const int row_lo = a.window > 0 ? pos - a.window + 1 : 0;
    // Tokens [all_lo, all_hi) are seen by every row of the warp.
    const int first_row = t.row0 + tile * 128 + quarter * 32, last_row = t.row0 + min(tile * 128 + quarter * 32 + 31, t.rows - 1);
    const int all_hi = a.causal ? min(hi, base_pos + first_row / a.group + 1) : hi;
    const int all_lo = a.window > 0 ? base_pos + last_row / a.group - a.window + 1 : 0;
    const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
    const uint32_t s_addr = tmem + lanes + Cfg::S_COL + tile * 128, o_addr = tmem + lanes + Cfg::O_COL + tile * 128;
    constexpr float kBias = AttnBias<TM>::value / 2;   // weights: at most 2^(8 + 4) in fp16
    float m = -INFINITY, l = 0.f;

    // Page of this lane's 16-token group of key tile i (lanes 0-7); 0 for tokens that no row sees.  Asked for a tile ahead and
    // looked at only then: the load would otherwise stand in the loop (600 of 3400 clocks a tile).
    auto page_of = [&](int i) -> int {
      const int j = (kt0 + i) * 128 + lane * 16;
      if (lane >= 8 || i >= n[tile] || j >= hi || j + 16 <= lo) return 0;
      return table[a.page_shift >= 0 ? j >> a.page_shift : j / a.page_size];
    };
    int page = page_of(0);
    for (int i = 0; i < n[tile]; ++i) {
      // Which of the groups are in the cache (bit g).
      const uint32_t there = __ballot_sync(0xffffffffu, page >= 0 && page < a.num_pages);
      page = page_of(i + 1);
      const int j0 = (kt0 + i) * 128;
      mbar_wait(&s_bar[tile], i & 1, dead);
      tc_fence_after();
      // e4m3: the tile's codes carry 2^(e_j - E) already, E the largest exponent of the tile (one for keys, one for values).
      // Further than 2^15 below, codes would lose bits in fp16: they carry 2^-15 and the token keeps a rest, values in the
      // exponent of the weight, keys in the factor of the score.
      float ct = c, add = 0.f, back = 1.f;
      const float* fac = nullptr;
      bool rests = false;
      if constexpr (Cfg::FP8) {
        mbar_wait(&exp_bar[i & 1], (i >> 1) & 1, dead);
        fac = reinterpret_cast<const float*>(smem + Cfg::EXP_OFF) + (i & 1) * Cfg::EXP_FLOATS;
        ct = fmaxf(c * fac[0], 1e-35f);               // never zero: masked scores stay -inf
        add = fac[1];
        back = fac[2];
        rests = reinterpret_cast<const int*>(fac)[3] != 0;
      }
      const float cs = rests ? 1.f : ct;
      const bool masked = there != 0xffffffffu || j0 + 128 > all_hi || j0 < all_lo;
      // Bit x: this row sees token j0 + 32 b + x.
      auto seen = [&](int b) -> uint32_t {
        const int h = row_hi - j0 - 32 * b, lw = row_lo - j0 - 32 * b;
        uint32_t bits = h >= 32 ? 0xffffffffu : h <= 0 ? 0u : (1u << h) - 1u;
        bits &= lw <= 0 ? 0xffffffffu : lw >= 32 ? 0u : ~((1u << lw) - 1u);
        return bits & (((there >> (2 * b)) & 1 ? 0xffffu : 0u) | ((there >> (2 * b + 1)) & 1 ? 0xffff0000u : 0u));
      };
      auto mask = [&](uint32_t (&w)[32], uint32_t bits) {
#pragma unroll
        for (int x = 0; x < 32; ++x) w[x] = (bits >> x) & 1 ? w[x] : 0xff800000u;      // -inf
      };
      // Masks and rests are rare and go through tensor memory, which keeps their code out of the loops below: with it the
      // loops ran out of the instruction cache (e4m3, two chunks over 12000 tokens: 467 us, without 311).
      if (masked || rests) {
#pragma unroll 1
        for (int b = 0; b < 4; ++b) {
          uint32_t w[32];
          tc_ld32(s_addr + b * 32, w);
          tc_wait_ld32(w);
          if (rests) {
#pragma unroll
            for (int x = 0; x < 32; x += 4) {
              const float4 k4 = *reinterpret_cast<const float4*>(fac + 132 + b * 32 + x), r4 = *reinterpret_cast<const float4*>(fac + 4 + b * 32 + x);
              w[x] = __float_as_uint(fmaf(__uint_as_float(w[x]), c * k4.x, r4.x));
              w[x + 1] = __float_as_uint(fmaf(__uint_as_float(w[x + 1]), c * k4.y, r4.y));
              w[x + 2] = __float_as_uint(fmaf(__uint_as_float(w[x + 2]), c * k4.z, r4.z));
              w[x + 3] = __float_as_uint(fmaf(__uint_as_float(w[x + 3]), c * k4.w, r4.w));
            }
          }
          mask(w, seen(b));
          tc_st32(s_addr + b * 32, w);
        }
        tc_wait_st();
      }
      // The whole row in registers; e4m3, where four more warps need some: read twice, 32 scores at a time and the next 32 on
      // their way, once for the maximum and once for the weights (a row held there spills; the other way round, a second
      // reading costs 4%: 8192-token prompt 551 -> 577 us).
      constexpr int HELD = Cfg::FP8 ? 2 : 4;
      uint32_t v[HELD][32];
      float mx = -INFINITY;
#pragma unroll
      for (int b = 0; b < HELD - 1; ++b) tc_ld32(s_addr + b * 32, v[b]);
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        uint32_t (&w)[32] = v[b % HELD];
        if (Cfg::FP8) {
          tc_wait_ld32(w);
          if (b < 3) tc_ld32(s_addr + (b + 1) * 32, v[(b + 1) % HELD]);
        } else if (b == 0) {
          tc_ld32(s_addr + 96, v[HELD - 1]);
#pragma unroll
          for (int x = 0; x < HELD; ++x) tc_wait_ld32(v[x]);
        }
        float m4[4];
#pragma unroll
        for (int x = 0; x < 4; ++x) m4[x] = max3(__uint_as_float(w[x]), __uint_as_float(w[x + 4]), __uint_as_float(w[x + 8]));
#pragma unroll
        for (int x = 12; x < 28; x += 8)
#pragma unroll
          for (int y = 0; y < 4; ++y) m4[y] = max3(m4[y], __uint_as_float(w[x + y]), __uint_as_float(w[x + 4 + y]));
#pragma unroll
        for (int y = 0; y < 4; ++y) mx = max3(mx, m4[y], __uint_as_float(w[28 + y]));
      }
      if (Cfg::FP8) tc_ld32(s_addr, v[0]);
      const float top = fmaf(mx, cs, add);
      const float m_new = fmaxf(m, top);
      if (__any_sync(0xffffffffu, m_new > m + 8.f)) {
        if (i > 0) {
          // This tile's S is complete, so its last O is too.
          const float alpha = m == -INFINITY ? 1.f : exp2_fast(m - m_new);        // nothing in O yet: nothing to scale
          l *= alpha;
#pragma unroll
          for (int b = 0; b < D / 32; ++b) {
            uint32_t o[32];
            tc_ld32(o_addr + b * 32, o);
            tc_wait_ld32(o);
#pragma unroll
            for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * alpha);
            tc_st32(o_addr + b * 32, o);
          }
        }
        m = m_new;
      }
      const float off = kBias + add - (m == -INFINITY ? 0.f : m);
      const float2 c2 = make_float2(cs, cs), off2 = make_float2(off, off);
      float2 sum = make_float2(0.f, 0.f);
      float rest_sum = 0.f;                           // of the weights without the values' exponents
      if (Cfg::FP8 && rests) {
#pragma unroll 1
        for (int b = 0; b < 4; ++b) {
          uint32_t w[32];
          tc_ld32(s_addr + b * 32, w);
          tc_wait_ld32(w);
#pragma unroll
          for (int x = 0; x < 32; x += 4) {
            const float4 r4 = *reinterpret_cast<const float4*>(fac + 4 + b * 32 + x);
            rest_sum += exp2_fast(__uint_as_float(w[x]) - r4.x + (off - add));
            rest_sum += exp2_fast(__uint_as_float(w[x + 1]) - r4.y + (off - add));
            rest_sum += exp2_fast(__uint_as_float(w[x + 2]) - r4.z + (off - add));
            rest_sum += exp2_fast(__uint_as_float(w[x + 3]) - r4.w + (off - add));
          }
        }
      }
#pragma unroll
      for (int b = 0; b < 4; ++b) {
        uint32_t (&w)[32] = v[b % HELD];
        if (Cfg::FP8) {
          tc_wait_ld32(w);
          if (b < 3) tc_ld32(s_addr + (b + 1) * 32, v[(b + 1) % HELD]);
        }
        uint32_t p[16];
#pragma unroll
        for (int x = 0; x < 16; ++x) {
          const float2 sc = make_float2(__uint_as_float(w[2 * x]), __uint_as_float(w[2 * x + 1]));
          float2 y = fma2(sc, c2, off2);
          y.x = exp2_fast(y.x);
          y.y = exp2_fast(y.y);
          sum = add2(sum, y);
          p[x] = pack2(y.x, y.y, TM());
        }
        tc_st16(s_addr + b * 16, p);                  // over scores that have been read
        if (b & 1) {
          tc_wait_st();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(&p_bar[2 * tile + (b >> 1)]);
        }
      }
      l = rests ? l + rest_sum : fmaf(sum.x + sum.y, back, l);
      if (Cfg::FP8 && lane == 0) mbar_arrive(&fac_free[i & 1]);
    }
    if (Cfg::FP8) {                                   // the other tile's last key tiles: this one has no use for them
      for (int i = n[tile]; i < n_all; ++i) {
        mbar_wait(&exp_bar[i & 1], (i >> 1) & 1, dead);
        if (lane == 0) mbar_arrive(&fac_free[i & 1]);
      }
    }
    // ------------------------------ epilogue ------------------------------
    if (n[tile] > 0) {
      mbar_wait(&o_bar[tile], 0, dead);
      tc_fence_after();
    } else {
      mbar_wait(q_bar, 0, dead);                      // the staging rows below are the queries' rows
    }
    // SPLIT: the ring takes [sender][row] of float [D + 4], then as many pairs of maximum and sum.
    constexpr int kRow = (D + 4) * 4;
    static_assert(224 * (kRow + 8) <= Cfg::EXP_OFF - Cfg::KV_OFF);
    const int share = SPLIT ? 8 / split : 8, owner = (tile * 4 + quarter) / share;
    const int sent = share * 32, at_row = (tile * 4 + quarter) % share * 32 + lane;       // rows per sender, this row among them
    const uint32_t in_o = smem_base + Cfg::KV_OFF, in_ml = in_o + (SPLIT ? (split - 1) * sent * kRow : 0);
    float f_own = 1.f;
    if constexpr (SPLIT) {
      __syncwarp();
      cluster_sync_all();                             // every MMA of every CTA has retired, so no load is under way: the rings are idle
      if (owner != rank) {
        const int slot = (rank - (rank > owner)) * sent + at_row;
#pragma unroll
        for (int b = 0; b < D / 32; ++b) {
          uint32_t o[32] = {};
          if (n[tile] > 0) {
            tc_ld32(o_addr + b * 32, o);
            tc_wait_ld32(o);
          }
          const uint32_t to = mapa_shared(in_o + slot * kRow + b * 128, owner);
#pragma unroll
          for (int x = 0; x < 32; x += 4) st_cluster_v4(to + x * 4, o[x], o[x + 1], o[x + 2], o[x + 3]);
        }
        const uint32_t to = mapa_shared(in_ml + slot * 8, owner);
        asm volatile("st.shared::cluster.v2.b32 [%0], {%1, %2};" ::"r"(to), "r"(__float_as_uint(m)), "r"(__float_as_uint(l)) : "memory");
      }
      __syncwarp();
      cluster_sync_all();
      if (owner == rank) {
        float top = m;
        for (int s = 0; s < split - 1; ++s) top = fmaxf(top, __uint_as_float(lds32(in_ml + (s * sent + at_row) * 8)));
        f_own = m == -INFINITY ? 0.f : exp2_fast(m - top);
        l *= f_own;
        for (int s = 0; s < split - 1; ++s) {
          const uint32_t at = in_ml + (s * sent + at_row) * 8;
          const float m2 = __uint_as_float(lds32(at)), f = m2 == -INFINITY ? 0.f : exp2_fast(m2 - top);
          l = fmaf(__uint_as_float(lds32(at + 4)), f, l);
          asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "f"(f) : "memory");   // only this thread reads it
        }
      }
    }
    if (!SPLIT || owner == rank) {
    // Every MMA of this tile has retired: its queries' rows take the output on its way to whole rows in memory.
    const float inv = l == 0.f ? 0.f : 1.f / l;
    const uint32_t patch = qtile + quarter * (32 * D * 2);
#pragma unroll
    for (int b = 0; b < D / 32; ++b) {
      uint32_t o[32] = {};
      if (n[tile] > 0) {
        tc_ld32(o_addr + b * 32, o);
        tc_wait_ld32(o);
      }
      if constexpr (SPLIT) {
#pragma unroll
        for (int x = 0; x < 32; ++x) o[x] = __float_as_uint(__uint_as_float(o[x]) * f_own);
        for (int s = 0; s < split - 1; ++s) {
          const float f = __uint_as_float(lds32(in_ml + (s * sent + at_row) * 8));
          const uint32_t from = in_o + (s * sent + at_row) * kRow + b * 128;
#pragma unroll
          for (int x = 0; x < 32; x += 4) {
            const uint4 z = lds128(from + x * 4);
            o[x] = __float_as_uint(fmaf(__uint_as_float(z.x), f, __uint_as_float(o[x])));
            o[x + 1] = __float_as_uint(fmaf(__uint_as_float(z.y), f, __uint_as_float(o[x + 1])));
            o[x + 2] = __float_as_uint(fmaf(__uint_as_float(z.z), f, __uint_as_float(o[x + 2])));
            o[x + 3] = __float_as_uint(fmaf(__uint_as_float(z.w), f, __uint_as_float(o[x + 3])));
          }
        }
      }
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        uint32_t w[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const float y0 = l == 0.f ? 0.f : __uint_as_float(o[x * 8 + e * 2]) * inv;
          const float y1 = l == 0.f ? 0.f : __uint_as_float(o[x * 8 + e * 2 + 1]) * inv;
          w[e] = pack2(y0, y1, T());
        }
        const uint32_t at = patch + attn_swizzle<D * 2>(lane, b * 4 + x);
        asm volatile("st.shared.v4.b32 [%0], {%1,%2,%3,%4};" ::"r"(at), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]) : "memory");
      }
    }
    __syncwarp();
    const long long out_at = on ? (long long)(t.q0 + qi) * a.o_tok + (long long)head * a.o_head : -1;
    constexpr int CH = D / 8;                         // 16-byte pieces of a row
#pragma unroll
    for (int x0 = 0; x0 < CH; x0 += 4) {
      uint4 w[4];
      long long at[4];
#pragma unroll
      for (int x = 0; x < 4; ++x) {
        const int r = (x0 + x) * (32 / CH) + lane / CH;
        at[x] = __shfl_sync(0xffffffffu, out_at, r);
        w[x] = lds128(patch + attn_swizzle<D * 2>(r, lane % CH));
      }
#pragma unroll
      for (int x = 0; x < 4; ++x)
        if (at[x] >= 0) *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + at[x] + (lane % CH) * 8) = w[x];
    }
    }
  }
  tc_fence_before();
  __syncthreads();
  if (warp == 8) {
    tc_fence_after();
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(Cfg::TMEM_COLS) : "memory");
  }
}

// The cache as (size, head, place, page), a box = 64 sizes of `box` tokens of one page and head, 128-byte swizzle.
// e4m3: all sizes of the tokens, not swizzled.
static bool make_map_cache(CUtensorMap* map, CUtensorMapDataType type, const void* base, const AttnArgs& a, int size, int box) {
  auto fn = get_encode_fn();
  if (!fn) return false;
  cuuint64_t dims[4] = {(cuuint64_t)size, (cuuint64_t)a.kv_heads, (cuuint64_t)a.page_size, (cuuint64_t)a.num_pages};
  const bool codes = type == CU_TENSOR_MAP_DATA_TYPE_UINT8;
  const cuuint64_t esz = codes ? 1 : 2;
  cuuint64_t strides[3] = {a.c_head * esz, a.c_tok * esz, a.c_page * esz};
  cuuint32_t boxes[4] = {codes ? (cuuint32_t)size : 64, 1, (cuuint32_t)box, 1};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  return fn(map, type, 4, const_cast<void*>(base), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
            codes ? CU_TENSOR_MAP_SWIZZLE_NONE : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
            CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Tokens of a TMA box: what divides both a page and a tile of 128 keys.
static int attn_tc_box(int page_size) {
  int box = page_size & -page_size;
  return box > 128 ? 128 : box;
}

// Whether the tensor-memory kernel takes the call: pages that hold whole groups of 16 tokens, strides that TMA takes.
static bool attn_tc_fits(bool single, int page_size, long long num_pages, long long page_stride, long long token_stride, long long head_stride) {
  if (single || attn_tc_box(page_size) < 16 || num_pages <= 0 || num_pages >= 0x7fffffffLL) return false;
  if (head_stride <= 0 || token_stride <= 0 || page_stride <= 0) return false;
  const long long most = 1LL << 38;                   // strides of a tensor map: below 2^40 bytes
  return head_stride < most && token_stride < most && page_stride < most;
}

template <class T, int D, bool FP8>
static int launch_attn_tc(const AttnArgs& a, int dev, cudaStream_t st) {
  using Cfg = AttnTcCfg<D, FP8>;
  const int box = attn_tc_box(a.page_size);
  CUtensorMap tk, tv;
  constexpr CUtensorMapDataType type = FP8 ? CU_TENSOR_MAP_DATA_TYPE_UINT8
                                       : std::is_same<T, __nv_bfloat16>::value ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  if (!make_map_cache(&tk, type, a.key_cache, a, D, box) || !make_map_cache(&tv, type, a.value_cache, a, D, box)) return TRB_ERR_CUDA;
  const long long per_token = (a.group + 255) / 256;
  long long tiles = ((long long)a.tokens * a.group + 255LL * a.seqs) / 256;      // every sequence's last tile may hold one row
  if (tiles > a.tokens * per_token) tiles = a.tokens * per_token;
  const long long grid = tiles * a.kv_heads;
  if (grid > 0x3fffffffLL) return TRB_ERR_PROB_SHAPE;
  // Few items over long keys: the largest cluster per item with which all clusters still run at once, two key tiles or more per
  // CTA, by the page table's width.  Below 8 key tiles sending the states costs more than it saves (32 heads over 8 of size 128,
  // bf16, one CTA -> a cluster: 128 tokens after 500: 18.5 -> 19.8 us; after 1000: 25.1 -> 23.0; after 2000: 38 -> 26.5; 64 tokens
  // after 8000: 116 -> 34.7; 256 after 4000: 65 -> 35.7; 512 after 4000: 65 -> 47).
  const long long key_tiles = ((long long)a.table_width * a.page_size + 127) / 128;
  for (int split = 8; split >= 2; split /= 2) {
    if (grid * split > sm_count(dev) || key_tiles < (split == 8 ? 16 : 8)) continue;
    static std::atomic<bool> shared[64];
    static std::atomic<int> fit[64][4];               // clusters that run at once
    if (!ensure_smem_attr(attn_tc_kernel<T, Cfg, true>, dev, Cfg::SMEM_ALLOC, shared)) return TRB_ERR_CUDA;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(grid * split));
    cfg.blockDim = dim3(Cfg::THREADS);
    cfg.dynamicSmemBytes = Cfg::SMEM_ALLOC;
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = split;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    std::atomic<int>& most = fit[dev < 64 ? dev : 0][split == 8 ? 3 : split / 2];
    int n = dev < 64 ? most.load(std::memory_order_relaxed) : 0;
    if (n == 0) {
      if (cudaOccupancyMaxActiveClusters(&n, attn_tc_kernel<T, Cfg, true>, &cfg) != cudaSuccess) return TRB_ERR_CUDA;
      most.store(n > 0 ? n : -1, std::memory_order_relaxed);
    }
    if (grid > n) continue;
    return cudaLaunchKernelEx(&cfg, attn_tc_kernel<T, Cfg, true>, tk, tv, a, (int)tiles, box, split) == cudaSuccess ? TRB_OK
                                                                                                                    : TRB_ERR_CUDA;
  }
  static std::atomic<bool> done[64];
  if (!ensure_smem_attr(attn_tc_kernel<T, Cfg, false>, dev, Cfg::SMEM_ALLOC, done)) return TRB_ERR_CUDA;
  attn_tc_kernel<T, Cfg, false><<<(unsigned)grid, Cfg::THREADS, Cfg::SMEM_ALLOC, st>>>(tk, tv, a, (int)tiles, box, 1);
  return cudaGetLastError() == cudaSuccess ? TRB_OK : TRB_ERR_CUDA;
}

}  // namespace trb
