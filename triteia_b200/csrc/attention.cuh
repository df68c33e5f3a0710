// Attention of new tokens over a paged cache.  The reference's attention files hold the decode and the extend form as
// two programs (triteia/triton/decode_attention.py:30-214, extend_attention.py:39-170); here one definition covers both:
//   query token i of the n of sequence b stands at p = length_b - n + i (its own key is in the cache already) and sees
//   the keys j < length_b with j <= p (causal) and j > p - window (window > 0);
//   o = sum_j softmax_j(scale q.k_j) v_j;  a row that sees nothing is zero.
// Query head h reads key head h / g, g = query heads per key head.  The cache is paged as kv_cache.cuh says, in the
// inputs' type or e4m3 with a power of two per token and head.
//
// A work tile is M rows of one sequence and one key head; a row is a (token, query head of the group), so that the g
// heads of a group share every key and value that is read.  This kernel serves the calls that reading the cache bounds
// (single and few tokens) and the caches that the tensor-memory kernel does not take.  Per 16 x 16 block of scores it
// issues two m16n8k16 MMAs for each 16 of the head size, one running maximum per row, and as many MMAs again with the
// values.
//   M = 16: the four warps of a CTA take different tokens (16 each of every 64) and keep softmax states of their own,
//           so that nothing in the loop is CTA-wide; the states meet at the end.
//   M = 64: a warp has 16 rows, and the four share the 64 tokens of a stage.
// The work is cut evenly whatever the sequences' lengths: all (tile, key head) items' units of 64 or 128 tokens stand in one
// line, every CTA of one resident wave takes an equal run of it, and the loads run ahead of the arithmetic across the items'
// borders.  An item inside a run is finished there; of one that a border cuts, the pieces' states (maximum, sum, weighted
// values) go to the caller's workspace, and a second launch joins them in the order of the tokens: no counters, nothing to
// clear, a fixed order of the sums.
// Measured in a graph (and as calls in a row through Python): 64 sequences of 100 to 8000 tokens, 32 heads over 8 of 128, bf16:
// 163 us (172), 6.0 TB/s of the 6.55 that a copy reaches; three of 90000 to 131072 tokens, e4m3: 135 to 140 us (148), 4.8 to 5.0
// TB/s -- there the conversions make the loop longer than the instruction cache takes well (two of three stalled cycles wait for
// instructions).  Clusters for all calls (one launch, no workspace)
// left half of the SMs idle with twelve CTAs each and unequal sequences unequal: 184 and 197 us.
// Loads are 16-byte cp.async with a row address per token (any page size and strides); a token outside the visible range
// or on a page outside the cache is filled with zeros and masked.
#pragma once

#include "kv_cache.cuh"
#include "lora.cuh"

namespace trb {

struct AttnArgs {
  const void* query;
  const void *key_cache, *value_cache;
  const uint8_t *key_exp, *value_exp;
  const int *page_table, *lengths, *query_starts;
  void* out;
  long long q_tok, q_head, o_tok, o_head;
  long long c_page, c_tok, c_head, e_page, e_tok, e_head;
  long long table_stride, num_pages;
  float scale_log2;                   // scale * log2(e)
  int tokens, seqs, kv_heads, group, page_size, table_width;
  int page_shift;                     // log2(page_size), -1 where that is no integer
  int causal, window;
  int clear;                          // rows of out that belong to no sequence become zero
};

// One work tile: rows [row0, row0 + M) of sequence `seq`, whose new tokens are rows of the query from `q0`.
struct AttnTile {
  int seq, row0, rows, q0, new_tokens, length;
};

// Query tokens [first, last) of a sequence, held within the batch and in order whatever the array says.
__device__ __forceinline__ void attn_query_range(const AttnArgs& a, int b, int& first, int& last) {
  if (a.query_starts == nullptr) {
    first = b;
    last = b + 1;
    return;
  }
  first = max(0, min(a.query_starts[b], a.tokens));
  last = max(first, min(a.query_starts[b + 1], a.tokens));
}

// Tokens in the cache, held within the page table.
__device__ __forceinline__ int attn_length(const AttnArgs& a, int b) {
  const long long most = (long long)a.table_width * a.page_size;
  return (int)max(0LL, min((long long)a.lengths[b], most));
}

// This CTA's share of the rows of out before the first and behind the last sequence; `thread` of `threads` take part.
template <class T, int D>
__device__ __forceinline__ void attn_clear_rest(const AttnArgs& a, int thread, int threads) {
  const int first = max(0, min(a.query_starts[0], a.tokens)), last = max(first, min(a.query_starts[a.seqs], a.tokens));
  const int rest = first + (a.tokens - last), pieces = a.kv_heads * a.group * (D / 8);      // pieces of 16 bytes
  for (int x = blockIdx.x; x < rest; x += gridDim.x) {
    T* row = static_cast<T*>(a.out) + (long long)(x < first ? x : last + (x - first)) * a.o_tok;
    for (int i = thread; i < pieces; i += threads)
      *reinterpret_cast<uint4*>(row + (long long)(i / (D / 8)) * a.o_head + i % (D / 8) * 8) = make_uint4(0, 0, 0, 0);
  }
}

// The same by itself, for a call without sequences.
template <class T, int D>
__global__ void __launch_bounds__(128) attn_clear_kernel(const AttnArgs a) {
  attn_clear_rest<T, D>(a, threadIdx.x, 128);
}

// The `index`-th tile of the batch; all lanes of a warp call it together.  False: there are fewer tiles.
template <int M>
__device__ __forceinline__ bool attn_find_tile(const AttnArgs& a, int index, AttnTile& t) {
  const int lane = threadIdx.x & 31;
  int first = 0, last = 0, before = 0;
  if (a.query_starts == nullptr) {
    const int per = (a.group + M - 1) / M;
    t.seq = index / per;
    if (t.seq >= a.seqs) return false;
    before = t.seq * per;
    attn_query_range(a, t.seq, first, last);
  } else {
    bool found = false;
    for (int base = 0; base < a.seqs && !found; base += 32) {
      int f = 0, l = 0;
      if (base + lane < a.seqs) attn_query_range(a, base + lane, f, l);
      const long long rows = (long long)(l - f) * a.group;
      const int n = (int)((rows + M - 1) / M);
      int inc = n;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      const unsigned past = __ballot_sync(0xffffffffu, before + inc > index);
      if (past) {
        const int at = __ffs(past) - 1;
        t.seq = base + at;
        first = __shfl_sync(0xffffffffu, f, at);
        last = __shfl_sync(0xffffffffu, l, at);
        before += __shfl_sync(0xffffffffu, inc - n, at);
        found = true;
      } else {
        before += __shfl_sync(0xffffffffu, inc, 31);
      }
    }
    if (!found) return false;
  }
  t.q0 = first;
  t.new_tokens = last - first;
  t.row0 = (index - before) * M;
  t.rows = min(M, t.new_tokens * a.group - t.row0);
  t.length = attn_length(a, t.seq);
  return true;
}

// Keys [lo, hi) that some row of the tile sees.
__device__ __forceinline__ void attn_key_range(const AttnArgs& a, const AttnTile& t, int& lo, int& hi) {
  lo = 0;
  hi = t.length;
  const int base = t.length - t.new_tokens;
  if (a.causal) hi = min(hi, base + (t.row0 + t.rows - 1) / a.group + 1);
  if (a.window > 0) lo = max(0, base + t.row0 / a.group - a.window + 1);
  if (hi < lo) hi = lo;
}

// A tile and a key head: units [u0, u0 + n) of UNIT tokens, at least one (which may hold nothing that a row sees).
struct AttnItem {
  AttnTile t;
  int kvh, lo, hi, u0, n;
};

template <int M, int UNIT>
__device__ __forceinline__ void attn_item_units(const AttnArgs& a, AttnItem& it) {
  attn_key_range(a, it.t, it.lo, it.hi);
  it.u0 = it.lo / UNIT;
  it.n = it.hi > it.lo ? (it.hi + UNIT - 1) / UNIT - it.u0 : 1;
}

// Units of one key head of sequence b.
template <int M, int UNIT>
__device__ __forceinline__ long long attn_seq_units(const AttnArgs& a, int b) {
  AttnItem it;
  if (a.query_starts == nullptr && a.group <= M) {    // one tile, and no divisions
    const int hi = attn_length(a, b), lo = a.window > 0 ? max(0, hi - a.window) : 0;
    return hi > lo ? (hi + UNIT - 1) / UNIT - lo / UNIT : 1;
  }
  int first, last;
  attn_query_range(a, b, first, last);
  it.t = AttnTile{b, 0, 0, first, last - first, attn_length(a, b)};
  long long n = 0;
  const int rows = (last - first) * a.group;
  for (int r = 0; r < rows; r += M) {
    it.t.row0 = r;
    it.t.rows = min(M, rows - r);
    attn_item_units<M, UNIT>(a, it);
    n += it.n;
  }
  return n;
}

// The line's length in units; all lanes of a warp together.  `own`: the units of this lane's sequence among the first 32.
template <int M, int UNIT>
__device__ __forceinline__ long long attn_total_units(const AttnArgs& a, long long& own) {
  const int lane = threadIdx.x & 31;
  own = lane < a.seqs ? attn_seq_units<M, UNIT>(a, lane) : 0;
  long long n = own;
  for (int b = lane + 32; b < a.seqs; b += 32) n += attn_seq_units<M, UNIT>(a, b);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
  return n * a.kv_heads;
}

// First unit of CTA x's run of the line: total * x / ctas, with one wide division for all x (a wide one takes 100 clocks).
struct AttnRuns {
  long long each;
  uint32_t left, ctas;
  __device__ __forceinline__ AttnRuns(long long total, int n) : ctas((uint32_t)n) {
    each = total <= 0xffffffffLL ? (long long)((uint32_t)total / ctas) : total / ctas;
    left = (uint32_t)(total - each * ctas);
  }
  __device__ __forceinline__ long long begin(int x) const { return each * x + left * (uint32_t)x / ctas; }      // below ctas^2 < 2^32
};

// The item that holds unit `flat` of the line (flat < total) and the unit's number in it; all lanes of a warp together.
template <int M, int UNIT>
__device__ __forceinline__ int attn_seek(const AttnArgs& a, long long flat, long long own, AttnItem& it) {
  const int lane = threadIdx.x & 31;
  int b = 0;
  for (int base = 0;; base += 32) {
    const long long n = (base == 0 ? own : base + lane < a.seqs ? attn_seq_units<M, UNIT>(a, base + lane) : 0) * a.kv_heads;
    long long inc = n;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, inc, o);
      if (lane >= o) inc += v;
    }
    const unsigned past = __ballot_sync(0xffffffffu, inc > flat);
    if (past) {
      const int at = __ffs(past) - 1;
      b = base + at;
      flat -= __shfl_sync(0xffffffffu, inc - n, at);
      break;
    }
    flat -= __shfl_sync(0xffffffffu, inc, 31);
    if (base + 32 >= a.seqs) return 0;                // not reached: flat < total
  }
  int first, last;
  attn_query_range(a, b, first, last);
  it.t = AttnTile{b, 0, 0, first, last - first, attn_length(a, b)};
  const int rows = (last - first) * a.group;
  for (int r = 0; r < rows; r += M) {
    it.t.row0 = r;
    it.t.rows = min(M, rows - r);
    attn_item_units<M, UNIT>(a, it);
    const long long all = (long long)it.n * a.kv_heads;
    if (flat < all) break;
    flat -= all;
  }
  it.kvh = (int)(flat / it.n);
  return (int)(flat - (long long)it.kvh * it.n);
}

// The next item of the line.  The caller knows that there is one.
template <int M, int UNIT>
__device__ __forceinline__ void attn_next(const AttnArgs& a, AttnItem& it) {
  if (++it.kvh < a.kv_heads) return;
  it.kvh = 0;
  it.t.row0 += M;
  if (it.t.row0 >= it.t.new_tokens * a.group) {
    int first = 0, last = 0, b = it.t.seq;
    do {
      ++b;
      if (b >= a.seqs) return;
      attn_query_range(a, b, first, last);
    } while (last <= first);
    it.t = AttnTile{b, 0, 0, first, last - first, attn_length(a, b)};
  }
  it.t.rows = min(M, it.t.new_tokens * a.group - it.t.row0);
  attn_item_units<M, UNIT>(a, it);
}

template <class T, bool FP8_, int D_, bool ROWS_>
struct AttnCfg {
  static constexpr bool FP8 = FP8_, ROWS = ROWS_;
  static constexpr int D = D_;
  static constexpr int M = ROWS ? 64 : 16;
  static constexpr int ROWB = FP8 ? D : 2 * D;                  // bytes of a token's key or value
  static constexpr int CHUNKS = ROWB / 16;
  static constexpr int NT = ROWS ? 4 : FP8 ? 2 : 1;             // a warp takes 16 * NT tokens at a time
  static constexpr int UNIT = ROWS ? 64 : 64 * NT;              // tokens of a stage, a quarter loaded by each warp
  static constexpr int WTOK = UNIT / 4;
  static constexpr int HALF_BYTES = UNIT * ROWB;                // keys; the values follow
  static constexpr int STAGE_BYTES = 2 * HALF_BYTES;
  // About 96 KB of loads in flight per CTA and two CTAs per SM: 6.5 TB/s for about 1.5 us of latency is 66 KB per SM.
  static constexpr int STAGES = 98304 / STAGE_BYTES > 6 ? 6 : 98304 / STAGE_BYTES;
  // uint32 [STAGES][4][2], per loading warp: tokens that count; e4m3: tokens that may have a value head of zeros
  static constexpr int MASK_OFF = STAGES * STAGE_BYTES;
  static constexpr int EXP_OFF = MASK_OFF + STAGES * 32;        // float [STAGES][3][UNIT]: 2^e of keys; e and 2^-e of values
  static constexpr int WML_OFF = EXP_OFF + (FP8 ? STAGES * 3 * UNIT * 4 : 0);   // float [4][16][2]: the warps' maxima and sums (M = 16)
  static constexpr int ML_OFF = WML_OFF + (ROWS ? 0 : 4 * 16 * 8);             // float [16][2]: the CTA's (M = 16)
  static constexpr int O_STRIDE = D + 4;                                       // floats
  static constexpr int O_OFF = ML_OFF + (ROWS ? 0 : 16 * 8);                   // float [16][O_STRIDE]: the CTA's weighted values
  static constexpr int SMEM_BYTES = O_OFF + (ROWS ? 0 : 16 * O_STRIDE * 4);
  static constexpr int PIECE_FLOATS = M * (D + 2);              // a piece in the workspace: values [M][D], maximum and sum [M][2]
  static constexpr int THREADS = 128;
};

// Byte of 16-byte chunk `c` of row `r` of a tile, spread so that eight rows of one chunk fall into different banks.
template <int ROWB>
__device__ __forceinline__ uint32_t attn_swizzle(int r, int c) {
  if constexpr (ROWB == 64) return r * 64 + ((c ^ ((r >> 1) & 3)) << 4);
  else return r * ROWB + ((c ^ (r & 7)) << 4);
}


__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <class TP>
__device__ __forceinline__ void attn_mma(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void attn_mma<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  mma_m16n8k16(d, a, b0, b1);
}
template <>
__device__ __forceinline__ void attn_mma<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  mma_m16n8k16_bf16(d, a, b0, b1);
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi, __half) {
  __half2 h = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t pack2(float lo, float hi, __nv_bfloat16) {
  __nv_bfloat162 h = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&h);
}

// Two e4m3 codes (low 16 bits) as two fp16 numbers: exact.
__device__ __forceinline__ uint32_t e4m3x2_to_half2(uint32_t two) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, lo;\n\t}" : "=r"(r) : "r"(two));
  return r;
}
__device__ __forceinline__ uint32_t e4m3x2_hi_to_half2(uint32_t two) {
  uint32_t r;
  asm("{\n\t.reg .b16 lo, hi;\n\tmov.b32 {lo, hi}, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, hi;\n\t}" : "=r"(r) : "r"(two));
  return r;
}

__device__ __forceinline__ float pow2_of_byte(int byte) { return __uint_as_float(byte <= 0 ? 0x00400000u : (uint32_t)byte << 23); }

__device__ __forceinline__ float ld_cluster_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ float4 ld_cluster_f32x4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}

// The e4m3 form computes in fp16 whatever T is: a code is exact in fp16, and a bf16 query row, scaled by a power of two
// to a largest magnitude of 2^9 .. 2^10, keeps all its bits down to 2^-25 of that; what is smaller is off by 2^-34 of the largest
// (half of fp16's last step), as a rule far less than the 32-bit sum of the score rounds off.  Weights are fp16 there (11 bits).
template <class T, bool FP8>
struct AttnMma { using type = T; };
template <class T>
struct AttnMma<T, true> { using type = __half; };

// Exponent field of the power of two that brings a bf16 row with the largest magnitude `top` to 2^9 .. 2^10.
__device__ __forceinline__ int attn_row_shift(float top) {
  const int field = (int)(__float_as_uint(top) >> 23);                  // top in [2^(field - 127), twice that)
  return top > 0.f ? min(max(127 + 127 + 9 - field, 1), 253) : 127;
}

// A value head of zeros has the exponent byte 127 (kv_cache.cuh).  Its product with a weight is zero whatever exponent it is
// given, but the running maximum below is over log2 weight + e: with e = 0 such a token would push the weights of values that
// are all much smaller out of fp16.  It takes this exponent instead, below any that matters (values under 2^-81 alone are less),
// while its weight times 2^90 enters the sum as ever: 2^(90 + 8) a token, far from the end of 32 bits for 2^17 tokens and more.
constexpr int kZeroValueExp = -90;

// Whether 16 codes are zeros, of either sign.
__device__ __forceinline__ bool attn_zero_codes(uint4 w) { return ((w.x | w.y | w.z | w.w) & 0x7f7f7f7fu) == 0; }

// Gives the tokens of `maybe` (byte 127) whose value codes in shared memory are zeros their exponent; a warp for itself.  Not
// inlined: the loop that hardly ever calls it has to stay in the instruction cache.
template <class Cfg>
__device__ __noinline__ void attn_zero_values(unsigned long long maybe, uint32_t vbase, float* exps, int lane) {
#pragma unroll 1
  for (int r = lane; r < 16 * Cfg::NT; r += 32) {
    bool zeros = (maybe >> r) & 1;
#pragma unroll 1
    for (int c = 0; zeros && c < Cfg::CHUNKS; ++c) zeros = attn_zero_codes(lds128(vbase + attn_swizzle<Cfg::ROWB>(r, c)));      // real values: once
    if (zeros) {
      exps[Cfg::UNIT + r] = (float)kZeroValueExp;
      exps[2 * Cfg::UNIT + r] = __uint_as_float((uint32_t)(127 - kZeroValueExp) << 23);
    }
  }
  __syncwarp();
}

// Softmax state of a warp's 16 rows; a lane has rows lane / 4 and lane / 4 + 8.
template <int D>
struct AttnState {
  float o[D / 8][4];
  float m[2], l[2];                   // maxima in powers of two; l: this lane's share of the sum
};

// fp16 weights are kept at 2^8 times their value, so that small ones stay clear of the subnormal range (the same
// factor is in l); bf16 has the exponents of 32-bit numbers.
template <class TM>
struct AttnBias { static constexpr float value = std::is_same<TM, __half>::value ? 8.f : 0.f; };

// 16 rows x (16 * NT) tokens: scores, masks, running maxima, weights, product with the values.
template <class T, class Cfg, int NT>
__device__ __forceinline__ void attn_block(AttnState<Cfg::D>& st, const uint32_t (&q)[Cfg::D / 16][4], const float (&c_row)[2],
                                           uint32_t kbase, uint32_t vbase, const float* exps, unsigned long long valid, int j0,
                                           const int (&row_hi)[2], const int (&row_lo)[2], bool need_mask, int lane) {
  using TM = typename AttnMma<T, Cfg::FP8>::type;
  constexpr int D = Cfg::D, ROWB = Cfg::ROWB;
  const int quad = lane & 3;
  float s[2 * NT][4];
#pragma unroll
  for (int i = 0; i < 2 * NT; ++i)
#pragma unroll
    for (int e = 0; e < 4; ++e) s[i][e] = 0.f;
  // ---- scores
  if constexpr (!Cfg::FP8) {
    const int r = (lane & 7) + ((lane >> 4) << 3), c = (lane >> 3) & 1;
#pragma unroll
    for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        uint32_t b[4];
        ldmatrix_x4(b, kbase + attn_swizzle<ROWB>(n * 16 + r, 2 * ks + c));
        attn_mma<TM>(s[2 * n], q[ks], b[0], b[1]);
        attn_mma<TM>(s[2 * n + 1], q[ks], b[2], b[3]);
      }
  } else {
    // A 16-byte chunk is 16 sizes = one MMA step; a lane's four bytes are sizes 4 quad .. + 3, and the query fragments
    // are loaded in that order.
    const int r = (lane & 7) + ((lane >> 4) << 3), c = (lane >> 3) & 1;
#pragma unroll
    for (int kp = 0; kp < D / 32; ++kp)
#pragma unroll
      for (int n = 0; n < NT; ++n) {
        uint32_t b[4];
        ldmatrix_x4(b, kbase + attn_swizzle<ROWB>(n * 16 + r, 2 * kp + c));
        attn_mma<TM>(s[2 * n], q[2 * kp], e4m3x2_to_half2(b[0]), e4m3x2_hi_to_half2(b[0]));
        attn_mma<TM>(s[2 * n + 1], q[2 * kp], e4m3x2_to_half2(b[2]), e4m3x2_hi_to_half2(b[2]));
        attn_mma<TM>(s[2 * n], q[2 * kp + 1], e4m3x2_to_half2(b[1]), e4m3x2_hi_to_half2(b[1]));
        attn_mma<TM>(s[2 * n + 1], q[2 * kp + 1], e4m3x2_to_half2(b[3]), e4m3x2_hi_to_half2(b[3]));
      }
  }
  // ---- scale.  With exponents the weight that meets the code of v_j is 2^(t_j - m), t_j = log2 weight + e_j, and m
  // runs over the t_j: the weights fit the MMA type whatever the values' magnitudes; the sum takes the 2^-e_j back out.
  float2 iv[2 * NT];
  if constexpr (Cfg::FP8) {
#pragma unroll
    for (int n = 0; n < 2 * NT; ++n) {
      const float2 kf = *reinterpret_cast<const float2*>(exps + n * 8 + 2 * quad);
      const float2 ev = *reinterpret_cast<const float2*>(exps + Cfg::UNIT + n * 8 + 2 * quad);
      iv[n] = *reinterpret_cast<const float2*>(exps + 2 * Cfg::UNIT + n * 8 + 2 * quad);
      // The row's and the key's factor first: they may be far from 1 on opposite sides.
      s[n][0] = fmaf(s[n][0], kf.x * c_row[0], ev.x);
      s[n][1] = fmaf(s[n][1], kf.y * c_row[0], ev.y);
      s[n][2] = fmaf(s[n][2], kf.x * c_row[1], ev.x);
      s[n][3] = fmaf(s[n][3], kf.y * c_row[1], ev.y);
    }
  } else {
#pragma unroll
    for (int n = 0; n < 2 * NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] *= c_row[e >> 1];
  }
  if (need_mask) {
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      // Bit x: this row sees token j0 + x; then those of this lane's columns.
      const int h = row_hi[r] - j0, w = row_lo[r] - j0;
      unsigned long long bits = h >= 64 ? valid : h <= 0 ? 0ull : valid & ((1ull << h) - 1);
      bits = w <= 0 ? bits : w >= 64 ? 0ull : bits & ~((1ull << w) - 1);
      bits >>= 2 * quad;
#pragma unroll
      for (int n = 0; n < 2 * NT; ++n) {
        const uint32_t two = (uint32_t)(bits >> (n * 8)) & 3;
        if (!(two & 1)) s[n][2 * r] = -INFINITY;
        if (!(two & 2)) s[n][2 * r + 1] = -INFINITY;
      }
    }
  }
  // ---- running maxima
  float mx[2] = {st.m[0], st.m[1]};
#pragma unroll
  for (int n = 0; n < 2 * NT; ++n) {
    mx[0] = fmaxf(mx[0], fmaxf(s[n][0], s[n][1]));
    mx[1] = fmaxf(mx[1], fmaxf(s[n][2], s[n][3]));
  }
#pragma unroll
  for (int o = 1; o <= 2; o <<= 1) {
    mx[0] = fmaxf(mx[0], __shfl_xor_sync(0xffffffffu, mx[0], o));
    mx[1] = fmaxf(mx[1], __shfl_xor_sync(0xffffffffu, mx[1], o));
  }
  if (__any_sync(0xffffffffu, mx[0] > st.m[0] || mx[1] > st.m[1])) {
    float alpha[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      alpha[r] = st.m[r] == -INFINITY ? 0.f : exp2_fast(st.m[r] - mx[r]);
      st.l[r] *= alpha[r];
      st.m[r] = mx[r];
    }
#pragma unroll
    for (int d = 0; d < D / 8; ++d) {
      st.o[d][0] *= alpha[0];
      st.o[d][1] *= alpha[0];
      st.o[d][2] *= alpha[1];
      st.o[d][3] *= alpha[1];
    }
  }
  // A row that has seen nothing yet has the maximum -inf; its weights have to come out as zero, not as NaN.
  const float base[2] = {(st.m[0] == -INFINITY ? 0.f : st.m[0]) - AttnBias<TM>::value, (st.m[1] == -INFINITY ? 0.f : st.m[1]) - AttnBias<TM>::value};
#pragma unroll
  for (int n = 0; n < 2 * NT; ++n)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      const float p = exp2_fast(s[n][e] - base[e >> 1]);
      s[n][e] = p;
      if constexpr (Cfg::FP8) st.l[e >> 1] = fmaf(p, e & 1 ? iv[n].y : iv[n].x, st.l[e >> 1]);
      else st.l[e >> 1] += p;
    }
  // ---- values: the weights are rounded to the MMA type (half a step, of random sign), the sum above is not.  That adds about as
  // much to the output's error as its own rounding (bf16 2.1e-3 of it in all against 1.7e-3, fp16 2.5e-4 against 2.0e-4); weights
  // in two parts would keep their bits for half as many MMAs again.
  const int r = (lane & 7) + (((lane >> 3) & 1) << 3), c = lane >> 4;
#pragma unroll
  for (int n = 0; n < NT; ++n) {
    const uint32_t p[4] = {pack2(s[2 * n][0], s[2 * n][1], TM()), pack2(s[2 * n][2], s[2 * n][3], TM()),
                           pack2(s[2 * n + 1][0], s[2 * n + 1][1], TM()), pack2(s[2 * n + 1][2], s[2 * n + 1][3], TM())};
    if constexpr (!Cfg::FP8) {
#pragma unroll
      for (int dp = 0; dp < D / 16; ++dp) {
        uint32_t b[4];
        ldmatrix_x4_trans(b, vbase + attn_swizzle<ROWB>(n * 16 + r, 2 * dp + c));
        attn_mma<TM>(st.o[2 * dp], p, b[0], b[1]);
        attn_mma<TM>(st.o[2 * dp + 1], p, b[2], b[3]);
      }
    } else {
      // A transposed lane has two sizes (2n, 2n + 1) of two tokens; the bytes of a size are brought together, and the
      // even and the odd sizes of a 16-byte chunk become two column tiles.
#pragma unroll
      for (int dp = 0; dp < D / 32; ++dp) {
        uint32_t b[4];
        ldmatrix_x4_trans(b, vbase + attn_swizzle<ROWB>(n * 16 + r, 2 * dp + c));
#pragma unroll
        for (int i = 0; i < 4; ++i) b[i] = __byte_perm(b[i], 0, 0x3120);
        attn_mma<TM>(st.o[4 * dp], p, e4m3x2_to_half2(b[0]), e4m3x2_to_half2(b[1]));
        attn_mma<TM>(st.o[4 * dp + 1], p, e4m3x2_hi_to_half2(b[0]), e4m3x2_hi_to_half2(b[1]));
        attn_mma<TM>(st.o[4 * dp + 2], p, e4m3x2_to_half2(b[2]), e4m3x2_to_half2(b[3]));
        attn_mma<TM>(st.o[4 * dp + 3], p, e4m3x2_hi_to_half2(b[2]), e4m3x2_hi_to_half2(b[3]));
      }
    }
  }
}

// A row's 4 or 8 numbers, divided by the sum and rounded once.
template <class T, int N>
__device__ __forceinline__ void attn_store_row(T* dst, const float* v, float l) {
  const float inv = l == 0.f ? 0.f : 1.f / l;
  uint32_t w[N / 2];
#pragma unroll
  for (int e = 0; e < N; e += 2) w[e / 2] = l == 0.f ? 0u : pack2(v[e] * inv, v[e + 1] * inv, T());
  if constexpr (N == 2) *reinterpret_cast<uint32_t*>(dst) = w[0];
  else if constexpr (N == 4) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
  else *reinterpret_cast<uint4*>(dst) = make_uint4(w[0], w[1], w[2], w[3]);
}
template <class T>
__device__ __forceinline__ T* attn_out_row(const AttnArgs& a, const AttnItem& it, int row) {
  const int rq = it.t.row0 + row, i = rq / a.group, head = it.kvh * a.group + (rq - i * a.group);
  return static_cast<T*>(a.out) + (long long)(it.t.q0 + i) * a.o_tok + (long long)head * a.o_head;
}

constexpr int kAttnParts = 8;           // CTAs of a cluster at most

// CLUSTER: a cluster shares one item (of a single-token call) instead, its CTAs' states meet through distributed shared memory,
// and there is no line to cut and no second launch.
template <class T, class Cfg, bool CLUSTER>
__global__ void __launch_bounds__(Cfg::THREADS, 2) attn_kernel(const AttnArgs a, float* pieces) {
  using TM = typename AttnMma<T, Cfg::FP8>::type;
  constexpr int D = Cfg::D, M = Cfg::M, STAGES = Cfg::STAGES, UNIT = Cfg::UNIT;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t smem_base = smem_u32(smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad = lane & 3;
  AttnItem it;                          // the item that is computed
  int skip;
  long long f0, f1;                     // this CTA's run of the line (CLUSTER: of the item)
  uint32_t parts = 1, part = 0;
  if constexpr (CLUSTER) {
    asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(parts));
    asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(part));
    const int item = blockIdx.x / parts;
    attn_find_tile<M>(a, item / a.kv_heads, it.t);
    it.kvh = item % a.kv_heads;
    attn_item_units<M, UNIT>(a, it);
    skip = (int)((uint32_t)it.n * part / parts);
    f0 = skip;
    f1 = (uint32_t)it.n * (part + 1) / parts;
  } else if (pieces == nullptr) {       // a CTA for each item
    if (a.clear) attn_clear_rest<T, D>(a, tid, Cfg::THREADS);
    if (!attn_find_tile<M>(a, blockIdx.x / a.kv_heads, it.t)) return;
    it.kvh = blockIdx.x % a.kv_heads;
    attn_item_units<M, UNIT>(a, it);
    skip = 0;
    f0 = 0;
    f1 = it.n;
  } else {
    pdl_launch_dependents();            // the joining launch waits for this one's end before it reads
    if (a.clear && gridDim.x == 1) attn_clear_rest<T, D>(a, tid, Cfg::THREADS);      // else the joining launch does
    long long own;
    const long long total = attn_total_units<M, UNIT>(a, own);
    const AttnRuns runs(total, gridDim.x);
    f0 = runs.begin(blockIdx.x);
    f1 = runs.begin(blockIdx.x + 1);
    if (f0 == f1) return;
    skip = attn_seek<M, UNIT>(a, f0, own, it);
  }
  long long flat = f0 - skip;           // the item's place in the line
  AttnItem ld = it;                     // the item whose loads are issued
  int ld_u = it.u0 + skip;
  long long ld_left = f1 - f0;          // units whose loads have not been issued

  const uint8_t* kc = static_cast<const uint8_t*>(a.key_cache);
  const uint8_t* vc = static_cast<const uint8_t*>(a.value_cache);
  constexpr int ESZ = Cfg::FP8 ? 1 : 2;
  uint2* masks = reinterpret_cast<uint2*>(smem + Cfg::MASK_OFF);
  float* exps = reinterpret_cast<float*>(smem + Cfg::EXP_OFF);
  constexpr int WTOK = Cfg::WTOK;                     // 16 or 32 tokens of a stage are this warp's to load
  const int tok = warp * WTOK + (lane & (WTOK - 1));  // this lane's among the unit's

  // Page, place and key head of this lane's token of unit ld_u (page -1: not visible, or not in the cache), found one unit ahead.
  struct Where { int page, place, kvh; };
  auto where = [&]() -> Where {
    const int j = ld_u * UNIT + tok;
    if (ld_left == 0 || j < ld.lo || j >= ld.hi) return {-1, 0, 0};
    const int p = a.page_shift >= 0 ? j >> a.page_shift : j / a.page_size;
    const int pg = a.page_table[ld.t.seq * a.table_stride + p];
    return {pg >= 0 && pg < a.num_pages ? pg : -1, j - p * a.page_size, ld.kvh};
  };
  Where ahead = where();
  int exp_slot = -1, kb = 126, vb = 126;              // e4m3: the bytes that the last issue() asked for, and their stage
  auto settle_exps = [&]() {
    if (exp_slot < 0) return;
    const unsigned maybe = __ballot_sync(0xffffffffu, vb == 127 && lane < WTOK);
    if (lane == 0) masks[exp_slot * 4 + warp].y = maybe;
    if (lane < WTOK) {
      float* e = exps + exp_slot * 3 * UNIT + tok;
      e[0] = pow2_of_byte(kb);
      e[UNIT] = (float)(vb - 127);
      e[2 * UNIT] = pow2_of_byte(254 - vb);
    }
  };
  constexpr int PER = 32 / Cfg::CHUNKS;               // rows per instruction
  const int c = lane % Cfg::CHUNKS, r0 = lane / Cfg::CHUNKS;
  const long long row_bytes = a.c_tok * ESZ;
  const bool paged16 = (a.page_size & 15) == 0;       // 16 tokens of a unit lie on one page
  // Loads this warp's tokens of the next unit into `slot`.
  auto issue = [&](int slot) {
    if constexpr (Cfg::FP8) settle_exps();
    exp_slot = -1;
    if (ld_left > 0) {
      const Where w = ahead;
      if (--ld_left > 0 && ++ld_u == ld.u0 + ld.n) {
        attn_next<M, UNIT>(a, ld);
        ld_u = ld.u0;
      }
      ahead = where();
      const bool there = w.page >= 0;
      long long off = there ? (long long)w.page * a.c_page + (long long)w.place * a.c_tok + (long long)w.kvh * a.c_head : 0;
      if constexpr (ESZ == 2) off *= 2;
      unsigned mask = __ballot_sync(0xffffffffu, there);
      if constexpr (WTOK == 16) mask &= 0xffffu;
      if (lane == 0) masks[slot * 4 + warp].x = mask;
      if constexpr (Cfg::FP8) {
        exp_slot = slot;
        kb = vb = 126;
        if (there) {
          const long long eo = (long long)w.page * a.e_page + (long long)w.place * a.e_tok + (long long)w.kvh * a.e_head;
          kb = a.key_exp[eo];
          vb = a.value_exp[eo];
        }
      }
      const uint32_t dst = smem_base + slot * Cfg::STAGE_BYTES;
      if (paged16 && mask == (WTOK == 16 ? 0xffffu : 0xffffffffu)) {
#pragma unroll
        for (int g = 0; g < WTOK / 16; ++g) {
          const long long base = __shfl_sync(0xffffffffu, off, g * 16) + r0 * row_bytes + c * 16;
          const uint8_t *kp = kc + base, *vp = vc + base;
#pragma unroll
          for (int i = 0; i < 16 / PER; ++i) {
            const uint32_t at = dst + attn_swizzle<Cfg::ROWB>(warp * WTOK + g * 16 + i * PER + r0, c);
            cp_async16(at, kp, true);
            cp_async16(at + Cfg::HALF_BYTES, vp, true);
            kp += PER * row_bytes;
            vp += PER * row_bytes;
          }
        }
      } else {
#pragma unroll 1
        for (int i = 0; i < WTOK / PER; ++i) {
          const int r = i * PER + r0;
          const long long ro = __shfl_sync(0xffffffffu, off, r) + c * 16;
          const bool ok = (mask >> r) & 1;
          const uint32_t at = dst + attn_swizzle<Cfg::ROWB>(warp * WTOK + r, c);
          cp_async16(at, kc + ro, ok);
          cp_async16(at + Cfg::HALF_BYTES, vc + ro, ok);
        }
      }
    }
    cp_async_commit();
  };
  int slot = 0, warm = STAGES - 1;      // stage of the next unit; stages that are to be filled before it can be computed
  for (long long f = f0; f < f1 || CLUSTER;) {        // CLUSTER: one round, with nothing in it if the share is empty
    // ---- a piece: units [u, u_end) of item `it`
    int u = it.u0 + (int)(f - flat);
    const int u_end = (int)min((long long)(it.u0 + it.n), u + (f1 - f));
    const bool whole = u == it.u0 && u_end == it.u0 + it.n;
    const AttnTile& t = it.t;
    const int hi = it.hi;
    // this warp's rows: query fragments, visible ranges
    const int wrow = Cfg::ROWS ? warp * 16 : 0;
    uint32_t q[D / 16][4];
    float c_row[2];
    int row_hi[2], row_lo[2];
#pragma unroll
    for (int rr = 0; rr < 2; ++rr) {
      const int row = wrow + (lane >> 2) + 8 * rr;
      const bool on = row < t.rows;
      const int rq = t.row0 + (on ? row : 0);
      const int i = rq / a.group, head = it.kvh * a.group + (rq - i * a.group);
      const T* qp = static_cast<const T*>(a.query) + (long long)(t.q0 + i) * a.q_tok + (long long)head * a.q_head;
      const int pos = t.length - t.new_tokens + i;
      row_hi[rr] = a.causal ? min(hi, pos + 1) : hi;
      row_lo[rr] = a.window > 0 ? pos - a.window + 1 : 0;
      c_row[rr] = a.scale_log2;
      if constexpr (!Cfg::FP8) {
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks)
#pragma unroll
          for (int h = 0; h < 2; ++h)
            q[ks][rr + 2 * h] = on ? *reinterpret_cast<const uint32_t*>(qp + ks * 16 + h * 8 + 2 * quad) : 0u;
      } else {
        float top = 0.f;
        uint2 raw[D / 16];
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          raw[ks] = on ? *reinterpret_cast<const uint2*>(qp + ks * 16 + 4 * quad) : make_uint2(0, 0);
          const T* e = reinterpret_cast<const T*>(&raw[ks]);
#pragma unroll
          for (int x = 0; x < 4; ++x) top = fmaxf(top, fabsf(Ew<T>::to_f(e[x])));
        }
        float up = 1.f;
        if constexpr (std::is_same<T, __nv_bfloat16>::value) {
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
          top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
          const int k = attn_row_shift(top);
          up = __uint_as_float((uint32_t)k << 23);
          c_row[rr] *= __uint_as_float((uint32_t)(254 - k) << 23);
        }
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
          const T* e = reinterpret_cast<const T*>(&raw[ks]);
          q[ks][rr] = pack2(Ew<T>::to_f(e[0]) * up, Ew<T>::to_f(e[1]) * up, __half());
          q[ks][rr + 2] = pack2(Ew<T>::to_f(e[2]) * up, Ew<T>::to_f(e[3]) * up, __half());
        }
      }
    }
    AttnState<D> st;
#pragma unroll
    for (int d = 0; d < D / 8; ++d)
#pragma unroll
      for (int e = 0; e < 4; ++e) st.o[d][e] = 0.f;
    st.m[0] = st.m[1] = -INFINITY;
    st.l[0] = st.l[1] = 0.f;
    // Tokens [all_lo, all_hi) are seen by every row of the warp.
    const int base_pos = t.length - t.new_tokens;
    const int last_row = min(wrow + 15, t.rows - 1);
    const int all_hi = a.causal ? min(hi, base_pos + (t.row0 + wrow) / a.group + 1) : hi;
    const int all_lo = a.window > 0 ? base_pos + (t.row0 + last_row) / a.group - a.window + 1 : 0;
    const bool idle = wrow >= t.rows;

    f += u_end - u;
    // The loads are issued in one place, the first stages' too: the loop has to stay in the instruction cache, whose misses
    // were the largest stall of this kernel while it held more.
    while (u < u_end) {
      if (warm == 0) {
        cp_async_wait<STAGES - 2>();
        if constexpr (Cfg::ROWS) __syncthreads();
        else __syncwarp();
      }
      issue(warm > 0 ? STAGES - 1 - warm : slot == 0 ? STAGES - 1 : slot - 1);
      if (warm > 0) {
        --warm;
        continue;
      }
      if (!idle) {
        constexpr int TOK = Cfg::NT * 16;
        const int own = Cfg::ROWS ? 0 : warp * WTOK;
        const int j0 = u * UNIT + own;
        const uint2* mk = masks + slot * 4;
        unsigned long long valid, maybe;
        if constexpr (Cfg::ROWS) {
          const uint2 m0 = mk[0], m1 = mk[1], m2 = mk[2], m3 = mk[3];
          valid = (unsigned long long)(m0.x | m1.x << 16) | (unsigned long long)(m2.x | m3.x << 16) << 32;
          maybe = (unsigned long long)(m0.y | m1.y << 16) | (unsigned long long)(m2.y | m3.y << 16) << 32;
        } else {
          const uint2 m = mk[warp];
          valid = m.x;
          maybe = m.y;
        }
        constexpr unsigned long long kAll = ~0ull >> (64 - TOK);
        if (valid != 0) {
          const bool need_mask = valid != kAll || j0 + TOK > all_hi || j0 < all_lo;
          const uint32_t kbase = smem_base + slot * Cfg::STAGE_BYTES + own * Cfg::ROWB;
          if constexpr (Cfg::FP8) {                   // the warps of the rows' form all mark all tokens, with the same values
            if (maybe != 0) attn_zero_values<Cfg>(maybe, kbase + Cfg::HALF_BYTES, exps + slot * 3 * UNIT + own, lane);
          }
          attn_block<T, Cfg, Cfg::NT>(st, q, c_row, kbase, kbase + Cfg::HALF_BYTES, exps + slot * 3 * UNIT + own, valid, j0, row_hi, row_lo,
                                      need_mask, lane);
        }
      }
      if constexpr (!Cfg::ROWS) __syncwarp();
      slot = slot + 1 == STAGES ? 0 : slot + 1;
      ++u;
    }

    // ---- the piece's state: to the output, or to the workspace (slot 2 c of CTA c for the item its run begins in, or with;
    // 2 c + 1 for another one)
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      st.l[r] += __shfl_xor_sync(0xffffffffu, st.l[r], 1);
      st.l[r] += __shfl_xor_sync(0xffffffffu, st.l[r], 2);
    }
    float* piece = pieces + (2LL * blockIdx.x + (f0 < flat ? 1 : 0)) * Cfg::PIECE_FLOATS;
    if constexpr (Cfg::ROWS) {
#pragma unroll
      for (int rr = 0; rr < 2; ++rr) {
        const int row = wrow + (lane >> 2) + 8 * rr;
        if (row >= t.rows) continue;
        T* dst = attn_out_row<T>(a, it, row);
        if (!whole && quad == 0) *reinterpret_cast<float2*>(piece + M * D + 2 * row) = make_float2(st.m[rr], st.l[rr]);
        constexpr int N = Cfg::FP8 ? 4 : 2;           // neighbouring sizes that a lane has
#pragma unroll
        for (int d = 0; d < D / (4 * N); ++d) {
          float v[N];
#pragma unroll
          for (int e = 0; e < N; ++e) v[e] = Cfg::FP8 ? st.o[2 * d + (e & 1)][2 * rr + (e >> 1)] : st.o[d][2 * rr + e];
          const int at = d * 4 * N + N * quad;
          if (whole) attn_store_row<T, N>(dst + at, v, st.l[rr]);
          else {
#pragma unroll
            for (int e = 0; e < N; ++e) piece[row * D + at + e] = v[e];
          }
        }
      }
    } else {
      float* obuf = reinterpret_cast<float*>(smem + Cfg::O_OFF);
      float2* ml = reinterpret_cast<float2*>(smem + Cfg::ML_OFF);
      float2* wml = reinterpret_cast<float2*>(smem + Cfg::WML_OFF);
      if constexpr (CLUSTER) {
        // No loads are under way: the warps' states go to the ring side by side and are added in one pass (a short call
        // feels every barrier).
        cp_async_wait<0>();
        __syncthreads();
        float* wbuf = reinterpret_cast<float*>(smem) + warp * 16 * Cfg::O_STRIDE;
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
          const int row = (lane >> 2) + 8 * rr;
          if (row >= t.rows) continue;
          if (quad == 0) wml[warp * 16 + row] = make_float2(st.m[rr], st.l[rr]);
          float* dst = wbuf + row * Cfg::O_STRIDE;
#pragma unroll
          for (int d = 0; d < D / 16; ++d) {
            // Sizes 4 quad .. + 3 of each 16 (e4m3), or 2 quad, + 1 of each 8.
            float2* p0 = reinterpret_cast<float2*>(dst + d * 16 + (Cfg::FP8 ? 4 : 2) * quad);
            float2* p1 = Cfg::FP8 ? p0 + 1 : p0 + 4;
            *p0 = Cfg::FP8 ? make_float2(st.o[2 * d][2 * rr], st.o[2 * d + 1][2 * rr]) : make_float2(st.o[2 * d][2 * rr], st.o[2 * d][2 * rr + 1]);
            *p1 = Cfg::FP8 ? make_float2(st.o[2 * d][2 * rr + 1], st.o[2 * d + 1][2 * rr + 1])
                           : make_float2(st.o[2 * d + 1][2 * rr], st.o[2 * d + 1][2 * rr + 1]);
          }
        }
        __syncthreads();
        for (int x = tid; x < t.rows * (D / 4); x += Cfg::THREADS) {
          const int row = x / (D / 4), d = (x % (D / 4)) * 4;
          float m = -INFINITY, l = 0.f;
          float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
          for (int w = 0; w < 4; ++w) m = fmaxf(m, wml[w * 16 + row].x);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const float2 ws = wml[w * 16 + row];
            const float f_w = ws.x == -INFINITY ? 0.f : exp2_fast(ws.x - m);
            const float4 v = *reinterpret_cast<const float4*>(reinterpret_cast<const float*>(smem) + (w * 16 + row) * Cfg::O_STRIDE + d);
            l = fmaf(ws.y, f_w, l);
            o = make_float4(fmaf(v.x, f_w, o.x), fmaf(v.y, f_w, o.y), fmaf(v.z, f_w, o.z), fmaf(v.w, f_w, o.w));
          }
          *reinterpret_cast<float4*>(obuf + row * Cfg::O_STRIDE + d) = o;
          if (d == 0) ml[row] = make_float2(m, l);
        }
      } else {
        if (quad == 0) {
          wml[warp * 16 + (lane >> 2)] = make_float2(st.m[0], st.l[0]);
          wml[warp * 16 + (lane >> 2) + 8] = make_float2(st.m[1], st.l[1]);
        }
        __syncthreads();
        float f_row[2];
#pragma unroll
        for (int rr = 0; rr < 2; ++rr) {
          const int row = (lane >> 2) + 8 * rr;
          float m = -INFINITY, l = 0.f;
#pragma unroll
          for (int w = 0; w < 4; ++w) m = fmaxf(m, wml[w * 16 + row].x);
#pragma unroll
          for (int w = 0; w < 4; ++w) {
            const float2 s = wml[w * 16 + row];
            if (s.x != -INFINITY) l = fmaf(s.y, exp2_fast(s.x - m), l);
          }
          f_row[rr] = st.m[rr] == -INFINITY ? 0.f : exp2_fast(st.m[rr] - m);
          if (warp == 0 && quad == 0) ml[row] = make_float2(m, l);
        }
        // The warps add their parts one after the other: a fixed order.
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          if (warp == w) {
#pragma unroll
            for (int rr = 0; rr < 2; ++rr) {
              float* dst = obuf + ((lane >> 2) + 8 * rr) * Cfg::O_STRIDE;
#pragma unroll
              for (int d = 0; d < D / 16; ++d) {
                // Sizes 4 quad .. + 3 of each 16 (e4m3), or 2 quad, + 1 of each 8.
                float4 v = Cfg::FP8 ? make_float4(st.o[2 * d][2 * rr], st.o[2 * d + 1][2 * rr], st.o[2 * d][2 * rr + 1], st.o[2 * d + 1][2 * rr + 1])
                                    : make_float4(st.o[2 * d][2 * rr], st.o[2 * d][2 * rr + 1], st.o[2 * d + 1][2 * rr], st.o[2 * d + 1][2 * rr + 1]);
                v = make_float4(v.x * f_row[rr], v.y * f_row[rr], v.z * f_row[rr], v.w * f_row[rr]);
                float2* p0 = reinterpret_cast<float2*>(dst + d * 16 + (Cfg::FP8 ? 4 : 2) * quad);
                float2* p1 = Cfg::FP8 ? p0 + 1 : p0 + 4;
                if (w > 0) {
                  v.x += p0->x, v.y += p0->y;
                  v.z += p1->x, v.w += p1->y;
                }
                *p0 = make_float2(v.x, v.y);
                *p1 = make_float2(v.z, v.w);
              }
            }
          }
          __syncthreads();
        }
      }
      if constexpr (CLUSTER) {
        cluster_sync_all();
        const uint32_t o_at = smem_base + Cfg::O_OFF, ml_at = smem_base + Cfg::ML_OFF;
        for (int x = (int)part * Cfg::THREADS + tid; x < t.rows * (D / 8); x += (int)parts * Cfg::THREADS) {
          const int row = x / (D / 8), d = (x % (D / 8)) * 8;
          // Two round trips, whatever the number of neighbours: every load of one is in flight before the first is used.
          float m = -INFINITY, v[8] = {}, l = 0.f, m_p[kAttnParts], l_p[kAttnParts];
#pragma unroll
          for (int p = 0; p < kAttnParts; ++p) {
            m_p[p] = p < parts ? ld_cluster_f32(mapa_shared(ml_at + row * 8, p)) : -INFINITY;
            l_p[p] = p < parts ? ld_cluster_f32(mapa_shared(ml_at + row * 8 + 4, p)) : 0.f;
          }
          float4 w0[kAttnParts], w1[kAttnParts];
#pragma unroll
          for (int p = 0; p < kAttnParts; ++p) {
            const uint32_t src = mapa_shared(o_at + (row * Cfg::O_STRIDE + d) * 4, p < parts ? p : 0);
            w0[p] = ld_cluster_f32x4(src);
            w1[p] = ld_cluster_f32x4(src + 16);
          }
#pragma unroll
          for (int p = 0; p < kAttnParts; ++p) m = fmaxf(m, m_p[p]);
#pragma unroll
          for (int p = 0; p < kAttnParts; ++p) {
            const float f_p = m_p[p] == -INFINITY ? 0.f : exp2_fast(m_p[p] - m);
            l = fmaf(l_p[p], f_p, l);
            const float w[8] = {w0[p].x, w0[p].y, w0[p].z, w0[p].w, w1[p].x, w1[p].y, w1[p].z, w1[p].w};
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = fmaf(w[e], f_p, v[e]);
          }
          attn_store_row<T, 8>(attn_out_row<T>(a, it, row) + d, v, l);
        }
        cluster_sync_all();             // nobody's shared memory goes before its neighbours have read it
        break;
      }
      for (int x = tid; x < t.rows * (D / 8); x += Cfg::THREADS) {
        const int row = x / (D / 8), d = (x % (D / 8)) * 8;
        const float4 v0 = *reinterpret_cast<const float4*>(obuf + row * Cfg::O_STRIDE + d),
                     v1 = *reinterpret_cast<const float4*>(obuf + row * Cfg::O_STRIDE + d + 4);
        if (whole) {
          const float v[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
          attn_store_row<T, 8>(attn_out_row<T>(a, it, row) + d, v, ml[row].y);
        } else {
          *reinterpret_cast<float4*>(piece + row * D + d) = v0;
          *reinterpret_cast<float4*>(piece + row * D + d + 4) = v1;
          if (d == 0) *reinterpret_cast<float2*>(piece + M * D + 2 * row) = ml[row];
        }
      }
    }
    flat += it.n;
    if (f < f1) attn_next<M, UNIT>(a, it);
  }
  cp_async_wait<0>();
}

// Joins the pieces of the items that a border of two CTAs' runs cuts; `ctas`: the grid of the launch before.  CTA (c, y) has
// every gridDim.y-th group of the (row, 8 sizes) cells of the item that the end of run c cuts first.  Few pieces: a thread
// for each cell.  Many (a long sequence has up to one for every CTA): 32 cells at a time, and eight warps share the pieces, so
// that they are read in a few round trips; their states meet in a fixed order.
constexpr int kJoinWarps = 8;
template <class T, class Cfg>
__global__ void __launch_bounds__(kJoinWarps * 32) attn_join_kernel(const AttnArgs a, const float* pieces, int ctas) {
  constexpr int D = Cfg::D, M = Cfg::M, UNIT = Cfg::UNIT;
  __shared__ float states[kJoinWarps][10][32];
  if (a.clear && blockIdx.y == 0) attn_clear_rest<T, D>(a, threadIdx.x, kJoinWarps * 32);
  long long own;
  const long long total = attn_total_units<M, UNIT>(a, own);
  const int c = blockIdx.x;
  const AttnRuns runs(total, ctas);
  const long long border = runs.begin(c + 1);
  AttnItem it = {};
  int at = 0;
  if (border < total && runs.begin(c) < border) at = attn_seek<M, UNIT>(a, border, own, it);
  pdl_wait();                                         // the pieces are there; and this launch never ends before that one
  const long long s = border - at, e = s + it.n;
  if (at == 0 || runs.begin(c) > s) return;                // nothing is cut here, or an earlier border cuts it too
  // Pieces of CTAs c .. c + n - 1; an empty run (fewer units than CTAs) has none.
  int n = 1;
  while (runs.begin(c + n) < e) ++n;
  const float* first = pieces + (2LL * c + (runs.begin(c) < s ? 1 : 0)) * Cfg::PIECE_FLOATS;
  const float* rest = pieces + 2LL * c * Cfg::PIECE_FLOATS;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const bool shared = n > 4;            // the warps share the pieces of a cell
  const int cells = it.t.rows * (D / 8), step = shared ? 32 : kJoinWarps * 32;
  for (int x0 = blockIdx.y * step; x0 < cells; x0 += gridDim.y * step) {
    const int x = x0 + (shared ? lane : (int)threadIdx.x);
    const bool on = x < cells;
    const int row = on ? x / (D / 8) : 0, d = (x % (D / 8)) * 8;
    float m = -INFINITY, l = 0.f, v[8] = {};
    // One state into the running one.
    auto add = [&](float m2, float l2, const float (&w)[8]) {
      const float top = fmaxf(m, m2);
      const float f = m == -INFINITY ? 0.f : exp2_fast(m - top), g = m2 == -INFINITY ? 0.f : exp2_fast(m2 - top);
      m = top;
      l = fmaf(l, f, l2 * g);
#pragma unroll
      for (int i = 0; i < 8; ++i) v[i] = fmaf(v[i], f, w[i] * g);
    };
    constexpr int AHEAD = 4;            // pieces whose loads are in flight together
    const int stride = shared ? kJoinWarps : 1;
    for (int k0 = shared ? warp : 0; k0 < n; k0 += stride * AHEAD) {
      float2 ml[AHEAD];
      float4 v0[AHEAD], v1[AHEAD];
#pragma unroll
      for (int y = 0; y < AHEAD; ++y) {
        const int k = k0 + y * stride;
        ml[y] = make_float2(-INFINITY, 0.f);
        v0[y] = v1[y] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (on && k < n && (runs.each > 0 || runs.begin(c + k + 1) > runs.begin(c + k))) {
          const float* p = k == 0 ? first : rest + 2LL * k * Cfg::PIECE_FLOATS;
          ml[y] = *reinterpret_cast<const float2*>(p + M * D + 2 * row);
          v0[y] = *reinterpret_cast<const float4*>(p + row * D + d);
          v1[y] = *reinterpret_cast<const float4*>(p + row * D + d + 4);
        }
      }
#pragma unroll
      for (int y = 0; y < AHEAD; ++y) {
        const float w[8] = {v0[y].x, v0[y].y, v0[y].z, v0[y].w, v1[y].x, v1[y].y, v1[y].z, v1[y].w};
        add(ml[y].x, ml[y].y, w);
      }
    }
    if (shared) {
      states[warp][0][lane] = m;
      states[warp][1][lane] = l;
#pragma unroll
      for (int i = 0; i < 8; ++i) states[warp][2 + i][lane] = v[i];
      __syncthreads();
      if (warp == 0) {
        for (int w = 1; w < kJoinWarps; ++w) {
          float z[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) z[i] = states[w][2 + i][lane];
          add(states[w][0][lane], states[w][1][lane], z);
        }
      }
    }
    if (on && (warp == 0 || !shared)) attn_store_row<T, 8>(attn_out_row<T>(a, it, row) + d, v, l);
    if (shared) __syncthreads();        // before the next cells' states
  }
}

// How a call is cut.  ctas > 0: runs of the line, one wave of two CTAs per SM.  parts > 0: clusters of that many.  Neither: a
// CTA for each item.
struct AttnCut {
  int ctas, parts;
  long long items;
};
template <class Cfg>
static AttnCut attn_cut(long long tokens, int seqs, int group, int kv_heads, bool single, long long most_tokens, int sms) {
  const long long rows = tokens * group, per_token = (group + Cfg::M - 1) / Cfg::M;
  // Tiles of the batch: at most one per token (or several where a group has more than M heads), and at most the full
  // ones and one more per sequence.
  long long tiles = single ? seqs * per_token : rows / Cfg::M + seqs;
  if (!single && tiles > tokens * per_token) tiles = tokens * per_token;
  const long long items = tiles * kv_heads, each = most_tokens > 0 ? (most_tokens + Cfg::UNIT - 1) / Cfg::UNIT : 1, slots = 2LL * sms;
  // Short single-token calls: a cluster of up to eight CTAs for each item, all of them resident at once, at least two units
  // and at most kShort for each CTA by the page table's width.
  constexpr int kShort = 8;
  if (single && !Cfg::ROWS && items * 2 <= slots) {
    long long parts = slots / items < kAttnParts ? slots / items : kAttnParts;
    if (parts > (each + 1) / 2) parts = (each + 1) / 2;
    if (parts >= 1 && each <= kShort * parts) return {0, (int)parts, items};
  }
  // Short items, a few waves of them at most: nothing to even out, and neither the scan of the batch nor the second launch
  // (8 sequences of 101 tokens, 8 heads, e4m3: 18.7 us with them, 10.0 without; 27 of 61 tokens, 32 heads: 20.4 and 12).
  if (each <= kShort && items <= 4 * slots) return {0, 0, items};
  const long long ctas = items * each / 2 < slots ? items * each / 2 : slots;
  return {ctas < 1 ? 1 : (int)ctas, 0, items};
}

template <class T, class Cfg>
static int launch_attn(const AttnArgs& a, void* workspace, size_t workspace_bytes, int dev, cudaStream_t st) {
  const AttnCut cut = attn_cut<Cfg>(a.tokens, a.seqs, a.group, a.kv_heads, a.query_starts == nullptr, (long long)a.table_width * a.page_size,
                                    sm_count(dev));
  cudaLaunchConfig_t cfg = {};
  cfg.stream = st;
  cudaLaunchAttribute attr;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if constexpr (!Cfg::ROWS) {
    if (cut.parts > 0) {
      static std::atomic<bool> done[64];
      if (!ensure_smem_attr(attn_kernel<T, Cfg, true>, dev, Cfg::SMEM_BYTES, done)) return TRB_ERR_CUDA;
      cfg.gridDim = dim3((unsigned)(cut.items * cut.parts));
      cfg.blockDim = dim3(Cfg::THREADS);
      cfg.dynamicSmemBytes = Cfg::SMEM_BYTES;
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = cut.parts;
      attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
      return cudaLaunchKernelEx(&cfg, attn_kernel<T, Cfg, true>, a, (float*)nullptr) == cudaSuccess ? TRB_OK : TRB_ERR_CUDA;
    }
  }
  static std::atomic<bool> done[64];
  if (!ensure_smem_attr(attn_kernel<T, Cfg, false>, dev, Cfg::SMEM_BYTES, done)) return TRB_ERR_CUDA;
  const bool line = cut.ctas > 0;
  if (line && (workspace == nullptr || workspace_bytes < 2ull * cut.ctas * Cfg::PIECE_FLOATS * 4)) return TRB_ERR_SCRATCH;
  attn_kernel<T, Cfg, false><<<line ? cut.ctas : (int)cut.items, Cfg::THREADS, Cfg::SMEM_BYTES, st>>>(a, line ? (float*)workspace : nullptr);
  if (cudaGetLastError() != cudaSuccess) return TRB_ERR_CUDA;
  if (cut.ctas <= 1) return TRB_OK;
  cfg.gridDim = dim3(cut.ctas - 1, Cfg::ROWS ? 4 : 1);
  cfg.blockDim = dim3(kJoinWarps * 32);
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  return cudaLaunchKernelEx(&cfg, attn_join_kernel<T, Cfg>, a, (const float*)workspace, cut.ctas) == cudaSuccess ? TRB_OK : TRB_ERR_CUDA;
}
}  // namespace trb
