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
// (single tokens, short chunks) and the caches that the tensor-memory kernel does not take.  Per 16 x 16 block of scores it
// issues two m16n8k16 MMAs for each 16 of the head size, one running maximum per row, and as many MMAs again with the
// values.
//   M = 16: the four warps of a CTA take different tokens (16 each of every 64) and keep softmax states of their own,
//           so that nothing in the loop is CTA-wide; the states meet at the end.
//   M = 64: a warp has 16 rows, and the four share the 64 tokens of a stage.
// The CTAs of a cluster share a tile along the tokens and join their states through distributed shared memory: one
// launch, no workspace, no counters, and a fixed order of the sums.
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
  const long long most = (long long)a.table_width * a.page_size;
  t.length = (int)max(0LL, min((long long)a.lengths[t.seq], most));
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
  static constexpr int MASK_OFF = STAGES * STAGE_BYTES;         // uint32 [STAGES][4]: tokens that count, per loading warp
  static constexpr int EXP_OFF = MASK_OFF + STAGES * 16;        // float [STAGES][3][UNIT]: 2^e of keys; e and 2^-e of values
  static constexpr int ML_OFF = EXP_OFF + (FP8 ? STAGES * 3 * UNIT * 4 : 0);   // float [M][2]: the CTA's maxima and sums
  static constexpr int WML_OFF = ML_OFF + M * 8;                // float [4][16][2]: the warps' (M = 16)
  static constexpr int SMEM_BYTES = WML_OFF + 4 * 16 * 8;
  static constexpr int O_STRIDE = D + 4;                        // floats; rows of the joined states (in the idle ring)
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
// to a largest magnitude of 2^9 .. 2^10, keeps all its bits down to 2^-25 of that.  Weights are fp16 there (11 bits).
template <class T, bool FP8>
struct AttnMma { using type = T; };
template <class T>
struct AttnMma<T, true> { using type = __half; };

// Exponent field of the power of two that brings a bf16 row with the largest magnitude `top` to 2^9 .. 2^10.
__device__ __forceinline__ int attn_row_shift(float top) {
  const int field = (int)(__float_as_uint(top) >> 23);                  // top in [2^(field - 127), twice that)
  return top > 0.f ? min(max(127 + 127 + 9 - field, 1), 253) : 127;
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
      s[n][0] = fmaf(s[n][0] * kf.x, c_row[0], ev.x);
      s[n][1] = fmaf(s[n][1] * kf.y, c_row[0], ev.y);
      s[n][2] = fmaf(s[n][2] * kf.x, c_row[1], ev.x);
      s[n][3] = fmaf(s[n][3] * kf.y, c_row[1], ev.y);
    }
  } else {
#pragma unroll
    for (int n = 0; n < 2 * NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) s[n][e] *= c_row[e >> 1];
  }
  if (need_mask) {
#pragma unroll
    for (int n = 0; n < 2 * NT; ++n)
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const int jl = n * 8 + 2 * quad + (e & 1), j = j0 + jl;
        if (!((valid >> jl) & 1) || j >= row_hi[e >> 1] || j < row_lo[e >> 1]) s[n][e] = -INFINITY;
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
  // ---- values: the weights are rounded to the MMA type (half a step, of random sign), the sum above is not.
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

template <class T, class Cfg>
__global__ void __launch_bounds__(Cfg::THREADS, 2) attn_kernel(const AttnArgs a) {
  using TM = typename AttnMma<T, Cfg::FP8>::type;
  constexpr int D = Cfg::D, M = Cfg::M, STAGES = Cfg::STAGES;
  extern __shared__ __align__(128) uint8_t smem[];
  const uint32_t smem_base = smem_u32(smem);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, quad = lane & 3;
  uint32_t parts, part;
  asm("mov.u32 %0, %%cluster_nctarank;" : "=r"(parts));
  asm("mov.u32 %0, %%cluster_ctarank;" : "=r"(part));
  const int item = blockIdx.x / parts;
  const int kvh = item % a.kv_heads;
  AttnTile t;
  if (!attn_find_tile<M>(a, item / a.kv_heads, t)) return;      // the whole cluster leaves
  int lo, hi;
  attn_key_range(a, t, lo, hi);
  // This CTA's units of 64 tokens.
  const int u_first = lo / Cfg::UNIT, u_all = hi > lo ? (hi + Cfg::UNIT - 1) / Cfg::UNIT - u_first : 0;
  const int u0 = u_first + (int)((long long)u_all * part / parts), u1 = u_first + (int)((long long)u_all * (part + 1) / parts);

  const int* table = a.page_table + t.seq * a.table_stride;
  const uint8_t* kc = static_cast<const uint8_t*>(a.key_cache);
  const uint8_t* vc = static_cast<const uint8_t*>(a.value_cache);
  constexpr int ESZ = Cfg::FP8 ? 1 : 2;
  uint32_t* masks = reinterpret_cast<uint32_t*>(smem + Cfg::MASK_OFF);
  float* exps = reinterpret_cast<float*>(smem + Cfg::EXP_OFF);
  constexpr int WTOK = Cfg::WTOK;                     // 16 or 32 tokens of a stage are this warp's to load
  const int tok = warp * WTOK + (lane & (WTOK - 1));  // this lane's among the unit's

  // Page and place of this lane's token of unit u (page -1: not visible, or not in the cache), found one unit ahead.
  struct Where { int page, place; };
  auto where = [&](int u) -> Where {
    const int j = u * Cfg::UNIT + tok;
    if (u >= u1 || j < lo || j >= hi) return {-1, 0};
    const int p = a.page_shift >= 0 ? j >> a.page_shift : j / a.page_size;
    const int pg = table[p];
    return {pg >= 0 && pg < a.num_pages ? pg : -1, j - p * a.page_size};
  };
  Where ahead = where(u0);
  int exp_slot = -1, kb = 127, vb = 127;              // e4m3: the bytes that the last issue() asked for, and their stage
  auto settle_exps = [&]() {
    if (exp_slot >= 0 && lane < WTOK) {
      float* e = exps + exp_slot * 3 * Cfg::UNIT + tok;
      e[0] = pow2_of_byte(kb);
      e[Cfg::UNIT] = (float)(vb - 127);
      e[2 * Cfg::UNIT] = pow2_of_byte(254 - vb);
    }
  };
  constexpr int PER = 32 / Cfg::CHUNKS;               // rows per instruction
  const int c = lane % Cfg::CHUNKS, r0 = lane / Cfg::CHUNKS;
  const long long row_bytes = a.c_tok * ESZ;
  const bool paged16 = (a.page_size & 15) == 0;       // 16 tokens of a unit lie on one page
  // Loads this warp's tokens of unit u into `slot`.
  auto issue = [&](int u, int slot) {
    if constexpr (Cfg::FP8) settle_exps();
    const Where w = ahead;
    ahead = where(u + 1);
    if (u < u1) {
      const bool there = w.page >= 0;
      long long off = there ? (long long)w.page * a.c_page + (long long)w.place * a.c_tok + (long long)kvh * a.c_head : 0;
      if constexpr (ESZ == 2) off *= 2;
      unsigned mask = __ballot_sync(0xffffffffu, there);
      if constexpr (WTOK == 16) mask &= 0xffffu;
      if (lane == 0) masks[slot * 4 + warp] = mask;
      if constexpr (Cfg::FP8) {
        exp_slot = slot;
        kb = vb = 127;
        if (there) {
          const long long eo = (long long)w.page * a.e_page + (long long)w.place * a.e_tok + (long long)kvh * a.e_head;
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
#pragma unroll
        for (int i = 0; i < WTOK / PER; ++i) {
          const int r = i * PER + r0;
          const long long ro = __shfl_sync(0xffffffffu, off, r) + c * 16;
          const bool ok = (mask >> r) & 1;
          const uint32_t at = dst + attn_swizzle<Cfg::ROWB>(warp * WTOK + r, c);
          cp_async16(at, kc + ro, ok);
          cp_async16(at + Cfg::HALF_BYTES, vc + ro, ok);
        }
      }
    } else {
      exp_slot = -1;
    }
    cp_async_commit();
  };
#pragma unroll
  for (int i = 0; i < STAGES - 1; ++i) issue(u0 + i, i);

  // ---- this warp's rows: query fragments, visible ranges
  const int wrow = Cfg::ROWS ? warp * 16 : 0;
  uint32_t q[D / 16][4];
  float c_row[2];
  int row_hi[2], row_lo[2];
#pragma unroll
  for (int rr = 0; rr < 2; ++rr) {
    const int row = wrow + (lane >> 2) + 8 * rr;
    const bool on = row < t.rows;
    const int rq = t.row0 + (on ? row : 0);
    const int i = rq / a.group, head = kvh * a.group + (rq - i * a.group);
    const T* qp = static_cast<const T*>(a.query) + (t.q0 + i) * a.q_tok + head * a.q_head;
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

  int slot = 0;
  for (int u = u0; u < u1; ++u) {
    cp_async_wait<STAGES - 2>();
    if constexpr (Cfg::ROWS) __syncthreads();
    else __syncwarp();
    issue(u + STAGES - 1, slot == 0 ? STAGES - 1 : slot - 1);
    if (!idle) {
      constexpr int TOK = Cfg::NT * 16;
      const int own = Cfg::ROWS ? 0 : warp * WTOK;
      const int j0 = u * Cfg::UNIT + own;
      const uint32_t* mk = masks + slot * 4;
      const unsigned long long valid =
          Cfg::ROWS ? (unsigned long long)(mk[0] | mk[1] << 16) | (unsigned long long)(mk[2] | mk[3] << 16) << 32 : mk[warp];
      constexpr unsigned long long kAll = ~0ull >> (64 - TOK);
      if (valid != 0) {
        const bool need_mask = valid != kAll || j0 + TOK > all_hi || j0 < all_lo;
        const uint32_t kbase = smem_base + slot * Cfg::STAGE_BYTES + own * Cfg::ROWB;
        attn_block<T, Cfg, Cfg::NT>(st, q, c_row, kbase, kbase + Cfg::HALF_BYTES, exps + slot * 3 * Cfg::UNIT + own, valid, j0, row_hi,
                                    row_lo, need_mask, lane);
      }
    }
    if constexpr (!Cfg::ROWS) __syncwarp();
    slot = slot + 1 == STAGES ? 0 : slot + 1;
  }
  cp_async_wait<0>();
  __syncthreads();                      // the ring is idle: it takes the states now

  // ---- states into shared memory: float o[rows][D + 4], {m, l} per row
#pragma unroll
  for (int r = 0; r < 2; ++r) {
    st.l[r] += __shfl_xor_sync(0xffffffffu, st.l[r], 1);
    st.l[r] += __shfl_xor_sync(0xffffffffu, st.l[r], 2);
  }
  float* obuf = reinterpret_cast<float*>(smem);
  float2* ml = reinterpret_cast<float2*>(smem + Cfg::ML_OFF);
  float2* wml = reinterpret_cast<float2*>(smem + Cfg::WML_OFF);
  {
#pragma unroll
    for (int rr = 0; rr < 2; ++rr) {
      const int row = warp * 16 + (lane >> 2) + 8 * rr;
      float* dst = obuf + row * Cfg::O_STRIDE;
      if (quad == 0) (Cfg::ROWS ? ml : wml)[row] = make_float2(st.m[rr], st.l[rr]);
      if constexpr (!Cfg::FP8) {
#pragma unroll
        for (int d = 0; d < D / 8; ++d)
          *reinterpret_cast<float2*>(dst + d * 8 + 2 * quad) = make_float2(st.o[d][2 * rr], st.o[d][2 * rr + 1]);
      } else {
#pragma unroll
        for (int d = 0; d < D / 16; ++d)
          *reinterpret_cast<float4*>(dst + d * 16 + 4 * quad) =
              make_float4(st.o[2 * d][2 * rr], st.o[2 * d + 1][2 * rr], st.o[2 * d][2 * rr + 1], st.o[2 * d + 1][2 * rr + 1]);
      }
    }
  }
  __syncthreads();
  if constexpr (!Cfg::ROWS) {
    // The four warps' states become the CTA's, in place of the first warp's: an element is read and written by one thread.
    for (int x = tid; x < 16 * (D / 4); x += Cfg::THREADS) {
      const int row = x / (D / 4), d = (x % (D / 4)) * 4;
      float m = -INFINITY;
#pragma unroll
      for (int w = 0; w < 4; ++w) m = fmaxf(m, wml[w * 16 + row].x);
      float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
      float l = 0.f;
#pragma unroll
      for (int w = 0; w < 4; ++w) {
        const float2 s = wml[w * 16 + row];
        const float f = s.x == -INFINITY ? 0.f : exp2_fast(s.x - m);
        const float4 v = *reinterpret_cast<const float4*>(obuf + (w * 16 + row) * Cfg::O_STRIDE + d);
        l = fmaf(s.y, f, l);
        o.x = fmaf(v.x, f, o.x);
        o.y = fmaf(v.y, f, o.y);
        o.z = fmaf(v.z, f, o.z);
        o.w = fmaf(v.w, f, o.w);
      }
      *reinterpret_cast<float4*>(obuf + row * Cfg::O_STRIDE + d) = o;
      if (d == 0) ml[row] = make_float2(m, l);
    }
  }
  if (parts > 1) cluster_sync_all();
  else __syncthreads();
  // ---- the cluster's states joined in the order of the tokens, divided, rounded once
  const uint32_t o_local = smem_base, ml_local = smem_base + Cfg::ML_OFF;
  for (int x = (int)part * Cfg::THREADS + tid; x < t.rows * (D / 8); x += (int)parts * Cfg::THREADS) {
    const int row = x / (D / 8), d = (x % (D / 8)) * 8;
    float m = -INFINITY;
    for (uint32_t p = 0; p < parts; ++p) m = fmaxf(m, ld_cluster_f32(mapa_shared(ml_local + row * 8, p)));
    float o[8] = {}, l = 0.f;
    if (m != -INFINITY) {
      for (uint32_t p = 0; p < parts; ++p) {
        const float f = exp2_fast(ld_cluster_f32(mapa_shared(ml_local + row * 8, p)) - m);
        l = fmaf(ld_cluster_f32(mapa_shared(ml_local + row * 8 + 4, p)), f, l);
        const uint32_t src = mapa_shared(o_local + (row * Cfg::O_STRIDE + d) * 4, p);
        const float4 v0 = ld_cluster_f32x4(src), v1 = ld_cluster_f32x4(src + 16);
        const float v[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = fmaf(v[e], f, o[e]);
      }
    }
    const float inv = l == 0.f ? 0.f : 1.f / l;
    uint4 packed;
    T* pe = reinterpret_cast<T*>(&packed);
#pragma unroll
    for (int e = 0; e < 8; ++e) pe[e] = Ew<T>::from_f(l == 0.f ? 0.f : o[e] * inv);
    const int rq = t.row0 + row, i = rq / a.group, head = kvh * a.group + (rq - i * a.group);
    *reinterpret_cast<uint4*>(static_cast<T*>(a.out) + (t.q0 + i) * a.o_tok + head * a.o_head + d) = packed;
  }
  if (parts > 1) cluster_sync_all();    // nobody's shared memory goes before its neighbours have read it
}

// CTAs of a cluster that share a tile: where the tiles alone would leave SMs idle (two CTAs fit an SM), as many as fill
// one wave, at most 16; several waves of tiles are cut into eight or so, so that sequences of different lengths even out.
static int attn_parts(long long tiles, long long most_tokens, int unit, int sms) {
  const long long slots = 2LL * sms, units = (most_tokens + unit - 1) / unit;
  long long parts = 2 * tiles <= slots ? slots / tiles : (8 * slots + tiles - 1) / tiles;
  parts = parts > 16 ? 16 : parts;
  if (2 * tiles > slots && parts > 8) parts = 8;
  if (parts > (units + 1) / 2) parts = (units + 1) / 2;      // two units each at least
  return parts < 1 ? 1 : (int)parts;
}

template <class T, class Cfg>
static int launch_attn(const AttnArgs& a, int dev, cudaStream_t st) {
  static std::atomic<bool> wide[64], done[64];
  if (dev < 0 || dev >= 64 || !wide[dev].load(std::memory_order_acquire)) {      // clusters of more than eight CTAs
    if (cudaFuncSetAttribute(attn_kernel<T, Cfg>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) return TRB_ERR_CUDA;
    if (dev >= 0 && dev < 64) wide[dev].store(true, std::memory_order_release);
  }
  if (!ensure_smem_attr(attn_kernel<T, Cfg>, dev, Cfg::SMEM_BYTES, done)) return TRB_ERR_CUDA;
  const long long rows = (long long)a.tokens * a.group;
  const long long per_token = (a.group + Cfg::M - 1) / Cfg::M;
  // Tiles of the batch: at most one per token (or several where a group has more than M heads), and at most the full
  // ones and one more per sequence.
  long long tiles = a.query_starts ? rows / Cfg::M + a.seqs : a.seqs * per_token;
  if (a.query_starts && tiles > a.tokens * per_token) tiles = a.tokens * per_token;
  if (tiles == 0) return TRB_OK;
  const int parts = attn_parts(tiles * a.kv_heads, (long long)a.table_width * a.page_size, Cfg::UNIT, sm_count(dev));
  const long long grid = tiles * a.kv_heads * parts;
  if (grid > 0x7fffffffLL) return TRB_ERR_PROB_SHAPE;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)grid);
  cfg.blockDim = dim3(Cfg::THREADS);
  cfg.dynamicSmemBytes = Cfg::SMEM_BYTES;
  cfg.stream = st;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeClusterDimension;
  attr.val.clusterDim.x = parts;
  attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  if (cudaLaunchKernelEx(&cfg, attn_kernel<T, Cfg>, a) != cudaSuccess) {
    cudaGetLastError();
    return TRB_ERR_CUDA;
  }
  return TRB_OK;
}

}  // namespace trb
