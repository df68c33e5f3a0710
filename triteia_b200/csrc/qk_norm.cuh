// Root-mean-square norm of every query and key head together with the position rotation, one pass over the rows
// of a fused q/k/v product.  Stands beside rotary_embedding (elementwise.cuh; the reference's
// triteia/csrc/ops/pos_encoding_kernels.cu:118-160), which models with normed heads cannot use alone.
//   r = 1 / sqrt(mean_d x_d^2 + eps),  y_d = x_d r w_d,  first rot_dim elements of y: (a, b) -> (a c - b s, b c + a s)
// for the pairs (i, i + rot_dim / 2) (NeoX) or (2i, 2i + 1) (GPT-J).  32-bit arithmetic, one rounding at the end.
//
// A group of G = head_size / 8 lanes (rounded up to a power of two) holds one head, 8 elements = 16 bytes a lane: the sum of
// squares is log2(G) shuffles, a NeoX partner's inputs come with four more.  A group has up to five heads of ONE token and
// asks for all of them, for the position and then for its cosines and sines at once, so that a CTA waits for memory twice and
// no more: with loops over the heads of a token (fewer and longer CTAs) 8191 x 80 heads took 80 to 90 us, now 57 in a graph (5.9
// TB/s; 63 as calls in a row; before the arithmetic went two numbers at a time 61 with five heads a group, 74 with four or eight).
// Five is the number for 40 heads of queries and of keys.  Other numbers leave places empty, most of all few key heads, which have
// CTAs of their own: 32 + 32 heads 50.6 us (5.3 TB/s), 64 + 8 66 (4.6), 32 + 8 39 (4.3).
#pragma once

#include "elementwise.cuh"

namespace trb {

// Makes `dev` current and puts the previous device back.
struct DeviceGuard {
  int old = -1;
  bool ok;
  explicit DeviceGuard(int dev) {
    ok = cudaGetDevice(&old) == cudaSuccess;
    if (ok && old != dev) ok = cudaSetDevice(dev) == cudaSuccess;
    else old = -1;
  }
  ~DeviceGuard() {
    if (old >= 0) cudaSetDevice(old);
  }
};

// Two 32-bit products, sums or multiply-adds in one instruction.
__device__ __forceinline__ float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmul.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tadd.rn.f32x2 w, x, y;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z, w;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 w, x, y, z;\n\tmov.b64 {%0, %1}, w;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}

// The two numbers of a word.
__device__ __forceinline__ float2 two_of(uint32_t w, __half) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
__device__ __forceinline__ float2 two_of(uint32_t w, __nv_bfloat16) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
__device__ __forceinline__ uint32_t word_of(float2 v, __half) {
  const __half2 h = __floats2half2_rn(v.x, v.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}
__device__ __forceinline__ uint32_t word_of(float2 v, __nv_bfloat16) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
  return *reinterpret_cast<const uint32_t*>(&h);
}

struct QkNormArgs {
  const int64_t* positions;
  const void *query, *key;            // key may be null (num_kv_heads 0 then)
  void *query_out, *key_out;
  const void *query_weight, *key_weight;   // null: ones
  const void* table;                  // [max_position, rot_dim]: cosines, then sines
  long long max_position, q_stride, qo_stride, k_stride, ko_stride;
  int rot_dim, num_heads, num_kv_heads, head_size;
  float eps;
};

constexpr int kQkThreads = 128;
constexpr int kQkHeads = 5;           // heads of a group, all loaded together
// NeoX and GPT-J; "Any": rot_dim / 2 is no multiple of 8 (4), or the table or the weights are not 16-byte aligned, so that
// cosines, sines and weights come one by one (and a NeoX partner through shared memory).  "Part": without a norm, sizes that are
// not turned pass as they are, so that 0 * infinity must not reach them (with a norm an infinity leaves nothing of its head);
// a form of its own because the test costs the others 2 % (8191 x 80 heads 57 -> 58 us).
enum RotMode { kNeox, kNeoxPart, kNeoxAny, kPairs, kPairsPart, kPairsAny };

__device__ __forceinline__ float table_value(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float table_value(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float table_value(const float* p) { return *p; }

// N numbers from an aligned address.
template <int N, class TC>
__device__ __forceinline__ void table_values(const TC* p, float* v) {
  constexpr int BYTES = N * (int)sizeof(TC), PIECE = BYTES < 16 ? 8 : 16;
  using Word = typename std::conditional<PIECE == 16, uint4, uint2>::type;
#pragma unroll
  for (int i = 0; i < BYTES / PIECE; ++i) {
    const Word w = reinterpret_cast<const Word*>(p)[i];
#pragma unroll
    for (int e = 0; e < PIECE / (int)sizeof(TC); ++e) v[i * (PIECE / (int)sizeof(TC)) + e] = table_value(reinterpret_cast<const TC*>(&w) + e);
  }
}

template <class T, class TC, int G, int MODE>
__global__ void __launch_bounds__(kQkThreads) qk_norm_rotary_kernel(const QkNormArgs a) {
  constexpr int GROUPS = kQkThreads / G;
  constexpr bool PAIRS = MODE == kPairs || MODE == kPairsPart || MODE == kPairsAny;
  constexpr bool NEOX = MODE == kNeox || MODE == kNeoxPart, PART = MODE != kNeox && MODE != kPairs;
  __shared__ uint4 swap[MODE == kNeoxAny ? GROUPS : 1][MODE == kNeoxAny ? G : 1];
  const long long t = blockIdx.x;
  const int li = threadIdx.x % G, grp = threadIdx.x / G;
  const int d0 = li * 8;              // first of this lane's elements
  const bool active = d0 < a.head_size;
  const bool is_key = blockIdx.z != 0;
  const int heads = is_key ? a.num_kv_heads : a.num_heads;
  const int step = gridDim.y * GROUPS, h0 = blockIdx.y * GROUPS + grp;
  if (h0 >= heads) return;
  const T* in = is_key ? static_cast<const T*>(a.key) + t * a.k_stride : static_cast<const T*>(a.query) + t * a.q_stride;
  T* out = is_key ? static_cast<T*>(a.key_out) + t * a.ko_stride : static_cast<T*>(a.query_out) + t * a.qo_stride;
  uint4 raw[kQkHeads];                // all loads in flight, before the position is known
#pragma unroll
  for (int u = 0; u < kQkHeads; ++u) {
    const int h = h0 + u * step;
    raw[u] = make_uint4(0, 0, 0, 0);
    if (active && h < heads) raw[u] = *reinterpret_cast<const uint4*>(in + (long long)h * a.head_size + d0);
  }
  const int64_t pos = a.positions[t];
  const T* w = static_cast<const T*>(is_key ? a.key_weight : a.query_weight);
  const int half = a.rot_dim / 2;
  const unsigned lanes = G == 32 ? 0xffffffffu : ((1u << G) - 1u) << ((threadIdx.x & 31) / G * G);
  // y_d = r (x_d own_d + x_partner other_d): own = weight x cosine, other = the partner's weight x sine with its sign.
  float own[8], other[8];
  const bool there = pos >= 0 && pos < a.max_position;        // not: a padding token
  const TC* row = static_cast<const TC*>(a.table) + (there ? pos : 0) * a.rot_dim;
  if constexpr (NEOX || (PAIRS && MODE != kPairsAny)) {
    // A lane's eight elements turn together or not at all.
    const bool turn = there && d0 < a.rot_dim;
    const int i = !turn ? 0 : PAIRS ? d0 >> 1 : d0 < half ? d0 : d0 - half;
    const int partner = !turn || PAIRS ? d0 : d0 < half ? d0 + half : d0 - half;
    float c[8], sn[8], ww[8], wp[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = 1.f, sn[e] = 0.f, ww[e] = wp[e] = 1.f;
    if (turn) {
      table_values<PAIRS ? 4 : 8>(row + i, c);
      table_values<PAIRS ? 4 : 8>(row + half + i, sn);
    }
    if (w && active) {
      table_values<8>(w + d0, ww);
      table_values<8>(w + partner, wp);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float ce = !turn ? 1.f : PAIRS ? c[e >> 1] : c[e], se = !turn ? 0.f : PAIRS ? sn[e >> 1] : sn[e];
      own[e] = ce * ww[e];
      other[e] = ((PAIRS ? (e & 1) == 0 : d0 < half) ? -se : se) * (PAIRS ? wp[e ^ 1] : wp[e]);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int d = d0 + e;
      const bool turn = there && d < a.rot_dim;
      const int i = !turn ? 0 : PAIRS ? d >> 1 : d < half ? d : d - half;
      const int partner = !turn ? d : PAIRS ? d ^ 1 : d < half ? d + half : d - half;
      const float c = turn ? table_value(row + i) : 1.f, sn = turn ? table_value(row + half + i) : 0.f;
      own[e] = c * (w && active ? Ew<T>::to_f(w[d]) : 1.f);
      other[e] = ((PAIRS ? (d & 1) == 0 : d < half) ? -sn : sn) * (w && active ? Ew<T>::to_f(w[partner]) : 1.f);
    }
  }
  if (!there) return;
  const float inv_size = 1.f / (float)a.head_size;
#pragma unroll
  for (int u = 0; u < kQkHeads; ++u) {
    const int h = h0 + u * step;
    if (h >= heads) break;
    // The partners' inputs come over as they are, two to a word; their factor of the norm is this head's too.
    uint4 them = raw[u];
    if constexpr (NEOX) {
      const int hl = half >> 3;
      const int src = li < hl ? li + hl : li < 2 * hl ? li - hl : li;
      them.x = __shfl_sync(lanes, raw[u].x, src, G);
      them.y = __shfl_sync(lanes, raw[u].y, src, G);
      them.z = __shfl_sync(lanes, raw[u].z, src, G);
      them.w = __shfl_sync(lanes, raw[u].w, src, G);
    } else if constexpr (MODE == kNeoxAny) {
      swap[grp][li] = raw[u];
      __syncwarp(lanes);
      T* te = reinterpret_cast<T*>(&them);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int d = d0 + e;
        te[e] = reinterpret_cast<const T*>(swap[grp])[d >= a.rot_dim ? d : d < half ? d + half : d - half];
      }
      __syncwarp(lanes);
    }
    uint32_t* mine = reinterpret_cast<uint32_t*>(&raw[u]);
    const uint32_t* theirs = reinterpret_cast<const uint32_t*>(&them);
    float2 x[4], sum2 = make_float2(0.f, 0.f);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      x[e] = two_of(mine[e], T());
      sum2 = fma2(x[e], x[e], sum2);
    }
    float sum = sum2.x + sum2.y;
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(lanes, sum, o);
    const float r = a.eps < 0.f ? 1.f : rsqrtf(sum * inv_size + a.eps);      // eps < 0: the rotation alone
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      float2 p = PAIRS ? make_float2(x[e].y, x[e].x) : two_of(theirs[e], T());
      if (PART && d0 + 2 * e >= a.rot_dim) p = make_float2(0.f, 0.f);
      const float2 y = fma2(x[e], make_float2(own[2 * e], own[2 * e + 1]), mul2(p, make_float2(other[2 * e], other[2 * e + 1])));
      mine[e] = word_of(mul2(y, make_float2(r, r)), T());
    }
    if (active) *reinterpret_cast<uint4*>(out + (long long)h * a.head_size + d0) = raw[u];
  }
}

template <class T, class TC, int G>
static void launch_qk_norm(const QkNormArgs& a, int mode, dim3 grid, cudaStream_t st) {
  if (mode == kNeox) qk_norm_rotary_kernel<T, TC, G, kNeox><<<grid, kQkThreads, 0, st>>>(a);
  else if (mode == kNeoxPart) qk_norm_rotary_kernel<T, TC, G, kNeoxPart><<<grid, kQkThreads, 0, st>>>(a);
  else if (mode == kNeoxAny) qk_norm_rotary_kernel<T, TC, G, kNeoxAny><<<grid, kQkThreads, 0, st>>>(a);
  else if (mode == kPairs) qk_norm_rotary_kernel<T, TC, G, kPairs><<<grid, kQkThreads, 0, st>>>(a);
  else if (mode == kPairsPart) qk_norm_rotary_kernel<T, TC, G, kPairsPart><<<grid, kQkThreads, 0, st>>>(a);
  else qk_norm_rotary_kernel<T, TC, G, kPairsAny><<<grid, kQkThreads, 0, st>>>(a);
}

template <class T, class TC>
static void launch_qk_norm(const QkNormArgs& a, int num_tokens, bool is_neox, int sms, cudaStream_t st) {
  int g = 1;
  while (g * 8 < a.head_size) g *= 2;
  const int groups = kQkThreads / g, heads = a.num_heads > a.num_kv_heads ? a.num_heads : a.num_kv_heads;
  // A CTA has the query's or the key's heads of a token, kQkHeads of them in a group; few tokens: fewer heads in a group,
  // until about four CTAs per SM run.
  const int most = (heads + groups - 1) / groups, least = (heads + kQkHeads * groups - 1) / (kQkHeads * groups);
  int y = (2 * sms + num_tokens - 1) / num_tokens;
  y = y < least ? least : y > most ? most : y;
  const dim3 grid(num_tokens, y, a.num_kv_heads > 0 ? 2 : 1);
  const bool aligned = (((uintptr_t)a.table | (uintptr_t)a.query_weight | (uintptr_t)a.key_weight) & 15) == 0;
  const bool part = a.eps < 0.f && a.rot_dim < a.head_size;
  const int mode = is_neox ? (!aligned || a.rot_dim % 16 != 0 ? kNeoxAny : part ? kNeoxPart : kNeox)
                           : (!aligned || a.rot_dim % 8 != 0 ? kPairsAny : part ? kPairsPart : kPairs);
  switch (g) {
    case 1: launch_qk_norm<T, TC, 1>(a, mode, grid, st); break;
    case 2: launch_qk_norm<T, TC, 2>(a, mode, grid, st); break;
    case 4: launch_qk_norm<T, TC, 4>(a, mode, grid, st); break;
    case 8: launch_qk_norm<T, TC, 8>(a, mode, grid, st); break;
    case 16: launch_qk_norm<T, TC, 16>(a, mode, grid, st); break;
    default: launch_qk_norm<T, TC, 32>(a, mode, grid, st); break;
  }
}

}  // namespace trb

extern "C" int trb_qk_norm_rotary(const void* positions, const void* query, void* query_out, const void* key, void* key_out,
                                  const void* query_weight, const void* key_weight, const void* cos_sin_cache, int cache_is_f32,
                                  long long max_position, int num_tokens, int rot_dim, long long query_stride,
                                  long long query_out_stride, long long key_stride, long long key_out_stride, int num_heads,
                                  int num_kv_heads, int head_size, float eps, int is_neox, int dtype, int dev, void* stream) {
  using namespace trb;
  if (num_tokens == 0) return TRB_OK;
  if (num_tokens < 0 || !positions || !query || !query_out || (!cos_sin_cache && rot_dim > 0) || max_position < 0 || num_heads <= 0 || num_kv_heads < 0 ||
      (num_kv_heads > 0 && (!key || !key_out)))
    return TRB_ERR_BAD_ARG;
  if (head_size <= 0 || head_size % 8 != 0 || head_size > 256 || rot_dim < 0 || rot_dim % 2 != 0 || rot_dim > head_size)
    return TRB_ERR_PROB_SHAPE;
  if (num_tokens == 1) query_stride = query_out_stride = key_stride = key_out_stride = 0;      // of one row: says nothing
  if (((uintptr_t)query | (uintptr_t)query_out) & 15 || ((query_stride | query_out_stride) & 7) != 0) return TRB_ERR_PROB_SHAPE;
  if (num_kv_heads > 0 && (((uintptr_t)key | (uintptr_t)key_out) & 15 || ((key_stride | key_out_stride) & 7) != 0)) return TRB_ERR_PROB_SHAPE;
  if (dtype != TRB_F16 && dtype != TRB_BF16) return TRB_ERR_KERN_SHAPE;
  DeviceGuard guard(dev);
  if (!guard.ok) return TRB_ERR_CUDA;
  const QkNormArgs a{(const int64_t*)positions, query, key, query_out, key_out, query_weight, key_weight, cos_sin_cache, max_position,
                     query_stride, query_out_stride, key_stride, key_out_stride, rot_dim, num_heads, num_kv_heads, head_size, eps};
  const int sms = sm_count(dev);
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == TRB_F16) {
    if (cache_is_f32) launch_qk_norm<__half, float>(a, num_tokens, is_neox != 0, sms, st);
    else launch_qk_norm<__half, __half>(a, num_tokens, is_neox != 0, sms, st);
  } else {
    if (cache_is_f32) launch_qk_norm<__nv_bfloat16, float>(a, num_tokens, is_neox != 0, sms, st);
    else launch_qk_norm<__nv_bfloat16, __nv_bfloat16>(a, num_tokens, is_neox != 0, sms, st);
  }
  return cudaGetLastError() == cudaSuccess ? TRB_OK : TRB_ERR_CUDA;
}
