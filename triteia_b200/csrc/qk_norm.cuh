// Root-mean-square norm of every query and key head together with the position rotation, one pass over the rows
// of a fused q/k/v product.  Stands beside rotary_embedding (elementwise.cuh; the reference's
// triteia/csrc/ops/pos_encoding_kernels.cu:118-160), which models with normed heads cannot use alone.
//   r = 1 / sqrt(mean_d x_d^2 + eps),  y_d = x_d r w_d,  first rot_dim elements of y: (a, b) -> (a c - b s, b c + a s)
// for the pairs (i, i + rot_dim / 2) (NeoX) or (2i, 2i + 1) (GPT-J).  32-bit arithmetic, one rounding at the end.
//
// A group of G = head_size / 8 lanes (rounded up to a power of two) holds one head, 8 elements = 16 bytes a lane:
// the sum of squares is log2(G) shuffles, a NeoX partner is one shuffle per element away.  A group goes through
// several heads of ONE token, so the token's cosines and sines and the weights are read once and stay in registers.
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
enum RotMode { kNeoxLanes, kNeoxAny, kPairs };   // NeoX with rot_dim / 2 a multiple of 8, any other NeoX, GPT-J

__device__ __forceinline__ float table_value(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ float table_value(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float table_value(const float* p) { return *p; }

template <class T, class TC, int G, int MODE>
__global__ void __launch_bounds__(kQkThreads) qk_norm_rotary_kernel(const QkNormArgs a) {
  constexpr int GROUPS = kQkThreads / G;
  constexpr int AHEAD = 4;            // heads whose loads are in flight together
  __shared__ float swap[MODE == kNeoxAny ? GROUPS : 1][MODE == kNeoxAny ? G * 8 : 1];
  const long long t = blockIdx.x;
  const int li = threadIdx.x % G, grp = threadIdx.x / G;
  const int d0 = li * 8;              // first of this lane's elements
  const bool active = d0 < a.head_size;
  const int64_t pos = a.positions[t];
  if (pos < 0 || pos >= a.max_position) return;     // a padding token
  const int half = a.rot_dim / 2;
  const TC* row = static_cast<const TC*>(a.table) + pos * a.rot_dim;
  float c[8], s[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int d = d0 + e;
    const bool turn = d < a.rot_dim;
    const int i = !turn ? 0 : MODE == kPairs ? d >> 1 : d < half ? d : d - half;
    c[e] = turn ? table_value(row + i) : 1.f;
    const float sn = turn ? table_value(row + half + i) : 0.f;
    s[e] = (MODE == kPairs ? (d & 1) == 0 : d < half) ? -sn : sn;   // the sign that goes with the partner
  }
  const int total = a.num_heads + a.num_kv_heads;
  const int step = gridDim.y * GROUPS;
  const unsigned lanes = G == 32 ? 0xffffffffu : ((1u << G) - 1u) << ((threadIdx.x & 31) / G * G);
  float wq[8], wk[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    wq[e] = active && a.query_weight ? Ew<T>::to_f(static_cast<const T*>(a.query_weight)[d0 + e]) : 1.f;
    wk[e] = active && a.key_weight ? Ew<T>::to_f(static_cast<const T*>(a.key_weight)[d0 + e]) : 1.f;
  }
  for (int h0 = blockIdx.y * GROUPS + grp; h0 < total; h0 += AHEAD * step) {
    uint4 raw[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int h = h0 + u * step;
      raw[u] = make_uint4(0, 0, 0, 0);
      if (active && h < total) {
        const T* p = h < a.num_heads ? static_cast<const T*>(a.query) + t * a.q_stride + (long long)h * a.head_size
                                     : static_cast<const T*>(a.key) + t * a.k_stride + (long long)(h - a.num_heads) * a.head_size;
        raw[u] = *reinterpret_cast<const uint4*>(p + d0);
      }
    }
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int h = h0 + u * step;
      if (h >= total) break;
      const bool is_q = h < a.num_heads;
      T* e16 = reinterpret_cast<T*>(&raw[u]);
      float x[8], sum = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = Ew<T>::to_f(e16[e]);
        sum = fmaf(x[e], x[e], sum);
      }
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) sum += __shfl_xor_sync(lanes, sum, o);
      const float r = rsqrtf(sum / (float)a.head_size + a.eps);
#pragma unroll
      for (int e = 0; e < 8; ++e) x[e] *= r * (is_q ? wq[e] : wk[e]);
      float y[8];
      if (MODE == kPairs) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = fmaf(x[e], c[e], x[e ^ 1] * s[e]);
      } else if (MODE == kNeoxLanes) {
        const int hl = half >> 3;
        const int src = li < hl ? li + hl : li < 2 * hl ? li - hl : li;
#pragma unroll
        for (int e = 0; e < 8; ++e) y[e] = fmaf(x[e], c[e], __shfl_sync(lanes, x[e], src, G) * s[e]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) swap[grp][d0 + e] = x[e];
        __syncwarp(lanes);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int d = d0 + e;
          const int from = d >= a.rot_dim ? d : d < half ? d + half : d - half;
          y[e] = fmaf(x[e], c[e], swap[grp][from] * s[e]);
        }
        __syncwarp(lanes);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e) e16[e] = Ew<T>::from_f(y[e]);
      if (active) {
        T* p = is_q ? static_cast<T*>(a.query_out) + t * a.qo_stride + (long long)h * a.head_size
                    : static_cast<T*>(a.key_out) + t * a.ko_stride + (long long)(h - a.num_heads) * a.head_size;
        *reinterpret_cast<uint4*>(p + d0) = raw[u];
      }
    }
  }
}

template <class T, class TC, int G>
static void launch_qk_norm(const QkNormArgs& a, int mode, dim3 grid, cudaStream_t st) {
  if (mode == kPairs) qk_norm_rotary_kernel<T, TC, G, kPairs><<<grid, kQkThreads, 0, st>>>(a);
  else if (mode == kNeoxLanes) qk_norm_rotary_kernel<T, TC, G, kNeoxLanes><<<grid, kQkThreads, 0, st>>>(a);
  else qk_norm_rotary_kernel<T, TC, G, kNeoxAny><<<grid, kQkThreads, 0, st>>>(a);
}

template <class T, class TC>
static void launch_qk_norm(const QkNormArgs& a, int num_tokens, bool is_neox, int sms, cudaStream_t st) {
  int g = 1;
  while (g * 8 < a.head_size) g *= 2;
  const int groups = kQkThreads / g, total = a.num_heads + a.num_kv_heads;
  // Few tokens: a token's heads go to several CTAs, down to one head per group, until about four CTAs per SM run.
  const int most = (total + groups - 1) / groups;
  int y = (4 * sms + num_tokens - 1) / num_tokens;
  y = y < 1 ? 1 : y > most ? most : y;
  const dim3 grid(num_tokens, y);
  const int mode = !is_neox ? kPairs : a.rot_dim % 16 == 0 ? kNeoxLanes : kNeoxAny;
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
