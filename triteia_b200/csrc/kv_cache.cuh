// Keys and values into a paged cache and back.  The reference has no cache; its attention files take one that the
// serving engine owns (triteia/triton/decode_attention.py:30-120), a slot per token.
//   slot = page * page_size + place; cache[page, place, head, :] with any page, token and head strides.
// A cache holds values of the inputs' type, or e4m3 with one power of two per token and head:
//   e = smallest integer with max |x| <= 448 * 2^e over the finite values (0 if there is none, at least -126),
//   code = e4m3(x * 2^-e), the product exact and the rounding to nearest even, exponent byte e + 127.
// A power of two costs no accuracy against max / 448 (e4m3 keeps 4 bits at every magnitude down to 2^-15 of the
// largest), takes a byte instead of four and makes reading back exact: code * 2^e is a number of the inputs' type
// (fp16: but for subnormals).  Infinities and NaN are stored as NaN.
//
// Bytes bound both kernels.  A group of G lanes moves one head, 16 bytes of inputs a lane; the maximum of a head is
// log2(G) shuffles, so a token is read once.  A CTA works on one token at a time: its slot is split into page and place
// once per token, not per head.
#pragma once

#include <cuda_fp8.h>

#include "qk_norm.cuh"

namespace trb {

struct KvArgs {
  const void *key, *value;            // write: [T, heads, head_size] with token and head strides
  void *key_out, *value_out;          // read: contiguous [T, heads, head_size]
  void *key_cache, *value_cache;
  uint8_t *key_exp, *value_exp;       // null: the cache holds the inputs' type
  const int64_t* slots;
  long long num_slots;
  long long k_tok, k_head, v_tok, v_head;
  long long c_page, c_tok, c_head, e_page, e_tok, e_head;
  int tokens, heads, head_size, page_size;
};

constexpr int kKvThreads = 128;

// Largest finite magnitude of a group's values -> e + 127.
__device__ __forceinline__ int kv_exponent_byte(float top) {
  if (top == 0.f) return 127;
  // Subnormal 32-bit numbers lie far below 448 * 2^-126: their exponent field of 0 ends at the bound like any small one.
  const uint32_t bits = __float_as_uint(top);
  // top = m * 2^(field - 126), m in [0.5, 1), and 448 = 0.875 * 2^9: one more where m is above 0.875.
  const int byte = (int)(bits >> 23) - 126 - 9 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0) + 127;
  return byte < 1 ? 1 : byte;
}

template <class T, bool FP8>
__device__ __forceinline__ void kv_store(uint4 raw, unsigned lanes, int g, bool active, bool first, void* cache, long long at,
                                         uint8_t* exps, long long exp_at) {
  if constexpr (!FP8) {
    if (active) *reinterpret_cast<uint4*>(static_cast<T*>(cache) + at) = raw;
  } else {
    const T* e16 = reinterpret_cast<const T*>(&raw);
    float x[8], top = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = Ew<T>::to_f(e16[e]);
      const float m = fabsf(x[e]);
      if (m <= 3.402823466e38f) top = fmaxf(top, m);
      else x[e] = __uint_as_float(0x7fffffffu);
    }
    for (int o = g / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(lanes, top, o));
    const int byte = kv_exponent_byte(top);
    const float inv = __uint_as_float((uint32_t)(254 - byte) << 23);      // 2^-(byte - 127): byte is 1 .. 247
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float2 p = make_float2(x[e] * inv, x[e + 1] * inv);
      w[e >> 2] |= (uint32_t)__nv_cvt_float2_to_fp8x2(p, __NV_SATFINITE, __NV_E4M3) << (8 * (e & 3));
    }
    if (active) *reinterpret_cast<uint2*>(static_cast<uint8_t*>(cache) + at) = make_uint2(w[0], w[1]);
    if (first) exps[exp_at] = (uint8_t)byte;
  }
}

template <class T, bool FP8>
__global__ void __launch_bounds__(kKvThreads) cache_write_kernel(const KvArgs a, int g) {
  const int li = threadIdx.x % g, grp = threadIdx.x / g, groups = kKvThreads / g;
  const bool active = li * 8 < a.head_size;
  const unsigned lanes = g == 32 ? 0xffffffffu : ((1u << g) - 1u) << ((threadIdx.x & 31) / g * g);
  for (long long t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    const int64_t slot = a.slots[t];
    if (slot < 0 || slot >= a.num_slots) continue;      // a padding token
    const long long page = slot / a.page_size, place = slot - page * a.page_size;
    const long long at = page * a.c_page + place * a.c_tok + li * 8, exp_at = page * a.e_page + place * a.e_tok;
    const T* kp = static_cast<const T*>(a.key) + t * a.k_tok + li * 8;
    const T* vp = static_cast<const T*>(a.value) + t * a.v_tok + li * 8;
    for (int h = blockIdx.y * groups + grp; h < a.heads; h += gridDim.y * groups) {
      uint4 k = make_uint4(0, 0, 0, 0), v = k;
      if (active) {
        k = *reinterpret_cast<const uint4*>(kp + h * a.k_head);
        v = *reinterpret_cast<const uint4*>(vp + h * a.v_head);
      }
      kv_store<T, FP8>(k, lanes, g, active, li == 0, a.key_cache, at + h * a.c_head, a.key_exp, exp_at + h * a.e_head);
      kv_store<T, FP8>(v, lanes, g, active, li == 0, a.value_cache, at + h * a.c_head, a.value_exp, exp_at + h * a.e_head);
    }
  }
}

// 8 e4m3 codes times 2^(byte - 127), rounded once to T.
template <class T>
__device__ __forceinline__ uint4 kv_decode(uint2 w, int byte) {
  const uint32_t b = (uint32_t)byte;
  const float p = __uint_as_float(b == 0 ? 0x00400000u : b << 23);        // byte 0 stands for 2^-127
  uint4 out;
  T* o = reinterpret_cast<T*>(&out);
#pragma unroll
  for (int e = 0; e < 8; e += 2) {
    const uint32_t word = e < 4 ? w.x : w.y;
    const __half2_raw h = __nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(word >> (8 * (e & 3))), __NV_E4M3);
    const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h));
    o[e] = Ew<T>::from_f(f.x * p);
    o[e + 1] = Ew<T>::from_f(f.y * p);
  }
  return out;
}

template <class T, bool FP8>
__global__ void __launch_bounds__(kKvThreads) cache_read_kernel(const KvArgs a, int g) {
  const int li = threadIdx.x % g, grp = threadIdx.x / g, groups = kKvThreads / g;
  if (li * 8 >= a.head_size) return;
  for (long long t = blockIdx.x; t < a.tokens; t += gridDim.x) {
    const int64_t slot = a.slots[t];
    const bool there = slot >= 0 && slot < a.num_slots;
    const long long page = there ? slot / a.page_size : 0, place = there ? slot - page * a.page_size : 0;
    const long long at = page * a.c_page + place * a.c_tok + li * 8, exp_at = page * a.e_page + place * a.e_tok;
    T* ko = static_cast<T*>(a.key_out) + t * a.heads * a.head_size + li * 8;
    T* vo = static_cast<T*>(a.value_out) + t * a.heads * a.head_size + li * 8;
    for (int h = blockIdx.y * groups + grp; h < a.heads; h += gridDim.y * groups) {
      uint4 k = make_uint4(0, 0, 0, 0), v = k;
      if (there) {
        if constexpr (FP8) {
          const uint2 kw = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.key_cache) + at + h * a.c_head);
          const uint2 vw = *reinterpret_cast<const uint2*>(static_cast<const uint8_t*>(a.value_cache) + at + h * a.c_head);
          const int kb = a.key_exp[exp_at + h * a.e_head], vb = a.value_exp[exp_at + h * a.e_head];
          k = kv_decode<T>(kw, kb);
          v = kv_decode<T>(vw, vb);
        } else {
          k = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.key_cache) + at + h * a.c_head);
          v = *reinterpret_cast<const uint4*>(static_cast<const T*>(a.value_cache) + at + h * a.c_head);
        }
      }
      *reinterpret_cast<uint4*>(ko + (long long)h * a.head_size) = k;
      *reinterpret_cast<uint4*>(vo + (long long)h * a.head_size) = v;
    }
  }
}

// Lanes of a group and the grid: a CTA per token; few tokens: a token's heads go to several CTAs.
static dim3 kv_grid(const KvArgs& a, int sms, int* g) {
  *g = 1;
  while (*g * 8 < a.head_size) *g *= 2;
  const int groups = kKvThreads / *g, most = (a.heads + groups - 1) / groups;
  int y = (4 * sms + a.tokens - 1) / a.tokens;
  y = y < 1 ? 1 : y > most ? most : y;
  return dim3(a.tokens, y);
}

static int kv_check(const KvArgs& a, long long num_pages, bool fp8) {
  if (a.tokens < 0 || a.heads <= 0 || num_pages < 0 || a.page_size <= 0) return TRB_ERR_BAD_ARG;
  if (a.head_size <= 0 || a.head_size % 8 != 0 || a.head_size > 256) return TRB_ERR_PROB_SHAPE;
  const uintptr_t cache_align = fp8 ? 7 : 15;
  if (((uintptr_t)a.key_cache | (uintptr_t)a.value_cache) & cache_align || ((a.c_page | a.c_tok | a.c_head) & 7)) return TRB_ERR_PROB_SHAPE;
  return TRB_OK;
}

}  // namespace trb

extern "C" int trb_cache_write(const void* key, const void* value, const void* slots, void* key_cache, void* value_cache,
                               void* key_exponents, void* value_exponents, int num_tokens, int heads, int head_size, int page_size,
                               long long num_pages, long long key_token_stride, long long key_head_stride,
                               long long value_token_stride, long long value_head_stride, long long page_stride,
                               long long token_stride, long long head_stride, long long exp_page_stride, long long exp_token_stride,
                               long long exp_head_stride, int dtype, int dev, void* stream) {
  using namespace trb;
  if (num_tokens == 0) return TRB_OK;
  const bool fp8 = key_exponents != nullptr;
  if (!key || !value || !slots || !key_cache || !value_cache || fp8 != (value_exponents != nullptr)) return TRB_ERR_BAD_ARG;
  const KvArgs a{key, value, nullptr, nullptr, key_cache, value_cache, (uint8_t*)key_exponents, (uint8_t*)value_exponents,
                 (const int64_t*)slots, num_pages * page_size, key_token_stride, key_head_stride, value_token_stride, value_head_stride,
                 page_stride, token_stride, head_stride, exp_page_stride, exp_token_stride, exp_head_stride, num_tokens, heads,
                 head_size, page_size};
  if (const int err = kv_check(a, num_pages, fp8)) return err;
  if (((uintptr_t)key | (uintptr_t)value) & 15 || ((key_token_stride | key_head_stride | value_token_stride | value_head_stride) & 7))
    return TRB_ERR_PROB_SHAPE;
  if (dtype != TRB_F16 && dtype != TRB_BF16) return TRB_ERR_KERN_SHAPE;
  DeviceGuard guard(dev);
  if (!guard.ok) return TRB_ERR_CUDA;
  int g;
  const dim3 grid = kv_grid(a, sm_count(dev), &g);
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == TRB_F16) {
    if (fp8) cache_write_kernel<__half, true><<<grid, kKvThreads, 0, st>>>(a, g);
    else cache_write_kernel<__half, false><<<grid, kKvThreads, 0, st>>>(a, g);
  } else {
    if (fp8) cache_write_kernel<__nv_bfloat16, true><<<grid, kKvThreads, 0, st>>>(a, g);
    else cache_write_kernel<__nv_bfloat16, false><<<grid, kKvThreads, 0, st>>>(a, g);
  }
  return cudaGetLastError() == cudaSuccess ? TRB_OK : TRB_ERR_CUDA;
}

extern "C" int trb_cache_read(const void* key_cache, const void* value_cache, const void* key_exponents, const void* value_exponents,
                              const void* slots, void* key_out, void* value_out, int num_tokens, int heads, int head_size,
                              int page_size, long long num_pages, long long page_stride, long long token_stride,
                              long long head_stride, long long exp_page_stride, long long exp_token_stride, long long exp_head_stride,
                              int dtype, int dev, void* stream) {
  using namespace trb;
  if (num_tokens == 0) return TRB_OK;
  const bool fp8 = key_exponents != nullptr;
  if (!key_out || !value_out || !slots || !key_cache || !value_cache || fp8 != (value_exponents != nullptr)) return TRB_ERR_BAD_ARG;
  const KvArgs a{nullptr, nullptr, key_out, value_out, const_cast<void*>(key_cache), const_cast<void*>(value_cache),
                 (uint8_t*)key_exponents, (uint8_t*)value_exponents, (const int64_t*)slots, num_pages * page_size, 0, 0, 0, 0,
                 page_stride, token_stride, head_stride, exp_page_stride, exp_token_stride, exp_head_stride, num_tokens, heads,
                 head_size, page_size};
  if (const int err = kv_check(a, num_pages, fp8)) return err;
  if (((uintptr_t)key_out | (uintptr_t)value_out) & 15) return TRB_ERR_PROB_SHAPE;
  if (dtype != TRB_F16 && dtype != TRB_BF16) return TRB_ERR_KERN_SHAPE;
  DeviceGuard guard(dev);
  if (!guard.ok) return TRB_ERR_CUDA;
  int g;
  const dim3 grid = kv_grid(a, sm_count(dev), &g);
  cudaStream_t st = (cudaStream_t)stream;
  if (dtype == TRB_F16) {
    if (fp8) cache_read_kernel<__half, true><<<grid, kKvThreads, 0, st>>>(a, g);
    else cache_read_kernel<__half, false><<<grid, kKvThreads, 0, st>>>(a, g);
  } else {
    if (fp8) cache_read_kernel<__nv_bfloat16, true><<<grid, kKvThreads, 0, st>>>(a, g);
    else cache_read_kernel<__nv_bfloat16, false><<<grid, kKvThreads, 0, st>>>(a, g);
  }
  return cudaGetLastError() == cudaSuccess ? TRB_OK : TRB_ERR_CUDA;
}
