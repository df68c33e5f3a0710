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
// log2(G) shuffles, so a token is read once.  A CTA works on one token: its slot is split into page and place once, and each
// group has the loads of up to five heads' keys or values in flight before the first is worked on.  8192 tokens x 40 heads of
// 128, fp16 and e4m3, in a graph: write 51 us (4.9 TB/s; its rounding and packing share the issue slots with the loads), read 41
// us (6.1 TB/s).  Five is the number for 40 heads; with 8 key heads a group has two loads in flight behind that of the slot
// (1500 tokens written and 4000 read, bf16: 3 and 5.5 us, 4.1 and 5.9 TB/s, most of it in L2).
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

// Page of a slot; 32-bit division where it does.
__device__ __forceinline__ long long kv_page(const KvArgs& a, int64_t slot) {
  return a.num_slots <= 0xffffffffLL ? (long long)((uint32_t)slot / (uint32_t)a.page_size) : slot / a.page_size;
}

// Largest finite magnitude of a group's values -> e + 127.
__device__ __forceinline__ int kv_exponent_byte(float top) {
  if (top == 0.f) return 127;
  // Subnormal 32-bit numbers lie far below 448 * 2^-126: their exponent field of 0 ends at the bound like any small one.
  const uint32_t bits = __float_as_uint(top);
  // top = m * 2^(field - 126), m in [0.5, 1), and 448 = 0.875 * 2^9: one more where m is above 0.875.
  const int byte = (int)(bits >> 23) - 126 - 9 + ((bits & 0x7fffffu) > 0x600000u ? 1 : 0) + 127;
  return byte < 1 ? 1 : byte;
}

template <class T, bool FP8, int G>
__device__ __forceinline__ void kv_store(uint4 raw, unsigned lanes, bool active, bool first, void* cache, long long at, uint8_t* byte_out) {
  if constexpr (!FP8) {
    if (active) *reinterpret_cast<uint4*>(static_cast<T*>(cache) + at) = raw;
  } else {
    // Magnitudes compare like the integers that their bits are, two at a time.
    constexpr uint32_t kInf = std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    const uint32_t word[4] = {raw.x, raw.y, raw.z, raw.w};
    uint32_t most = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) most = __vmaxu2(most, word[e] & 0x7fff7fffu);
#pragma unroll
    for (int o = G / 2; o > 0; o >>= 1) most = __vmaxu2(most, __shfl_xor_sync(lanes, most, o));
    most = max(most & 0xffffu, most >> 16);
    float2 x[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = two_of(word[e], T());
    float top = two_of(most, T()).x;
    if (most >= kInf) {                                 // infinities or NaN in the head: the largest of the others
      top = 0.f;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float mx = fabsf(x[e].x), my = fabsf(x[e].y);
        if (mx <= 3.402823466e38f) top = fmaxf(top, mx);
        else x[e].x = __uint_as_float(0x7fffffffu);
        if (my <= 3.402823466e38f) top = fmaxf(top, my);
        else x[e].y = __uint_as_float(0x7fffffffu);
      }
#pragma unroll
      for (int o = G / 2; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(lanes, top, o));
    }
    const int byte = kv_exponent_byte(top);
    const float inv = __uint_as_float((uint32_t)(254 - byte) << 23);      // 2^-(byte - 127): byte is 1 .. 247
    uint32_t w[2] = {0, 0};
#pragma unroll
    for (int e = 0; e < 4; ++e)
      w[e >> 1] |= (uint32_t)__nv_cvt_float2_to_fp8x2(mul2(x[e], make_float2(inv, inv)), __NV_SATFINITE, __NV_E4M3) << (16 * (e & 1));
    if (active) *reinterpret_cast<uint2*>(static_cast<uint8_t*>(cache) + at) = make_uint2(w[0], w[1]);
    if (first) *byte_out = (uint8_t)byte;
  }
}

constexpr int kKvAhead = 5;           // heads' keys or values of a group, all loaded together

template <class T, bool FP8, int G>
__global__ void __launch_bounds__(kKvThreads) cache_write_kernel(const KvArgs a) {
  constexpr int GROUPS = kKvThreads / G;
  __shared__ uint8_t bytes[kKvAhead][GROUPS];
  const long long t = blockIdx.x;
  const int li = threadIdx.x % G, grp = threadIdx.x / G;
  const bool active = li * 8 < a.head_size;
  const unsigned lanes = G == 32 ? 0xffffffffu : ((1u << G) - 1u) << ((threadIdx.x & 31) / G * G);
  const T* kp = static_cast<const T*>(a.key) + t * a.k_tok + li * 8;
  const T* vp = static_cast<const T*>(a.value) + t * a.v_tok + li * 8;
  // Unit u: the keys of head u, or the values of head u - heads.
  const int step = gridDim.y * GROUPS, units = 2 * a.heads, u0 = blockIdx.y * GROUPS + grp;
  uint4 raw[kKvAhead];                                // the slot is not waited for
#pragma unroll
  for (int x = 0; x < kKvAhead; ++x) {
    const int u = u0 + x * step;
    raw[x] = make_uint4(0, 0, 0, 0);
    if (active && u < units) raw[x] = *reinterpret_cast<const uint4*>(u < a.heads ? kp + u * a.k_head : vp + (u - a.heads) * a.v_head);
  }
  const int64_t slot = a.slots[t];
  if (slot < 0 || slot >= a.num_slots) return;        // a padding token
  const long long page = kv_page(a, slot), place = slot - page * a.page_size;
  const long long at = page * a.c_page + place * a.c_tok + li * 8, exp_at = page * a.e_page + place * a.e_tok;
#pragma unroll
  for (int x = 0; x < kKvAhead; ++x) {
    const int u = u0 + x * step;
    if (u >= units) break;
    const bool is_k = u < a.heads;
    const int h = is_k ? u : u - a.heads;
    kv_store<T, FP8, G>(raw[x], lanes, active, li == 0, is_k ? a.key_cache : a.value_cache, at + h * a.c_head, &bytes[x][grp]);
  }
  if constexpr (FP8) {
    // Neighbouring heads' bytes leave together: one by one they were a seventh of the write transactions.
    __syncthreads();
    for (int i = threadIdx.x; i < kKvAhead * GROUPS; i += kKvThreads) {
      const int x = i / GROUPS, g = i % GROUPS, u = blockIdx.y * GROUPS + g + x * step;
      if (u >= units) continue;
      const bool is_k = u < a.heads;
      (is_k ? a.key_exp : a.value_exp)[exp_at + (is_k ? u : u - a.heads) * a.e_head] = bytes[x][g];
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

template <class T, bool FP8, int G>
__global__ void __launch_bounds__(kKvThreads) cache_read_kernel(const KvArgs a) {
  constexpr int GROUPS = kKvThreads / G;
  using Raw = typename std::conditional<FP8, uint2, uint4>::type;      // a lane's 8 codes or numbers
  constexpr int ESZ = FP8 ? 1 : 2;
  const long long t = blockIdx.x;
  const int li = threadIdx.x % G, grp = threadIdx.x / G;
  if (li * 8 >= a.head_size) return;
  const int64_t slot = a.slots[t];
  const bool there = slot >= 0 && slot < a.num_slots;
  const long long page = there ? kv_page(a, slot) : 0, place = there ? slot - page * a.page_size : 0;
  const long long at = page * a.c_page + place * a.c_tok + li * 8, exp_at = page * a.e_page + place * a.e_tok;
  const long long out_at = t * a.heads * a.head_size + li * 8;
  const int step = gridDim.y * GROUPS, units = 2 * a.heads, u0 = blockIdx.y * GROUPS + grp;      // as in cache_write_kernel
  Raw raw[kKvAhead];
  int byte[kKvAhead];
#pragma unroll
  for (int x = 0; x < kKvAhead; ++x) {
    const int u = u0 + x * step;
    raw[x] = Raw();
    byte[x] = 127;
    if (there && u < units) {
      const bool is_k = u < a.heads;
      const int h = is_k ? u : u - a.heads;
      raw[x] = *reinterpret_cast<const Raw*>(static_cast<const uint8_t*>(is_k ? a.key_cache : a.value_cache) + (at + h * a.c_head) * ESZ);
      if constexpr (FP8) byte[x] = (is_k ? a.key_exp : a.value_exp)[exp_at + h * a.e_head];
    }
  }
#pragma unroll
  for (int x = 0; x < kKvAhead; ++x) {
    const int u = u0 + x * step;
    if (u >= units) break;
    const bool is_k = u < a.heads;
    const int h = is_k ? u : u - a.heads;
    uint4 w;
    if constexpr (FP8) w = kv_decode<T>(raw[x], byte[x]);
    else w = raw[x];
    *reinterpret_cast<uint4*>(static_cast<T*>(is_k ? a.key_out : a.value_out) + out_at + (long long)h * a.head_size) = w;
  }
}

// A CTA has kKvAhead units of a token in a group; few tokens: fewer, until about four CTAs per SM run.
template <class T, bool FP8, int G>
static void launch_kv(const KvArgs& a, bool write, int sms, cudaStream_t st) {
  constexpr int GROUPS = kKvThreads / G;
  const int most = (2 * a.heads + GROUPS - 1) / GROUPS, least = (2 * a.heads + kKvAhead * GROUPS - 1) / (kKvAhead * GROUPS);
  int y = (4 * sms + a.tokens - 1) / a.tokens;
  y = y < least ? least : y > most ? most : y;
  const dim3 grid(a.tokens, y);
  if (write) cache_write_kernel<T, FP8, G><<<grid, kKvThreads, 0, st>>>(a);
  else cache_read_kernel<T, FP8, G><<<grid, kKvThreads, 0, st>>>(a);
}

template <class T, bool FP8>
static void launch_kv(const KvArgs& a, bool write, int sms, cudaStream_t st) {
  int g = 1;
  while (g * 8 < a.head_size) g *= 2;
  switch (g) {
    case 1: launch_kv<T, FP8, 1>(a, write, sms, st); break;
    case 2: launch_kv<T, FP8, 2>(a, write, sms, st); break;
    case 4: launch_kv<T, FP8, 4>(a, write, sms, st); break;
    case 8: launch_kv<T, FP8, 8>(a, write, sms, st); break;
    case 16: launch_kv<T, FP8, 16>(a, write, sms, st); break;
    default: launch_kv<T, FP8, 32>(a, write, sms, st); break;
  }
}

static int launch_kv(const KvArgs& a, bool fp8, bool write, int dtype, int dev, cudaStream_t st) {
  DeviceGuard guard(dev);
  if (!guard.ok) return TRB_ERR_CUDA;
  const int sms = sm_count(dev);
  if (dtype == TRB_F16) {
    if (fp8) launch_kv<__half, true>(a, write, sms, st);
    else launch_kv<__half, false>(a, write, sms, st);
  } else {
    if (fp8) launch_kv<__nv_bfloat16, true>(a, write, sms, st);
    else launch_kv<__nv_bfloat16, false>(a, write, sms, st);
  }
  return cudaGetLastError() == cudaSuccess ? TRB_OK : TRB_ERR_CUDA;
}

static int kv_check(KvArgs& a, long long num_pages, bool fp8) {
  // The stride of a dimension of one entry says nothing.
  if (a.heads == 1) a.c_head = a.k_head = a.v_head = 0;
  if (a.page_size == 1) a.c_tok = 0;
  if (num_pages == 1) a.c_page = 0;
  if (a.tokens == 1) a.k_tok = a.v_tok = 0;
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
  KvArgs a{key, value, nullptr, nullptr, key_cache, value_cache, (uint8_t*)key_exponents, (uint8_t*)value_exponents,
                 (const int64_t*)slots, num_pages * page_size, key_token_stride, key_head_stride, value_token_stride, value_head_stride,
                 page_stride, token_stride, head_stride, exp_page_stride, exp_token_stride, exp_head_stride, num_tokens, heads,
                 head_size, page_size};
  if (const int err = kv_check(a, num_pages, fp8)) return err;
  if (((uintptr_t)key | (uintptr_t)value) & 15 || ((a.k_tok | a.k_head | a.v_tok | a.v_head) & 7)) return TRB_ERR_PROB_SHAPE;
  if (dtype != TRB_F16 && dtype != TRB_BF16) return TRB_ERR_KERN_SHAPE;
  return launch_kv(a, fp8, true, dtype, dev, (cudaStream_t)stream);
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
  KvArgs a{nullptr, nullptr, key_out, value_out, const_cast<void*>(key_cache), const_cast<void*>(value_cache),
                 (uint8_t*)key_exponents, (uint8_t*)value_exponents, (const int64_t*)slots, num_pages * page_size, 0, 0, 0, 0,
                 page_stride, token_stride, head_stride, exp_page_stride, exp_token_stride, exp_head_stride, num_tokens, heads,
                 head_size, page_size};
  if (const int err = kv_check(a, num_pages, fp8)) return err;
  if (((uintptr_t)key_out | (uintptr_t)value_out) & 15) return TRB_ERR_PROB_SHAPE;
  if (dtype != TRB_F16 && dtype != TRB_BF16) return TRB_ERR_KERN_SHAPE;
  return launch_kv(a, fp8, false, dtype, dev, (cudaStream_t)stream);
}
