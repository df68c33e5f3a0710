// Host side of paged attention: the choice of the kernel and the C entry point.
#pragma once

#include "attention_tc.cuh"

namespace trb {

// Which kernel takes a call, by the rows (token, query head of a group) of an average sequence: up to 16 the warps of a CTA split
// the tokens; more go to the tensor-memory kernel where its page and stride rules hold, and else to CTAs whose warps split the
// rows.  Tensor memory against split rows, bf16, heads 32 over 8 of size 128: 8 tokens of one sequence after 8000: 28.8 and 34.6
// us, 24 of each of 32 after 2000: 64 and 118, 700 after 800 next to 127 single ones after 1000: 150 and 228; 6 of each of 200
// after 900: 217 and 221, of size 64 e4m3 122 and 112, its worst.  Below 17 rows splitting the tokens wins (4 of each of 128 after
// 1000: 134 and 103).
// The host knows the average alone.  A chunk beside so many single or empty sequences that the average stays below 17 rows walks
// its keys 16 rows at a time: in a graph, against the chunk and the rest as two calls, 512 of 1512 next to 63 single ones, 32 heads
// over 32, bf16: 228 us against 193; 700 of 1500 next to 240 single ones, 32 over 8: 276 against 197; 900 of 12000 next to 63
// single ones, 32 over 32: 1425 against 367, next to 63 empty ones 1204 against 200.  Two calls are the better way there.
enum AttnKind { kAttnSplit, kAttnRows, kAttnTensor };
static AttnKind attn_kind(long long tokens, int seqs, int group, bool single, bool tensor_fits) {
  const long long rows = single ? (long long)group * seqs : tokens * group;
  if (rows <= 16LL * seqs) return kAttnSplit;
  return !single && tensor_fits ? kAttnTensor : kAttnRows;
}

// The stride of a dimension of one entry says nothing.
static void attn_settle_strides(long long num_pages, int page_size, int kv_heads, int head_size, long long& page, long long& token,
                                long long& head) {
  if (kv_heads == 1) head = head_size;
  if (page_size == 1) token = head_size;
  if (num_pages == 1) page = head_size;
}

// Calls f with the configuration of the kernel for short calls.
template <class T, class F>
static auto attn_with_cfg(bool fp8, int head_size, bool rows, F f) {
  if (head_size == 128) {
    if (fp8) return rows ? f(AttnCfg<T, true, 128, true>()) : f(AttnCfg<T, true, 128, false>());
    return rows ? f(AttnCfg<T, false, 128, true>()) : f(AttnCfg<T, false, 128, false>());
  }
  if (fp8) return rows ? f(AttnCfg<T, true, 64, true>()) : f(AttnCfg<T, true, 64, false>());
  return rows ? f(AttnCfg<T, false, 64, true>()) : f(AttnCfg<T, false, 64, false>());
}

template <class T>
static int launch_attn(const AttnArgs& a, int head_size, void* workspace, size_t workspace_bytes, int dev, cudaStream_t st) {
  const bool fp8 = a.key_exp != nullptr;
  if (a.seqs == 0) {
    const unsigned ctas = a.tokens < 4096 ? a.tokens : 4096;
    if (head_size == 128) attn_clear_kernel<T, 128><<<ctas, 128, 0, st>>>(a);
    else attn_clear_kernel<T, 64><<<ctas, 128, 0, st>>>(a);
    return cudaGetLastError() == cudaSuccess ? TRB_OK : TRB_ERR_CUDA;
  }
  const bool single = a.query_starts == nullptr;
  const AttnKind kind =
      attn_kind(a.tokens, a.seqs, a.group, single, attn_tc_fits(single, a.page_size, a.num_pages, a.c_page, a.c_tok, a.c_head));
  if (kind == kAttnTensor) {
    if (head_size == 128) return fp8 ? launch_attn_tc<T, 128, true>(a, dev, st) : launch_attn_tc<T, 128, false>(a, dev, st);
    return fp8 ? launch_attn_tc<T, 64, true>(a, dev, st) : launch_attn_tc<T, 64, false>(a, dev, st);
  }
  return attn_with_cfg<T>(fp8, head_size, kind == kAttnRows,
                          [&](auto cfg) { return launch_attn<T, decltype(cfg)>(a, workspace, workspace_bytes, dev, st); });
}

}  // namespace trb

extern "C" size_t trb_paged_attention_workspace_bytes(int num_tokens, int num_seqs, int num_heads, int num_kv_heads, int head_size,
                                                      int page_size, int table_width, int single, int e4m3, int dev) {
  using namespace trb;
  if (num_tokens <= 0 || num_seqs <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 || page_size <= 0 || table_width < 0)
    return 0;
  const int group = num_heads / num_kv_heads;
  // The tensor-memory kernel needs none: the other bound says which calls it takes.
  const bool rows = attn_kind(num_tokens, num_seqs, group, single != 0, false) == kAttnRows;
  return attn_with_cfg<__half>(e4m3 != 0, head_size, rows, [&](auto cfg) -> size_t {
    using Cfg = decltype(cfg);
    const int ctas = attn_cut<Cfg>(num_tokens, num_seqs, group, num_kv_heads, single != 0, (long long)table_width * page_size, sm_count(dev)).ctas;
    return 2ull * ctas * Cfg::PIECE_FLOATS * 4;
  });
}

extern "C" size_t trb_paged_attention_cache_workspace_bytes(int num_tokens, int num_seqs, int num_heads, int num_kv_heads, int head_size,
                                                            int page_size, long long num_pages, int table_width, long long page_stride,
                                                            long long token_stride, long long head_stride, int single, int e4m3, int dev) {
  using namespace trb;
  if (num_tokens <= 0 || num_seqs <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads != 0 || page_size <= 0) return 0;
  attn_settle_strides(num_pages, page_size, num_kv_heads, head_size, page_stride, token_stride, head_stride);
  const bool fits = attn_tc_fits(single != 0, page_size, num_pages, page_stride, token_stride, head_stride);
  if (attn_kind(num_tokens, num_seqs, num_heads / num_kv_heads, single != 0, fits) == kAttnTensor) return 0;
  return trb_paged_attention_workspace_bytes(num_tokens, num_seqs, num_heads, num_kv_heads, head_size, page_size, table_width, single, e4m3, dev);
}

extern "C" int trb_paged_attention_clear(const void* query, const void* key_cache, const void* value_cache,
                                         const void* key_exponents, const void* value_exponents, const void* page_table,
                                         const void* lengths, const void* query_starts, void* out, int num_tokens, int num_seqs,
                                         int num_heads, int num_kv_heads, int head_size, int page_size, long long num_pages,
                                         long long table_stride, int table_width, long long query_token_stride,
                                         long long query_head_stride, long long out_token_stride, long long out_head_stride,
                                         long long page_stride, long long token_stride, long long head_stride,
                                         long long exp_page_stride, long long exp_token_stride, long long exp_head_stride,
                                         float scale, int causal, int window, int dtype, void* workspace, size_t workspace_bytes,
                                         int dev, void* stream, int clear) {
  using namespace trb;
  if (num_tokens == 0 || (num_seqs == 0 && !clear)) return TRB_OK;
  const bool fp8 = key_exponents != nullptr;
  if (num_tokens < 0 || num_seqs < 0 || !query || !key_cache || !value_cache || (!lengths && num_seqs > 0) || !out || fp8 != (value_exponents != nullptr) ||
      num_heads <= 0 || num_kv_heads <= 0 || page_size <= 0 || num_pages < 0 || table_width < 0 || (!page_table && table_width > 0 && num_seqs > 0) || window < 0)
    return TRB_ERR_BAD_ARG;
  if (!query_starts && (num_tokens != num_seqs || clear)) return TRB_ERR_BAD_ARG;
  attn_settle_strides(num_pages, page_size, num_kv_heads, head_size, page_stride, token_stride, head_stride);
  if (num_tokens == 1) query_token_stride = out_token_stride = 0;
  if (num_heads == 1) query_head_stride = out_head_stride = 0;
  if (num_heads % num_kv_heads != 0 || (window > 0 && !causal)) return TRB_ERR_PROB_SHAPE;
  const int esz = fp8 ? 1 : 2;
  if (((uintptr_t)query | (uintptr_t)out | (uintptr_t)key_cache | (uintptr_t)value_cache | (uintptr_t)workspace) & 15) return TRB_ERR_PROB_SHAPE;
  if ((query_token_stride | query_head_stride | out_token_stride | out_head_stride) & 7) return TRB_ERR_PROB_SHAPE;
  if (((page_stride | token_stride | head_stride) * esz) & 15) return TRB_ERR_PROB_SHAPE;
  // Positions are 32-bit numbers; the largest unit starts below length + 64.
  const long long most = (long long)table_width * page_size;
  if (most > 0x7fff0000LL || (long long)num_tokens * (num_heads / num_kv_heads) > 0x7fff0000LL) return TRB_ERR_PROB_SHAPE;
  const float scale_log2 = scale * 1.4426950408889634f;
  if (!(fabsf(scale_log2) <= 3.402823466e38f)) return TRB_ERR_BAD_ARG;
  // A window as wide as the table hides nothing.  A narrower one is subtracted from positions down to -num_tokens (more new tokens
  // than the cache has).
  if (window >= most) window = 0;
  if (window > 0 && most + num_tokens > 0x7fff0000LL) return TRB_ERR_PROB_SHAPE;
  if (dtype != TRB_F16 && dtype != TRB_BF16) return TRB_ERR_KERN_SHAPE;
  if (head_size != 64 && head_size != 128) return TRB_ERR_KERN_SHAPE;
  DeviceGuard guard(dev);
  if (!guard.ok) return TRB_ERR_CUDA;
  const AttnArgs a{query, key_cache, value_cache, (const uint8_t*)key_exponents, (const uint8_t*)value_exponents,
                   (const int*)page_table, (const int*)lengths, (const int*)query_starts, out, query_token_stride, query_head_stride,
                   out_token_stride, out_head_stride, page_stride, token_stride, head_stride, exp_page_stride, exp_token_stride,
                   exp_head_stride, table_stride, num_pages, scale_log2, num_tokens, num_seqs, num_kv_heads,
                   num_heads / num_kv_heads, page_size, table_width,
                   (page_size & (page_size - 1)) == 0 ? __builtin_ctz((unsigned)page_size) : -1, causal, window, clear != 0};
  if (dtype == TRB_F16) return launch_attn<__half>(a, head_size, workspace, workspace_bytes, dev, (cudaStream_t)stream);
  return launch_attn<__nv_bfloat16>(a, head_size, workspace, workspace_bytes, dev, (cudaStream_t)stream);
}

extern "C" int trb_paged_attention(const void* query, const void* key_cache, const void* value_cache, const void* key_exponents,
                                   const void* value_exponents, const void* page_table, const void* lengths,
                                   const void* query_starts, void* out, int num_tokens, int num_seqs, int num_heads,
                                   int num_kv_heads, int head_size, int page_size, long long num_pages, long long table_stride,
                                   int table_width, long long query_token_stride, long long query_head_stride,
                                   long long out_token_stride, long long out_head_stride, long long page_stride,
                                   long long token_stride, long long head_stride, long long exp_page_stride,
                                   long long exp_token_stride, long long exp_head_stride, float scale, int causal, int window,
                                   int dtype, void* workspace, size_t workspace_bytes, int dev, void* stream) {
  return trb_paged_attention_clear(query, key_cache, value_cache, key_exponents, value_exponents, page_table, lengths, query_starts,
                                   out, num_tokens, num_seqs, num_heads, num_kv_heads, head_size, page_size, num_pages,
                                   table_stride, table_width, query_token_stride, query_head_stride, out_token_stride,
                                   out_head_stride, page_stride, token_stride, head_stride, exp_page_stride, exp_token_stride,
                                   exp_head_stride, scale, causal, window, dtype, workspace, workspace_bytes, dev, stream, 0);
}
