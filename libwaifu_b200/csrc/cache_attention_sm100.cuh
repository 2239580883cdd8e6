// Attention over a decoder's key-value cache for sm_100a: a length per sequence, a sliding window with
// first keys that stay visible, a prefix that a batch shares, and the sum of each key's weights.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

namespace flsm100 {

// q (batch, heads, q_len, head_dim), k and v (batch, kv_heads, kv_len, head_dim), out like q; heads a
// multiple of kv_heads. Sequence n holds len = kv_lens[n] keys (kv_len where there is no kv_lens; what lies
// outside 0 .. kv_len is taken as the nearer of the two). Query i sits at position p = i + len - q_len and
// sees the keys j <= p with j > p - window or j < sinks; with a prefix, all of its prefix_len keys before.
struct CacheAttentionArgs {
  const void *q, *k, *v;
  void *out;
  int is_bf16;  // else half
  int batch, heads, kv_heads, q_len, kv_len, head_dim;
  int64_t q_stride[3], k_stride[3], v_stride[3], out_stride[3];  // batch, head, position, in elements
  const int32_t *kv_lens;  // (batch) or null
  int window, sinks;
  const void *prefix_k, *prefix_v;  // (kv_heads, prefix_len, head_dim), null without a prefix
  int64_t prefix_k_stride[2], prefix_v_stride[2];  // head, position
  int prefix_len;
  // The keys' weights, (batch, kv_heads, kv_len): weights_out = weights_in + this call's; null without.
  const float *weights_in;
  float *weights_out;
  int64_t weights_in_stride[2], weights_out_stride[2];
  uint8_t *workspace;   // cache_attention_workspace_bytes()
  uint32_t *counters;   // kCacheCounters words, zero between calls
  uint32_t *status;     // device word: a wait that gave up is recorded there
  cudaStream_t stream;
};

constexpr int kCacheCounters = 4096;

bool cache_attention_supported(const CacheAttentionArgs &a, const char **why);
size_t cache_attention_workspace_bytes(const CacheAttentionArgs &a);
// Counts the kernels it launched in *launches.
cudaError_t cache_attention(const CacheAttentionArgs &a, const char **why, int *launches);

// What stays of a cache: per sequence and key-value head the `recent` last keys and, of the others, the
// keep - recent of the largest weight (of equal ones the first; one that is not a number counts least), in
// the order of their positions; every key where there are no more than keep.
struct CacheEvictArgs {
  const void *k, *v;  // (batch, kv_heads, kv_len, row_bytes), rows of row_bytes
  void *k_out, *v_out;  // (batch, kv_heads, out_len >= keep, row_bytes)
  int batch, kv_heads, kv_len, out_len, row_bytes;
  int64_t k_stride[3], v_stride[3], k_out_stride[3], v_out_stride[3];  // in bytes
  const float *weights;  // (batch, kv_heads, kv_len), the last dimension contiguous
  float *weights_out;    // (batch, kv_heads, out_len): zeros past the new length
  int64_t weights_stride[2], weights_out_stride[2];
  const int32_t *kv_lens;  // (batch) or null
  int32_t *lens_out;       // (batch) or null; may be kv_lens
  int32_t *kept;           // (batch, kv_heads, keep): the kept keys' positions, -1 past the new length
  int keep, recent;
  cudaStream_t stream;
};
cudaError_t cache_evict(const CacheEvictArgs &a);

}  // namespace flsm100
