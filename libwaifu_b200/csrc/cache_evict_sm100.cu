// Eviction from a key-value cache by accumulated attention weight: which keys stay, and their rows gathered.
//
// One CTA per sequence and key-value head finds the weight of the last key that stays by its bits, eight at a time
// from the top (a histogram of the keys that agree so far, then the bin in which the wanted rank falls), and
// lists the keys above it and the first of those equal to it in the order of their positions (a scan over the CTA).
// The rows are then copied by a kernel over the whole GPU, sixteen bytes a thread. Both are bound by memory: a weight is
// read once and a kept row once, and written once.
#include "cache_attention_sm100.cuh"

#include "cache_common_sm100.cuh"
#include "ptx_sm100.cuh"

namespace flsm100 {

namespace {

constexpr int kSelectThreads = 1024;

// An unsigned number that orders like the weight: NaN below everything, -0 equal to 0.
__device__ __forceinline__ uint32_t order_of(float w) {
  const uint32_t bits = __float_as_uint(w);
  if ((bits & 0x7FFFFFFFu) > 0x7F800000u) return 0u;
  if (bits == 0x80000000u) return 0x80000000u;
  return (bits & 0x80000000u) ? ~bits : (bits | 0x80000000u);
}

struct SelectParams {
  const float *weights;
  int64_t weights_stride[2];
  float *weights_out;
  int64_t weights_out_stride[2];
  const int32_t *kv_lens;
  int32_t *kept;
  int kv_heads, kv_len, out_len, keep, recent;
};

// The exclusive sum of `mine` over the CTA's threads in order, and the total.
__device__ __forceinline__ int scan_cta(int mine, int *warp_sums, int *total) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  int sum = mine;
#pragma unroll
  for (int x = 1; x < 32; x <<= 1) {
    const int y = __shfl_up_sync(0xffffffffu, sum, x);
    if (lane >= x) sum += y;
  }
  __syncthreads();  // (an earlier scan's sums have been read)
  if (lane == 31) warp_sums[warp] = sum;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int w = 0; w < kSelectThreads / 32; ++w) {
    if (w < warp) before += warp_sums[w];
    all += warp_sums[w];
  }
  *total = all;
  return before + sum - mine;
}

__global__ void __launch_bounds__(kSelectThreads) select_kept_kernel(const SelectParams p) {
  __shared__ uint32_t bins[256];
  __shared__ int warp_sums[kSelectThreads / 32];
  __shared__ uint32_t found_bin;
  __shared__ int found_rank;
  const int run = blockIdx.x, seq = run / p.kv_heads, head = run % p.kv_heads;
  const int len = sequence_length(p.kv_lens, seq, p.kv_len);
  const float *weights = p.weights + seq * p.weights_stride[0] + head * p.weights_stride[1];
  float *weights_out = p.weights_out + seq * p.weights_out_stride[0] + head * p.weights_out_stride[1];
  int32_t *kept = p.kept + static_cast<int64_t>(run) * p.keep;
  griddep_launch_dependents();

  const int old = len <= p.keep ? 0 : len - p.recent;  // the keys that have to earn their place
  int wanted = p.keep - p.recent;                       // how many of them stay
  uint32_t prefix = 0, mask = 0;
  if (old > 0 && wanted > 0) {
    for (int shift = 24; shift >= 0; shift -= 8) {
      for (int i = threadIdx.x; i < 256; i += kSelectThreads) bins[i] = 0;
      __syncthreads();
      for (int i = threadIdx.x; i < old; i += kSelectThreads) {
        const uint32_t o = order_of(weights[i]);
        if ((o & mask) == prefix) atomicAdd(&bins[(o >> shift) & 255], 1u);
      }
      __syncthreads();
      if (threadIdx.x == 0) {
        int rank = wanted;
        int b = 255;
        for (; b > 0; --b) {
          const int here = static_cast<int>(bins[b]);
          if (rank <= here) break;
          rank -= here;
        }
        found_bin = static_cast<uint32_t>(b);
        found_rank = rank;
      }
      __syncthreads();
      prefix |= found_bin << shift;
      mask |= 255u << shift;
      wanted = found_rank;
    }
  }
  // Of the old keys those above `prefix` stay, and the first `wanted` that equal it.
  const bool choose = old > 0 && p.keep > p.recent;
  int placed = 0, equal_before = 0;
  for (int base = 0; base < len; base += kSelectThreads) {
    const int i = base + threadIdx.x;
    const float w = i < len ? weights[i] : 0.0f;
    const uint32_t o = order_of(w);
    const bool is_old = i < old;
    const bool equal = choose && is_old && o == prefix;
    int total = 0;
    const int equal_here = equal_before + scan_cta(equal ? 1 : 0, warp_sums, &total);
    equal_before += total;
    const bool stays = i < len && (!is_old || (choose && (o > prefix || (equal && equal_here < wanted))));
    const int to = placed + scan_cta(stays ? 1 : 0, warp_sums, &total);
    placed += total;
    if (stays) {
      kept[to] = i;
      weights_out[to] = w;
    }
  }
  for (int i = placed + threadIdx.x; i < p.out_len; i += kSelectThreads) {
    if (i < p.keep) kept[i] = -1;
    weights_out[i] = 0.0f;
  }
}

struct GatherParams {
  const uint8_t *k, *v;
  uint8_t *k_out, *v_out;
  int64_t k_stride[3], v_stride[3], k_out_stride[3], v_out_stride[3];
  const int32_t *kept, *kv_lens;
  int32_t *lens_out;
  int kv_heads, kv_len, keep, pieces;  // 16-byte pieces of a row
  int64_t total;                       // batch * kv_heads * keep * pieces
};

__global__ void __launch_bounds__(256) gather_kept_kernel(const GatherParams p) {
  griddep_wait();
  const int64_t step = static_cast<int64_t>(gridDim.x) * 256;
  for (int64_t at = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x; at < p.total; at += step) {
    const int piece = static_cast<int>(at % p.pieces);
    const int64_t slot = at / p.pieces;
    const int to = static_cast<int>(slot % p.keep);
    const int run = static_cast<int>(slot / p.keep), seq = run / p.kv_heads, head = run % p.kv_heads;
    const int from = p.kept[slot];
    if (head == 0 && to == 0 && piece == 0 && p.lens_out != nullptr) p.lens_out[seq] = min(sequence_length(p.kv_lens, seq, p.kv_len), p.keep);
    if (from < 0) continue;
    const uint4 x = *reinterpret_cast<const uint4 *>(p.k + seq * p.k_stride[0] + head * p.k_stride[1] + from * p.k_stride[2] + piece * 16);
    const uint4 y = *reinterpret_cast<const uint4 *>(p.v + seq * p.v_stride[0] + head * p.v_stride[1] + from * p.v_stride[2] + piece * 16);
    *reinterpret_cast<uint4 *>(p.k_out + seq * p.k_out_stride[0] + head * p.k_out_stride[1] + to * p.k_out_stride[2] + piece * 16) = x;
    *reinterpret_cast<uint4 *>(p.v_out + seq * p.v_out_stride[0] + head * p.v_out_stride[1] + to * p.v_out_stride[2] + piece * 16) = y;
  }
}

}  // namespace

cudaError_t cache_evict(const CacheEvictArgs &a) {
  SelectParams s = {};
  s.weights = a.weights;
  s.weights_out = a.weights_out;
  for (int i = 0; i < 2; ++i) {
    s.weights_stride[i] = a.weights_stride[i];
    s.weights_out_stride[i] = a.weights_out_stride[i];
  }
  s.kv_lens = a.kv_lens;
  s.kept = a.kept;
  s.kv_heads = a.kv_heads;
  s.kv_len = a.kv_len;
  s.out_len = a.out_len;
  s.keep = a.keep;
  s.recent = a.recent;
  select_kept_kernel<<<static_cast<unsigned>(a.batch * a.kv_heads), kSelectThreads, 0, a.stream>>>(s);
  cudaError_t e = cudaGetLastError();
  if (e != cudaSuccess) return e;

  GatherParams g = {};
  g.k = static_cast<const uint8_t *>(a.k);
  g.v = static_cast<const uint8_t *>(a.v);
  g.k_out = static_cast<uint8_t *>(a.k_out);
  g.v_out = static_cast<uint8_t *>(a.v_out);
  for (int i = 0; i < 3; ++i) {
    g.k_stride[i] = a.k_stride[i];
    g.v_stride[i] = a.v_stride[i];
    g.k_out_stride[i] = a.k_out_stride[i];
    g.v_out_stride[i] = a.v_out_stride[i];
  }
  g.kept = a.kept;
  g.kv_lens = a.kv_lens;
  g.lens_out = a.lens_out;
  g.kv_heads = a.kv_heads;
  g.kv_len = a.kv_len;
  g.keep = a.keep;
  g.pieces = a.row_bytes / 16;
  g.total = static_cast<int64_t>(a.batch) * a.kv_heads * a.keep * g.pieces;
  cudaLaunchConfig_t cfg = {};
  const int64_t ctas = (g.total + 255) / 256, most = static_cast<int64_t>(sm_count()) * 32;
  cfg.gridDim = dim3(static_cast<unsigned>(ctas < most ? ctas : most), 1, 1);
  cfg.blockDim = dim3(256, 1, 1);
  cfg.stream = a.stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, gather_kept_kernel, g);
}

}  // namespace flsm100
