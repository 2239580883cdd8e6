// Eviction from a key-value cache by accumulated attention weight: which keys stay, and their rows gathered.
//
// One CTA per sequence and key-value head finds the weight of the last key that stays by its bits, and lists the keys above it
// and the first of those equal to it in the order of their positions (a scan over the CTA). A pass counts the keys in
// 2048 bins that divide the range in question in equal parts, at first that from the lightest key to the heaviest, and goes on
// with the bin in which the wanted rank falls, until that bin is one number or all of its keys stay: three passes at most. The
// weights are read once, into shared memory as far as they fit. What bounds a CTA is its instructions, so the
// passes are short: a key's bin, and one atomic without a result, which the hardware adds up for
// the lanes that share a bin (16 x 8 heads of 8192 keys and their rows 85.8 us, all weights equal 83.0; with bins at fixed bits,
// lanes grouped by votes and the keys of the bin found listed for the next pass 89.1; bit by bit over keys in registers, a
// barrier a bit, 94.4).
// The rows are then copied by a kernel over the whole GPU, sixteen bytes a thread. Both are bound by memory: a weight is
// read once and a kept row once, and written once.
#include "cache_attention_sm100.cuh"

#include <algorithm>

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
  int cached_keys;  // room for so many in shared memory
};

constexpr int kKeysPerThread = 4;  // of the scan
constexpr int kMaxCachedKeys = 48 * 1024;  // in shared memory
constexpr int kBins = 2048;

__global__ void __launch_bounds__(kSelectThreads, 1) select_kept_kernel(const __grid_constant__ SelectParams p) {
  extern __shared__ __align__(16) uint32_t cache[];
  __shared__ uint32_t bins[kBins];
  __shared__ uint32_t warp_counts[kSelectThreads / 32];
  __shared__ uint32_t warp_low[kSelectThreads / 32], warp_high[kSelectThreads / 32];
  __shared__ uint32_t found_bin;
  __shared__ int found_rank, found_keys;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  griddep_wait();
  griddep_launch_dependents();
  const int run = blockIdx.x, seq = run / p.kv_heads, head = run % p.kv_heads;
  const int len = sequence_length(p.kv_lens, seq, p.kv_len);
  const float *weights = p.weights + seq * p.weights_stride[0] + head * p.weights_stride[1];
  float *weights_out = p.weights_out + seq * p.weights_out_stride[0] + head * p.weights_out_stride[1];
  int32_t *kept = p.kept + static_cast<int64_t>(run) * p.keep;

  const int old = len <= p.keep ? 0 : len - p.recent;  // the keys that have to earn their place
  const bool choose = old > 0 && p.keep > p.recent;
  int wanted = p.keep - p.recent;  // how many of them stay
  uint32_t last = 0;               // the order of the lightest that does
  const int cached = choose ? min(old, p.cached_keys) : 0;
  auto order_at = [&](int i) -> uint32_t { return i < cached ? cache[i] : order_of(weights[i]); };
  if (choose) {
    uint32_t low = 0xffffffffu, high = 0u;
#pragma unroll 4
    for (int i = threadIdx.x; i < old; i += kSelectThreads) {
      const uint32_t o = order_of(weights[i]);
      if (i < cached) cache[i] = o;
      low = min(low, o);
      high = max(high, o);
    }
    low = __reduce_min_sync(0xffffffffu, low);
    high = __reduce_max_sync(0xffffffffu, high);
    if (lane == 0) warp_low[warp] = low, warp_high[warp] = high;
    __syncthreads();
    low = __reduce_min_sync(0xffffffffu, warp_low[lane]);
    high = __reduce_max_sync(0xffffffffu, warp_high[lane]);
    // The bins of a pass divide [low, low + (width << shift)), which holds the wanted key, in equal parts: at first from the
    // lightest key to the heaviest.
    int shift = max(0, 21 - __clz(static_cast<int>(high - low)));
    uint32_t width = kBins;
#pragma unroll 1
    while (true) {
      for (int i = threadIdx.x; i < kBins; i += kSelectThreads) bins[i] = 0;
      __syncthreads();
#pragma unroll 4
      for (int i = threadIdx.x; i < old; i += kSelectThreads) {
        const uint32_t bin = (order_at(i) - low) >> shift;  // (of a key below `low`, which the first pass has not, beyond the bins)
        if (bin < width) atomicAdd(&bins[bin], 1u);
      }
      __syncthreads();
      // Two bins a thread, the highest first: the bin in which the rank falls, and what is left of the rank there.
      const int top = kBins - 1 - 2 * static_cast<int>(threadIdx.x);
      const int here[2] = {static_cast<int>(bins[top]), static_cast<int>(bins[top - 1])};
      int upto = here[0] + here[1];
#pragma unroll
      for (int x = 1; x < 32; x <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, upto, x);
        if (lane >= x) upto += y;
      }
      if (lane == 31) warp_counts[warp] = static_cast<uint32_t>(upto);
      __syncthreads();
      const int before = __reduce_add_sync(0xffffffffu, lane < warp ? static_cast<int>(warp_counts[lane]) : 0);
      const int rank = wanted - (before + upto - here[0] - here[1]);
      if (rank > 0 && rank <= here[0] + here[1]) {
        const int second = rank > here[0] ? 1 : 0;
        found_bin = static_cast<uint32_t>(top - second);
        found_rank = second ? rank - here[0] : rank;
        found_keys = here[second];
      }
      __syncthreads();
      wanted = found_rank;
      low += found_bin << shift;
      last = low;
      if (shift == 0) break;
      if (found_keys == wanted) {  // all that are left
        last = low - 1;
        wanted = 0;
        break;
      }
      const int next_shift = max(0, shift - 11);
      width = 1u << (shift - next_shift);
      shift = next_shift;
    }
  }
  // Of the old keys those above `last` stay, and the first `wanted` that equal it; of the others all.
  int sure = 0, equal = 0;  // before this thread's keys
  for (int base = 0; base < len; base += kSelectThreads * kKeysPerThread) {
    const int first = base + static_cast<int>(threadIdx.x) * kKeysPerThread;
    uint32_t mine = 0;  // how many stay for sure (upper half) and how many equal the last (lower half): 4096 a round at most
    bool is_sure[kKeysPerThread], is_equal[kKeysPerThread];
#pragma unroll
    for (int k = 0; k < kKeysPerThread; ++k) {
      const int i = first + k;
      const uint32_t o = choose && i < old ? order_at(i) : 0u;
      is_sure[k] = i < len && (i >= old || (choose && o > last));
      is_equal[k] = choose && i < old && o == last;
      mine += (is_sure[k] ? 0x10000u : 0u) + (is_equal[k] ? 1u : 0u);
    }
    uint32_t upto = mine;
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, upto, x);
      if (lane >= x) upto += y;
    }
    if (lane == 31) warp_counts[warp] = upto;
    __syncthreads();
    uint32_t of_warps = warp_counts[lane];
#pragma unroll
    for (int x = 1; x < 32; x <<= 1) {
      const uint32_t y = __shfl_up_sync(0xffffffffu, of_warps, x);
      if (lane >= x) of_warps += y;
    }
    const uint32_t total = __shfl_sync(0xffffffffu, of_warps, 31);
    const uint32_t before = (warp == 0 ? 0u : __shfl_sync(0xffffffffu, of_warps, max(warp - 1, 0))) + upto - mine;
    int my_sure = sure + static_cast<int>(before >> 16), my_equal = equal + static_cast<int>(before & 0xffffu);
#pragma unroll
    for (int k = 0; k < kKeysPerThread; ++k) {
      if (is_sure[k] || (is_equal[k] && my_equal < wanted)) {
        const int to = my_sure + min(my_equal, wanted);
        kept[to] = first + k;
        weights_out[to] = weights[first + k];
      }
      my_sure += is_sure[k];
      my_equal += is_equal[k];
    }
    sure += static_cast<int>(total >> 16);
    equal += static_cast<int>(total & 0xffffu);
    __syncthreads();  // (the warps' counts have been read)
  }
  for (int i = min(len, p.keep) + threadIdx.x; i < p.out_len; i += kSelectThreads) {
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
  griddep_launch_dependents();
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
  static const cudaError_t attr_set = cudaFuncSetAttribute(select_kept_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kMaxCachedKeys * 4);
  if (attr_set != cudaSuccess) return attr_set;
  // (a cache that holds no more than stays has nothing to choose from)
  s.cached_keys = a.kv_len <= a.keep ? 0 : std::min(a.kv_len, kMaxCachedKeys);
  cudaError_t e = launch_overlapped(select_kept_kernel, static_cast<int64_t>(a.batch) * a.kv_heads, kSelectThreads,
                                    static_cast<size_t>(s.cached_keys) * 4, a.stream, s);
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
  const int64_t ctas = (g.total + 255) / 256, most = static_cast<int64_t>(sm_count()) * 32;
  return launch_overlapped(gather_kept_kernel, ctas < most ? ctas : most, 256, 0, a.stream, g);
}

}  // namespace flsm100
