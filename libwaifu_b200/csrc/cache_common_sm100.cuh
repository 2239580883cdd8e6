// What the kernels over a key-value cache share: which keys a run of queries sees, 16-bit pairs, and the sum of
// parts of a row's output that are relative to different maxima.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "gemm_sm100.cuh"

namespace flsm100 {

constexpr int kFewRowsTile = 16;

__device__ __forceinline__ int sequence_length(const int32_t *kv_lens, int seq, int kv_len) {
  return kv_lens == nullptr ? kv_len : min(max(kv_lens[seq], 0), kv_len);
}

// Keys 0 .. sinks - 1 and begin .. end - 1, counted through.
struct KeyRange {
  int sinks, begin, end;
  __device__ __forceinline__ int count() const { return sinks + end - begin; }
  __device__ __forceinline__ int key(int at) const { return at < sinks ? at : at - sinks + begin; }
};

// The keys that queries at positions first .. last see between them. (window <= kv_len, so nothing leaves 32 bits.)
__device__ __forceinline__ KeyRange visible_keys(int first, int last, int len, int window, int sinks) {
  KeyRange r;
  r.end = max(0, min(len, last + 1));
  r.begin = min(max(0, first - window + 1), r.end);
  r.sinks = min(sinks, r.begin);
  return r;
}

// 2^x by the hardware's function (relative error 2^-22), -inf -> 0.
__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <bool BF16>
__device__ __forceinline__ uint32_t pack_pair(float a, float b) {
  if constexpr (BF16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
  } else {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
}

template <bool BF16>
__device__ __forceinline__ float2 widen_pair(uint32_t w) {
  if constexpr (BF16) {
    return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162 *>(&w));
  } else {
    return __half22float2(*reinterpret_cast<const __half2 *>(&w));
  }
}

// a and b rounded, and what the rounding took.
template <bool BF16>
__device__ __forceinline__ void split_pair(float a, float b, uint32_t *hi, uint32_t *lo) {
  *hi = pack_pair<BF16>(a, b);
  const float2 h = widen_pair<BF16>(*hi);
  *lo = pack_pair<BF16>(a - h.x, b - h.y);
}

// Does a word of two 16-bit values hold an infinity or a NaN (an exponent of ones)? A mask of the halves that do.
template <bool BF16>
__device__ __forceinline__ uint32_t nonfinite_halves(uint32_t w) {
  constexpr uint32_t kExponent = BF16 ? 0x7F807F80u : 0x7C007C00u;
  return __vcmpeq2(w & kExponent, kExponent);
}
template <bool BF16>
__device__ __forceinline__ bool has_nonfinite(uint4 w) {
  return (nonfinite_halves<BF16>(w.x) | nonfinite_halves<BF16>(w.y) | nonfinite_halves<BF16>(w.z) | nonfinite_halves<BF16>(w.w)) != 0;
}
template <bool BF16>
__device__ __forceinline__ uint4 without_nonfinite(uint4 w) {
  return make_uint4(w.x & ~nonfinite_halves<BF16>(w.x), w.y & ~nonfinite_halves<BF16>(w.y), w.z & ~nonfinite_halves<BF16>(w.z),
                    w.w & ~nonfinite_halves<BF16>(w.w));
}

// C columns of a row's output and its sum, relative to the maximum m (log2 units), from parts that have their own:
// the maxima are seen first (raise), then the parts added, which scales them down to m once. What was there before is
// scaled when a later maximum raises m.
template <int C>
struct RowSum {
  float m, l, o[C];
  __device__ __forceinline__ void clear() {
    m = -INFINITY;
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < C; ++i) o[i] = 0.0f;
  }
  __device__ __forceinline__ void raise(float part_max) {
    if (part_max > m) {
      const float f = exp2f(m - part_max);
      m = part_max;
      l *= f;
#pragma unroll
      for (int i = 0; i < C; ++i) o[i] *= f;
    }
  }
  // (A part whose rows saw no finite score has the maximum -inf: its sum is 0 or NaN, taken as it is.)
  __device__ __forceinline__ float factor(float part_max) const { return part_max == -INFINITY ? 1.0f : exp2f(part_max - m); }
  __device__ __forceinline__ void add(float2 part, const float *part_out) {
    const float f = factor(part.x);
    l = fmaf(part.y, f, l);
#pragma unroll
    for (int i = 0; i < C; i += 4) {
      const float4 x = *reinterpret_cast<const float4 *>(part_out + i);
      o[i] = fmaf(x.x, f, o[i]);
      o[i + 1] = fmaf(x.y, f, o[i + 1]);
      o[i + 2] = fmaf(x.z, f, o[i + 2]);
      o[i + 3] = fmaf(x.w, f, o[i + 3]);
    }
  }
  // The same from global memory that another CTA wrote.
  __device__ __forceinline__ void add_parts(float2 part, const float *part_out) {
    const float f = factor(part.x);
    l = fmaf(part.y, f, l);
#pragma unroll
    for (int i = 0; i < C; i += 4) {
      const float4 x = __ldcg(reinterpret_cast<const float4 *>(part_out + i));
      o[i] = fmaf(x.x, f, o[i]);
      o[i + 1] = fmaf(x.y, f, o[i + 1]);
      o[i + 2] = fmaf(x.z, f, o[i + 2]);
      o[i + 3] = fmaf(x.w, f, o[i + 3]);
    }
  }
  __device__ __forceinline__ void store(float *dst) const {
#pragma unroll
    for (int i = 0; i < C; i += 4) *reinterpret_cast<float4 *>(dst + i) = make_float4(o[i], o[i + 1], o[i + 2], o[i + 3]);
  }
  __device__ __forceinline__ float2 max_and_sum() const { return make_float2(m, l); }
};

}  // namespace flsm100
