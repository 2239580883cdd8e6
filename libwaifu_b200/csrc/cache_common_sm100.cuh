// What the kernels over a key-value cache share: which keys a run of queries sees, 16-bit pairs, and the sum of
// parts of a row's output that are relative to different maxima.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <utility>

#include "gemm_sm100.cuh"

namespace flsm100 {

// Division by a number that the host knows, of numbers below 2^31, by a multiplication (Granlund and Montgomery's division by invariant
// integers): with 2^s >= d > 2^(s - 1) and m = ceil(2^(32 + s) / d) - 2^32 the
// quotient is (n m / 2^32 + n) / 2^s, rounded down twice. A unit's place takes a dozen divisions, which at some 40
// instructions each were a microsecond and more at the beginning of a kernel.
struct Divisor {
  uint32_t d, m;
  int s;
  static Divisor of(uint32_t d) {
    Divisor r = {d, 0, 0};
    while ((uint64_t{1} << r.s) < d) ++r.s;
    r.m = static_cast<uint32_t>(((uint64_t{1} << (32 + r.s)) + d - 1) / d - (uint64_t{1} << 32));
    return r;
  }
  __device__ __forceinline__ int quotient(int n) const {
    return static_cast<int>((__umulhi(static_cast<uint32_t>(n), m) + static_cast<uint32_t>(n)) >> s);
  }
  // n becomes the quotient, and the remainder is returned.
  __device__ __forceinline__ int take(int *n) const {
    const int q = quotient(*n), r = *n - q * static_cast<int>(d);
    *n = q;
    return r;
  }
};

// Half probabilities are 2^7 times what they are relative to a row's maximum, and the row's sum and output with them. The maximum lags by
// 2^8 at most (see the kernels), so the largest is 2^15; the least that does not round to zero is 2^-32 instead of 2^-25. A
// million keys below 2^-25 have up to 3 % of a row's weight, below 2^-32 less than a half's rounding. (bfloat16 has float's range.)
template <bool BF16>
constexpr float kProbabilityShift = BF16 ? 0.0f : 7.0f;

// Eight 32-bit values to 32-byte aligned memory: a whole sector from one lane.
__device__ __forceinline__ void store_32_bytes(void *dst, uint32_t a, uint32_t b, uint32_t c, uint32_t d, uint32_t e, uint32_t f, uint32_t g,
                                               uint32_t h) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(dst), "r"(a), "r"(b), "r"(c), "r"(d), "r"(e), "r"(f), "r"(g), "r"(h)
               : "memory");
}

// (Read past L1: a kernel that starts under the end of another may find a line there from before the lengths were written.)
__device__ __forceinline__ int sequence_length(const int32_t *kv_lens, int seq, int kv_len) {
  return kv_lens == nullptr ? kv_len : min(max(__ldcg(kv_lens + seq), 0), kv_len);
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

// Zeros (of either sign) go on as such, through eight finite values: zero times an infinity or a NaN is a NaN, which stays.
template <bool BF16>
__device__ __forceinline__ uint32_t probe_nonfinite(uint4 w, uint32_t zeros) {
  const uint32_t each[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (BF16) {
      asm("fma.rn.bf16x2 %0, %1, %2, %0;" : "+r"(zeros) : "r"(each[i]), "r"(0u));
    } else {
      asm("fma.rn.f16x2 %0, %1, %2, %0;" : "+r"(zeros) : "r"(each[i]), "r"(0u));
    }
  }
  return zeros;
}

template <bool BF16>
__device__ __forceinline__ uint4 without_nonfinite(uint4 w) {
  return make_uint4(w.x & ~nonfinite_halves<BF16>(w.x), w.y & ~nonfinite_halves<BF16>(w.y), w.z & ~nonfinite_halves<BF16>(w.z),
                    w.w & ~nonfinite_halves<BF16>(w.w));
}

// Four columns of a row's output and its sum, relative to the maximum m (log2 units), from parts that have their own:
// a part's maximum is seen (raise) before the part is added, which scales it down to m; what was there is scaled when m rises.
struct RowSum {
  float m, l;
  float4 o;
  __device__ __forceinline__ void clear() {
    m = -INFINITY;
    l = 0.0f;
    o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
  }
  __device__ __forceinline__ void raise(float part_max) {
    if (part_max > m) {
      const float f = exp2f(m - part_max);
      m = part_max;
      l *= f;
      o = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
    }
  }
  // (A part whose rows saw no finite score has the maximum -inf: its sum is 0 or NaN, taken as it is.)
  __device__ __forceinline__ void add(float2 part, float4 x) {
    const float f = part.x == -INFINITY ? 1.0f : exp2f(part.x - m);
    l = fmaf(part.y, f, l);
    o = make_float4(fmaf(x.x, f, o.x), fmaf(x.y, f, o.y), fmaf(x.z, f, o.z), fmaf(x.w, f, o.w));
  }
};

// Adds four columns of `count` parts that other CTAs wrote, part c at row place(c), in their order, eight of them on their way
// at a time.
template <int D, typename Place>
__device__ __forceinline__ void add_parts(int count, const float2 *sums, const float *outs, int col, RowSum *sum, Place &&place) {
  constexpr int kAtOnce = 8;
  for (int c0 = 0; c0 < count; c0 += kAtOnce) {
    float2 part[kAtOnce];
    float4 out[kAtOnce];
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      const int64_t at = place(min(c0 + i, count - 1));
      part[i] = __ldcg(&sums[at]);
      out[i] = __ldcg(reinterpret_cast<const float4 *>(outs + at * D + col));
    }
    float top = part[0].x;
#pragma unroll
    for (int i = 1; i < kAtOnce; ++i) top = fmaxf(top, part[i].x);
    sum->raise(top);
#pragma unroll
    for (int i = 0; i < kAtOnce; ++i) {
      if (c0 + i < count) sum->add(part[i], out[i]);
    }
  }
}

// Launches a kernel that may start under the end of the one before it in the stream. Every kernel here waits for that one
// (griddep_wait) before it reads or writes global memory, and only then lets the next one start: so whatever starts
// early finds the inputs of the call complete. The kernels that follow another one of the same call wait where
// they need its results.
template <typename... Params, typename... Args>
cudaError_t launch_overlapped(void (*kernel)(Params...), int64_t ctas, int threads, size_t smem, cudaStream_t stream, Args &&...args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas), 1, 1);
  cfg.blockDim = dim3(static_cast<unsigned>(threads), 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, std::forward<Args>(args)...);
}

}  // namespace flsm100
