// What the attention kernels on tcgen05 share: tiles of 128 queries against blocks of 128 keys, both products'
// instructions, the online softmax of a block from and to tensor memory, and the operands' tensor maps.
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "ptx_sm100.cuh"

namespace flsm100 {

namespace {

constexpr int kBlockQ = 128;   // queries per CTA = lanes of tensor memory
constexpr int kBlockKv = 128;  // keys per step
constexpr int kAtomBytes = 128;  // one swizzle atom: 64 16-bit elements of K
constexpr int kAtomElems = 64;
constexpr int kMmaKBytes = 32;   // one kind::f16 instruction: 16 elements of K
constexpr int kTiles = 2;
constexpr int kTileWarps = 4;

// A block's probabilities are handed over in so many parts of its keys. At head_dim 128 the product of
// the first half runs under the exponentials of the second (2 x 24 x 4352: 396 -> 386 us); at 64,
// where the products are half as long, one hand-over less is worth more (2 x 8 x 1000 x 2000: 34.6 us
// in halves, 32.1 whole).
template <int D>
constexpr int kPartsOf = D == 128 ? 2 : 1;

__device__ __forceinline__ void tma_load_4d(void *smem_dst, const CUtensorMap *desc, uint64_t *bar, int32_t c0,
                                            int32_t c1, int32_t c2, int32_t c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5, %6}], [%2];"
      ::"r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(desc)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2),
      "r"(c3)
      : "memory");
}

__device__ __forceinline__ void tma_load_3d(void *smem_dst, const CUtensorMap *desc, uint64_t *bar, int32_t c0,
                                            int32_t c1, int32_t c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(desc)), "r"(smem_u32(bar)), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}

// 2^x for x <= 2^kRescaleStep's exponent: the hardware approximation (relative error 2^-22), -inf -> 0.
__device__ __forceinline__ float fast_exp2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 2^x for a pair of exponents x <= 2^kRescaleStep's, without the special-function unit: that unit
// delivers 16 results a cycle and SM, so the 128 x 128 exponentials of a block would hold it for
// 1024 cycles; one pair in four of a row goes through here instead, on the multiply-add pipes
// (with one softmax warp per scheduler at work at a time, more than that costs more issue slots
// than it frees special-function cycles).
// x = n + f with n = round(x) (the low mantissa bits of x + 1.5 * 2^23) and f in [-0.5, 0.5]; 2^f
// by a cubic (relative error 7.5e-5, below the 16-bit rounding the probabilities get); n added
// into the exponent field. Exponents below -126 (masked keys are -inf) give 2^-126 or 0.
__device__ __forceinline__ void exp2_pair_poly(uint64_t x, float *e0, float *e1) {
  float x0, x1;
  f2_unpack(x, &x0, &x1);
  x = f2_pack(fmaxf(x0, -126.0f), fmaxf(x1, -126.0f));
  const uint64_t t = f2_add(x, f2_pack(12582912.0f, 12582912.0f));
  const uint64_t n = f2_add(t, f2_pack(-12582912.0f, -12582912.0f));
  const uint64_t f = f2_fma(n, f2_pack(-1.0f, -1.0f), x);
  uint64_t q = f2_fma(f, f2_pack(0.05517162f, 0.05517162f), f2_pack(0.24261113f, 0.24261113f));
  q = f2_fma(q, f, f2_pack(0.69326097f, 0.69326097f));
  q = f2_fma(q, f, f2_pack(0.99992806f, 0.99992806f));
  float q0, q1, t0, t1;
  f2_unpack(q, &q0, &q1);
  f2_unpack(t, &t0, &t1);
  *e0 = __int_as_float(__float_as_int(q0) + (__float_as_int(t0) << 23));
  *e1 = __int_as_float(__float_as_int(q1) + (__float_as_int(t1) << 23));
}

// max(a, b, c) in one instruction.
__device__ __forceinline__ float max3(float a, float b, float c) {
  float r;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

// The same, NaN where one of them is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ uint32_t pack16(float a, float b, int is_bf16) {
  if (is_bf16) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
  }
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t *>(&h);
}

// Asks for a CTA of this grid that has not started: sixteen bytes of answer, counted on `bar`.
__device__ __forceinline__ void claim_next_cta(uint4 *answer, uint64_t *bar) {
  asm volatile("clusterlaunchcontrol.try_cancel.async.shared::cta.mbarrier::complete_tx::bytes.b128 [%0], [%1];"
               ::"r"(smem_u32(answer)), "r"(smem_u32(bar))
               : "memory");
}

// The block indices of the CTA that was taken over, w = 1; w = 0 where none was left.
__device__ __forceinline__ int4 claimed_cta(const uint4 *answer) {
  int4 c;
  asm volatile(
      "{\n\t"
      ".reg .b128 r;\n\t"
      ".reg .pred p;\n\t"
      ".reg .b32 x, y, z, u;\n\t"
      "ld.shared.b128 r, [%4];\n\t"
      "clusterlaunchcontrol.query_cancel.is_canceled.pred.b128 p, r;\n\t"
      "selp.b32 %3, 1, 0, p;\n\t"
      "mov.b32 x, 0;\n\t"
      "mov.b32 y, 0;\n\t"
      "mov.b32 z, 0;\n\t"
      "@p clusterlaunchcontrol.query_cancel.get_first_ctaid.v4.b32.b128 {x, y, z, u}, r;\n\t"
      "mov.b32 %0, x;\n\t"
      "mov.b32 %1, y;\n\t"
      "mov.b32 %2, z;\n\t"
      "}"
      : "=r"(c.x), "=r"(c.y), "=r"(c.z), "=r"(c.w)
      : "r"(smem_u32(answer))
      : "memory");
  return c;
}

// Zeros in the rows of `ATOMS` atoms of 128 that boxes of `rows` rows never fill: what lies there takes part in no result, but a
// row's garbage would have its warp rescale when other garbage would not, and the results differ in their last bits.
template <int ATOMS>
__device__ __forceinline__ void clear_empty_places(uint8_t *atoms, int rows, int threads) {
  const int pieces = (kBlockQ - rows) * (kAtomBytes / 16);  // of an atom
#pragma unroll 1
  for (int a = 0; a < ATOMS; ++a) {
    for (int i = threadIdx.x; i < pieces; i += threads) {
      *reinterpret_cast<uint4 *>(atoms + a * kBlockQ * kAtomBytes + rows * kAtomBytes + i * 16) = make_uint4(0, 0, 0, 0);
    }
  }
  fence_proxy_async_smem();
}

// The tiles in shared and tensor memory.
template <int D>
struct TileLayout {
  static constexpr int kQAtoms = D / kAtomElems;
  static constexpr int kQBytes = kQAtoms * kBlockQ * kAtomBytes;  // one tile's queries
  static constexpr int kSlotBytes = kQAtoms * kBlockKv * kAtomBytes;  // a block of K: 128 keys x head_dim
  static constexpr int kVAtoms = kBlockKv / kAtomElems;
  static constexpr int kVAtomBytes = D * kAtomBytes;
  static_assert(kVAtoms * kVAtomBytes == kSlotBytes, "a block of V^T fills a slot exactly as a block of K does");
  static constexpr int kSCols = kBlockKv;           // tile t's scores at column t * kSCols, its P over their first half
  static constexpr int kOCol = kTiles * kSCols;     // tile t's output at kOCol + t * D
  static constexpr int kTmemCols = 512;
  static_assert(kOCol + kTiles * D <= kTmemCols, "tensor memory holds 512 columns");
};

// Block j of the keys for one query (a lane's row of the tile): its scores from tensor memory, the running
// maximum and sum, and the probabilities back into tensor memory, part by part. `hide(scores)` sets those of the
// keys the row does not see to -inf; `first` is the tile's first block, whose output need not be rescaled.
// The probabilities, their sum and the output are 2^shift times what they are relative to *m_used_io.
// Where a seen score that is NaN or +inf has to make the row NaN (CARRY_NAN), the maximum carries it into the sum: the
// cubic exponential does not.
template <int D, bool CARRY_NAN, typename Hide>
__device__ __forceinline__ void softmax_block(float scale_log2, int is_bf16, float shift, uint32_t t_scores, uint32_t t_out, bool first,
                                              Hide &&hide, uint64_t *p_full_bar, uint32_t lane, float *m_used_io, float *l_run_io) {
  constexpr int kPParts = kPartsOf<D>;
  constexpr int kChunks = kBlockKv / 32;
  static_assert(kChunks == 4, "four chunks of scores pack into the first two");
  constexpr float kRescaleStep = 8.0f;
  float m_used = *m_used_io, l_run = *l_run_io;
  uint32_t sc[kChunks][32];  // the row's scores of the block, in one round trip
#pragma unroll
  for (int c = 0; c < kChunks; ++c) tmem_ld_32x32(t_scores + c * 32, sc[c]);
#pragma unroll
  for (int c = 0; c < kChunks; ++c) tmem_ld_wait(sc[c]);
  float m4[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
  hide(sc);
#pragma unroll
  for (int c = 0; c < kChunks; ++c) {
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      m4[(i >> 1) & 3] = CARRY_NAN ? max3_nan(m4[(i >> 1) & 3], __uint_as_float(sc[c][i]), __uint_as_float(sc[c][i + 1]))
                                   : max3(m4[(i >> 1) & 3], __uint_as_float(sc[c][i]), __uint_as_float(sc[c][i + 1]));
    }
  }
  const float m_blk = (CARRY_NAN ? max3_nan(max3_nan(m4[0], m4[1], m4[2]), m4[3], m4[3]) : fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]))) * scale_log2;
  if (CARRY_NAN && !(m_blk < INFINITY)) l_run = NAN;
  if (__any_sync(0xffffffffu, m_blk > m_used + kRescaleStep)) {
    const float m_new = fmaxf(m_used, m_blk);
    const float alpha = exp2f(m_used - ((m_new == -INFINITY) ? 0.0f : m_new));
    l_run *= alpha;
    if (!first) {
#pragma unroll 1
      for (int c = 0; c < D / 16; ++c) {  // sixteen columns at a time: the block's scores stay in registers
        uint32_t v[16];
        tmem_ld_32x16(t_out + c * 16, v);
        tmem_ld_wait(v);
#pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * alpha);
        tmem_st_32x16(t_out + c * 16, v);
      }
    }
    m_used = m_new;
  }
  const float m_sub = (m_used == -INFINITY) ? 0.0f : m_used;
  // The probabilities, packed in place: pair i of the row's keys becomes column i of its P
  // (a slot whose scores have been used by then).
  // They are rounded to the operands' type, which the product takes: half a step each at most (2^-8 of it in bfloat16, 2^-11 in half), of
  // either sign, so that a result is off by about as much as its own rounding makes it (bfloat16 2.3e-3 of relative error in all
  // where 1.7e-3 is the result's rounding, half 2.9e-4 and 2.1e-4). A second product with what the rounding took, as the
  // few-row kernel has it, would be half as many instructions again on the tensor pipe. The sums are of the values before.
  const uint64_t scale2 = f2_pack(scale_log2, scale_log2), neg_m2 = f2_pack(shift - m_sub, shift - m_sub);
  uint64_t sums[2] = {0, 0};  // (pairs of float32 zeros)
  auto emit = [&](auto bf16_tag, int part) {
    constexpr int kBf16 = decltype(bf16_tag)::value ? 1 : 0;
#pragma unroll
    for (int h = 0; h < kChunks / kPParts; ++h) {
      const int c = part * (kChunks / kPParts) + h;
#pragma unroll
      for (int i = 0; i < 32; i += 2) {
        const uint64_t x = f2_fma(f2_pack(__uint_as_float(sc[c][i]), __uint_as_float(sc[c][i + 1])), scale2, neg_m2);
        float e0, e1;
        if ((i & 6) != 6) {  // one pair in four goes through the cubic, the others through the special-function unit
          float x0, x1;
          f2_unpack(x, &x0, &x1);
          e0 = fast_exp2(x0);
          e1 = fast_exp2(x1);
        } else {
          exp2_pair_poly(x, &e0, &e1);
        }
        sums[(i >> 1) & 1] = f2_add(sums[(i >> 1) & 1], f2_pack(e0, e1));
        sc[c >> 1][(c & 1) * 16 + (i >> 1)] = pack16(e0, e1, kBf16);
      }
    }
  };
  // Each half of the block's keys is handed over as soon as it is there: its product runs under
  // the exponentials of the other half.
#pragma unroll
  for (int part = 0; part < kPParts; ++part) {
    if (is_bf16) {
      emit(std::true_type{}, part);
    } else {
      emit(std::false_type{}, part);
    }
    tmem_st_32x32(t_scores + part * 32, sc[part]);
    if (kPParts == 1) tmem_st_32x32(t_scores + 32, sc[1]);
    tmem_st_wait();          // the probabilities and a rescaled output are in tensor memory
    tc_fence_before_sync();  // before the MMAs that the hand-over starts
    __syncwarp();
    if (lane == 0) mbar_arrive(&p_full_bar[part]);
  }
  float s0, s1, s2, s3;
  f2_unpack(sums[0], &s0, &s1);
  f2_unpack(sums[1], &s2, &s3);
  l_run += (s0 + s1) + (s2 + s3);
  *m_used_io = m_used;
  *l_run_io = l_run;
}

// The instructions of a tile's two products. The whole warp calls, the elected lane issues.
template <int D>
struct TileMmas {
  using L = TileLayout<D>;
  static constexpr uint64_t kMmaStep = kMmaKBytes >> 4;
  static constexpr int kMmasPerAtom = kAtomBytes / kMmaKBytes;
  static constexpr int kScoreMmas = L::kQAtoms * kMmasPerAtom;
  static constexpr int kOutMmas = L::kVAtoms * kMmasPerAtom;  // one per 16 keys: 8 columns of P each
  uint32_t tmem_base, idesc_s, idesc_o, idesc_o_mn;
  uint64_t qdesc0, mn_fields;
  bool issuer, v_direct;

  // With v as it lies, a slot's rows are keys: an instruction's 16 keys are 16 rows of 128 bytes on, the
  // operand is MN-major (bit 16 of the instruction descriptor) and its runs of 64 head_dim positions
  // lie a 128-key atom apart.
  __device__ __forceinline__ TileMmas(int is_bf16, bool v_as_it_lies, uint32_t tmem, uint32_t q_smem, bool elected)
      : tmem_base(tmem), qdesc0(umma_desc_sw128(q_smem)),
        mn_fields(umma_desc_sw128_mn(0, kBlockKv * kAtomBytes) ^ umma_desc_sw128(0)), issuer(elected), v_direct(v_as_it_lies) {
    const uint32_t fmt = is_bf16 ? 1u : 0u;
    idesc_s = umma_idesc(kBlockQ, kBlockKv, fmt, fmt);
    idesc_o = umma_idesc(kBlockQ, D, fmt, fmt);
    idesc_o_mn = idesc_o | (1u << 16);
  }

  __device__ __forceinline__ void scores(int i, uint64_t kd) const {  // S_i = Q_i K^T
    const uint32_t s_tmem = tmem_base + i * L::kSCols;
    const uint64_t qd = qdesc0 + static_cast<uint64_t>(i * (L::kQBytes >> 4));
#pragma unroll
    for (int m = 0; m < kScoreMmas; ++m) {
      const int a = m / kMmasPerAtom, s = m % kMmasPerAtom;
      const uint64_t qa = qd + (((a * kBlockQ * kAtomBytes) >> 4) + s * kMmaStep);
      const uint64_t ka = kd + (((a * kBlockKv * kAtomBytes) >> 4) + s * kMmaStep);
      if (issuer) umma_ss<kKindF16>(s_tmem, qa, ka, idesc_s, m != 0 ? 1u : 0u);
    }
  }

  // O_i += P_i V over one part of the block's keys
  __device__ __forceinline__ void product(int i, int part, uint64_t vd, uint32_t first_block) const {
    const uint32_t o_tmem = tmem_base + L::kOCol + i * D;
    const uint32_t p_tmem = tmem_base + i * L::kSCols;
    constexpr int kPartMmas = kOutMmas / kPartsOf<D>;
    if (v_direct) {
#pragma unroll
      for (int k = 0; k < kPartMmas; ++k) {
        const int m = part * kPartMmas + k;
        const uint64_t va = (vd ^ mn_fields) + static_cast<uint64_t>(m * ((16 * kAtomBytes) >> 4));
        if (issuer) umma_ts_f16(o_tmem, p_tmem + m * 8, va, idesc_o_mn, m != 0 ? 1u : (first_block ^ 1u));
      }
    } else {
#pragma unroll
      for (int k = 0; k < kPartMmas; ++k) {
        const int m = part * kPartMmas + k;
        const int a = m / kMmasPerAtom, s = m % kMmasPerAtom;
        if (issuer) umma_ts_f16(o_tmem, p_tmem + m * 8, vd + (((a * L::kVAtomBytes) >> 4) + s * kMmaStep), idesc_o,
                    m != 0 ? 1u : (first_block ^ 1u));
      }
    }
  }
};

using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                   const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_fn() {
  static EncodeTiledFn fn = [] {
    void *ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess) {
      return reinterpret_cast<EncodeTiledFn>(ptr);
    }
    return static_cast<EncodeTiledFn>(nullptr);
  }();
  return fn;
}

// A byte tensor of `rank` dimensions, innermost contiguous, read in boxes of 128 bytes x box[0] x box[1] x box[2] of
// the others, 128-byte swizzle, zeros outside.
inline bool make_tmap(CUtensorMap *map, const void *base, int rank, const uint64_t *dims, const uint64_t *strides_bytes,
                      const uint32_t (&rows)[3]) {
  EncodeTiledFn fn = encode_fn();
  if (!fn) return false;
  cuuint64_t d[4];
  cuuint64_t s[3];
  cuuint32_t box[4] = {static_cast<cuuint32_t>(kAtomBytes), rows[0], rows[1], rows[2]};
  cuuint32_t estr[4] = {1, 1, 1, 1};
  for (int i = 0; i < rank; ++i) d[i] = dims[i];
  for (int i = 0; i + 1 < rank; ++i) s[i] = strides_bytes[i];
  CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, static_cast<cuuint32_t>(rank), const_cast<void *>(base), d, s, box,
                  estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS;
}

// The same in boxes of 128 bytes x box_rows of the second dimension.
inline bool make_tmap(CUtensorMap *map, const void *base, int rank, const uint64_t *dims, const uint64_t *strides_bytes,
                      uint32_t box_rows) {
  const uint32_t rows[3] = {box_rows, 1, 1};
  return make_tmap(map, base, rank, dims, strides_bytes, rows);
}

// Queries, keys or values as (head_dim bytes, positions, heads, batch), strides in elements, in boxes of box_rows positions.
inline bool row_map(CUtensorMap *map, const void *base, int head_dim, int len, int heads, int batch, int64_t batch_stride, int64_t head_stride,
             int64_t position_stride, uint32_t box_rows) {
  const uint64_t dims[4] = {static_cast<uint64_t>(head_dim) * 2, static_cast<uint64_t>(len), static_cast<uint64_t>(heads), static_cast<uint64_t>(batch)};
  // (the stride of a dimension of extent 1 is never used, but has to pass the encoder's checks)
  auto bytes = [&](int64_t s) { return static_cast<uint64_t>(s > 0 ? s : head_dim) * 2; };
  const uint64_t strides[3] = {bytes(len > 1 ? position_stride : 0), bytes(heads > 1 ? head_stride : 0), bytes(batch > 1 ? batch_stride : 0)};
  return make_tmap(map, base, 4, dims, strides, box_rows);
}

}  // namespace

}  // namespace flsm100
