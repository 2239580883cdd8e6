// How much each key of a cache is attended to by many queries, on tcgen05.
//
// The attention kernel has left each query row's maximum m and 1 / sum; a key's weight from a row is
// exp2(score - m) / sum, and its scores are computed again: storing them would move heads x queries x keys x 4 bytes
// twice, more than the product takes. Here the keys are the rows of the product, S^T = K Q^T: a CTA owns two tiles of 128
// keys of one key-value head and walks the rows of the heads that share it, packed as the tile kernel packs them, up to
// 128 at a time, so a thread owns a key and adds up over the columns of its row in tensor memory; nothing has to meet another thread. The scores of two blocks lie in
// tensor memory at a time, so that a block's product runs under the exponentials of the one before it. The
// walks of a key's tiles are divided over CTAs, whose sums the last one to arrive adds in their order.
//
// What bounds it is the special-function unit: 16 exponentials a cycle and SM against 128 x 128 of them a tile and block, 23 of
// the 37 us that 2 x 16 heads of 2048 queries and keys take. They are all the hardware's (2^-22), unlike the attention
// kernel's, whose cubic (7.5e-5 in one of four) a row's sum carries.
#include "cache_weights_sm100.cuh"

#include <cuda_runtime.h>

#include <algorithm>

#include "attention_sm100.cuh"
#include "attention_tile_sm100.cuh"
#include "cache_common_sm100.cuh"

namespace flsm100 {

namespace {

constexpr int kKeysPerCta = kTiles * kBlockKv;
constexpr int kSumWarps = kTiles * kTileWarps;
constexpr int kProducerWarp = kSumWarps;
constexpr int kMmaWarp = kSumWarps + 1;
constexpr int kThreads = (kSumWarps + 2) * 32;
constexpr int kMaxSlots = 6;
constexpr int kNormBytes = kBlockQ * 8;

struct Tail {
  uint64_t k_full_bar;
  uint64_t slot_full_bar[kMaxSlots], slot_empty_bar[kMaxSlots];
  uint64_t s_full_bar[kTiles][2], s_empty_bar[kTiles][2];
  uint32_t tmem_base_slot;
  uint32_t abort_flag;
  int is_last;
};

template <int D>
struct Layout : TileLayout<D> {
  using T = TileLayout<D>;
  static constexpr int kKeysOff = 0;
  static constexpr int kSlotBytes = T::kQBytes + kNormBytes;  // 128 queries and their rows' maxima and 1 / sums
  static constexpr int kRoom = (227 * 1024 - kTiles * T::kSlotBytes - static_cast<int>(sizeof(Tail))) / kSlotBytes;
  static constexpr int kSlots = kRoom < kMaxSlots ? kRoom : kMaxSlots;
  static constexpr int kQueriesOff = kKeysOff + kTiles * T::kSlotBytes;
  static constexpr int kNormsOff = kQueriesOff + kSlots * T::kQBytes;
  static constexpr int kTailOff = kNormsOff + kSlots * kNormBytes;
  static constexpr int kSmemBytes = kTailOff + static_cast<int>(sizeof(Tail));
  static_assert(kSlots >= 2 && kSmemBytes <= 227 * 1024, "shared memory");
};

// Two tiles of keys and the blocks of rows that see some of them.
struct Unit {
  int run, head, seq, part, pair;
  int key0, len, offset;     // query i sits at i + offset
  int first, count, active;  // blocks of this part
  __device__ __forceinline__ Unit(const WeightsParams &p, int at) {
    // The first keys, which most queries see, first.
    run = at % p.runs;
    at /= p.runs;
    part = at % p.parts;
    pair = at / p.parts;
    head = run % p.kv_heads;
    seq = run / p.kv_heads;
    key0 = pair * kKeysPerCta;
    len = sequence_length(p.kv_lens, seq, p.kv_len);
    offset = len - p.q_len;
    const int first_block = p.by_positions.quotient(max(0, key0 - offset)), blocks = p.by_positions.quotient(p.q_len + p.positions - 1);
    const int total = key0 < len ? max(0, blocks - first_block) : 0;
    active = max(1, (total + p.part_blocks - 1) / p.part_blocks);
    first = first_block + part * p.part_blocks;
    count = max(0, min(p.part_blocks, total - part * p.part_blocks));
  }
  // Does a query of block b see a key of tile i?
  __device__ __forceinline__ bool meets(const WeightsParams &p, int b, int i) const {
    return key0 + i * kBlockKv < len && (first + b + 1) * p.positions - 1 + offset >= key0 + i * kBlockKv;
  }
};

// A key's sum over this part's rows that came out as NaN. The columns of a block that hold no row are zeros, their 1 / sum too, but
// zero times a key's infinity is a NaN. A row that sees such a key scores it -inf, or +inf or NaN, which make that row's own sum a NaN:
// the key's weight from it is zero, or a NaN as are all weights from a row without a sum. (Looked at here, and not where the columns
// are added up: a bound on each exponent that drops the NaN took 72.5 us where this takes 70.7, weights_prefill.)
template <int D>
__device__ __noinline__ float sum_without_empty_columns(const WeightsParams &p, const Unit &u, int key, const uint8_t *key_row, float sum) {
  bool infinite = false;
  for (int a = 0; a < D / kAtomElems; ++a) {  // (the pieces of a row lie in another order: here it is all the same)
    const uint16_t *w = reinterpret_cast<const uint16_t *>(key_row + a * kBlockKv * kAtomBytes);
    const int infinity = p.is_bf16 ? 0x7F80 : 0x7C00;
    for (int d = 0; d < kAtomElems; ++d) {
      const int magnitude = w[d] & 0x7FFF;
      if (magnitude > infinity) return sum;
      infinite |= magnitude == infinity;
    }
  }
  if (!infinite) return sum;
  for (int b = u.first; b < u.first + u.count; ++b) {
    const int query0 = b * p.positions, from = max(0, key - u.offset - query0), to = min(p.positions, p.q_len - query0);
    const float2 *norm = p.row_norm + static_cast<int64_t>(u.run) * p.norm_pitch + b * kBlockQ;
    for (int c = from * p.group; c < to * p.group; ++c) {
      const float inv = __ldcg(&norm[c]).y;
      if (inv != inv) return sum;
    }
  }
  return 0.0f;
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
cache_weights_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k,
                     const __grid_constant__ WeightsParams p) {
  using L = Layout<D>;
  constexpr int S = L::kSlots;
  extern __shared__ __align__(1024) uint8_t smem[];
  Tail &t = *reinterpret_cast<Tail *>(smem + L::kTailOff);
  volatile uint32_t &abort_flag = *reinterpret_cast<volatile uint32_t *>(&t.abort_flag);
  const uint32_t warp = threadIdx.x >> 5;
  const uint32_t lane = threadIdx.x & 31;
  if ((smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0) atomicCAS(p.status, 0u, kStatusAttentionLayout);
    return;
  }
  const Unit u(p, blockIdx.x);
  if (u.part >= u.active) return;

  if (threadIdx.x == 0) {
    t.abort_flag = 0;
    mbar_init(&t.k_full_bar, 1);
    for (int i = 0; i < S; ++i) {
      mbar_init(&t.slot_full_bar[i], 1);
      mbar_init(&t.slot_empty_bar[i], 1 + kSumWarps);
    }
    for (int i = 0; i < kTiles; ++i) {
      for (int b = 0; b < 2; ++b) {
        mbar_init(&t.s_full_bar[i][b], 1);
        mbar_init(&t.s_empty_bar[i][b], kTileWarps);
      }
    }
    fence_barrier_init();
  }
  if (warp == kProducerWarp && lane == 0) {
    tma_prefetch_desc(&tmap_q);
    tma_prefetch_desc(&tmap_k);
  }
  if (warp == kMmaWarp) {
    tmem_alloc<1>(&t.tmem_base_slot, L::kTmemCols);
    tmem_relinquish<1>();
  }
  clear_empty_places<L::kQAtoms * S>(smem + L::kQueriesOff, p.tile_rows, kThreads);  // (their maxima and 1 / sums are zeros too)
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = t.tmem_base_slot;
  griddep_wait();  // the rows' maxima and sums
  griddep_launch_dependents();

  if (warp < kSumWarps) {
    // ------------------------------------------------------------------ a key's sum
    const int tile = static_cast<int>(warp >> 2);
    const uint32_t quarter = warp & 3;
    const int in_cta = tile * kBlockKv + static_cast<int>(quarter) * 32 + static_cast<int>(lane);
    const int key = u.key0 + in_cta;
    const uint32_t t_lane = tmem_base + ((quarter * 32u) << 16) + tile * L::kSCols;
    const int tile_last = u.key0 + tile * kBlockKv + kBlockKv - 1;
    float sum = 0.0f;
    bool ok = true;
    int met = 0;
    for (int b = 0; b < u.count && ok; ++b) {
      const int st = b % S;
      ok = __all_sync(0xffffffffu, mbar_wait(&t.slot_full_bar[st], (b / S) & 1, &abort_flag));
      if (!ok) break;
      if (u.meets(p, b, tile)) {
        ok = __all_sync(0xffffffffu, mbar_wait(&t.s_full_bar[tile][met & 1], (met >> 1) & 1, &abort_flag));
        if (!ok) break;
        tc_fence_after_sync();
        uint32_t sc[4][32];
        const uint32_t t_scores = t_lane + (met & 1) * kTiles * L::kSCols;
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_32x32(t_scores + c * 32, sc[c]);
#pragma unroll
        for (int c = 0; c < 4; ++c) tmem_ld_wait(sc[c]);
        tc_fence_before_sync();
        __syncwarp();
        if (lane == 0) mbar_arrive(&t.s_empty_bar[tile][met & 1]);
        ++met;
        const float4 *norm = reinterpret_cast<const float4 *>(smem + L::kNormsOff + st * kNormBytes);  // two queries each
        const int query0 = (u.first + b) * p.positions;
        float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        if (query0 + u.offset >= tile_last) {  // every row of the block sees every key of the tile
#pragma unroll
          for (int c = 0; c < 4; ++c) {
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const float4 n = norm[(c * 32 + i) / 2];
              part[i & 3] = fmaf(fast_exp2(fmaf(__uint_as_float(sc[c][i]), p.scale_log2, -n.x)), n.y, part[i & 3]);
              part[(i + 1) & 3] = fmaf(fast_exp2(fmaf(__uint_as_float(sc[c][i + 1]), p.scale_log2, -n.z)), n.w, part[(i + 1) & 3]);
            }
          }
        } else {
          const int begin = max(0, key - u.offset - query0) * p.group;  // the first column that sees the key
#pragma unroll
          for (int c = 0; c < 4; ++c) {
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const float4 n = norm[(c * 32 + i) / 2];
              const int col = c * 32 + i;
              if (col >= begin) part[i & 3] = fmaf(fast_exp2(fmaf(__uint_as_float(sc[c][i]), p.scale_log2, -n.x)), n.y, part[i & 3]);
              if (col + 1 >= begin) {
                part[(i + 1) & 3] = fmaf(fast_exp2(fmaf(__uint_as_float(sc[c][i + 1]), p.scale_log2, -n.z)), n.w, part[(i + 1) & 3]);
              }
            }
          }
        }
        sum += (part[0] + part[1]) + (part[2] + part[3]);
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&t.slot_empty_bar[st]);
    }
    if (ok && sum != sum && key < u.len && mbar_wait(&t.k_full_bar, 0, &abort_flag)) {
      sum = sum_without_empty_columns<D>(p, u, key, smem + L::kKeysOff + tile * L::T::kSlotBytes + (in_cta % kBlockKv) * kAtomBytes, sum);
    }
    if (u.active > 1) {
      float *parts = p.part_sums + (static_cast<int64_t>(u.run) * p.pairs + u.pair) * p.parts * kKeysPerCta + in_cta;
      parts[u.part * kKeysPerCta] = sum;
      asm volatile("bar.sync 1, %0;" ::"n"(kSumWarps * 32) : "memory");
      if (threadIdx.x == 0) {
        __threadfence();
        uint32_t *counter = &p.counters[u.run * p.pairs + u.pair];
        const uint32_t before = atomicAdd(counter, 1u);
        t.is_last = before + 1 == static_cast<uint32_t>(u.active);
        if (t.is_last) *counter = 0;
        __threadfence();
      }
      asm volatile("bar.sync 1, %0;" ::"n"(kSumWarps * 32) : "memory");
      if (t.is_last) {
        sum = 0.0f;
        for (int s = 0; s < u.active; ++s) sum += __ldcg(parts + s * kKeysPerCta);
      }
    }
    if (ok && key < p.kv_len && (u.active == 1 || t.is_last)) {
      const float before = p.weights_in[u.seq * p.in_stride[0] + u.head * p.in_stride[1] + key];
      p.weights_out[u.seq * p.out_stride[0] + u.head * p.out_stride[1] + key] = key < u.len ? before + sum : before;
    }
    if (!ok && lane == 0) {
      abort_flag = 1;
      atomicCAS(p.status, 0u, kStatusAttentionTimeout);
    }
  } else if (warp == kProducerWarp) {
    // ------------------------------------------------------------------ producer
    if (elect_one()) {
      bool ok = true;
      if (u.count > 0) {
        mbar_arrive_expect_tx(&t.k_full_bar, kTiles * L::T::kSlotBytes);
#pragma unroll
        for (int i = 0; i < kTiles; ++i) {
#pragma unroll
          for (int a = 0; a < L::kQAtoms; ++a) {
            tma_load_4d(smem + L::kKeysOff + i * L::T::kSlotBytes + a * kBlockKv * kAtomBytes, &tmap_k, &t.k_full_bar, a * kAtomBytes,
                        u.key0 + i * kBlockKv, u.head, u.seq);
          }
        }
      }
      for (int b = 0; b < u.count && ok; ++b) {
        const int st = b % S;
        if (!mbar_wait(&t.slot_empty_bar[st], ((b / S) & 1) ^ 1, &abort_flag)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(&t.slot_full_bar[st], static_cast<uint32_t>(p.tile_rows) * D * 2 + kNormBytes);
#pragma unroll
        for (int a = 0; a < L::kQAtoms; ++a) {
          tma_load_4d(smem + L::kQueriesOff + st * L::kQBytes + a * kBlockQ * kAtomBytes, &tmap_q, &t.slot_full_bar[st], a * kAtomBytes, u.head * p.group,
                      (u.first + b) * p.positions, u.seq);
        }
        bulk_load_1d(smem + L::kNormsOff + st * kNormBytes, p.row_norm + static_cast<int64_t>(u.run) * p.norm_pitch + (u.first + b) * kBlockQ,
                     kNormBytes, &t.slot_full_bar[st]);
      }
      if (!ok) {
        abort_flag = 1;
        atomicCAS(p.status, 0u, kStatusAttentionTimeout);
      }
    }
  } else {
    // ------------------------------------------------------------------ MMA issuer
    const bool issuer = elect_one();
    const uint32_t keys = smem_u32(smem + L::kKeysOff);
    const TileMmas<D> mma[2] = {{p.is_bf16, true, tmem_base, keys, issuer}, {p.is_bf16, true, tmem_base + kTiles * L::kSCols, keys, issuer}};
    const uint64_t qdesc0 = umma_desc_sw128(smem_u32(smem + L::kQueriesOff));
    bool ok = u.count == 0 || mbar_wait(&t.k_full_bar, 0, &abort_flag);
    int met[kTiles] = {0, 0};
    for (int b = 0; b < u.count && ok; ++b) {
      const int st = b % S;
      ok = mbar_wait(&t.slot_full_bar[st], (b / S) & 1, &abort_flag);
      const uint64_t qd = qdesc0 + static_cast<uint64_t>(st * (L::kQBytes >> 4));
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        if (!ok || !u.meets(p, b, i)) continue;
        ok = mbar_wait(&t.s_empty_bar[i][met[i] & 1], ((met[i] >> 1) & 1) ^ 1, &abort_flag);
        if (!ok) continue;
        tc_fence_after_sync();
        if (met[i] & 1) {
          mma[1].scores(i, qd);
        } else {
          mma[0].scores(i, qd);
        }
        if (issuer) umma_commit(&t.s_full_bar[i][met[i] & 1]);
        ++met[i];
      }
      if (ok && issuer) umma_commit(&t.slot_empty_bar[st]);
    }
    if (!ok && issuer) {
      abort_flag = 1;
      atomicCAS(p.status, 0u, kStatusAttentionTimeout);
    }
  }

  // ---------------------------------------------------------------------- teardown
  tc_fence_before_sync();
  __syncthreads();
  if (abort_flag != 0) {
    for (int i = 0; i < 64; ++i) __nanosleep(2000);
    __syncthreads();
  }
  if (warp == kMmaWarp) {
    tc_fence_after_sync();
    tmem_dealloc<1>(tmem_base, L::kTmemCols);
  }
}

template <int D>
cudaError_t launch(const CUtensorMap &tq, const CUtensorMap &tk, const WeightsParams &p, int64_t ctas, cudaStream_t stream) {
  using L = Layout<D>;
  auto kernel = cache_weights_kernel<D>;
  static const cudaError_t attr_set = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmemBytes);
  if (attr_set != cudaSuccess) return attr_set;
  return launch_overlapped(kernel, ctas, kThreads, L::kSmemBytes, stream, tq, tk, p);
}

}  // namespace

int cache_weights_norm_pitch(int rows, int tile_rows) { return (rows + kTiles * tile_rows - 1) / (kTiles * tile_rows) * kTiles * kBlockQ; }

WeightsPlan cache_weights_plan(const CacheAttentionArgs &a, int tile_rows, int most_units) {
  WeightsPlan plan;
  const int64_t runs = static_cast<int64_t>(a.batch) * a.kv_heads;
  plan.pairs = (a.kv_len + kKeysPerCta - 1) / kKeysPerCta;
  const int positions = tile_rows / (a.heads / a.kv_heads);  // of a block
  const int64_t longest = (a.q_len + positions - 1) / positions;  // blocks of the first keys' walk
  plan.part_blocks = static_cast<int>(longest);
  if (runs * plan.pairs <= most_units) {
    // The shortest parts (eight blocks at least) of which there are no more than SMs, for sequences that fill the cache: one
    // round of CTAs (2 x 4 runs of 2048 keys, four heads and 2048 queries each: parts of 14 blocks in three rounds 53 us, of 20 in one 37).
    auto parts_of = [&](int64_t part) {
      int64_t sum = 0;
      for (int pair = 0; pair < plan.pairs; ++pair) {
        const int64_t first = std::max<int64_t>(0, static_cast<int64_t>(pair) * kKeysPerCta - (a.kv_len - a.q_len)) / positions;
        sum += (std::max<int64_t>(0, longest - first) + part - 1) / part;
      }
      return sum * runs;
    };
    int64_t low = std::min<int64_t>(8, longest), high = longest;
    while (low < high) {
      const int64_t middle = (low + high) / 2;
      if (parts_of(middle) <= sm_count()) {
        high = middle;
      } else {
        low = middle + 1;
      }
    }
    plan.part_blocks = static_cast<int>(low);
  }
  plan.parts = static_cast<int>((longest + plan.part_blocks - 1) / plan.part_blocks);
  plan.part_bytes = plan.parts > 1 ? static_cast<size_t>(runs) * plan.pairs * plan.parts * kKeysPerCta * 4 : 0;
  plan.ctas = runs * plan.pairs * plan.parts;
  return plan;
}

cudaError_t cache_weights(const WeightsParams &p, const CacheAttentionArgs &a, const char **why) {
  CUtensorMap tq, tk;
  const uint64_t dims[4] = {static_cast<uint64_t>(a.head_dim) * 2, static_cast<uint64_t>(a.heads), static_cast<uint64_t>(a.q_len),
                            static_cast<uint64_t>(a.batch)};
  auto bytes = [&](int64_t s, int extent) { return static_cast<uint64_t>(extent > 1 ? s : a.head_dim) * 2; };
  const uint64_t strides[3] = {bytes(a.q_stride[1], a.heads), bytes(a.q_stride[2], a.q_len), bytes(a.q_stride[0], a.batch)};
  const uint32_t box[3] = {static_cast<uint32_t>(p.group), static_cast<uint32_t>(p.positions), 1};
  if (!make_tmap(&tq, a.q, 4, dims, strides, box) ||
      !row_map(&tk, a.k, a.head_dim, a.kv_len, a.kv_heads, a.batch, a.k_stride[0], a.k_stride[1], a.k_stride[2], kBlockKv)) {
    *why = "cuTensorMapEncodeTiled refused q or k";
    return cudaErrorInvalidValue;
  }
  *why = "launching the keys' weights";
  const int64_t ctas = static_cast<int64_t>(p.runs) * p.pairs * p.parts;
  return a.head_dim == 64 ? launch<64>(tq, tk, p, ctas, a.stream) : launch<128>(tq, tk, p, ctas, a.stream);
}

}  // namespace flsm100
