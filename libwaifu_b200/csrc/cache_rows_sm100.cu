// Attention over a key-value cache for few query rows (single tokens): the keys of a sequence are split over
// the GPU, and a key's row is read once for all the query heads that share it.
//
// The rows of one key-value head, its group of query heads times the queries, are packed into tiles of 16, the M
// of mma.sync m16n8k16. A unit is such a tile with its keys; its keys are divided over `splits` CTAs of four
// warps, and a warp walks 16 keys at a time on its own: its own ring of shared-memory stages filled by 16-byte
// asynchronous copies (a key's address is computed by itself, so sinks, window and any strides need no tile of
// their own), its own running maximum, sum and output. No barrier stands in the loop. The four meet in
// shared memory at the end, the CTAs of a unit in the workspace, where the last one to arrive adds the parts in
// the order of the splits: the result does not depend on which came last.
//
// What bounds it is the keys' way from HBM: 2 head_dim bytes twice per key, against 16 x head_dim x 4 operations.
#include "cache_attention_sm100.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "cache_common_sm100.cuh"
#include "cache_tiles_sm100.cuh"
#include "cache_weights_sm100.cuh"
#include "ptx_sm100.cuh"

namespace flsm100 {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kTileKeys = 16;  // keys a warp takes at a time
constexpr int kStages = 3;
constexpr int kStepKeys = kWarps * kTileKeys;
constexpr int kRows = kFewRowsTile;

template <int D>
struct RowsLayout {
  static constexpr int kRowBytes = D * 2;
  static constexpr int kTileBytes = kTileKeys * kRowBytes;
  static constexpr int kStageBytes = 2 * kTileBytes;  // K and V of 16 keys
  static constexpr int kQOff = 0;
  static constexpr int kRingOff = kRows * kRowBytes;
  static constexpr int kSmemBytes = kRingOff + kWarps * kStages * kStageBytes;
  static_assert(kWarps * kRows * D * 4 <= kWarps * kStages * kStageBytes, "the warps' outputs fit the ring");
  static_assert(2 * (kSmemBytes + 2048) <= 227 * 1024, "two CTAs an SM");
};

// Where 16-byte piece c of row r lies in a tile: eight rows of one piece fall into different banks.
template <int D>
__device__ __forceinline__ int piece_offset(int r, int c) {
  return r * (D * 2) + ((c ^ (r & 7)) << 4);
}

__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}

template <bool BF16>
__device__ __forceinline__ void mma_16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  if constexpr (BF16) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  } else {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}

template <int N>
__device__ __forceinline__ void cp_async_wait_group() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

struct RowsParams {
  const uint16_t *q, *k, *v;
  uint16_t *out;
  int64_t q_stride[3], k_stride[3], v_stride[3], out_stride[3];
  const int32_t *kv_lens;
  int kv_heads, group, q_len, kv_len;
  int window, sinks;
  float scale_log2;
  // Rows of the whole batch over keys that all of them see (a shared prefix): parts only.
  bool over_batch;
  int rows;       // packed rows of a key-value head: group * q_len, times the batch over a prefix
  int row_tiles;  // of 16
  int splits;
  float *part_out;   // (unit, split, 16, D), or (kv_head, split, rows, D) over a prefix
  float2 *part_sum;  // the same without D: maximum in log2 units, sum
  uint32_t *counters;
  // The parts over the prefix that an earlier kernel left, as above; 0 splits without.
  const float *prefix_out;
  const float2 *prefix_sum;
  int prefix_splits, prefix_rows;
  // For the keys' weights: the scores (batch * kv_heads, rows, kv_len) in log2 units and each row's maximum and 1 / sum.
  float *scores;
  float2 *row_norm;
};

template <int D, bool BF16>
__global__ void __launch_bounds__(kThreads, 2) few_rows_kernel(const RowsParams p) {
  using L = RowsLayout<D>;
  constexpr int kPieces = D / 8;       // of a row
  constexpr int kColTiles = D / 8;     // of the output, eight columns each
  constexpr int kMyCols = D / 8;       // columns a thread finishes: eight threads a row
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float2 warp_sum[kWarps][kRows];
  __shared__ int is_last;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int at = blockIdx.x;
  const int tile = at % p.row_tiles;
  at /= p.row_tiles;
  const int split = at % p.splits;
  at /= p.splits;  // the run: (sequence, key-value head), or the head alone over a prefix
  const int run = at;
  const int head = at % p.kv_heads, seq = at / p.kv_heads;
  const int row0 = tile * kRows;
  const int live = min(kRows, p.rows - row0);

  griddep_launch_dependents();

  KeyRange range;
  int len = p.kv_len, first_pos = 0, last_pos = 0;
  if (p.over_batch) {
    range = KeyRange{0, 0, p.kv_len};
  } else {
    len = sequence_length(p.kv_lens, seq, p.kv_len);
    first_pos = row0 / p.group + len - p.q_len;
    last_pos = (row0 + live - 1) / p.group + len - p.q_len;
    range = visible_keys(first_pos, last_pos, len, p.window, p.sinks);
  }
  const int total = range.count();
  const int steps = (total + kStepKeys - 1) / kStepKeys;
  const int per_split = max(1, (steps + p.splits - 1) / p.splits);
  const int active = max(1, (steps + per_split - 1) / per_split);  // splits that have keys (one where there are none)
  if (split >= active) return;
  const int tile_begin = split * per_split * kWarps;
  const int tile_end = min((split + 1) * per_split * kWarps, (total + kTileKeys - 1) / kTileKeys);

  const uint16_t *k_base = p.k + head * p.k_stride[1] + (p.over_batch ? 0 : seq * p.k_stride[0]);
  const uint16_t *v_base = p.v + head * p.v_stride[1] + (p.over_batch ? 0 : seq * p.v_stride[0]);
  uint8_t *ring = smem + L::kRingOff + warp * kStages * L::kStageBytes;

  auto load_tile = [&](int t, int stage) {
    uint8_t *dst = ring + stage * L::kStageBytes;
    constexpr int kRowsAtOnce = 32 / kPieces;
    const int c = lane % kPieces;
#pragma unroll
    for (int i = 0; i < kTileKeys / kRowsAtOnce; ++i) {
      const int r = i * kRowsAtOnce + lane / kPieces;
      const int at = t * kTileKeys + r;
      const bool there = at < total;
      const int64_t key = there ? range.key(at) : 0;
      const int off = piece_offset<D>(r, c);
      cp_async_16(dst + off, k_base + key * p.k_stride[2] + c * 8, there ? 16 : 0);
      cp_async_16(dst + L::kTileBytes + off, v_base + key * p.v_stride[2] + c * 8, there ? 16 : 0);
    }
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    const int t = tile_begin + warp + s * kWarps;
    if (t < tile_end) load_tile(t, s);
    asm volatile("cp.async.commit_group;" ::: "memory");
  }

  // The queries: eight threads a row, then each warp's A operand.
  {
    const int r = threadIdx.x >> 3;
    const uint16_t *src = nullptr;
    if (r < live) {
      int n = seq, in_seq = row0 + r;
      if (p.over_batch) {
        n = in_seq / (p.group * p.q_len);
        in_seq -= n * p.group * p.q_len;
      }
      const int i = in_seq / p.group, g = in_seq - i * p.group;
      src = p.q + n * p.q_stride[0] + static_cast<int64_t>(head * p.group + g) * p.q_stride[1] + i * p.q_stride[2];
    }
#pragma unroll
    for (int c = threadIdx.x & 7; c < kPieces; c += 8) {
      *reinterpret_cast<uint4 *>(smem + L::kQOff + piece_offset<D>(r, c)) =
          src ? *reinterpret_cast<const uint4 *>(src + c * 8) : make_uint4(0, 0, 0, 0);
    }
  }
  __syncthreads();
  uint32_t qf[D / 16][4];
#pragma unroll
  for (int s = 0; s < D / 16; ++s) {
    ldmatrix_x4(qf[s], smem_u32(smem + L::kQOff + piece_offset<D>(lane & 15, 2 * s + (lane >> 4))));
  }

  // This thread's two rows of the tile (fragment rows lane / 4 and + 8), and where they sit.
  const int my_row = lane >> 2;
  const int pos0 = (row0 + my_row) / p.group + len - p.q_len, pos1 = (row0 + my_row + 8) / p.group + len - p.q_len;
  auto sees = [&](int key, int pos) { return p.over_batch || (key <= pos && (key > pos - p.window || key < p.sinks)); };

  float o[kColTiles][4] = {};
  float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.0f, l1 = 0.0f;
  int stage = 0;
  for (int t = tile_begin + warp; t < tile_end; t += kWarps) {
    cp_async_wait_group<kStages - 2>();
    __syncwarp();
    {
      const int ahead = t + (kStages - 1) * kWarps;
      if (ahead < tile_end) load_tile(ahead, stage == 0 ? kStages - 1 : stage - 1);
      asm volatile("cp.async.commit_group;" ::: "memory");
    }
    uint8_t *k_tile = ring + stage * L::kStageBytes;
    uint8_t *v_tile = k_tile + L::kTileBytes;
    stage = stage + 1 == kStages ? 0 : stage + 1;

    float sc[2][4] = {};  // keys 0 .. 7 and 8 .. 15 of the tile: (row, key), (row, key + 1), (row + 8, key), ...
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      uint32_t b[4];
      ldmatrix_x4(b, smem_u32(k_tile + piece_offset<D>((lane & 7) + ((lane >> 4) << 3), 2 * s + ((lane >> 3) & 1))));
      mma_16<BF16>(sc[0], qf[s], b[0], b[1]);
      mma_16<BF16>(sc[1], qf[s], b[2], b[3]);
    }
    const int at0 = t * kTileKeys;
    const int key_lo = range.key(at0), key_hi = range.key(min(at0 + kTileKeys, total) - 1);
    // Does some row not see some key here? (The keys between key_lo and key_hi may jump from the sinks to the window.)
    const bool differ = !p.over_batch && (key_hi > first_pos || (key_hi >= p.sinks && key_lo <= last_pos - p.window));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[h][i] *= p.scale_log2;
    }
    if (differ || at0 + kTileKeys > total) {
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int at = at0 + h * 8 + (lane & 3) * 2 + (i & 1);
          if (at >= total || !sees(range.key(at), i < 2 ? pos0 : pos1)) sc[h][i] = -INFINITY;
        }
      }
    }
    if (p.scores != nullptr) {  // (no window there: a key's place is the key)
      float *dst = p.scores + (static_cast<int64_t>(run) * p.rows + row0 + my_row) * p.kv_len;
#pragma unroll
      for (int h = 0; h < 2; ++h) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int key = at0 + h * 8 + (lane & 3) * 2 + (i & 1);
          if (key < total && my_row + (i < 2 ? 0 : 8) < live) dst[(i < 2 ? 0 : 8) * static_cast<int64_t>(p.kv_len) + key] = sc[h][i];
        }
      }
    }
    float b0 = fmaxf(fmaxf(sc[0][0], sc[0][1]), fmaxf(sc[1][0], sc[1][1]));
    float b1 = fmaxf(fmaxf(sc[0][2], sc[0][3]), fmaxf(sc[1][2], sc[1][3]));
#pragma unroll
    for (int x = 1; x <= 2; x <<= 1) {
      b0 = fmaxf(b0, __shfl_xor_sync(0xffffffffu, b0, x));
      b1 = fmaxf(b1, __shfl_xor_sync(0xffffffffu, b1, x));
    }
    // The output and the sum are relative to a maximum that follows the rows' own only when one has grown by more
    // than 2^8: until then the exponentials stay below what every type here holds.
    if (__any_sync(0xffffffffu, b0 > m0 + 8.0f || b1 > m1 + 8.0f)) {
      const float n0 = fmaxf(m0, b0), n1 = fmaxf(m1, b1);
      const float f0 = n0 == -INFINITY ? 1.0f : exp2f(m0 - n0), f1 = n1 == -INFINITY ? 1.0f : exp2f(m1 - n1);
      l0 *= f0;
      l1 *= f1;
#pragma unroll
      for (int c = 0; c < kColTiles; ++c) {
        o[c][0] *= f0;
        o[c][1] *= f0;
        o[c][2] *= f1;
        o[c][3] *= f1;
      }
      m0 = n0;
      m1 = n1;
    }
    const float s0 = m0 == -INFINITY ? 0.0f : m0, s1 = m1 == -INFINITY ? 0.0f : m1;
    // The probabilities enter the second product as two 16-bit values each, the rounded one and what it lost: the
    // product is not what bounds the walk (see above), and the result keeps the precision of its own rounding.
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[h][i] = exp2f(sc[h][i] - (i < 2 ? s0 : s1));
      l0 += sc[h][0] + sc[h][1];
      l1 += sc[h][2] + sc[h][3];
#pragma unroll
      for (int i = 0; i < 2; ++i) split_pair<BF16>(sc[h][2 * i], sc[h][2 * i + 1], &hi[2 * h + i], &lo[2 * h + i]);
    }
    // Infinities and NaN in the values of a key that one row sees and another does not: zero times such a value is
    // not zero, so they leave the tile, and the rows that see them get their products by hand.
    if (differ) {
      bool odd = false;
#pragma unroll
      for (int i = 0; i < L::kTileBytes / 512; ++i) {
        odd |= has_nonfinite<BF16>(*reinterpret_cast<const uint4 *>(v_tile + (i * 32 + lane) * 16));
      }
      if (__any_sync(0xffffffffu, odd)) {
        for (int kk = 0; kk < kTileKeys; ++kk) {
          const int from = (lane & ~3) | ((kk & 7) >> 1);
          const float e0 = __shfl_sync(0xffffffffu, kk < 8 ? ((kk & 1) ? sc[0][1] : sc[0][0]) : ((kk & 1) ? sc[1][1] : sc[1][0]), from);
          const float e1 = __shfl_sync(0xffffffffu, kk < 8 ? ((kk & 1) ? sc[0][3] : sc[0][2]) : ((kk & 1) ? sc[1][3] : sc[1][2]), from);
          const int key = at0 + kk < total ? range.key(at0 + kk) : 0;
          const bool see0 = at0 + kk < total && sees(key, pos0), see1 = at0 + kk < total && sees(key, pos1);
#pragma unroll
          for (int c = 0; c < kColTiles; ++c) {
            const uint32_t w = *reinterpret_cast<const uint32_t *>(v_tile + piece_offset<D>(kk, c) + (lane & 3) * 4);
            const float2 x = widen_pair<BF16>(w);
            const bool odd0 = !(fabsf(x.x) < INFINITY), odd1 = !(fabsf(x.y) < INFINITY);
            if (odd0 && see0) o[c][0] += e0 * x.x;
            if (odd1 && see0) o[c][1] += e0 * x.y;
            if (odd0 && see1) o[c][2] += e1 * x.x;
            if (odd1 && see1) o[c][3] += e1 * x.y;
          }
        }
        __syncwarp();
#pragma unroll 1
        for (int i = 0; i < L::kTileBytes / 512; ++i) {
          uint4 *w = reinterpret_cast<uint4 *>(v_tile + (i * 32 + lane) * 16);
          *w = without_nonfinite<BF16>(*w);
        }
        __syncwarp();
      }
    }
#pragma unroll
    for (int c = 0; c < kColTiles; c += 2) {
      uint32_t b[4];
      ldmatrix_x4_trans(b, smem_u32(v_tile + piece_offset<D>(lane & 15, c + (lane >> 4))));
      mma_16<BF16>(o[c], hi, b[0], b[1]);
      mma_16<BF16>(o[c + 1], hi, b[2], b[3]);
      mma_16<BF16>(o[c], lo, b[0], b[1]);
      mma_16<BF16>(o[c + 1], lo, b[2], b[3]);
    }
  }

  // The four warps' outputs meet over the ring.
  cp_async_wait_all();
  __syncthreads();
#pragma unroll
  for (int x = 1; x <= 2; x <<= 1) {
    l0 += __shfl_xor_sync(0xffffffffu, l0, x);
    l1 += __shfl_xor_sync(0xffffffffu, l1, x);
  }
  if ((lane & 3) == 0) {
    warp_sum[warp][my_row] = make_float2(m0, l0);
    warp_sum[warp][my_row + 8] = make_float2(m1, l1);
  }
  float *warp_out = reinterpret_cast<float *>(smem + L::kRingOff);
#pragma unroll
  for (int c = 0; c < kColTiles; ++c) {
    float *dst = warp_out + (warp * kRows + my_row) * D + c * 8 + (lane & 3) * 2;
    *reinterpret_cast<float2 *>(dst) = make_float2(o[c][0], o[c][1]);
    *reinterpret_cast<float2 *>(dst + 8 * D) = make_float2(o[c][2], o[c][3]);
  }
  __syncthreads();

  const int r = threadIdx.x >> 3, col = (threadIdx.x & 7) * kMyCols;
  RowSum<kMyCols> sum;
  sum.clear();
#pragma unroll
  for (int w = 0; w < kWarps; ++w) sum.raise(warp_sum[w][r].x);
#pragma unroll
  for (int w = 0; w < kWarps; ++w) sum.add(warp_sum[w][r], warp_out + (w * kRows + r) * D + col);

  if (p.over_batch) {
    if (r < live) {
      const int64_t part = (static_cast<int64_t>(head) * p.splits + split) * p.rows + row0 + r;
      sum.store(p.part_out + part * D + col);
      if ((threadIdx.x & 7) == 0) p.part_sum[part] = sum.max_and_sum();
    }
    return;
  }
  if (active > 1) {
    const int64_t unit = static_cast<int64_t>(run) * p.row_tiles + tile;
    const int64_t part = (unit * p.splits + split) * kRows + r;
    if (r < live) {
      sum.store(p.part_out + part * D + col);
      if ((threadIdx.x & 7) == 0) p.part_sum[part] = sum.max_and_sum();
    }
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
      const uint32_t before = atomicAdd(&p.counters[unit], 1u);
      is_last = before + 1 == static_cast<uint32_t>(active);
      if (is_last) p.counters[unit] = 0;
    }
    __syncthreads();
    if (!is_last) return;
    __threadfence();
    if (r < live) {
      sum.clear();
      const int64_t first = unit * p.splits * kRows + r;
      for (int s = 0; s < active; ++s) sum.raise(__ldcg(&p.part_sum[first + s * kRows]).x);
#pragma unroll 4
      for (int s = 0; s < active; ++s) sum.add_parts(__ldcg(&p.part_sum[first + s * kRows]), p.part_out + (first + s * kRows) * D + col);
    }
  }
  if (p.prefix_splits > 0) {
    griddep_wait();  // the parts over the prefix
    if (r < live) {
      const int64_t first = static_cast<int64_t>(head) * p.prefix_splits * p.prefix_rows + static_cast<int64_t>(seq) * p.rows + row0 + r;
      for (int s = 0; s < p.prefix_splits; ++s) sum.raise(__ldcg(&p.prefix_sum[first + static_cast<int64_t>(s) * p.prefix_rows]).x);
#pragma unroll 4
      for (int s = 0; s < p.prefix_splits; ++s) {
        const int64_t part = first + static_cast<int64_t>(s) * p.prefix_rows;
        sum.add_parts(__ldcg(&p.prefix_sum[part]), p.prefix_out + part * D + col);
      }
    }
  }
  if (r >= live) return;
  const int i = (row0 + r) / p.group, g = (row0 + r) - i * p.group;
  // A query that sees no key: zeros. (Where it sees some and their exponentials sum to zero or to NaN, that is its result.)
  const bool empty = p.prefix_splits == 0 && i + len - p.q_len < 0;
  const float inv = empty ? 0.0f : 1.0f / sum.l;
  uint16_t *dst = p.out + seq * p.out_stride[0] + static_cast<int64_t>(head * p.group + g) * p.out_stride[1] + i * p.out_stride[2] + col;
#pragma unroll
  for (int c = 0; c < kMyCols; c += 8) {
    uint4 w;
    w.x = pack_pair<BF16>(sum.o[c] * inv, sum.o[c + 1] * inv);
    w.y = pack_pair<BF16>(sum.o[c + 2] * inv, sum.o[c + 3] * inv);
    w.z = pack_pair<BF16>(sum.o[c + 4] * inv, sum.o[c + 5] * inv);
    w.w = pack_pair<BF16>(sum.o[c + 6] * inv, sum.o[c + 7] * inv);
    *reinterpret_cast<uint4 *>(dst + c) = empty ? make_uint4(0, 0, 0, 0) : w;
  }
  if (p.row_norm != nullptr && (threadIdx.x & 7) == 0) {
    p.row_norm[static_cast<int64_t>(run) * p.rows + row0 + r] = make_float2(sum.m, inv);
  }
}

// weights_out = weights_in + the sum over the rows of a key-value head of exp2(score - maximum) / sum.
__global__ void __launch_bounds__(256) add_weights_kernel(const float *__restrict__ scores, const float2 *__restrict__ row_norm, int rows,
                                                          int group, int q_len, int kv_len, int kv_heads, const int32_t *kv_lens,
                                                          const float *weights_in, int64_t in_seq, int64_t in_head, float *weights_out,
                                                          int64_t out_seq, int64_t out_head) {
  griddep_wait();
  const int chunks = (kv_len + 255) / 256;
  const int run = blockIdx.x / chunks, seq = run / kv_heads, head = run % kv_heads;
  const int key = (blockIdx.x % chunks) * 256 + threadIdx.x;
  if (key >= kv_len) return;
  const int len = sequence_length(kv_lens, seq, kv_len);
  float sum = 0.0f;
  if (key < len) {
    // The first query at or behind the key's own position.
    const int first = max(0, key - len + q_len) * group;
    for (int r = first; r < rows; ++r) {
      const float2 norm = row_norm[static_cast<int64_t>(run) * rows + r];
      sum += exp2f(scores[(static_cast<int64_t>(run) * rows + r) * kv_len + key] - norm.x) * norm.y;
    }
  }
  weights_out[seq * out_seq + head * out_head + key] = weights_in[seq * in_seq + head * in_head + key] + sum;
}

// How many CTAs divide a unit's keys: enough for about four waves of two CTAs an SM, so that sequences of different
// lengths even out, but no fewer than 256 keys each.
int splits_for(int64_t units, int keys) {
  const int64_t wanted = units > 0 ? (8ll * sm_count() + units - 1) / units : 1;
  const int most = keys / 256;
  return static_cast<int>(wanted < 1 || most < 1 ? 1 : (wanted < most ? wanted : most));
}

size_t round_256(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

// From so many packed rows of a key-value head on a run takes the tiles of the tensor cores: up to there the tiles of 16
// rows read the keys again from L2 at most three times.
constexpr int kTilesFromRows = 64;

// Which kernels a call takes, and its workspace.
struct CachePlan {
  int rows;         // packed rows of a run
  bool tiles;       // the sequences' own keys (and a prefix before them in the same walk) on the tile kernel
  int row_tiles;    // of 16, or pairs of 128
  int splits;
  bool prefix_apart;  // a kernel of its own over the prefix for the rows of the whole batch
  bool prefix_tiles;
  int prefix_rows, prefix_row_tiles, prefix_splits;
  WeightsPlan weights;  // with `tiles`
  size_t part_out, part_sum, prefix_out, prefix_sum, scores, row_norm, bytes;  // (scores: or the sums of their parts)
};

CachePlan cache_plan(const CacheAttentionArgs &a) {
  CachePlan p = {};
  const int group = a.heads / a.kv_heads;
  const int64_t d = a.head_dim;
  p.rows = group * a.q_len;
  p.tiles = p.rows >= kTilesFromRows;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t off = at;
    at += round_256(bytes);
    return off;
  };
  int64_t most = a.kv_len;  // keys that the rows of a tile see between them
  if (static_cast<int64_t>(a.window) + a.sinks + a.q_len < most) most = static_cast<int64_t>(a.window) + a.sinks + a.q_len;
  const int64_t runs = static_cast<int64_t>(a.batch) * a.kv_heads;
  size_t part_rows = 0;
  if (p.tiles) {
    p.row_tiles = cache_tiles_pairs(p.rows);
    p.splits = cache_tiles_splits(runs * p.row_tiles, static_cast<int>(std::min<int64_t>(most + a.prefix_len, INT32_MAX)), kCacheCounters);
    part_rows = p.splits > 1 ? cache_tiles_part_rows(runs * p.row_tiles, p.splits) : 0;
  } else {
    p.row_tiles = (p.rows + kRows - 1) / kRows;
    const int64_t units = runs * p.row_tiles;
    p.splits = units <= kCacheCounters ? splits_for(units, static_cast<int>(most)) : 1;
    part_rows = p.splits > 1 ? static_cast<size_t>(units) * p.splits * kRows : 0;
  }
  if (part_rows > 0) {
    p.part_out = take(part_rows * d * 4);
    p.part_sum = take(part_rows * 8);
  }
  if (a.prefix_len > 0 && !p.tiles) {
    p.prefix_apart = true;
    p.prefix_rows = a.batch * p.rows;
    p.prefix_tiles = p.prefix_rows >= kTilesFromRows;
    if (p.prefix_tiles) {
      p.prefix_row_tiles = cache_tiles_pairs(p.prefix_rows);
      p.prefix_splits = cache_tiles_splits(static_cast<int64_t>(a.kv_heads) * p.prefix_row_tiles, a.prefix_len, INT32_MAX);
    } else {
      p.prefix_row_tiles = (p.prefix_rows + kRows - 1) / kRows;
      // (as many as the kernel finds keys for: every part that the merge reads is written)
      const int steps = (a.prefix_len + kStepKeys - 1) / kStepKeys;
      const int wanted = splits_for(static_cast<int64_t>(a.kv_heads) * p.prefix_row_tiles, a.prefix_len);
      const int per_split = (steps + wanted - 1) / wanted;
      p.prefix_splits = (steps + per_split - 1) / per_split;
    }
    p.prefix_out = take(static_cast<size_t>(a.kv_heads) * p.prefix_splits * p.prefix_rows * d * 4);
    p.prefix_sum = take(static_cast<size_t>(a.kv_heads) * p.prefix_splits * p.prefix_rows * 8);
  }
  if (a.weights_out != nullptr && p.tiles) {
    p.weights = cache_weights_plan(a, kCacheCounters);
    p.row_norm = take(static_cast<size_t>(runs) * group * cache_weights_norm_pitch(a.q_len) * 8);
    p.scores = take(p.weights.part_bytes);
  } else if (a.weights_out != nullptr) {
    p.scores = take(static_cast<size_t>(runs) * p.rows * a.kv_len * 4);
    p.row_norm = take(static_cast<size_t>(runs) * p.rows * 8);
  }
  p.bytes = at;
  return p;
}

template <int D, bool BF16>
cudaError_t launch_rows(const RowsParams &p, int64_t ctas, bool dependent, cudaStream_t stream) {
  using L = RowsLayout<D>;
  auto kernel = few_rows_kernel<D, BF16>;
  static const cudaError_t attr_set = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmemBytes);
  if (attr_set != cudaSuccess) return attr_set;
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(ctas), 1, 1);
  cfg.blockDim = dim3(kThreads, 1, 1);
  cfg.dynamicSmemBytes = L::kSmemBytes;
  cfg.stream = stream;
  cudaLaunchAttribute attr;
  attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr.val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = &attr;
  cfg.numAttrs = dependent ? 1 : 0;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

cudaError_t launch_rows(const CacheAttentionArgs &a, const RowsParams &p, int64_t ctas, bool dependent) {
  if (a.head_dim == 64) {
    return a.is_bf16 ? launch_rows<64, true>(p, ctas, dependent, a.stream) : launch_rows<64, false>(p, ctas, dependent, a.stream);
  }
  return a.is_bf16 ? launch_rows<128, true>(p, ctas, dependent, a.stream) : launch_rows<128, false>(p, ctas, dependent, a.stream);
}

}  // namespace

bool cache_attention_supported(const CacheAttentionArgs &a, const char **why) {
  const int64_t most = INT32_MAX;
  if (static_cast<int64_t>(a.batch) * a.heads * a.q_len > most) {
    *why = "more than 2^31 - 1 query rows";
    return false;
  }
  const CachePlan plan = cache_plan(a);
  if (static_cast<int64_t>(a.batch) * a.kv_heads * plan.row_tiles * plan.splits > most || plan.weights.ctas > most ||
      static_cast<int64_t>(a.batch) * a.kv_heads * ((static_cast<int64_t>(a.kv_len) + 255) / 256) > most) {
    *why = "more work than one launch indexes";
    return false;
  }
  return true;
}

size_t cache_attention_workspace_bytes(const CacheAttentionArgs &a) { return cache_plan(a).bytes; }

// The fields that both kernels' parameters have alike.
template <typename Params>
void fill_params(const CacheAttentionArgs &a, Params *p) {
  p->q = static_cast<const uint16_t *>(a.q);
  p->k = static_cast<const uint16_t *>(a.k);
  p->v = static_cast<const uint16_t *>(a.v);
  p->out = static_cast<uint16_t *>(a.out);
  for (int i = 0; i < 3; ++i) {
    p->q_stride[i] = a.q_stride[i];
    p->k_stride[i] = a.k_stride[i];
    p->v_stride[i] = a.v_stride[i];
    p->out_stride[i] = a.out_stride[i];
  }
  p->kv_lens = a.kv_lens;
  p->kv_heads = a.kv_heads;
  p->group = a.heads / a.kv_heads;
  p->q_len = a.q_len;
  p->kv_len = a.kv_len;
  p->window = a.window;
  p->sinks = a.sinks;
  p->scale_log2 = 1.4426950408889634f / sqrtf(static_cast<float>(a.head_dim));
  p->counters = a.counters;
}

cudaError_t cache_attention(const CacheAttentionArgs &a, const char **why, int *launches) {
  *why = "";
  const CachePlan plan = cache_plan(a);
  auto floats = [&](size_t off) { return reinterpret_cast<float *>(a.workspace + off); };
  auto pairs = [&](size_t off) { return reinterpret_cast<float2 *>(a.workspace + off); };
  cudaError_t e;
  TilesParams tiles = {};
  fill_params(a, &tiles);
  tiles.is_bf16 = a.is_bf16;
  tiles.status = a.status;
  tiles.prefix_len = a.prefix_len;
  if (plan.tiles) {
    tiles.runs = a.batch * a.kv_heads;
    tiles.rows = plan.rows;
    tiles.row_pairs = plan.row_tiles;
    tiles.splits = plan.splits;
    tiles.part_out = floats(plan.part_out);
    tiles.part_sum = pairs(plan.part_sum);
    if (a.weights_out != nullptr) {
      tiles.row_norm = pairs(plan.row_norm);
      tiles.norm_pitch = cache_weights_norm_pitch(a.q_len);
    }
    e = cache_tiles(tiles, a, why);
    *launches += e == cudaSuccess;
    if (e != cudaSuccess || a.weights_out == nullptr) return e;
    WeightsParams w = {};
    w.kv_lens = a.kv_lens;
    w.is_bf16 = a.is_bf16;
    w.kv_heads = a.kv_heads;
    w.group = tiles.group;
    w.q_len = a.q_len;
    w.kv_len = a.kv_len;
    w.runs = tiles.runs;
    w.pairs = plan.weights.pairs;
    w.parts = plan.weights.parts;
    w.part_blocks = plan.weights.part_blocks;
    w.scale_log2 = tiles.scale_log2;
    w.row_norm = tiles.row_norm;
    w.norm_pitch = tiles.norm_pitch;
    w.part_sums = floats(plan.scores);
    w.counters = a.counters;
    w.weights_in = a.weights_in;
    w.weights_out = a.weights_out;
    for (int i = 0; i < 2; ++i) {
      w.in_stride[i] = a.weights_in_stride[i];
      w.out_stride[i] = a.weights_out_stride[i];
    }
    w.status = a.status;
    e = cache_weights(w, a, why);
    *launches += e == cudaSuccess;
    return e;
  }

  RowsParams p = {};
  fill_params(a, &p);
  p.rows = plan.rows;
  p.row_tiles = plan.row_tiles;
  p.splits = plan.splits;
  p.part_out = floats(plan.part_out);
  p.part_sum = pairs(plan.part_sum);
  if (a.weights_out != nullptr) {
    p.scores = floats(plan.scores);
    p.row_norm = pairs(plan.row_norm);
  }
  if (plan.prefix_apart) {
    if (plan.prefix_tiles) {
      tiles.over_batch = true;
      tiles.runs = a.kv_heads;
      tiles.rows = plan.prefix_rows;
      tiles.row_pairs = plan.prefix_row_tiles;
      tiles.splits = plan.prefix_splits;
      tiles.part_out = floats(plan.prefix_out);
      tiles.part_sum = pairs(plan.prefix_sum);
      e = cache_tiles(tiles, a, why);
    } else {
      RowsParams s = p;
      s.over_batch = true;
      s.k = static_cast<const uint16_t *>(a.prefix_k);
      s.v = static_cast<const uint16_t *>(a.prefix_v);
      for (int i = 0; i < 2; ++i) {
        s.k_stride[i + 1] = a.prefix_k_stride[i];
        s.v_stride[i + 1] = a.prefix_v_stride[i];
      }
      s.kv_len = a.prefix_len;
      s.rows = plan.prefix_rows;
      s.row_tiles = plan.prefix_row_tiles;
      s.splits = plan.prefix_splits;
      s.part_out = floats(plan.prefix_out);
      s.part_sum = pairs(plan.prefix_sum);
      *why = "launching the prefix's part";
      e = launch_rows(a, s, static_cast<int64_t>(a.kv_heads) * s.row_tiles * s.splits, false);
    }
    if (e != cudaSuccess) return e;
    ++*launches;
    p.prefix_out = floats(plan.prefix_out);
    p.prefix_sum = pairs(plan.prefix_sum);
    p.prefix_splits = plan.prefix_splits;
    p.prefix_rows = plan.prefix_rows;
  }
  e = launch_rows(a, p, static_cast<int64_t>(a.batch) * a.kv_heads * p.row_tiles * p.splits, plan.prefix_apart);
  if (e != cudaSuccess) {
    *why = "launching the few-row kernel";
    return e;
  }
  ++*launches;
  if (a.weights_out != nullptr) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<unsigned>((a.kv_len + 255) / 256) * static_cast<unsigned>(a.batch * a.kv_heads), 1, 1);
    cfg.blockDim = dim3(256, 1, 1);
    cfg.stream = a.stream;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, add_weights_kernel, static_cast<const float *>(p.scores), static_cast<const float2 *>(p.row_norm), p.rows, p.group,
                           a.q_len, a.kv_len, a.kv_heads, a.kv_lens, a.weights_in, a.weights_in_stride[0], a.weights_in_stride[1], a.weights_out,
                           a.weights_out_stride[0], a.weights_out_stride[1]);
    if (e != cudaSuccess) {
      *why = "launching the keys' weights";
      return e;
    }
    ++*launches;
  }
  return cudaSuccess;
}

}  // namespace flsm100
