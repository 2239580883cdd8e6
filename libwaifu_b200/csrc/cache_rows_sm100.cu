// Attention over a key-value cache for few query rows (single tokens): the keys of a sequence are split over
// the GPU, and a key's row is read once for all the query heads that share it.
//
// The rows of one key-value head, its group of query heads times the queries, are packed into tiles of 8 or 16, the N of
// mma.sync m16n8k16, once or twice; the keys of a tile are its M (S^T = K Q^T), and so are the columns of the output
// (O^T = V^T P^T): a decode step has a few rows to a head, and would leave most of an M of 16 empty. A unit is such a tile with the keys its sequence's queries see, in steps of 64. The steps of
// all units, one after the other, are dealt out in equal runs over two CTAs an SM, whatever the sequences'
// lengths: a CTA takes the end of one unit, whole units, the beginning of another. Its four warps walk 16 keys
// of a step each on their own: a ring of shared-memory stages per warp, filled by 16-byte asynchronous copies that run
// on into the next unit (a key's address is computed by itself, so sinks, window and any strides need no tile of
// their own), and a running maximum, sum and output per warp. No barrier stands in the loop. At a unit's end the four
// meet over the stages they have just read; a unit that several CTAs share meets in the workspace, where the last one to
// arrive adds the parts in their order: the result does not depend on which came last.
//
// What bounds it is the keys' way from HBM: 2 head_dim bytes twice per key, against 8 or 16 x head_dim x 4 operations. A warp
// has about 350 cycles of it per 16 keys at head_dim 128, times the eight warps of an SM, for its own instructions.
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
constexpr int kMaxRows = 16;
constexpr int kLeastSteps = 4;  // that are worth a CTA of their own

template <int D>
struct RowsLayout {
  static constexpr int kRowBytes = D * 2;
  static constexpr int kTileBytes = kTileKeys * kRowBytes;
  static constexpr int kStageBytes = 2 * kTileBytes;  // K and V of 16 keys
  static constexpr int kQOff = 0;
  static constexpr int kQBytes = kMaxRows * kRowBytes;
  static constexpr int kRingOff = 2 * kQBytes;  // the queries of the unit that comes, and of the one behind it
  static constexpr int kSmemBytes = kRingOff + kWarps * kStages * kStageBytes;
  static_assert(kMaxRows * D * 4 == kStageBytes, "a warp's outputs fit the stage that it has read");
  static_assert(2 * (kSmemBytes + 2048) <= 227 * 1024, "two CTAs an SM");
};

// Where 16-byte piece c of row r lies in a tile: eight rows of one piece fall into different banks.
template <int D>
__device__ __forceinline__ int piece_offset(int r, int c) {
  return r * (D * 2) + ((c ^ (r & 7)) << 4);
}

// Where column `col` of row r of a warp's output lies, in floats: lanes that hold two rows each apart write to different banks.
template <int D>
__device__ __forceinline__ int out_offset(int r, int col) {
  return r * D + (col ^ ((r & 6) << 2));
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

// An 8 x 8 matrix of 16-bit values, a pair of one row per lane, transposed.
__device__ __forceinline__ uint32_t transpose_8x8(uint32_t x) {
  uint32_t y;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
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
  Divisor by_kv_heads, by_group, by_row_tiles, by_sequence_rows;  // (the last: group * q_len)
  int window, sinks;
  float scale_log2;
  // Rows of the whole batch over keys that all of them see (a shared prefix): parts only.
  bool over_batch;
  int batch;
  int rows;       // packed rows of a key-value head: group * q_len, times the batch over a prefix
  int row_tiles;  // of 8 or 16
  int splits;     // over a prefix: CTAs that divide a unit
  int ctas;       // else: CTAs that the steps are dealt out to
  float *part_out;   // (CTA, 2, rows of a tile, D): a unit's end, and a unit's beginning; (kv_head, split, rows, D) over a prefix
  float2 *part_sum;  // the same without D: maximum in log2 units, sum
  uint32_t *counters;  // of the unit that the CTA's last run of steps begins
  // Behind a prefix's tile kernel, which a third kernel joins with this one: a row's output and sum, (batch * kv_heads, rows, D).
  float *own_out;
  float2 *own_sum;
  // The parts over the prefix that an earlier kernel of few rows left, as above; 0 splits without.
  const float *prefix_out;
  const float2 *prefix_sum;
  int prefix_splits, prefix_rows;
  // For the keys' weights: the scores (batch * kv_heads, rows, score_pitch) in log2 units and each row's maximum and 1 / sum.
  float *scores;
  int64_t score_pitch;
  float2 *row_norm;
};

// Where a CTA's walk over the units' steps stands. Units lie in the order of their sequences, heads and tiles; those of a
// sequence walk the same keys, what its first to its last query sees.
struct Cursor {
  int seq, head, tile, step, steps, len;
  KeyRange range;

  __device__ __forceinline__ void enter_sequence(const RowsParams &p) {
    if (p.over_batch) {
      len = 0;
      range = KeyRange{0, 0, p.kv_len};
    } else {
      len = sequence_length(p.kv_lens, seq, p.kv_len);
      range = visible_keys(len - p.q_len, len - 1, len, p.window, p.sinks);
    }
    steps = max(1, (range.count() + kStepKeys - 1) / kStepKeys);  // (a unit without keys still has its result to write)
  }
  // True where the step begins another unit.
  __device__ __forceinline__ bool advance(const RowsParams &p) {
    if (++step < steps) return false;
    step = 0;
    if (++tile == p.row_tiles) {
      tile = 0;
      if (++head == p.kv_heads) {
        head = 0;
        if (++seq < p.batch) enter_sequence(p);
      }
    }
    return true;
  }
};

template <int D, bool BF16, int NB>
__global__ void __launch_bounds__(kThreads, 2) few_rows_kernel(const __grid_constant__ RowsParams p) {
  using L = RowsLayout<D>;
  constexpr int kRows = NB * 8;
  constexpr int kPieces = D / 8;     // of a row
  constexpr int kColTiles = D / 16;  // of the output, sixteen columns each
  constexpr int kQuads = D / 4;      // of a row: a thread finishes four columns at a time
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float2 warp_sum[kWarps][NB * 8];
  __shared__ int is_last;

  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  // (Behind a prefix's kernel the inputs are complete: only its parts are waited for.)
  if (p.prefix_splits == 0 && p.own_out == nullptr) griddep_wait();
  griddep_launch_dependents();
  if (static_cast<int>(blockIdx.x) == p.ctas) {  // the kernel that joins the two waits for this one: so this one ends behind the prefix's
    griddep_wait();
    return;
  }

  // ---- this CTA's run of steps
  Cursor load;
  int64_t begin, per_cta;
  int count;
  if (p.over_batch) {
    load.seq = 0;
    load.enter_sequence(p);
    int at = blockIdx.x;
    load.tile = p.by_row_tiles.take(&at);
    load.head = p.by_kv_heads.take(&at);
    per_cta = (load.steps + p.splits - 1) / p.splits;
    begin = load.step = at * static_cast<int>(per_cta);
    count = min(static_cast<int>(per_cta), load.steps - load.step);
  } else {
    const int units = p.kv_heads * p.row_tiles;
    // Four steps each at least, or one unit where they are shorter.
    auto deal_out = [&](int64_t total, int most) {
      per_cta = max((total + p.ctas - 1) / p.ctas, static_cast<int64_t>(min(kLeastSteps, most)));
      begin = blockIdx.x * per_cta;
      count = static_cast<int>(max(static_cast<int64_t>(0), min(per_cta, total - begin)));
    };
    int64_t before = 0;
    if (p.kv_lens == nullptr || p.batch == 1) {  // all alike
      load.seq = 0;
      load.enter_sequence(p);
      const int64_t each = static_cast<int64_t>(load.steps) * units;
      deal_out(each * p.batch, load.steps);
      if (count == 0) return;
      load.seq = static_cast<int>(begin / each);
      before = load.seq * each;
    } else {
      // The steps of the whole batch, and then the sequence in which this CTA's begin: every warp for itself, a lane a sequence.
      int64_t total = 0;
      int most = 1;
      for (load.seq = lane; load.seq < p.batch; load.seq += 32) {
        load.enter_sequence(p);
        total += static_cast<int64_t>(load.steps) * units;
        most = max(most, load.steps);
      }
#pragma unroll
      for (int x = 1; x < 32; x <<= 1) {
        total += __shfl_xor_sync(0xffffffffu, total, x);
        most = max(most, __shfl_xor_sync(0xffffffffu, most, x));
      }
      deal_out(total, most);
      if (count == 0) return;
      for (int first = 0;; first += 32) {
        load.seq = first + lane;
        int64_t here = 0;
        if (load.seq < p.batch) {
          load.enter_sequence(p);
          here = static_cast<int64_t>(load.steps) * units;
        }
        int64_t upto = here;
#pragma unroll
        for (int x = 1; x < 32; x <<= 1) {
          const int64_t y = __shfl_up_sync(0xffffffffu, upto, x);
          if (lane >= x) upto += y;
        }
        const uint32_t past = __ballot_sync(0xffffffffu, before + upto > begin);
        if (past != 0) {
          const int at = __ffs(static_cast<int>(past)) - 1;
          before += __shfl_sync(0xffffffffu, upto - here, at);
          load.seq = first + at;
          break;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
      }
    }
    load.enter_sequence(p);
    const int64_t in_seq = begin - before;
    load.head = static_cast<int>(in_seq / load.steps);
    load.step = static_cast<int>(in_seq - static_cast<int64_t>(load.head) * load.steps);
    load.tile = p.by_row_tiles.take(&load.head);
  }
  Cursor at = load;

  // ---- the ring
  uint8_t *ring = smem + L::kRingOff + warp * kStages * L::kStageBytes;
  constexpr int kRowsAtOnce = 32 / kPieces;
  const int lane_row = lane / kPieces, lane_piece = lane % kPieces;
  int loaded = 0, load_stage = 0;
  const uint16_t *k_base, *v_base;  // of the unit that is loaded, and this lane's piece
  auto find_unit = [&]() {
    k_base = p.k + load.head * p.k_stride[1] + (p.over_batch ? 0 : load.seq * p.k_stride[0]) + lane_piece * 8;
    v_base = p.v + load.head * p.v_stride[1] + (p.over_batch ? 0 : load.seq * p.v_stride[0]) + lane_piece * 8;
  };
  find_unit();
  // The queries of the unit that is loaded come with its first tile, eight rows or sixteen by all threads.
  int load_unit = 0;
  auto load_queries = [&]() {
    constexpr int kCopies = kRows * kPieces;
#pragma unroll
    for (int i = 0; i < (kCopies + kThreads - 1) / kThreads; ++i) {
      const int c = i * kThreads + threadIdx.x, in_tile = c / kPieces, piece = c % kPieces;
      if (kCopies % kThreads != 0 && c >= kCopies) break;
      const int r = load.tile * kRows + in_tile;
      int n = load.seq, q = min(r, p.rows - 1);
      if (p.over_batch) {
        n = q;
        q = p.by_sequence_rows.take(&n);
      }
      const int g = p.by_group.take(&q);
      cp_async_16(smem + L::kQOff + (load_unit & 1) * L::kQBytes + piece_offset<D>(in_tile, piece),
                  p.q + n * p.q_stride[0] + static_cast<int64_t>(load.head * p.group + g) * p.q_stride[1] + q * p.q_stride[2] + piece * 8,
                  r < p.rows ? 16 : 0);
    }
    ++load_unit;
  };
  bool load_begins = true;
  auto load_tile = [&]() {
    if (loaded < count) {
      if (load_begins) load_queries();
      load_begins = false;
      uint8_t *dst = ring + load_stage * L::kStageBytes;
      const int at0 = (load.step * kWarps + warp) * kTileKeys, total = load.range.count();
      if (at0 + kTileKeys <= total && (at0 >= load.range.sinks || at0 + kTileKeys <= load.range.sinks)) {  // one run of keys
        const int key = load.range.key(at0) + lane_row;
        const uint16_t *k = k_base + key * p.k_stride[2], *v = v_base + key * p.v_stride[2];
#pragma unroll
        for (int i = 0; i < kTileKeys / kRowsAtOnce; ++i) {
          const int off = piece_offset<D>(i * kRowsAtOnce + lane_row, lane_piece);
          cp_async_16(dst + off, k, 16);
          cp_async_16(dst + L::kTileBytes + off, v, 16);
          k += kRowsAtOnce * p.k_stride[2];
          v += kRowsAtOnce * p.v_stride[2];
        }
      } else {
#pragma unroll 1
        for (int i = 0; i < kTileKeys / kRowsAtOnce; ++i) {
          const int r = i * kRowsAtOnce + lane_row;
          const bool there = at0 + r < total;
          const int64_t key = there ? load.range.key(at0 + r) : 0;
          const int off = piece_offset<D>(r, lane_piece);
          cp_async_16(dst + off, k_base + key * p.k_stride[2], there ? 16 : 0);
          cp_async_16(dst + L::kTileBytes + off, v_base + key * p.v_stride[2], there ? 16 : 0);
        }
      }
      ++loaded;
      load_stage = load_stage + 1 == kStages ? 0 : load_stage + 1;
      if (loaded < count && load.advance(p)) {
        find_unit();
        load_begins = true;
      }
    }
    asm volatile("cp.async.commit_group;" ::: "memory");
  };
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) load_tile();

  // Of the fragments of S^T and O^T this lane has the rows (keys, columns) lane / 4 and + 8, and of every eight query rows
  // the two from my_row on.
  const int my_key = lane >> 2, my_row = (lane & 3) * 2;
  uint32_t qf[D / 16][NB][2];
  float o[kColTiles][NB][4];
  float m[NB][2], l[NB][2];
  int first_pos, last_pos, pos[NB][2];  // of the tile's rows, and of this thread's
  int unit_step;                        // the first step that this CTA takes of the unit
  int begun = 0;
  auto begin_unit = [&]() {
    const uint8_t *queries = smem + L::kQOff + (begun & 1) * L::kQBytes;
    ++begun;
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      if constexpr (NB == 2) {
        uint32_t b[4];
        ldmatrix_x4(b, smem_u32(queries + piece_offset<D>((lane & 7) + ((lane >> 4) << 3), 2 * s + ((lane >> 3) & 1))));
        qf[s][0][0] = b[0], qf[s][0][1] = b[1], qf[s][NB - 1][0] = b[2], qf[s][NB - 1][1] = b[3];
      } else if ((s & 1) == 0) {
        uint32_t b[4];
        ldmatrix_x4(b, smem_u32(queries + piece_offset<D>(lane & 7, 2 * s + (lane >> 3))));
        qf[s][0][0] = b[0], qf[s][0][1] = b[1], qf[s + 1][0][0] = b[2], qf[s + 1][0][1] = b[3];
      }
    }
#pragma unroll
    for (int c = 0; c < kColTiles; ++c) {
#pragma unroll
      for (int n = 0; n < NB; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) o[c][n][i] = 0.0f;
      }
    }
    const int row0 = at.tile * kRows, offset = at.len - p.q_len;
    first_pos = p.by_group.quotient(row0) + offset;
    last_pos = p.by_group.quotient(min(row0 + kRows, p.rows) - 1) + offset;
#pragma unroll
    for (int n = 0; n < NB; ++n) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        m[n][i] = -INFINITY;
        l[n][i] = 0.0f;
        pos[n][i] = p.by_group.quotient(row0 + n * 8 + my_row + i) + offset;
      }
    }
    unit_step = at.step;
  };
  auto sees = [&](int key, int pos) { return p.over_batch || (key <= pos && (key > pos - p.window || key < p.sinks)); };
  cp_async_wait_group<kStages - 2>();
  __syncthreads();  // the first unit's queries are there
  begin_unit();
  __syncthreads();  // ... and have been read: behind two units of one step the third one's come to their place with the next load

  int stage = 0;
  for (int done = 0; done < count; ++done) {
    cp_async_wait_group<kStages - 2>();
    __syncwarp();
    load_tile();
    uint8_t *k_tile = ring + stage * L::kStageBytes;
    uint8_t *v_tile = k_tile + L::kTileBytes;
    stage = stage + 1 == kStages ? 0 : stage + 1;

    const int at0 = (at.step * kWarps + warp) * kTileKeys, total = at.range.count();
    if (at0 < total) {
      float sc[NB][4] = {};  // (key, row), (key, row + 1), (key + 8, row), (key + 8, row + 1)
#pragma unroll
      for (int s = 0; s < D / 16; ++s) {
        uint32_t a[4];
        ldmatrix_x4(a, smem_u32(k_tile + piece_offset<D>(lane & 15, 2 * s + (lane >> 4))));
#pragma unroll
        for (int n = 0; n < NB; ++n) mma_16<BF16>(sc[n], a, qf[s][n][0], qf[s][n][1]);
      }
      const int key_lo = at.range.key(at0), key_hi = at.range.key(min(at0 + kTileKeys, total) - 1);
      // Does some row not see some key here? (The keys between key_lo and key_hi may jump from the sinks to the window.)
      const bool differ = !p.over_batch && (key_hi > first_pos || (key_hi >= p.sinks && key_lo <= last_pos - p.window));
#pragma unroll
      for (int n = 0; n < NB; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[n][i] *= p.scale_log2;
      }
      if (differ || at0 + kTileKeys > total) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const int place = at0 + h * 8 + my_key, key = place < total ? at.range.key(place) : 0;
#pragma unroll
          for (int n = 0; n < NB; ++n) {
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              if (place >= total || !sees(key, pos[n][i])) sc[n][2 * h + i] = -INFINITY;
            }
          }
        }
      }
      if (p.scores != nullptr) {  // (no window there: a key's place is the key)
        const int row0 = at.tile * kRows;
        float *dst = p.scores + ((static_cast<int64_t>(at.seq) * p.kv_heads + at.head) * p.rows + row0) * p.score_pitch + at0 + my_key;
#pragma unroll
        for (int n = 0; n < NB; ++n) {
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = n * 8 + my_row + (i & 1);
            if (at0 + (i >> 1) * 8 + my_key < total && row0 + row < p.rows) dst[row * p.score_pitch + (i >> 1) * 8] = sc[n][i];
          }
        }
      }
      // The output and the sum are relative to a maximum that follows the rows' own only when one has grown by more
      // than 2^8: until then the exponentials stay below what every type here holds (2^15 in half), and no lane has to know another's.
      bool grown = false;
#pragma unroll
      for (int n = 0; n < NB; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) grown |= sc[n][i] > m[n][i & 1] + 8.0f;
      }
      if (__any_sync(0xffffffffu, grown)) {
#pragma unroll
        for (int n = 0; n < NB; ++n) {
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            float top = fmaxf(m[n][i], fmaxf(sc[n][i], sc[n][2 + i]));
#pragma unroll
            for (int x = 4; x <= 16; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
            const float f = top == -INFINITY ? 1.0f : exp2f(m[n][i] - top);
            m[n][i] = top;
            l[n][i] *= f;
#pragma unroll
            for (int c = 0; c < kColTiles; ++c) {
              o[c][n][i] *= f;
              o[c][n][2 + i] *= f;
            }
          }
        }
      }
      // The probabilities enter the second product as two 16-bit values each, the rounded one and what it lost: the
      // product is not what bounds the walk (see above), and the result keeps the precision of its own rounding.
      uint32_t hi[NB][2], lo[NB][2];
#pragma unroll
      for (int n = 0; n < NB; ++n) {
        constexpr float kShift = kProbabilityShift<BF16>;
        const float s0 = m[n][0] == -INFINITY ? 0.0f : m[n][0] - kShift, s1 = m[n][1] == -INFINITY ? 0.0f : m[n][1] - kShift;
#pragma unroll
        for (int i = 0; i < 4; ++i) sc[n][i] = exp2_approx(sc[n][i] - ((i & 1) ? s1 : s0));
        l[n][0] += sc[n][0] + sc[n][2];
        l[n][1] += sc[n][1] + sc[n][3];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          split_pair<BF16>(sc[n][2 * h], sc[n][2 * h + 1], &hi[n][h], &lo[n][h]);
          hi[n][h] = transpose_8x8(hi[n][h]);
          lo[n][h] = transpose_8x8(lo[n][h]);
        }
      }
      // Infinities and NaN in the values leave the tile, and the rows that see them get their products by hand: zero times
      // such a value is not zero, whether the zero is the probability of a key that the row does not see or what rounding
      // left of one that it does, and a negative rest would take an infinity back.
      {
        uint32_t odd = 0;
#pragma unroll
        for (int i = 0; i < L::kTileBytes / 512; ++i) {
          odd = probe_nonfinite<BF16>(*reinterpret_cast<const uint4 *>(v_tile + (i * 32 + lane) * 16), odd);
        }
        if (__any_sync(0xffffffffu, (odd & 0x7FFF7FFFu) != 0)) {
          for (int kk = 0; kk < kTileKeys; ++kk) {
            const int from = ((kk & 7) << 2) | (lane & 3);
            const int key = at0 + kk < total ? at.range.key(at0 + kk) : 0;
#pragma unroll
            for (int n = 0; n < NB; ++n) {
#pragma unroll
              for (int i = 0; i < 2; ++i) {
                const float e = __shfl_sync(0xffffffffu, kk < 8 ? sc[n][i] : sc[n][2 + i], from);
                if (at0 + kk >= total || !sees(key, pos[n][i])) continue;
#pragma unroll
                for (int c = 0; c < 2 * kColTiles; ++c) {
                  const uint16_t w = *reinterpret_cast<const uint16_t *>(v_tile + piece_offset<D>(kk, c) + my_key * 2);
                  const float x = widen_pair<BF16>(w).x;
                  if (!(fabsf(x) < INFINITY)) o[c >> 1][n][(c & 1) * 2 + i] += e * x;
                }
              }
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
      for (int c = 0; c < kColTiles; ++c) {
        uint32_t a[4];  // columns by keys
        ldmatrix_x4_trans(a, smem_u32(v_tile + piece_offset<D>((lane & 7) + ((lane >> 4) << 3), 2 * c + ((lane >> 3) & 1))));
#pragma unroll
        for (int n = 0; n < NB; ++n) {
          mma_16<BF16>(o[c][n], a, hi[n][0], hi[n][1]);
          mma_16<BF16>(o[c][n], a, lo[n][0], lo[n][1]);
        }
      }
    }

    const Cursor unit = at;
    if (done + 1 < count && !at.advance(p)) continue;

    // ---- the end of the unit, or of this CTA's part of it. The four warps' outputs meet over the stages that they
    // have just read, which no load fills before the next step's turn.
#pragma unroll
    for (int n = 0; n < NB; ++n) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int x = 4; x <= 16; x <<= 1) l[n][i] += __shfl_xor_sync(0xffffffffu, l[n][i], x);
        if (lane < 4) warp_sum[warp][n * 8 + my_row + i] = make_float2(m[n][i] - kProbabilityShift<BF16>, l[n][i]);
      }
    }
    __syncwarp();  // (every lane has read its stage)
#pragma unroll
    for (int c = 0; c < kColTiles; ++c) {
#pragma unroll
      for (int n = 0; n < NB; ++n) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int row = n * 8 + my_row + (i & 1);
          reinterpret_cast<float *>(k_tile)[out_offset<D>(row, c * 16 + (i >> 1) * 8 + my_key)] = o[c][n][i];
        }
      }
    }
    cp_async_wait_group<kStages - 2>();  // the next unit's queries, with its first tile
    __syncthreads();

    const int row0 = unit.tile * kRows, live = min(kRows, p.rows - row0);
    // The CTAs that share it: so many runs of steps before this one's, and so many behind.
    const int run = static_cast<int>(per_cta), before = unit.step - done, behind = done + unit.steps - unit.step - run;
    const int here = static_cast<int>(blockIdx.x);
    const int first_cta = before > 0 ? here - (before + run - 1) / run : here, last_cta = behind > 0 ? here + (behind + run - 1) / run : here;
    const bool shared = !p.over_batch && last_cta > first_cta;
    const uint8_t *stages = smem + L::kRingOff + (k_tile - ring);  // the first warp's
    auto own_part = [&](int r, int col, RowSum *sum) {
      sum->clear();
#pragma unroll
      for (int w = 0; w < kWarps; ++w) sum->raise(warp_sum[w][r].x);
#pragma unroll
      for (int w = 0; w < kWarps; ++w) {
        sum->add(warp_sum[w][r], *reinterpret_cast<const float4 *>(reinterpret_cast<const float *>(stages + w * kStages * L::kStageBytes) +
                                                                   out_offset<D>(r, col)));
      }
    };
    if (p.over_batch || shared) {
      const int64_t part = p.over_batch ? (static_cast<int64_t>(unit.head) * p.splits + unit_step / per_cta) * p.rows + row0
                                        : (static_cast<int64_t>(blockIdx.x) * 2 + (unit_step == 0 ? 1 : 0)) * kRows;
      for (int i = threadIdx.x; i < live * kQuads; i += kThreads) {
        const int r = i / kQuads, col = i % kQuads * 4;
        RowSum sum;
        own_part(r, col, &sum);
        *reinterpret_cast<float4 *>(p.part_out + (part + r) * D + col) = sum.o;
        if (col == 0) p.part_sum[part + r] = make_float2(sum.m, sum.l);
      }
    }
    bool finish = !p.over_batch;
    if (shared) {
      __syncthreads();
      if (threadIdx.x == 0) {
        __threadfence();
        const uint32_t before = atomicAdd(&p.counters[first_cta], 1u);
        is_last = before == static_cast<uint32_t>(last_cta - first_cta);
        if (is_last) p.counters[first_cta] = 0;
        __threadfence();
      }
      __syncthreads();
      finish = is_last;
    }
    if (finish) {
      if (p.prefix_splits > 0) griddep_wait();  // the parts over the prefix
      for (int i = threadIdx.x; i < live * kQuads; i += kThreads) {
        const int r = i / kQuads, col = i % kQuads * 4;
        RowSum sum;
        if (shared) {
          sum.clear();
          add_parts<D>(last_cta - first_cta + 1, p.part_sum, p.part_out, col, &sum,
                       [&](int c) { return (static_cast<int64_t>(first_cta + c) * 2 + (c == 0 ? 1 : 0)) * kRows + r; });
        } else {
          own_part(r, col, &sum);
        }
        if (p.prefix_splits > 0) {
          const int64_t first = static_cast<int64_t>(unit.head) * p.prefix_splits * p.prefix_rows + static_cast<int64_t>(unit.seq) * p.rows + row0 + r;
          add_parts<D>(p.prefix_splits, p.prefix_sum, p.prefix_out, col, &sum,
                       [&](int c) { return first + static_cast<int64_t>(c) * p.prefix_rows; });
        }
        if (p.own_out != nullptr) {
          const int64_t row = (static_cast<int64_t>(unit.seq) * p.kv_heads + unit.head) * p.rows + row0 + r;
          *reinterpret_cast<float4 *>(p.own_out + row * D + col) = sum.o;
          if (col == 0) p.own_sum[row] = make_float2(sum.m, sum.l);
          continue;
        }
        int q = row0 + r;
        const int g = p.by_group.take(&q);
        // A query that sees no key: zeros. (Where it sees some and their exponentials sum to zero or to NaN, that is its result.)
        const bool empty = p.prefix_splits == 0 && q + unit.len - p.q_len < 0;
        const float inv = empty ? 0.0f : 1.0f / sum.l;
        const uint2 w = make_uint2(pack_pair<BF16>(sum.o.x * inv, sum.o.y * inv), pack_pair<BF16>(sum.o.z * inv, sum.o.w * inv));
        *reinterpret_cast<uint2 *>(p.out + unit.seq * p.out_stride[0] + static_cast<int64_t>(unit.head * p.group + g) * p.out_stride[1] +
                                   q * p.out_stride[2] + col) = empty ? make_uint2(0, 0) : w;
        if (p.row_norm != nullptr && col == 0) {
          p.row_norm[(static_cast<int64_t>(unit.seq) * p.kv_heads + unit.head) * p.rows + row0 + r] = make_float2(sum.m, inv);
        }
      }
    }
    if (done + 1 < count) {
      begin_unit();
      __syncthreads();  // the stages have been read
    }
  }
}

struct JoinParams {
  const float *own_out, *prefix_out;
  const float2 *own_sum, *prefix_sum;
  uint16_t *out;
  int64_t out_stride[3];
  Divisor by_rows, by_kv_heads, by_group;
  int rows, prefix_rows, prefix_splits, group;
  int64_t total;  // rows of all runs times the fours of a row's columns
};

// A row's own part and its parts over the prefix, in their order: four columns a thread.
template <int D, bool BF16>
__global__ void __launch_bounds__(128) join_prefix_kernel(const __grid_constant__ JoinParams p) {
  griddep_wait();
  griddep_launch_dependents();
  constexpr int kQuads = D / 4;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 128 + threadIdx.x;
  if (at >= p.total) return;
  const int col = static_cast<int>(at % kQuads) * 4;
  const int row = static_cast<int>(at / kQuads);
  int run = row;
  const int r = p.by_rows.take(&run);
  int seq = run;
  const int head = p.by_kv_heads.take(&seq);
  RowSum sum;
  sum.clear();
  const float2 own = __ldcg(&p.own_sum[row]);
  sum.raise(own.x);
  sum.add(own, __ldcg(reinterpret_cast<const float4 *>(p.own_out + static_cast<int64_t>(row) * D + col)));
  const int64_t first = static_cast<int64_t>(head) * p.prefix_splits * p.prefix_rows + static_cast<int64_t>(seq) * p.rows + r;
  add_parts<D>(p.prefix_splits, p.prefix_sum, p.prefix_out, col, &sum, [&](int c) { return first + static_cast<int64_t>(c) * p.prefix_rows; });
  const float inv = sum.m == -INFINITY ? NAN : 1.0f / sum.l;  // (a row whose every score is -inf has no softmax)
  int q = r;
  const int g = p.by_group.take(&q);
  *reinterpret_cast<uint2 *>(p.out + seq * p.out_stride[0] + static_cast<int64_t>(head * p.group + g) * p.out_stride[1] + q * p.out_stride[2] + col) =
      make_uint2(pack_pair<BF16>(sum.o.x * inv, sum.o.y * inv), pack_pair<BF16>(sum.o.z * inv, sum.o.w * inv));
}

constexpr int kKeysAtOnce = 4;  // of a thread
constexpr int kAddThreads = 128;

// weights_out = weights_in + the sum over the rows of a key-value head of exp2(score - maximum) / sum, in the order of the rows.
__global__ void __launch_bounds__(kAddThreads) add_weights_kernel(const float *scores, int64_t score_pitch, const float2 *row_norm, int rows,
                                                                  Divisor by_chunks, Divisor by_kv_heads, int group, int q_len, int kv_len,
                                                                  const int32_t *kv_lens, const float *weights_in, int64_t in_seq,
                                                                  int64_t in_head, float *weights_out, int64_t out_seq, int64_t out_head) {
  int run = blockIdx.x;
  const int key = (by_chunks.take(&run) * kAddThreads + threadIdx.x) * kKeysAtOnce;
  // (The weights up to here and the lengths are complete: the kernel before has waited for what wrote them. They are read past L1.)
  int seq = run;
  const int head = by_kv_heads.take(&seq);
  const float *in = weights_in + seq * in_seq + head * in_head + key;
  float *out = weights_out + seq * out_seq + head * out_head + key;
  float before[kKeysAtOnce], sum[kKeysAtOnce] = {};
#pragma unroll
  for (int k = 0; k < kKeysAtOnce; ++k) before[k] = key + k < kv_len ? __ldcg(in + k) : 0.0f;
  const int len = sequence_length(kv_lens, seq, kv_len);
  griddep_wait();  // the scores, and the rows' maxima and sums
  griddep_launch_dependents();
  if (key < len) {
    // Query i sees the keys up to i + len - q_len; the rows' scores of others were not written.
    const float *score = scores + static_cast<int64_t>(run) * rows * score_pitch + key;
    const int offset = len - q_len, first = max(0, key - offset) * group;
    int query = max(0, key - offset), in_query = 0;
#pragma unroll 4
    for (int r = first; r < rows; ++r) {
      const float2 norm = row_norm[static_cast<int64_t>(run) * rows + r];
      const float4 s = *reinterpret_cast<const float4 *>(score + r * score_pitch);
      const float each[kKeysAtOnce] = {s.x, s.y, s.z, s.w};
#pragma unroll
      for (int k = 0; k < kKeysAtOnce; ++k) {
        if (key + k <= query + offset) sum[k] += exp2f(each[k] - norm.x) * norm.y;
      }
      if (++in_query == group) {
        in_query = 0;
        ++query;
      }
    }
  }
#pragma unroll
  for (int k = 0; k < kKeysAtOnce; ++k) {
    if (key + k < kv_len) out[k] = before[k] + sum[k];
  }
}

constexpr int kCtasPerSm = 2;

// How many CTAs divide a prefix for one of `units` tiles of rows: together two an SM, but no fewer than 256 keys each.
int prefix_splits(int64_t units, int keys) {
  const int64_t wanted = kCtasPerSm * static_cast<int64_t>(sm_count()) / units;
  const int most = keys / 256;
  return static_cast<int>(wanted < 1 || most < 1 ? 1 : (wanted < most ? wanted : most));
}

size_t round_256(size_t x) { return (x + 255) & ~static_cast<size_t>(255); }

// From so many packed rows of a key-value head on a run takes the tensor cores' tiles, as soon as there are two tiles of 16
// rows that would each walk the keys (microseconds, 16-row tiles and tensor cores, 8 x 8 heads over 2000 keys: 20 rows 25.6 and
// 24.3, 36 rows 32.5 and 24.7, 68 rows 46.6 and 25.9; one sequence: 36 rows 16.0 and 14.0).
constexpr int kMostTileHeads = 128;
constexpr int kTilesFromRows = 17;
// With the keys' weights, for which the tensor cores compute the scores a second time and the few-row kernel stores them, from
// so many (32 x 8 heads over 2000 keys: 36 rows 122 and 171 us, 68 rows 197 and 173), or where the scores took over 256 MiB.
constexpr int kWeightTilesFromRows = 64;
constexpr int64_t kMostScores = int64_t{64} << 20;

int64_t score_pitch_of(int kv_len) { return (static_cast<int64_t>(kv_len) + kKeysAtOnce - 1) / kKeysAtOnce * kKeysAtOnce; }

// The blocks of 128 keys of a prefix to a CTA of the tile kernel: it takes some 11 us to begin and to write its parts, and 2.3 us a
// block, while the kernel over the own keys has the other SMs (64 sequences behind 8192 keys: parts of four blocks 60 us, of
// eight 50; of sixteen 72 before the two overlapped).
constexpr int kPrefixBlocks = 8;
// A run's own blocks are divided into parts of so many where there are SMs for them.
constexpr int kOwnBlocks = 4;
// Up to two tiles of 16 rows over less than so many keys of all heads stay with the few-row kernel (24 rows of one head, 257
// keys: 8.6 us, on the tensor cores 12.1, one launch more; 24 rows of eight heads over 5000 keys 26.2 and 20.7).
constexpr int kFewPrefixRows = 32;
constexpr int64_t kFewPrefixKeys = 16384;

bool prefix_on_tiles(const CacheAttentionArgs &a, int rows) {  // of a run; the batch's together over the prefix
  const int64_t together = static_cast<int64_t>(a.batch) * rows;
  if (together < kTilesFromRows || rows > kMostTileHeads) return false;
  return together > kFewPrefixRows || static_cast<int64_t>(a.kv_heads) * a.prefix_len >= kFewPrefixKeys;
}

int tile_rows_of(int rows) { return rows <= 8 ? 8 : 16; }

// Which kernels a call takes, and its workspace.
struct CachePlan {
  int rows;         // packed rows of a run
  bool tiles;       // the sequences' own keys (and a prefix before them in the same walk) on the tile kernel
  int tile_rows;    // of the few-row kernel: 8 or 16; of the tile kernel up to 128
  int row_tiles;    // of so many, or pairs of them
  int splits;       // of a pair of tiles
  int ctas;         // of the few-row kernel
  bool prefix_apart;  // a kernel of its own over the prefix for the rows of the whole batch
  bool prefix_tiles;
  int prefix_rows, prefix_tile_rows, prefix_row_tiles, prefix_splits;
  WeightsPlan weights;  // with `tiles`
  size_t own_out, own_sum;  // with `prefix_tiles`
  size_t part_out, part_sum, prefix_out, prefix_sum, scores, row_norm, bytes;  // (scores: or the sums of their parts)
};

CachePlan cache_plan(const CacheAttentionArgs &a) {
  CachePlan p = {};
  const int group = a.heads / a.kv_heads;
  const int64_t d = a.head_dim;
  p.rows = group * a.q_len;
  // (a tile holds whole queries, so their heads have to go into it)
  const int64_t scores = static_cast<int64_t>(a.batch) * a.kv_heads * p.rows * a.kv_len;
  const bool many_rows = p.rows >= kTilesFromRows && (a.weights_out == nullptr || p.rows >= kWeightTilesFromRows || scores > kMostScores);
  p.tiles = many_rows && group <= kMostTileHeads;
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
    most = std::min<int64_t>(a.kv_len, static_cast<int64_t>(a.window) + a.sinks + std::min(a.q_len, cache_tiles_positions(group)));
    p.tile_rows = cache_tile_rows(group);
    p.row_tiles = cache_tiles_pairs(p.rows, p.tile_rows);
    p.splits = cache_tiles_splits(runs * p.row_tiles, static_cast<int>(std::min<int64_t>(most + a.prefix_len, INT32_MAX)), kOwnBlocks);
    part_rows = p.splits > 1 ? cache_tiles_part_rows(runs * p.row_tiles, p.splits, p.tile_rows) : 0;
  } else {
    p.tile_rows = tile_rows_of(p.rows);
    p.row_tiles = (p.rows + p.tile_rows - 1) / p.tile_rows;
    const int64_t steps = (most + kStepKeys - 1) / kStepKeys, least = std::min<int64_t>(kLeastSteps, steps);  // of a unit, and of a CTA
    // (beside a prefix's tile kernel, whose CTAs hold their SMs for a while, in two rounds: the SMs it leaves free take more of them)
    const bool beside_tiles = a.prefix_len > 0 && prefix_on_tiles(a, p.rows);
    p.ctas = static_cast<int>(std::min<int64_t>((beside_tiles ? 2 : 1) * kCtasPerSm * sm_count(), (runs * p.row_tiles * steps + least - 1) / least));
    part_rows = static_cast<size_t>(p.ctas) * 2 * p.tile_rows;
  }
  if (part_rows > 0) {
    p.part_out = take(part_rows * d * 4);
    p.part_sum = take(part_rows * 8);
  }
  if (a.prefix_len > 0 && !p.tiles) {
    p.prefix_apart = true;
    p.prefix_rows = a.batch * p.rows;
    p.prefix_tiles = prefix_on_tiles(a, p.rows);
    if (p.prefix_tiles) {
      p.own_out = take(static_cast<size_t>(runs) * p.rows * d * 4);
      p.own_sum = take(static_cast<size_t>(runs) * p.rows * 8);
      p.prefix_tile_rows = cache_tile_rows(p.rows);
      p.prefix_row_tiles = cache_tiles_pairs(p.prefix_rows, p.prefix_tile_rows);
      p.prefix_splits = cache_tiles_splits(static_cast<int64_t>(a.kv_heads) * p.prefix_row_tiles, a.prefix_len, kPrefixBlocks);
    } else {
      p.prefix_tile_rows = tile_rows_of(p.prefix_rows);
      p.prefix_row_tiles = (p.prefix_rows + p.prefix_tile_rows - 1) / p.prefix_tile_rows;
      // (as many as the kernel finds keys for: every part that the merge reads is written)
      const int steps = (a.prefix_len + kStepKeys - 1) / kStepKeys;
      const int wanted = prefix_splits(static_cast<int64_t>(a.kv_heads) * p.prefix_row_tiles, a.prefix_len);
      const int per_split = (steps + wanted - 1) / wanted;
      p.prefix_splits = (steps + per_split - 1) / per_split;
    }
    p.prefix_out = take(static_cast<size_t>(a.kv_heads) * p.prefix_splits * p.prefix_rows * d * 4);
    p.prefix_sum = take(static_cast<size_t>(a.kv_heads) * p.prefix_splits * p.prefix_rows * 8);
  }
  if (a.weights_out != nullptr && p.tiles) {
    p.weights = cache_weights_plan(a, p.tile_rows, kCacheCounters);
    p.row_norm = take(static_cast<size_t>(runs) * cache_weights_norm_pitch(p.rows, p.tile_rows) * 8);
    p.scores = take(p.weights.part_bytes);
  } else if (a.weights_out != nullptr) {
    p.scores = take(static_cast<size_t>(runs) * p.rows * score_pitch_of(a.kv_len) * 4);
    p.row_norm = take(static_cast<size_t>(runs) * p.rows * 8);
  }
  p.bytes = at;
  return p;
}

template <int D, bool BF16, int NB>
cudaError_t launch_rows(const RowsParams &p, int64_t ctas, cudaStream_t stream) {
  using L = RowsLayout<D>;
  auto kernel = few_rows_kernel<D, BF16, NB>;
  static const cudaError_t attr_set = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmemBytes);
  if (attr_set != cudaSuccess) return attr_set;
  return launch_overlapped(kernel, ctas, kThreads, L::kSmemBytes, stream, p);
}

template <int D, bool BF16>
cudaError_t launch_rows(const RowsParams &p, int tile_rows, int64_t ctas, cudaStream_t stream) {
  return tile_rows == 8 ? launch_rows<D, BF16, 1>(p, ctas, stream) : launch_rows<D, BF16, 2>(p, ctas, stream);
}

cudaError_t launch_rows(const CacheAttentionArgs &a, const RowsParams &p, int tile_rows, int64_t ctas) {
  if (a.head_dim == 64) {
    return a.is_bf16 ? launch_rows<64, true>(p, tile_rows, ctas, a.stream) : launch_rows<64, false>(p, tile_rows, ctas, a.stream);
  }
  return a.is_bf16 ? launch_rows<128, true>(p, tile_rows, ctas, a.stream) : launch_rows<128, false>(p, tile_rows, ctas, a.stream);
}

}  // namespace

bool cache_attention_supported(const CacheAttentionArgs &a, const char **why) {
  const int64_t most = INT32_MAX;
  if (static_cast<int64_t>(a.batch) * a.heads * a.q_len > most) {
    *why = "more than 2^31 - 1 query rows";
    return false;
  }
  const CachePlan plan = cache_plan(a);
  const int64_t steps = (static_cast<int64_t>(a.kv_len) + kStepKeys - 1) / kStepKeys * a.batch * a.kv_heads * plan.row_tiles;  // at most
  if ((!plan.tiles && steps / plan.ctas >= most) || (plan.tiles && static_cast<int64_t>(a.batch) * a.kv_heads * plan.row_tiles * plan.splits > most) || plan.weights.ctas > most ||
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
  p->by_kv_heads = Divisor::of(static_cast<uint32_t>(p->kv_heads));
  p->by_group = Divisor::of(static_cast<uint32_t>(p->group));
  p->by_sequence_rows = Divisor::of(static_cast<uint32_t>(p->group * a.q_len));
  p->q_len = a.q_len;
  p->kv_len = a.kv_len;
  p->window = a.window;
  p->sinks = a.sinks;
  p->scale_log2 = 1.4426950408889634f / sqrtf(static_cast<float>(a.head_dim));
}

cudaError_t cache_attention(const CacheAttentionArgs &a, const char **why, int *launches) {
  *why = "";
  const CachePlan plan = cache_plan(a);
  auto floats = [&](size_t off) { return reinterpret_cast<float *>(a.workspace + off); };
  auto pairs = [&](size_t off) { return reinterpret_cast<float2 *>(a.workspace + off); };
  cudaError_t e;
  TilesParams tiles = {};
  fill_params(a, &tiles);

  tiles.status = a.status;
  tiles.prefix_len = a.prefix_len;
  if (plan.tiles) {
    tiles.runs = a.batch * a.kv_heads;
    tiles.rows = plan.rows;
    tiles.tile_rows = plan.tile_rows;
    tiles.row_pairs = plan.row_tiles;
    tiles.splits = plan.splits;
    tiles.part_out = floats(plan.part_out);
    tiles.part_sum = pairs(plan.part_sum);
    if (a.weights_out != nullptr) {
      tiles.row_norm = pairs(plan.row_norm);
      tiles.norm_pitch = cache_weights_norm_pitch(plan.rows, plan.tile_rows);
    }
    e = cache_tiles(tiles, a, why);
    *launches += e == cudaSuccess ? (plan.splits > 1 ? 2 : 1) : 0;
    if (e != cudaSuccess || a.weights_out == nullptr) return e;
    WeightsParams w = {};
    w.kv_lens = a.kv_lens;
    w.is_bf16 = a.is_bf16;
    w.kv_heads = a.kv_heads;
    w.group = tiles.group;
    w.q_len = a.q_len;
    w.kv_len = a.kv_len;
    w.runs = tiles.runs;
    w.rows = plan.rows;
    w.tile_rows = plan.tile_rows;
    w.positions = plan.tile_rows / w.group;
    w.by_positions = Divisor::of(static_cast<uint32_t>(w.positions));
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
  p.by_row_tiles = Divisor::of(static_cast<uint32_t>(p.row_tiles));
  p.counters = a.counters;
  p.batch = a.batch;
  p.ctas = plan.ctas;
  p.part_out = floats(plan.part_out);
  p.part_sum = pairs(plan.part_sum);
  if (a.weights_out != nullptr) {
    p.scores = floats(plan.scores);
    p.score_pitch = score_pitch_of(a.kv_len);
    p.row_norm = pairs(plan.row_norm);
  }
  if (plan.prefix_apart) {
    if (plan.prefix_tiles) {
      tiles.over_batch = true;
      tiles.runs = a.kv_heads;
      tiles.rows = plan.prefix_rows;
      tiles.tile_rows = plan.prefix_tile_rows;
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
      s.by_row_tiles = Divisor::of(static_cast<uint32_t>(s.row_tiles));
      s.splits = plan.prefix_splits;
      s.ctas = INT32_MAX;
      s.part_out = floats(plan.prefix_out);
      s.part_sum = pairs(plan.prefix_sum);
      *why = "launching the prefix's part";
      e = launch_rows(a, s, plan.prefix_tile_rows, static_cast<int64_t>(a.kv_heads) * s.row_tiles * s.splits);
    }
    if (e != cudaSuccess) return e;
    ++*launches;
    if (plan.prefix_tiles) {
      p.own_out = floats(plan.own_out);
      p.own_sum = pairs(plan.own_sum);
    } else {
      p.prefix_out = floats(plan.prefix_out);
      p.prefix_sum = pairs(plan.prefix_sum);
      p.prefix_splits = plan.prefix_splits;
      p.prefix_rows = plan.prefix_rows;
    }
  }
  e = launch_rows(a, p, plan.tile_rows, plan.ctas + (p.own_out != nullptr ? 1 : 0));
  if (e != cudaSuccess) {
    *why = "launching the few-row kernel";
    return e;
  }
  ++*launches;
  if (plan.prefix_apart && plan.prefix_tiles) {
    JoinParams j = {};
    j.own_out = p.own_out;
    j.own_sum = p.own_sum;
    j.prefix_out = floats(plan.prefix_out);
    j.prefix_sum = pairs(plan.prefix_sum);
    j.out = p.out;
    for (int i = 0; i < 3; ++i) j.out_stride[i] = p.out_stride[i];
    j.by_rows = Divisor::of(static_cast<uint32_t>(p.rows));
    j.by_kv_heads = p.by_kv_heads;
    j.by_group = p.by_group;
    j.rows = p.rows;
    j.prefix_rows = plan.prefix_rows;
    j.prefix_splits = plan.prefix_splits;
    j.group = p.group;
    j.total = static_cast<int64_t>(a.batch) * a.kv_heads * p.rows * (a.head_dim / 4);
    auto join = a.head_dim == 64 ? (a.is_bf16 ? join_prefix_kernel<64, true> : join_prefix_kernel<64, false>)
                                 : (a.is_bf16 ? join_prefix_kernel<128, true> : join_prefix_kernel<128, false>);
    e = launch_overlapped(join, (j.total + 127) / 128, 128, 0, a.stream, j);
    if (e != cudaSuccess) {
      *why = "launching the kernel that joins the prefix's part";
      return e;
    }
    ++*launches;
  }
  if (a.weights_out != nullptr) {
    constexpr int kPerCta = kAddThreads * kKeysAtOnce;
    const int chunks = (a.kv_len + kPerCta - 1) / kPerCta;
    e = launch_overlapped(add_weights_kernel, static_cast<int64_t>(chunks) * a.batch * a.kv_heads, kAddThreads, 0, a.stream, p.scores, p.score_pitch,
                          p.row_norm, p.rows, Divisor::of(static_cast<uint32_t>(chunks)), p.by_kv_heads, p.group, a.q_len, a.kv_len, a.kv_lens,
                          a.weights_in, a.weights_in_stride[0], a.weights_in_stride[1], a.weights_out, a.weights_out_stride[0],
                          a.weights_out_stride[1]);
    if (e != cudaSuccess) {
      *why = "launching the keys' weights";
      return e;
    }
    ++*launches;
  }
  return cudaSuccess;
}

}  // namespace flsm100
