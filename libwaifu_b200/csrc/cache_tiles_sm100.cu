// Attention over a key-value cache for many query rows (prompts, and the rows of a whole batch over a prefix that
// it shares): both products on tcgen05, in the way of the two-tile attention kernel.
//
// A CTA owns two tiles of up to 128 rows of one key-value head. The rows are packed: row r is query r / group of query
// head r % group of the ones that share the head, so that a block of keys is read once for all of them and a
// tile's rows sit close together (under a window a tile walks its 128 / group positions and the window, not 128
// and the window). Over a prefix, which all of a batch sees, the rows of every sequence are packed one after the other.
// A tile holds whole queries (or whole sequences), as many as go into 128 rows, and so is a box of the queries' tensor.
// K and V blocks of 128 keys arrive by TMA into one ring of slots. The walk is a list of blocks: those of a prefix, then the
// sinks and the keys from the first window's start to the last query's position, one after the other and cut every 128
// keys (a block that holds both comes in boxes of 16 rows, the sinks filled up to whole ones): 8192 tokens under a window of
// 1024 keys and 16 sinks walk 9 blocks a unit so, and 10.4 in blocks at multiples of 128.
//
// A block that some row does not see whole (past the sequence's end, at a window's edge, on the diagonal) passes two
// helping warps before its product: they clear the values of keys that no row sees and take infinities, NaN and values of
// another size than any sum's out of the others, because what stands for a probability of zero times such a value is not
// zero (TooLarge). Rows that do see them have them added by hand at the end.
//
// A running CTA takes over units whose own CTA has not started (clusterlaunchcontrol.try_cancel): the next unit's keys,
// queries and first scores come under the last products and the output of the one before. Walks are short here (a window's,
// a chunk's), and a unit's own start and end would be a third of them.
//
// Few units are divided along the keys: each CTA leaves its rows' outputs relative to their own maxima, and a kernel over
// all rows adds them in the order of the splits. (The last CTA of a unit to arrive did that first: 256 rows on one SM took longer
// than the launch.)
#include "cache_tiles_sm100.cuh"

#include <cuda_runtime.h>

#include <algorithm>

#include "attention_sm100.cuh"
#include "attention_tile_sm100.cuh"
#include "cache_common_sm100.cuh"

namespace flsm100 {

namespace {

constexpr int kSoftmaxWarps = kTiles * kTileWarps;
constexpr int kProducerWarp = kSoftmaxWarps;
constexpr int kMmaWarp = kSoftmaxWarps + 1;
constexpr int kHelpWarp = kSoftmaxWarps + 2;  // and the one after it
constexpr int kHelpWarps = 2;
// Three warpgroups launched with 168 registers a thread; the one that loads, issues and helps gives its own up to the
// two of the softmax, which hold a row of 128 scores: 128 x 96 + 256 x 200 < 384 x 168.
constexpr int kThreads = (kSoftmaxWarps + 4) * 32;
constexpr int kIssueRegs = 96, kSoftmaxRegs = 200;
static_assert(128 * kIssueRegs + kSoftmaxWarps * 32 * kSoftmaxRegs <= kThreads * 168, "no more than the block was launched with");
constexpr int kMaxSlots = 6;

// The blocks of a walk that hold keys some row does not see: from one up to another (sinks, the windows' starts), and from one
// on (the rows' own positions, the end).
struct Dirty {
  int begin, end, from;
  __device__ __forceinline__ bool has(int j) const { return (j >= begin && j < end) || j >= from; }
};

constexpr int kBoxRows = 16;  // of the boxes in which a block of sinks and window keys comes

// The blocks of keys a pair of tiles walks, and what its rows see of them. The own keys have places 0 .. total - 1: the sinks
// from 0 on, hidden keys up to `pad`, then the keys from `begin` on. (pad is 0 where sinks and window meet, and without sinks.)
struct Walk {
  int prefix_blocks, prefix_len;
  int pad, begin, total;
  int first, count;         // blocks of this split
  int first_pos, last_pos;  // of the pair's rows
  int window, sinks;
  Dirty dirty;              // (keys past a prefix's end come as zeros: its blocks never are)

  // The blocks of own keys that some row at first .. last does not see whole.
  __device__ __forceinline__ Dirty dirty_for(int first_row_pos, int last_row_pos) const {
    const int own = prefix_blocks - first;  // the walk's first own block, in this split
    auto block_of = [](int place) { return place < 0 ? 0 : place / kBlockKv; };
    Dirty d;
    d.begin = own + block_of(pad > 0 ? sinks : sinks - begin);
    d.end = own + (last_row_pos - window - begin + pad < 0 ? 0 : block_of(last_row_pos - window - begin + pad) + 1);
    d.from = own + block_of(first_row_pos + 1 + pad - begin);
    return d;
  }
  __device__ __forceinline__ bool in_prefix(int j) const { return first + j < prefix_blocks; }
  __device__ __forceinline__ int place0(int j) const { return (first + j - prefix_blocks) * kBlockKv; }
  __device__ __forceinline__ int key_at(int place) const { return place < pad ? place : place - pad + begin; }
  // No row sees the key at this place (of its own keys).
  __device__ __forceinline__ bool hidden(int place) const { return place >= total || (place >= sinks && place < pad); }
  // Some rows see it and others do not (of keys that are not hidden).
  __device__ __forceinline__ bool mixed(int place) const {
    const int key = key_at(place);
    return key > first_pos || (key <= last_pos - window && key >= sinks);
  }
  // How many blocks of the whole walk hold keys up to `position`.
  __device__ __forceinline__ int blocks_up_to(int position) const {
    return prefix_blocks + (position < 0 ? 0 : (position - begin + pad) / kBlockKv + 1);
  }
};

struct Tail {
  uint4 claim;         // the answer to the last try_cancel
  uint64_t claim_bar;  // ... which has arrived
  uint64_t unit_full_bar[2], unit_empty_bar[2];  // producer -> all: the next unit is in next_unit[slot]; all -> producer
  int next_unit[2];                              // -1 when there is none left
  uint64_t q_full_bar[kTiles], q_empty_bar[kTiles];
  uint64_t slot_full_bar[kMaxSlots], slot_empty_bar[kMaxSlots], slot_clean_bar[kMaxSlots];
  uint64_t s_full_bar[kTiles];     // MMA -> softmax: the tile's scores are in tensor memory
  uint64_t p_full_bar[kTiles][2];  // softmax -> MMA: that part of the tile's probabilities is in tensor memory
  uint64_t pv_done_bar[kTiles];    // MMA -> softmax: the last block is in the tile's output
  uint32_t tmem_base_slot;
  uint32_t abort_flag;
  // The last unit of a count (mod 4) that had values taken out of a block. The helping warps may be two units ahead of the
  // softmax (one without blocks between), so two places would not do.
  uint32_t patch_flag[4];
  Walk walk[kSoftmaxWarps];  // of the unit that the warp works on
};

template <int D>
struct Layout : TileLayout<D> {
  using T = TileLayout<D>;
  static constexpr int kRoom = (227 * 1024 - kTiles * T::kQBytes - static_cast<int>(sizeof(Tail))) / T::kSlotBytes;
  static constexpr int kSlots = kRoom < kMaxSlots ? kRoom : kMaxSlots;
  static_assert(kSlots >= 3, "K of the next block, V of this one and a load in flight");
  static constexpr int kQOff = 0;
  static constexpr int kSlotOff = kQOff + kTiles * T::kQBytes;
  static constexpr int kTailOff = kSlotOff + kSlots * T::kSlotBytes;
  static constexpr int kSmemBytes = kTailOff + static_cast<int>(sizeof(Tail));
  static_assert(kSmemBytes <= 227 * 1024, "shared memory");
};

struct Unit {
  int index, run, head, seq, pair, split, active;
  int row0;  // of the pair
  int len;
  Walk walk;
  int blocks[kTiles];  // how many of the split's blocks each tile walks

  __device__ __forceinline__ Unit(const TilesParams &p, int at) : index(at) {
    // The longest walks first: the last pair of every run, then the one before it.
    run = p.by_runs.take(&at);
    split = p.by_splits.take(&at);
    pair = p.row_pairs - 1 - at;
    seq = run;
    head = p.by_kv_heads.take(&seq);
    row0 = pair * kTiles * p.tile_rows;
    const int last_row = min(row0 + kTiles * p.tile_rows, p.rows) - 1;
    walk.prefix_len = p.prefix_len;
    walk.prefix_blocks = (p.prefix_len + kBlockKv - 1) / kBlockKv;
    walk.window = p.window;
    walk.sinks = p.sinks;
    len = 0;
    walk.first_pos = walk.last_pos = walk.pad = walk.begin = walk.total = 0;
    if (!p.over_batch) {
      len = sequence_length(p.kv_lens, seq, p.kv_len);
      walk.first_pos = p.by_group.quotient(row0) + len - p.q_len;
      walk.last_pos = p.by_group.quotient(last_row) + len - p.q_len;
      const KeyRange range = visible_keys(walk.first_pos, walk.last_pos, len, p.window, p.sinks);
      const bool apart = range.sinks > 0 && range.sinks < range.begin;
      walk.pad = apart ? (range.sinks + kBoxRows - 1) / kBoxRows * kBoxRows : 0;
      walk.begin = apart || range.sinks == 0 ? range.begin : 0;
      walk.total = walk.pad + range.end - walk.begin;
    }
    const int total = walk.prefix_blocks + (walk.total + kBlockKv - 1) / kBlockKv;
    const int per_split = max(1, p.by_splits.quotient(total + p.splits - 1));
    active = p.splits == 1 ? 1 : max(1, (total + per_split - 1) / per_split);
    walk.first = split * per_split;
    walk.count = max(0, min(per_split, total - walk.first));  // (0 past the active splits)
    walk.dirty = p.over_batch ? Dirty{0, 0, INT32_MAX} : walk.dirty_for(walk.first_pos, walk.last_pos);
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      const int first_row = row0 + i * p.tile_rows, last = min(first_row + p.tile_rows, p.rows) - 1;
      const int mine = p.over_batch ? total : min(total, walk.blocks_up_to(p.by_group.quotient(last) + len - p.q_len));
      blocks[i] = first_row >= p.rows ? 0 : max(0, min(walk.count, mine - walk.first));
    }
  }
};

// What the issuing warp has to know of a unit.
struct Todo {
  int blocks[kTiles], total;
  Dirty dirty;
  __device__ __forceinline__ Todo() : blocks{0, 0}, total(0) {}
  __device__ __forceinline__ explicit Todo(const Unit &u) : blocks{u.blocks[0], u.blocks[1]}, total(u.walk.count), dirty(u.walk.dirty) {}
};

// Bits 0 .. n - 1.
__device__ __forceinline__ uint32_t bits_below(int n) { return n <= 0 ? 0u : (n >= 32 ? 0xffffffffu : (1u << n) - 1u); }

// Sets the scores of the keys of block j that the row at `pos` does not see to -inf, where there are any for its tile. What
// it takes of the walk lies in shared memory: the softmax has no registers to spare for it.
struct HideUnseen {
  bool edge;
  const Walk *walk;
  int j, pos;
  __device__ __forceinline__ void operator()(uint32_t (&sc)[kBlockKv / 32][32]) const {
    if (!edge) return;
    int key0, last, before, sinks;  // of the block's keys, from key0 on, the row sees those up to `last` behind `before`, and the first `sinks`
    if (walk->in_prefix(j)) {
      key0 = (walk->first + j) * kBlockKv;
      last = walk->prefix_len - 1;
      before = -1;
      sinks = 0;
    } else {
      const int x0 = walk->place0(j);
      key0 = x0 - walk->pad + walk->begin;
      last = pos;
      before = pos - walk->window;
      sinks = walk->sinks - key0;
      if (x0 < walk->pad) {  // sinks, and what follows them
        before = max(before, walk->begin - 1);
        sinks = walk->sinks - x0;
      }
    }
#pragma unroll
    for (int c = 0; c < kBlockKv / 32; ++c) {
      const int base = key0 + c * 32;
      const uint32_t seen = bits_below(last + 1 - base) & (~bits_below(before + 1 - base) | bits_below(sinks - c * 32));
#pragma unroll
      for (int i = 0; i < 32; ++i) {
        if (!((seen >> i) & 1u)) sc[c][i] = __float_as_uint(-INFINITY);
      }
    }
  }
};

// The address of packed row r of a head's queries (or results).
__device__ __forceinline__ int64_t row_offset(const TilesParams &p, const int64_t (&stride)[3], int head, int seq, int r) {
  if (p.over_batch) {
    seq = r;
    r = p.by_sequence_rows.take(&seq);
  }
  int i = r;
  const int g = p.by_group.take(&i);
  return seq * stride[0] + static_cast<int64_t>(head * p.group + g) * stride[1] + i * stride[2];
}

// The values that a key loses where some row of the tile does not see it: infinities and NaN, which a probability of zero does not
// stop, and of bfloat16 what is 2^64 or more, because the cubic's probability of an unseen key is 2^-126 (no half, but a
// bfloat16; to give it a zero cost 69.6 -> 72.5 us on prefix_extend). A mask of such halves, by a carry out of their exponents.
template <bool BF16>
struct TooLarge {
  static constexpr uint32_t kExponent = BF16 ? 0x7F807F80u : 0x7C007C00u;
  static constexpr uint32_t kCarry = BF16 ? 0x20802080u : 0x04000400u;  // from an exponent field of 191, of 31 on
  // Into the sign bits.
  static __device__ __forceinline__ uint32_t signs(uint32_t w) { return (w & kExponent) + kCarry; }
  static __device__ __forceinline__ uint32_t halves(uint32_t w) { return ((signs(w) >> 15) & 0x00010001u) * 0xFFFFu; }
  static __device__ __forceinline__ bool any(uint4 w) { return ((signs(w.x) | signs(w.y) | signs(w.z) | signs(w.w)) & 0x80008000u) != 0; }
  static __device__ __forceinline__ uint4 without(uint4 w) {
    return make_uint4(w.x & ~halves(w.x), w.y & ~halves(w.y), w.z & ~halves(w.z), w.w & ~halves(w.w));
  }
};

// Adds what a row sees of the values that were taken out of its blocks: rare, and as slow as it is plain.
template <int D, bool BF16>
__device__ __noinline__ void patch_row(const TilesParams &p, int unit, int pos, const uint16_t *q, float m, float l, uint16_t *out, float *part) {
  const Unit u(p, unit);
  auto pieces_of = [](const uint16_t *row) { return reinterpret_cast<const uint4 *>(row); };  // eight values each
  float sum[D];
#pragma unroll
  for (int d = 0; d < D; ++d) sum[d] = 0.0f;
  for (int j = 0; j < u.walk.count; ++j) {
    if (!u.walk.dirty.has(j)) continue;
    for (int x = u.walk.place0(j); x < u.walk.place0(j) + kBlockKv; ++x) {
      const int key = u.walk.key_at(x);
      if (u.walk.hidden(x) || !u.walk.mixed(x) || key > pos || !(key > pos - p.window || key < p.sinks)) continue;
      const uint4 *v = pieces_of(p.v + u.seq * p.v_stride[0] + u.head * p.v_stride[1] + key * p.v_stride[2]);
      bool found = false;
#pragma unroll
      for (int c = 0; c < D / 8; ++c) found |= TooLarge<BF16>::any(v[c]);
      if (!found) continue;
      const uint4 *k = pieces_of(p.k + u.seq * p.k_stride[0] + u.head * p.k_stride[1] + key * p.k_stride[2]);
      float s = 0.0f;
#pragma unroll 4
      for (int c = 0; c < D / 8; ++c) {
        const uint4 a = pieces_of(q)[c], b = k[c];
        const uint32_t as[4] = {a.x, a.y, a.z, a.w}, bs[4] = {b.x, b.y, b.z, b.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 y = widen_pair<BF16>(as[i]), z = widen_pair<BF16>(bs[i]);
          s = fmaf(y.x, z.x, fmaf(y.y, z.y, s));
        }
      }
      const float w = exp2f(s * p.scale_log2 - m);
#pragma unroll 1
      for (int c = 0; c < D / 8; ++c) {
        const uint4 y = v[c];
        const uint32_t ys[4] = {y.x, y.y, y.z, y.w};
        for (int i = 0; i < 4; ++i) {
          const uint32_t large = TooLarge<BF16>::halves(ys[i]);
          const float2 z = widen_pair<BF16>(ys[i]);
          if (large & 0xFFFFu) sum[c * 8 + 2 * i] += w * z.x;
          if (large >> 16) sum[c * 8 + 2 * i + 1] += w * z.y;
        }
      }
    }
  }
#pragma unroll 1
  for (int d = 0; d < D; ++d) {
    if (sum[d] == 0.0f) continue;
    if (part != nullptr) {
      part[d] += sum[d];
    } else {
      out[d] = static_cast<uint16_t>(pack_pair<BF16>(widen_pair<BF16>(out[d]).x + sum[d] / l, 0.0f));
    }
  }
}

// A row's result, or its part of it: output and sum are relative to m.
template <int D, bool BF16>
__device__ __forceinline__ void finish_row(const TilesParams &p, const Unit &u, uint32_t t_out, int tile, int in_tile, int pos, int my_blocks,
                                           bool ok, bool patch, float m, float l_run) {
  const int row = u.row0 + tile * p.tile_rows + in_tile;
  const bool live = in_tile < p.tile_rows && row < p.rows;
  const bool parts = p.over_batch || u.active > 1;
  // The index of this row's part of split s: (kv_head, split, rows) over a prefix, (unit, split, rows of a pair) else.
  const int64_t part_row0 = p.over_batch ? static_cast<int64_t>(u.head) * p.splits * p.rows + row
                                         : (static_cast<int64_t>(u.run) * p.row_pairs + u.pair) * p.splits * kTiles * p.tile_rows + (row - u.row0);
  const int64_t part_step = p.over_batch ? p.rows : kTiles * p.tile_rows;
  const bool empty = p.prefix_len == 0 && pos < 0;  // sees no key: zeros
  uint16_t *dst = live && !p.over_batch ? p.out + row_offset(p, p.out_stride, u.head, u.seq, row) : nullptr;
  float *part_dst = p.part_out + (part_row0 + u.split * part_step) * D;
  const int64_t norm_at = static_cast<int64_t>(u.run) * p.norm_pitch + (u.pair * kTiles + tile) * kBlockQ + in_tile;
  // (a row whose every score is -inf has no softmax)
  const float inv = empty ? 0.0f : (m == -INFINITY ? NAN : 1.0f / l_run);
  if (ok) {
#pragma unroll 1
    for (int c = 0; c < D / 32; ++c) {
      uint32_t v[32];
      if (my_blocks > 0) {
        tmem_ld_32x32(t_out + c * 32, v);
        tmem_ld_wait(v);
      } else {
#pragma unroll
        for (int i = 0; i < 32; ++i) v[i] = 0;
      }
      if (live && parts) {
#pragma unroll
        for (int g = 0; g < 32; g += 8) {
          store_32_bytes(part_dst + c * 32 + g, v[g], v[g + 1], v[g + 2], v[g + 3], v[g + 4], v[g + 5], v[g + 6], v[g + 7]);
        }
      } else if (live) {
#pragma unroll
        for (int g = 0; g < 4; ++g) {
          uint4 w;
          w.x = pack16(__uint_as_float(v[g * 8 + 0]) * inv, __uint_as_float(v[g * 8 + 1]) * inv, BF16);
          w.y = pack16(__uint_as_float(v[g * 8 + 2]) * inv, __uint_as_float(v[g * 8 + 3]) * inv, BF16);
          w.z = pack16(__uint_as_float(v[g * 8 + 4]) * inv, __uint_as_float(v[g * 8 + 5]) * inv, BF16);
          w.w = pack16(__uint_as_float(v[g * 8 + 6]) * inv, __uint_as_float(v[g * 8 + 7]) * inv, BF16);
          *reinterpret_cast<uint4 *>(dst + c * 32 + g * 8) = empty ? make_uint4(0, 0, 0, 0) : w;
        }
      }
    }
    if (live && patch && m != -INFINITY && l_run == l_run) {
      const uint16_t *q = p.q + row_offset(p, p.q_stride, u.head, u.seq, row);
      patch_row<D, BF16>(p, u.index, pos, q, m, l_run, dst, parts ? part_dst : nullptr);
    }
    // (the cubic's smallest exponentials keep a part that saw nothing from summing to zero)
    if (live && parts) p.part_sum[part_row0 + u.split * part_step] = make_float2(m, m == -INFINITY && l_run == l_run ? 0.0f : l_run);
    // (of a tile's empty places zeros, whose rows then weigh nothing)
    if (p.row_norm != nullptr && (!live || !parts)) p.row_norm[norm_at] = live ? make_float2(m, inv) : make_float2(0.0f, 0.0f);
  }
}

// The results of rows whose unit several CTAs shared: four columns a thread.
template <int D, bool BF16>
__global__ void __launch_bounds__(128) join_tiles_kernel(const __grid_constant__ TilesParams p, const Divisor by_rows, const Divisor by_tile_rows, int64_t total) {
  griddep_wait();
  griddep_launch_dependents();
  constexpr int kQuads = D / 4;
  const int64_t at = static_cast<int64_t>(blockIdx.x) * 128 + threadIdx.x;
  if (at >= total) return;
  const int col = static_cast<int>(at % kQuads) * 4;
  int run = static_cast<int>(at / kQuads);
  const int row = by_rows.take(&run), tile = by_tile_rows.quotient(row), pair = tile / kTiles;
  const Unit u(p, run + p.runs * p.splits * (p.row_pairs - 1 - pair));  // (its first split)
  if (u.active == 1) return;
  RowSum sum;
  sum.clear();
  const int pair_rows = kTiles * p.tile_rows;
  const int64_t first = (static_cast<int64_t>(run) * p.row_pairs + pair) * p.splits * pair_rows + (row - u.row0);
  add_parts<D>(u.active, p.part_sum, p.part_out, col, &sum, [&](int c) { return first + c * pair_rows; });
  const bool empty = p.prefix_len == 0 && p.by_group.quotient(row) + u.len - p.q_len < 0;  // sees no key: zeros
  // (a row whose every score is -inf has no softmax)
  const float inv = empty ? 0.0f : (sum.m == -INFINITY ? NAN : 1.0f / sum.l);
  const uint2 w = make_uint2(pack_pair<BF16>(sum.o.x * inv, sum.o.y * inv), pack_pair<BF16>(sum.o.z * inv, sum.o.w * inv));
  *reinterpret_cast<uint2 *>(p.out + row_offset(p, p.out_stride, u.head, u.seq, row) + col) = empty ? make_uint2(0, 0) : w;
  if (p.row_norm != nullptr && col == 0) p.row_norm[static_cast<int64_t>(run) * p.norm_pitch + tile * kBlockQ + row - tile * p.tile_rows] = make_float2(sum.m, inv);
}

template <int D, bool BF16>
__global__ void __launch_bounds__(kThreads, 1)
cache_tiles_kernel(const __grid_constant__ CUtensorMap tmap_q, const __grid_constant__ CUtensorMap tmap_k, const __grid_constant__ CUtensorMap tmap_v,
                   const __grid_constant__ CUtensorMap tmap_k16, const __grid_constant__ CUtensorMap tmap_v16,
                   const __grid_constant__ CUtensorMap tmap_pk, const __grid_constant__ CUtensorMap tmap_pv,
                   const __grid_constant__ TilesParams p) {
  using L = Layout<D>;
  constexpr int S = L::kSlots;
  constexpr int kPParts = kPartsOf<D>;
  extern __shared__ __align__(1024) uint8_t smem[];
  Tail &t = *reinterpret_cast<Tail *>(smem + L::kTailOff);
  volatile uint32_t &abort_flag = *reinterpret_cast<volatile uint32_t *>(&t.abort_flag);

  const uint32_t warp = threadIdx.x >> 5;
  const uint32_t lane = threadIdx.x & 31;
  if ((smem_u32(smem) & 1023u) != 0) {
    if (threadIdx.x == 0) atomicCAS(p.status, 0u, kStatusAttentionLayout);
    return;
  }
  if (threadIdx.x == 0) {
    t.abort_flag = 0;
    for (uint32_t &flag : t.patch_flag) flag = 0;
    mbar_init(&t.claim_bar, 1);
    for (int i = 0; i < 2; ++i) {
      mbar_init(&t.unit_full_bar[i], 1);
      mbar_init(&t.unit_empty_bar[i], kSoftmaxWarps + 1 + kHelpWarps);
    }
    for (int i = 0; i < S; ++i) {
      mbar_init(&t.slot_full_bar[i], 1);
      mbar_init(&t.slot_empty_bar[i], 1 + kHelpWarps);
      mbar_init(&t.slot_clean_bar[i], kHelpWarps);
    }
    for (int i = 0; i < kTiles; ++i) {
      mbar_init(&t.q_full_bar[i], 1);
      mbar_init(&t.q_empty_bar[i], 1);
      mbar_init(&t.s_full_bar[i], 1);
      for (int h = 0; h < kPParts; ++h) mbar_init(&t.p_full_bar[i][h], kTileWarps);
      mbar_init(&t.pv_done_bar[i], 1);
    }
    fence_barrier_init();
  }
  if (warp == kProducerWarp && lane == 0) {
    tma_prefetch_desc(&tmap_q);
    tma_prefetch_desc(&tmap_k);
    tma_prefetch_desc(&tmap_v);
  }
  if (warp == kMmaWarp) {
    tmem_alloc<1>(&t.tmem_base_slot, L::kTmemCols);
    tmem_relinquish<1>();
  }
  clear_empty_places<L::kQAtoms * kTiles>(smem + L::kQOff, p.tile_rows, kThreads);
  tc_fence_before_sync();
  __syncthreads();
  tc_fence_after_sync();
  const uint32_t tmem_base = t.tmem_base_slot;
  griddep_wait();
  griddep_launch_dependents();

  auto q_tile = [&](int i) { return smem + L::kQOff + i * L::kQBytes; };
  auto slot = [&](int i) { return smem + L::kSlotOff + i * L::kSlotBytes; };
  // Unit number `count` of this CTA (from 1 on), once the producer has put it there; -1: none left. The warp's lanes call together.
  auto next_unit = [&](int count, int *unit) -> bool {
    if (!__all_sync(0xffffffffu, mbar_wait(&t.unit_full_bar[count & 1], ((count - 1) >> 1) & 1, &abort_flag))) return false;
    *unit = *reinterpret_cast<volatile int *>(&t.next_unit[count & 1]);
    __syncwarp();
    if (lane == 0) mbar_arrive(&t.unit_empty_bar[count & 1]);
    return true;
  };

  // Load n of the ring, counted over all of the CTA's units (K of a block, V of it, K of the next), goes to slot n % S.
  if (warp < kSoftmaxWarps) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
    // ------------------------------------------------------------------ softmax and output
    const int tile = static_cast<int>(warp >> 2);
    const uint32_t quarter = warp & 3;
    const uint32_t t_lane = tmem_base + ((quarter * 32u) << 16);
    const uint32_t t_scores = t_lane + tile * L::kSCols;  // the row's 128 scores, then its 128 probabilities in 64 columns
    const uint32_t t_out = t_lane + L::kOCol + tile * D;
    bool ok = true;
    uint32_t s_phase = 0, pv_phase = 0;  // of the tile's scores and of its finished outputs
    int unit = blockIdx.x;
#pragma unroll 1
    for (int count = 1; ok && unit >= 0; ++count) {
      // What the loop needs of the unit; the rest is worked out again behind it.
      int my_blocks, pos;
      Dirty edges;
      bool active;
      {
        const Unit u(p, unit);
        active = u.split < u.active;
        my_blocks = tile == 0 ? u.blocks[0] : u.blocks[1];
        const int tile_row0 = u.row0 + tile * p.tile_rows, tile_end = min(tile_row0 + p.tile_rows, p.rows), offset = u.len - p.q_len;
        pos = p.by_group.quotient(max(0, min(tile_row0 + static_cast<int>(threadIdx.x % kBlockQ), tile_end - 1))) + offset;
        const int first = p.by_group.quotient(tile_row0) + offset, last = p.by_group.quotient(max(0, tile_end - 1)) + offset;
        edges = u.walk.dirty_for(first, last);
        if (p.prefix_len > 0) {  // (no window there)
          edges.end = u.walk.prefix_blocks - u.walk.first;
          edges.begin = edges.end - (p.prefix_len % kBlockKv != 0 ? 1 : 0);
          if (p.over_batch) edges.from = INT32_MAX;
        }
        if (lane == 0) t.walk[warp] = u.walk;
        __syncwarp();
      }
      float m_used = -INFINITY;
      float l_run = 0.0f;
      for (int j = 0; j < my_blocks && ok; ++j) {
        // (Scores of block j are issued behind the product of block j - 1: once they are here the tile's
        // output is complete up to that block.)
        ok = __all_sync(0xffffffffu, mbar_wait(&t.s_full_bar[tile], s_phase, &abort_flag));
        if (!ok) break;
        s_phase ^= 1;
        tc_fence_after_sync();
        const HideUnseen hide{edges.has(j), &t.walk[warp], j, pos};
        softmax_block<D, true>(p.scale_log2, BF16, kProbabilityShift<BF16>, t_scores, t_out, j == 0, hide, t.p_full_bar[tile], lane, &m_used, &l_run);
      }
      // The last product.
      if (ok && my_blocks > 0) {
        ok = __all_sync(0xffffffffu, mbar_wait(&t.pv_done_bar[tile], pv_phase, &abort_flag));
        pv_phase ^= 1;
        tc_fence_after_sync();
      }
      if (active) {
        asm volatile("" : "+r"(unit));  // (or what is worked out here would stay in registers from above)
        const Unit u(p, unit);
        const bool patch = *reinterpret_cast<volatile uint32_t *>(&t.patch_flag[count & 3]) == static_cast<uint32_t>(count);
        finish_row<D, BF16>(p, u, t_out, tile, static_cast<int>(threadIdx.x % kBlockQ), pos, my_blocks, ok, patch, m_used - kProbabilityShift<BF16>, l_run);
        // The next unit's first product overwrites this output: it waits for probabilities that the tile's
        // four warps hand over only after these reads.
        tc_fence_before_sync();
      }
      if (ok) ok = next_unit(count, &unit);
    }
    if (!ok && lane == 0) {
      abort_flag = 1;
      atomicCAS(p.status, 0u, kStatusAttentionTimeout);
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kIssueRegs));
    if (warp == kProducerWarp) {
      // ------------------------------------------------------------------ producer
      if (elect_one()) {
        bool ok = true;
        int n = 0;  // loads of the ring so far
        uint32_t q_phase = 0;  // bit i: of tile i's queries
        int unit = blockIdx.x;
        for (int count = 1; ok && unit >= 0; ++count) {
          const Unit u(p, unit);
          for (int i = 0; i < 2 * u.walk.count && ok; ++i, ++n) {
            const int st = n % S, j = i >> 1;
            if (!mbar_wait(&t.slot_empty_bar[st], ((n / S) & 1) ^ 1, &abort_flag)) {
              ok = false;
              break;
            }
            mbar_arrive_expect_tx(&t.slot_full_bar[st], L::kSlotBytes);
            const bool prefix = u.walk.in_prefix(j), keys = (i & 1) == 0;
            const int x0 = u.walk.place0(j);
            if (!prefix && x0 < u.walk.pad && x0 + kBlockKv > u.walk.pad) {
              const CUtensorMap *map = keys ? &tmap_k16 : &tmap_v16;
              for (int r = 0; r < kBlockKv; r += kBoxRows) {
#pragma unroll
                for (int a = 0; a < L::kQAtoms; ++a) {
                  tma_load_4d(slot(st) + a * kBlockKv * kAtomBytes + r * kAtomBytes, map, &t.slot_full_bar[st], a * kAtomBytes, u.walk.key_at(x0 + r),
                              u.head, u.seq);
                }
              }
            } else {
              const CUtensorMap *map = keys ? (prefix ? &tmap_pk : &tmap_k) : (prefix ? &tmap_pv : &tmap_v);
              const int key0 = prefix ? (u.walk.first + j) * kBlockKv : u.walk.key_at(x0);
#pragma unroll
              for (int a = 0; a < L::kQAtoms; ++a) {
                tma_load_4d(slot(st) + a * kBlockKv * kAtomBytes, map, &t.slot_full_bar[st], a * kAtomBytes, key0, u.head, prefix ? 0 : u.seq);
              }
            }
            // The queries behind the first block of keys, once the last scores of the unit before have been computed.
            for (int q = 0; i == 0 && q < kTiles && ok; ++q) {
              if ((q == 0 ? u.blocks[0] : u.blocks[1]) == 0) continue;
              if (!mbar_wait(&t.q_empty_bar[q], ((q_phase >> q) & 1) ^ 1, &abort_flag)) {
                ok = false;
                break;
              }
              q_phase ^= 1u << q;
              mbar_arrive_expect_tx(&t.q_full_bar[q], static_cast<uint32_t>(p.tile_rows) * D * 2);
              const int row = u.row0 + q * p.tile_rows;
              const int seq = p.over_batch ? p.by_sequence_rows.quotient(row) : u.seq, query = p.over_batch ? 0 : p.by_group.quotient(row);
#pragma unroll
              for (int a = 0; a < L::kQAtoms; ++a) {
                tma_load_4d(q_tile(q) + a * kBlockQ * kAtomBytes, &tmap_q, &t.q_full_bar[q], a * kAtomBytes, u.head * p.group, query, seq);
              }
            }
          }
          if (!ok) break;
          // The next unit is claimed once the last block of this one is on its way: as late as its own
          // loads allow, so that the CTA that is ahead takes it.
          mbar_arrive_expect_tx(&t.claim_bar, sizeof(t.claim));
          claim_next_cta(&t.claim, &t.claim_bar);
          if (!mbar_wait(&t.claim_bar, (count - 1) & 1, &abort_flag) ||
              !mbar_wait(&t.unit_empty_bar[count & 1], (((count - 1) >> 1) & 1) ^ 1, &abort_flag)) {
            ok = false;
            break;
          }
          const int4 at = claimed_cta(&t.claim);
          unit = at.w != 0 ? at.x : -1;
          fence_proxy_async_smem();  // the answer has been read before the next one overwrites it
          *reinterpret_cast<volatile int *>(&t.next_unit[count & 1]) = unit;
          mbar_arrive(&t.unit_full_bar[count & 1]);
        }
        if (!ok) {
          abort_flag = 1;
          atomicCAS(p.status, 0u, kStatusAttentionTimeout);
        }
      }
    } else if (warp == kMmaWarp) {
      // ------------------------------------------------------------------ MMA issuer
      // The whole warp walks the loop and an elected lane issues.
      const bool issuer = elect_one();
      const TileMmas<D> mma(BF16, true, tmem_base, smem_u32(q_tile(0)), issuer);
      const uint64_t sdesc0 = umma_desc_sw128(smem_u32(slot(0)));
      bool ok = true;
      uint32_t clean_phase = 0;  // bit i: the parity of the next unclean values in slot i
      uint32_t q_phase[kTiles] = {0, 0}, p_phase[kTiles] = {0, 0};
      auto commit = [&](uint64_t *bar) {
        if (issuer) umma_commit(bar);
      };
      auto wait_full = [&](int n) -> bool { return mbar_wait(&t.slot_full_bar[n % S], (n / S) & 1, &abort_flag); };
      auto desc_of = [&](int n) -> uint64_t { return sdesc0 + static_cast<uint64_t>((n % S) * (L::kSlotBytes >> 4)); };
      int n = 0;  // the ring's load that holds K of the unit's first block
      int unit = blockIdx.x;
      Todo now(Unit(p, unit));
      // Tile i's scores with the keys in load nk; after the last of them its queries may be replaced.
      auto issue_scores = [&](int i, int nk, bool last) {
        tc_fence_after_sync();
        mma.scores(i, desc_of(nk));
        commit(&t.s_full_bar[i]);
        if (last) commit(&t.q_empty_bar[i]);
      };
      auto first_scores = [&](int i, int nk, bool last) -> bool {
        const bool there = mbar_wait(&t.q_full_bar[i], q_phase[i], &abort_flag) && wait_full(nk);
        q_phase[i] ^= 1;
        if (there) issue_scores(i, nk, last);
        return there;
      };
      bool started[kTiles] = {false, false};  // the tile's first scores of the unit are under way
      for (int count = 1; ok && unit >= 0; ++count) {
        if (now.total > 0) {
#pragma unroll
          for (int i = 0; i < kTiles; ++i) {
            if (ok && !started[i] && now.blocks[i] > 0) ok = first_scores(i, n, now.blocks[i] == 1);
          }
          if (!ok) break;
          commit(&t.slot_empty_bar[n % S]);
        }
        started[0] = started[1] = false;
        bool known = false;
        Todo next;
        auto find_next = [&]() -> bool {
          known = true;
          if (!next_unit(count, &unit)) return false;
          if (unit >= 0) next = Todo(Unit(p, unit));
          return true;
        };
        for (int j = 0; j < now.total && ok; ++j) {
          const bool more = j + 1 < now.total;
          const int nv = n + 2 * j + 1, nk = nv + 1;  // (nk: of this unit's next block or the next unit's first)
          if (!wait_full(nv)) ok = false;
          bool unclean = now.dirty.has(j);
#pragma unroll
          for (int i = 0; i < kTiles; ++i) {
            if (!ok || j >= now.blocks[i]) continue;
            // The product reads P from the columns the next scores overwrite: the instructions of one
            // thread run in the order they were issued.
#pragma unroll
            for (int part = 0; part < kPParts; ++part) {
              if (unclean) {
                ok = mbar_wait(&t.slot_clean_bar[nv % S], (clean_phase >> (nv % S)) & 1, &abort_flag);
                clean_phase ^= 1u << (nv % S);
                unclean = false;
              }
              if (ok) ok = mbar_wait(&t.p_full_bar[i][part], p_phase[i], &abort_flag);
              if (!ok) break;
              tc_fence_after_sync();
              mma.product(i, part, desc_of(nv), j == 0 ? 1u : 0u);
            }
            if (!ok) continue;
            p_phase[i] ^= 1;
            if (j + 1 < now.blocks[i]) {
              if (!wait_full(nk)) {  // (seen by the first tile's turn, for the second's too)
                ok = false;
              } else {
                issue_scores(i, nk, j + 2 == now.blocks[i]);
              }
              continue;
            }
            commit(&t.pv_done_bar[i]);  // (a block's scores, which the softmax waits for, follow its product)
            if (more) continue;
            // Through with the unit: on with the first scores of the next one, which run under the
            // other tile's last product and this one's output.
            if (!known) ok = find_next();
            if (ok && next.blocks[i] > 0) {
              started[i] = true;
              ok = first_scores(i, nk, next.blocks[i] == 1);
            }
          }
          if (!ok) break;
          commit(&t.slot_empty_bar[nv % S]);  // both tiles have read the two slots
          if (more) commit(&t.slot_empty_bar[nk % S]);
        }
        n += 2 * now.total;
        if (ok && !known) ok = find_next();
        now = next;
      }
      if (!ok && issuer) {
        abort_flag = 1;
        atomicCAS(p.status, 0u, kStatusAttentionTimeout);
      }
    } else {
      // ------------------------------------------------------------------ values that are not seen by all
      using Large = TooLarge<BF16>;
      const int which = static_cast<int>(warp) - kHelpWarp;
      bool ok = true;
      int n = 0;
      int unit = blockIdx.x;
      for (int count = 1; ok && unit >= 0; ++count) {
        const Unit u(p, unit);
        // (Every load is waited for and its slot given back, so that none is filled again before its turn here.)
        for (int j = 0; j < u.walk.count && ok; ++j) {
          const int nk = n + 2 * j, nv = nk + 1;
          ok = __all_sync(0xffffffffu, mbar_wait(&t.slot_full_bar[nk % S], (nk / S) & 1, &abort_flag));
          if (ok && lane == 0) mbar_arrive(&t.slot_empty_bar[nk % S]);
          ok = ok && __all_sync(0xffffffffu, mbar_wait(&t.slot_full_bar[nv % S], (nv / S) & 1, &abort_flag));
          if (!ok) break;
          if (!u.walk.dirty.has(j)) {
            if (lane == 0) mbar_arrive(&t.slot_empty_bar[nv % S]);
            continue;
          }
          uint8_t *block = slot(nv % S) + lane * 16;
          const int x0 = u.walk.place0(j);
          uint32_t odd = 0;  // sign bits
#pragma unroll 1  // (unrolled by four: 157 us instead of 151, 8192 tokens under a window; the kernel's instructions no longer fit so well)
          for (int r = which * 4; r < kBlockKv; r += kHelpWarps * 4) {  // four keys' 128 bytes of an atom
            const int x = x0 + r + static_cast<int>(lane >> 3);
            const bool hidden = u.walk.hidden(x), mixed = !hidden && u.walk.mixed(x);
#pragma unroll
            for (int a = 0; a < L::kQAtoms; ++a) {
              uint4 *at = reinterpret_cast<uint4 *>(block + a * kBlockKv * kAtomBytes + r * kAtomBytes);
              if (hidden) *at = make_uint4(0, 0, 0, 0);
              if (mixed) {
                const uint4 w = *at;
                odd |= Large::signs(w.x) | Large::signs(w.y) | Large::signs(w.z) | Large::signs(w.w);
              }
            }
          }
          bool taken = false;
          if (__any_sync(0xffffffffu, (odd & 0x80008000u) != 0)) {
#pragma unroll 1
            for (int r = which * 4; r < kBlockKv; r += kHelpWarps * 4) {
              if (u.walk.hidden(x0 + r + static_cast<int>(lane >> 3)) || !u.walk.mixed(x0 + r + static_cast<int>(lane >> 3))) continue;
              for (int a = 0; a < L::kQAtoms; ++a) {
                uint4 *at = reinterpret_cast<uint4 *>(block + a * kBlockKv * kAtomBytes + r * kAtomBytes);
                const uint4 w = *at;
                *at = Large::without(w);
                taken = taken || Large::any(w);
              }
            }
          }
          if (taken) *reinterpret_cast<volatile uint32_t *>(&t.patch_flag[count & 3]) = static_cast<uint32_t>(count);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            mbar_arrive(&t.slot_clean_bar[nv % S]);
            mbar_arrive(&t.slot_empty_bar[nv % S]);
          }
        }
        n += 2 * u.walk.count;
        if (ok) ok = next_unit(count, &unit);
      }
      if (!ok && lane == 0) {
        abort_flag = 1;
        atomicCAS(p.status, 0u, kStatusAttentionTimeout);
      }
    }
  }

  // ---------------------------------------------------------------------- teardown
  tc_fence_before_sync();
  __syncthreads();
  if (abort_flag != 0) {
    // A wait gave up: copies that may still be in flight land before the shared memory they target is released.
    for (int i = 0; i < 64; ++i) __nanosleep(2000);
    __syncthreads();
  }
  if (warp == kMmaWarp) {
    tc_fence_after_sync();
    tmem_dealloc<1>(tmem_base, L::kTmemCols);
  }
}

template <int D, bool BF16>
cudaError_t launch(const CUtensorMap &tq, const CUtensorMap (&maps)[6], const TilesParams &p, int64_t ctas, cudaStream_t stream) {
  using L = Layout<D>;
  auto kernel = cache_tiles_kernel<D, BF16>;
  static const cudaError_t attr_set = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, L::kSmemBytes);
  if (attr_set != cudaSuccess) return attr_set;
  return launch_overlapped(kernel, ctas, kThreads, L::kSmemBytes, stream, tq, maps[0], maps[1], maps[2], maps[3], maps[4], maps[5], p);
}

}  // namespace

int cache_tile_rows(int whole) { return kBlockQ / whole * whole; }

int cache_tiles_pairs(int rows, int tile_rows) { return (rows + kTiles * tile_rows - 1) / (kTiles * tile_rows); }

int cache_tiles_positions(int group) { return kTiles * (kBlockQ / group); }

int cache_tiles_splits(int64_t units, int keys, int part_blocks) {
  const int blocks = (keys + kBlockKv - 1) / kBlockKv;
  if (units >= sm_count()) return 1;
  // One CTA an SM, and no more of them than SMs.
  const int wanted = static_cast<int>(std::min<int64_t>(sm_count() / units, std::max(1, (blocks + part_blocks - 1) / part_blocks)));
  const int per_split = (blocks + wanted - 1) / wanted;
  return (blocks + per_split - 1) / per_split;
}

size_t cache_tiles_part_rows(int64_t units, int splits, int tile_rows) { return static_cast<size_t>(units) * splits * kTiles * tile_rows; }

cudaError_t cache_tiles(TilesParams p, const CacheAttentionArgs &a, const char **why) {
  CUtensorMap tq, maps[6];  // of q; of k and v, the same in boxes of 16 positions, of the prefix
  p.by_runs = Divisor::of(static_cast<uint32_t>(p.runs));
  p.by_splits = Divisor::of(static_cast<uint32_t>(p.splits));
  {  // A tile's rows as a box: the heads of a group, a run of queries, and over a prefix a run of sequences.
    const uint64_t dims[4] = {static_cast<uint64_t>(a.head_dim) * 2, static_cast<uint64_t>(a.heads), static_cast<uint64_t>(a.q_len),
                              static_cast<uint64_t>(a.batch)};
    auto bytes = [&](int64_t s, int extent) { return static_cast<uint64_t>(extent > 1 ? s : a.head_dim) * 2; };
    const uint64_t strides[3] = {bytes(a.q_stride[1], a.heads), bytes(a.q_stride[2], a.q_len), bytes(a.q_stride[0], a.batch)};
    const int queries = p.over_batch ? a.q_len : p.tile_rows / p.group;
    const uint32_t box[3] = {static_cast<uint32_t>(p.group), static_cast<uint32_t>(queries), static_cast<uint32_t>(p.tile_rows / (p.group * queries))};
    if (!make_tmap(&tq, a.q, 4, dims, strides, box)) {
      *why = "cuTensorMapEncodeTiled refused q";
      return cudaErrorInvalidValue;
    }
  }
  const bool own = !p.over_batch, prefix = p.prefix_len > 0;
  for (int i = 0; own && i < 4; ++i) {
    const int64_t *stride = i % 2 == 0 ? a.k_stride : a.v_stride;
    if (!row_map(&maps[i], i % 2 == 0 ? a.k : a.v, a.head_dim, a.kv_len, a.kv_heads, a.batch, stride[0], stride[1], stride[2], i < 2 ? kBlockKv : kBoxRows)) {
      *why = "cuTensorMapEncodeTiled refused k or v";
      return cudaErrorInvalidValue;
    }
  }
  if (prefix && (!row_map(&maps[4], a.prefix_k, a.head_dim, a.prefix_len, a.kv_heads, 1, 0, a.prefix_k_stride[0], a.prefix_k_stride[1], kBlockKv) ||
                 !row_map(&maps[5], a.prefix_v, a.head_dim, a.prefix_len, a.kv_heads, 1, 0, a.prefix_v_stride[0], a.prefix_v_stride[1], kBlockKv))) {
    *why = "cuTensorMapEncodeTiled refused the prefix";
    return cudaErrorInvalidValue;
  }
  // (the others are not used)
  if (!own) maps[0] = maps[2] = maps[4], maps[1] = maps[3] = maps[5];
  if (!prefix) maps[4] = maps[0], maps[5] = maps[1];
  const int64_t ctas = static_cast<int64_t>(p.runs) * p.row_pairs * p.splits;
  *why = "launching the tile kernel";
  cudaError_t e = a.head_dim == 64 ? (a.is_bf16 ? launch<64, true>(tq, maps, p, ctas, a.stream) : launch<64, false>(tq, maps, p, ctas, a.stream))
                                   : (a.is_bf16 ? launch<128, true>(tq, maps, p, ctas, a.stream) : launch<128, false>(tq, maps, p, ctas, a.stream));
  if (e != cudaSuccess || p.over_batch || p.splits == 1) return e;
  *why = "launching the kernel that adds the parts";
  const int64_t total = static_cast<int64_t>(p.runs) * p.rows * (a.head_dim / 4);
  auto join = a.head_dim == 64 ? (a.is_bf16 ? join_tiles_kernel<64, true> : join_tiles_kernel<64, false>)
                               : (a.is_bf16 ? join_tiles_kernel<128, true> : join_tiles_kernel<128, false>);
  return launch_overlapped(join, (total + 127) / 128, 128, 0, a.stream, p, Divisor::of(static_cast<uint32_t>(p.rows)), Divisor::of(static_cast<uint32_t>(p.tile_rows)), total);
}

}  // namespace flsm100
