// The kernel over a key-value cache for many query rows (cache_tiles_sm100.cu), as cache_rows_sm100.cu plans and launches it.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "cache_attention_sm100.cuh"
#include "cache_common_sm100.cuh"

namespace flsm100 {

struct TilesParams {
  const uint16_t *q, *k, *v;
  uint16_t *out;
  int64_t q_stride[3], k_stride[3], v_stride[3], out_stride[3];
  const int32_t *kv_lens;
  int kv_heads, group, q_len, kv_len;
  int window, sinks;
  int prefix_len;   // keys that every row sees, walked first; 0 without
  bool over_batch;  // the rows of the whole batch over the prefix alone: parts only
  int runs;         // (sequence, key-value head), or the heads alone
  int rows;         // packed rows of a run
  int tile_rows;    // cache_tile_rows()
  int row_pairs;    // pairs of tiles of so many of them
  int splits;       // CTAs that divide a pair's blocks of keys
  Divisor by_kv_heads, by_group, by_sequence_rows;  // (the last: group * q_len)
  Divisor by_runs, by_splits;  // set by cache_tiles()
  float scale_log2;
  float *part_out;   // (kv_head, split, rows, D) over a prefix, (run, pair, split, rows of a pair, D) else
  float2 *part_sum;  // the same without D: maximum in log2 units, sum
  float2 *row_norm;  // (run, norm_pitch), 128 to a tile: a row's maximum and 1 / sum, or null
  int norm_pitch;
  uint32_t *status;
};

// The rows of a tile: as many as go into 128 of `whole` rows each (a query's heads; over a prefix a sequence's rows).
int cache_tile_rows(int whole);
int cache_tiles_pairs(int rows, int tile_rows);
int cache_tiles_positions(int group);  // the most that the rows of a pair lie on
// `keys`: the most that a pair's rows see between them; parts of about `part_blocks` blocks of 128 of them, longer ones where
// there were more than SMs.
int cache_tiles_splits(int64_t units, int keys, int part_blocks);
size_t cache_tiles_part_rows(int64_t units, int splits, int tile_rows);
// Two launches where a pair's blocks are divided and the rows are not those of a whole batch over a prefix: the second adds the parts.
cudaError_t cache_tiles(TilesParams p, const CacheAttentionArgs &a, const char **why);

}  // namespace flsm100
