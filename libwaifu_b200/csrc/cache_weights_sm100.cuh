// The sums of the keys' weights over many queries (cache_weights_sm100.cu), as cache_rows_sm100.cu plans and launches them.
#pragma once

#include <cuda_runtime.h>
#include <stdint.h>

#include "cache_attention_sm100.cuh"
#include "cache_common_sm100.cuh"

namespace flsm100 {

struct WeightsParams {
  const int32_t *kv_lens;
  int is_bf16;
  int kv_heads, group, q_len, kv_len;
  int runs;         // (sequence, key-value head)
  int pairs;        // of 128 keys
  int rows;         // packed rows of a run: query r / group of head r % group
  int tile_rows;    // of a block of them: whole queries
  int positions;    // tile_rows / group
  Divisor by_positions;
  int parts;        // CTAs that divide a pair's blocks of rows, part_blocks each
  int part_blocks;
  float scale_log2;
  const float2 *row_norm;  // (run, norm_pitch), 128 to a block: a row's maximum in log2 units and 1 / sum
  int norm_pitch;
  float *part_sums;  // (run, pair, part, 256)
  uint32_t *counters;
  const float *weights_in;
  float *weights_out;
  int64_t in_stride[2], out_stride[2];
  uint32_t *status;
};

struct WeightsPlan {
  int pairs, parts, part_blocks;
  size_t part_bytes;
  int64_t ctas;
};

int cache_weights_norm_pitch(int rows, int tile_rows);  // 128 to a block, and to an even number of them
// At most `most_units` walks may be divided.
WeightsPlan cache_weights_plan(const CacheAttentionArgs &a, int tile_rows, int most_units);
cudaError_t cache_weights(const WeightsParams &p, const CacheAttentionArgs &a, const char **why);

}  // namespace flsm100
