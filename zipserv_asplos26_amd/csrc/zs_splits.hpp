// zs_splits.hpp -- the partial results of an attention whose sequences are cut
// into splits, and their merge (zs_splits.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "zs_device.hpp"

namespace zs {

constexpr int kMergeWaves = 4;  // of a row's workgroup

// Row r is new token r % new_tokens of (sequence, head) r / new_tokens: that is also
// the order of lse; out is [sequence][new token][head][D].
struct SplitMerge {
  const float* ws_o;   // [row][split][D], not divided by the split's sum
  const float* ws_ml;  // [row][split][2]: maximum (log2 domain) and sum
  uint16_t* out;
  float* lse;          // or null
  int splits, rows, heads;
  FastDiv new_tokens, over_heads;

  static SplitMerge of(const float* ws_o, const float* ws_ml, uint16_t* out, float* lse, int splits, int rows,
                       int heads, int new_tokens) {
    return SplitMerge{ws_o, ws_ml, out, lse, splits, rows, heads, FastDiv::of(new_tokens), FastDiv::of(heads)};
  }
};

hipError_t merge_splits(hipStream_t stream, const SplitMerge& p, int head_dim);

}  // namespace zs
