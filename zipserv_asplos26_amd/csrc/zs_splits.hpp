// zs_splits.hpp -- the partial results of an attention whose sequences are cut
// into splits, and their merge (zs_splits.hip).
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "zs_device.hpp"

namespace zs {

constexpr int kMergeWaves = 4;  // of a row's workgroup

// Row r is (sequence, head) r, its splits are in the slots r * splits and up.
struct SplitMerge {
  const float* ws_o;   // [slot][D], not divided by the split's sum
  const float* ws_ml;  // [slot][2]: maximum (log2 domain) and sum
  uint16_t* out;       // [row][D]
  float* lse;          // [row], or null
  int splits, rows;
};

hipError_t merge_splits(hipStream_t stream, const SplitMerge& p, int head_dim);

// ln(sum 2^m), -inf for no sum.  (The sum's exponent goes to m, in 64 bits, so that neither
// the size of the sum nor that of m costs digits.)
__device__ __forceinline__ float natural_log_sum(float m, double sum) {
  const double log2 = ((double)m + __builtin_amdgcn_frexp_exp(sum)) + __log2f((float)__builtin_amdgcn_frexp_mant(sum));
  return sum == 0. ? -INFINITY : (float)(log2 * 0.69314718055994530942);
}

// Slots of [heads_k][columns] rows, a column being new token * group + head of the
// group, a row the result over the slot's tokens and the sum of their weights, relative to
// a power of two; out is [sequence][new token][head][D], lse [sequence][head][new token].  A
// sequence's slots are b * splits and up, or with a plan, (first, number) a sequence,
// the first and then first / 2 * 2 + 2, + 4, ...; a sequence of one is written already.
struct PartMerge {
  const float* ws_o;   // [slot][row][D]
  const float* ws_ml;  // [slot][row][2]: the power's log2 (-FLT_MAX for no weight), the sum
  const int2* plan;    // or null
  uint16_t* out;
  float* lse;
  int splits, columns, new_tokens;
  FastDiv over_group, over_heads_k, over_pieces;  // (the last two are set by the call)
};

constexpr int kPartMergeThreads = 512;  // of each of merge_parts_groups() workgroups
int64_t merge_parts_groups(int batch, int heads_k, int64_t columns);
hipError_t merge_parts(hipStream_t stream, PartMerge p, int batch, int heads_k, int head_dim);

}  // namespace zs
