// zs_splits.hip -- the merge of an attention's splits (gfx950).
#include "zs_splits.hpp"

namespace zs {

__device__ __forceinline__ int64_t out_row(const SplitMerge& p, int64_t row) {
  if (p.new_tokens.d == 1) return row;
  const uint32_t bh = p.new_tokens.div((uint32_t)row), i = (uint32_t)row - bh * p.new_tokens.d;
  const uint32_t b = p.over_heads.div(bh), h = bh - b * p.over_heads.d;
  return ((int64_t)b * p.new_tokens.d + i) * p.heads + h;
}

// The splits of one row merged by four waves: their weights by a
// lane each, then a wave takes every fourth split, eight loads in flight.
constexpr int kMergeChunk = 256;

template <int D>
__global__ __launch_bounds__(kMergeWaves * 64) void merge_kernel(SplitMerge p) {
  constexpr int kV = D / 64;  // values a lane
  __shared__ float weight[kMergeChunk];
  __shared__ float red[kMergeWaves];
  __shared__ float part[kMergeWaves][D];
  const int64_t head = blockIdx.x;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = lane_id();
  const float2* ml = reinterpret_cast<const float2*>(p.ws_ml) + head * p.splits;
  const float* o = p.ws_o + head * p.splits * D + kV * l;
  float m_run = -INFINITY, sum = 0.f, acc[kV] = {};
  for (int c0 = 0; c0 < p.splits; c0 += kMergeChunk) {
    const int n = min(p.splits - c0, kMergeChunk);
    const float2 own = tid < n ? ml[c0 + tid] : float2{-INFINITY, 0.f};
    float x[8][kV];
    auto load = [&](int s0) {
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int s = s0 + kMergeWaves * j;
#pragma unroll
        for (int i = 0; i < kV; ++i) x[j][i] = s < n ? o[(int64_t)(c0 + s) * D + i] : 0.f;
      }
    };
    load(w);
    float m = own.x;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
    __syncthreads();  // the last chunk's weights are read
    if (l == 0) red[w] = m;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kMergeWaves; ++i) m = fmaxf(m, red[i]);
    m = fmaxf(m, m_run);
    const float m_use = m == -INFINITY ? 0.f : m;
    const float alpha = __builtin_amdgcn_exp2f(m_run - m_use);
    const float f = __builtin_amdgcn_exp2f(own.x - m_use);
    weight[tid] = f;
    sum = sum * alpha + own.y * f;  // this thread's splits
#pragma unroll
    for (int i = 0; i < kV; ++i) acc[i] *= alpha;
    m_run = m;
    __syncthreads();
    for (int s0 = w; s0 < n; s0 += 8 * kMergeWaves) {
      if (s0 > w) load(s0);
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const float g = s0 + kMergeWaves * j < n ? weight[s0 + kMergeWaves * j] : 0.f;
#pragma unroll
        for (int i = 0; i < kV; ++i) acc[i] += x[j][i] * g;
      }
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
  __syncthreads();
  if (l == 0) red[w] = sum;
#pragma unroll
  for (int i = 0; i < kV; ++i) part[w][kV * l + i] = acc[i];
  __syncthreads();
  if (tid >= D / 2) return;
  sum = 0.f;
  float2 x = {0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kMergeWaves; ++i) {
    sum += red[i];
    x.x += part[i][2 * tid];
    x.y += part[i][2 * tid + 1];
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  *reinterpret_cast<uint32_t*>(p.out + out_row(p, head) * D + 2 * tid) = pack_bf16x2(x.x * inv, x.y * inv);
  if (p.lse && tid == 0) p.lse[head] = sum == 0.f ? -INFINITY : (m_run + __log2f(sum)) * 0.6931471805599453f;
}

hipError_t merge_splits(hipStream_t stream, const SplitMerge& p, int head_dim) {
  const dim3 grid((unsigned)p.rows), block(kMergeWaves * 64);
  if (head_dim == 128)
    hipLaunchKernelGGL(merge_kernel<128>, grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL(merge_kernel<64>, grid, block, 0, stream, p);
  return hipGetLastError();
}

}  // namespace zs
