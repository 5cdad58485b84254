// zs_splits.hip -- the merge of an attention's splits (gfx950).
#include "zs_splits.hpp"

#include <cfloat>
#include <type_traits>

namespace zs {

// The splits of one row merged by four waves: their weights by a
// lane each, then a wave takes every fourth split, eight loads in flight.
constexpr int kMergeChunk = 256;

template <int D>
__global__ __launch_bounds__(kMergeWaves * 64) void merge_kernel(SplitMerge p) {
  constexpr int kV = D / 64;  // values a lane
  __shared__ float weight[kMergeChunk];
  __shared__ float red[kMergeWaves];
  __shared__ float part[kMergeWaves][D];
  const int64_t row = blockIdx.x;
  const int tid = threadIdx.x, w = __builtin_amdgcn_readfirstlane(tid >> 6), l = lane_id();
  const float2* ml = reinterpret_cast<const float2*>(p.ws_ml) + row * p.splits;
  const float* o = p.ws_o + row * p.splits * D + kV * l;
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
  *reinterpret_cast<uint32_t*>(p.out + row * D + 2 * tid) = pack_bf16x2(x.x * inv, x.y * inv);
  if (p.lse && tid == 0) p.lse[row] = sum == 0.f ? -INFINITY : (m_run + __log2f(sum)) * 0.6931471805599453f;
}

// Eight columns of a (sequence, KV head) by eight waves: a wave has a column, or where there
// are fewer several share one, every kShare-th split each.  Most workgroups of a
// batch whose sequences are whole have nothing to do, so there are few of them.
constexpr int kPartWaves = kPartMergeThreads / 64;

template <int D, int kShare>
__global__ __launch_bounds__(kPartWaves * 64) void merge_parts_kernel(PartMerge p) {
  constexpr int kV = D / 64, kColumns = kPartWaves / kShare, kAtOnce = 8;
  __shared__ double part[kPartWaves][D + 2];
  const uint32_t bh = p.over_pieces.div(blockIdx.x), piece = blockIdx.x - bh * p.over_pieces.d;
  const uint32_t b = p.over_heads_k.div(bh), h = bh - b * p.over_heads_k.d;
  int first = b * p.splits, next = first + 1, step = 1, splits = p.splits;
  if (p.plan) {
    const int2 mine = p.plan[b];
    first = mine.x;
    next = (first & ~1) + 2;
    step = 2;
    splits = mine.y;
  }
  if (splits <= 1) return;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id();
  const int column = piece * kColumns + w / kShare, share = w % kShare;
  const bool live = column < p.columns;
  const int64_t rows = (int64_t)p.over_heads_k.d * p.columns, at = (int64_t)h * p.columns + column;
  auto slot = [&](int i) { return (i == 0 ? first : next + (i - 1) * step) * rows + at; };
  // Sums in 64 bits: a sum of weights times a result that fits fp32 need not, and powers of two
  // apart by any number of a split's are exact.
  auto scaled = [](double x, float log2) { return ldexp(x, (int)fmaxf(log2, -4000.f)); };
  float m_run = -FLT_MAX;
  double sum = 0., acc[kV] = {};
  for (int c0 = share; live && c0 < splits; c0 += 64 * kShare) {
    // 64 splits of this wave's: a lane's own reference and sum, then their results
    const int n = min((splits - c0 + kShare - 1) / kShare, 64);
    const float2* ml = reinterpret_cast<const float2*>(p.ws_ml);
    const float2 own = l < n ? ml[slot(c0 + l * kShare)] : float2{-FLT_MAX, 0.f};
    float x[kAtOnce][kV];
    auto load = [&](int s0) {
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        const float* o = p.ws_o + slot(c0 + min(s0 + j, n - 1) * kShare) * D + kV * l;
#pragma unroll
        for (int i = 0; i < kV; ++i) x[j][i] = o[i];
      }
    };
    load(0);
    float m = own.x;
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) m = fmaxf(m, __shfl_xor(m, off));
    m = fmaxf(m, m_run);
    const double f = scaled(own.y, own.x - m);
    sum = scaled(sum, m_run - m) + f;  // of this lane's splits (0 past the last)
#pragma unroll
    for (int i = 0; i < kV; ++i) acc[i] = scaled(acc[i], m_run - m);
    m_run = m;
    const uint64_t bits = __builtin_bit_cast(uint64_t, f);
    for (int s0 = 0; s0 < n; s0 += kAtOnce) {
      if (s0) load(s0);
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        const uint32_t lower = __builtin_amdgcn_readlane((uint32_t)bits, min(s0 + j, 63));
        const uint32_t upper = __builtin_amdgcn_readlane((uint32_t)(bits >> 32), min(s0 + j, 63));
        const double g = __builtin_bit_cast(double, (uint64_t)upper << 32 | lower);
#pragma unroll
        for (int i = 0; i < kV; ++i) acc[i] = s0 + j < n ? fma((double)x[j][i], g, acc[i]) : acc[i];
      }
    }
  }
#pragma unroll
  for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off);
  if constexpr (kShare > 1) {
#pragma unroll
    for (int i = 0; i < kV; ++i) part[w][kV * l + i] = acc[i];
    if (l == 0) part[w][D] = m_run, part[w][D + 1] = sum;
    __syncthreads();
    if (share != 0) return;
    float m = -FLT_MAX;
#pragma unroll
    for (int i = 0; i < kShare; ++i) m = fmaxf(m, (float)part[w + i][D]);
    sum = 0.;
#pragma unroll
    for (int i = 0; i < kV; ++i) acc[i] = 0.;
#pragma unroll
    for (int i = 0; i < kShare; ++i) {
      const float less = (float)part[w + i][D] - m;
      sum += scaled(part[w + i][D + 1], less);
#pragma unroll
      for (int j = 0; j < kV; ++j) acc[j] += scaled(part[w + i][kV * l + j], less);
    }
    m_run = m;
  }
  if (!live) return;
  const double inv = sum == 0. ? 0. : 1. / sum;
  const int fresh = (int)p.over_group.div((uint32_t)column), group = (int)p.over_group.d;
  const int heads = group * (int)p.over_heads_k.d, head = h * group + column - fresh * group;
  uint16_t* out = p.out + (((int64_t)b * p.new_tokens + fresh) * heads + head) * D;
  if constexpr (kV == 2)
    *reinterpret_cast<uint32_t*>(out + 2 * l) = pack_bf16x2((float)(acc[0] * inv), (float)(acc[1] * inv));
  else
    out[l] = (uint16_t)pack_bf16x2((float)(acc[0] * inv), 0.f);
  if (p.lse && l == 0)
    p.lse[((int64_t)b * heads + head) * p.new_tokens + fresh] = natural_log_sum(m_run, sum);
}

hipError_t merge_splits(hipStream_t stream, const SplitMerge& p, int head_dim) {
  const dim3 grid((unsigned)p.rows), block(kMergeWaves * 64);
  if (head_dim == 128)
    hipLaunchKernelGGL(merge_kernel<128>, grid, block, 0, stream, p);
  else
    hipLaunchKernelGGL(merge_kernel<64>, grid, block, 0, stream, p);
  return hipGetLastError();
}

// Columns of a workgroup: one, where there are so few rows that eight waves for each
// leave CUs idle (32 rows of 64 splits: 4 us, 6 with two waves for each), else eight.
static int columns_at_once(int batch, int heads_k, int64_t columns) {
  return (int64_t)batch * heads_k * columns <= 512 ? 1 : 8;
}

int64_t merge_parts_groups(int batch, int heads_k, int64_t columns) {
  const int at_once = columns_at_once(batch, heads_k, columns);
  return (int64_t)batch * heads_k * ((columns + at_once - 1) / at_once);
}

hipError_t merge_parts(hipStream_t stream, PartMerge p, int batch, int heads_k, int head_dim) {
  const int at_once = columns_at_once(batch, heads_k, p.columns);
  p.over_heads_k = FastDiv::of(heads_k);
  p.over_pieces = FastDiv::of((p.columns + at_once - 1) / at_once);
  const dim3 grid((unsigned)merge_parts_groups(batch, heads_k, p.columns)), block(kPartMergeThreads);
  auto launch = [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    if (at_once == 1)
      hipLaunchKernelGGL((merge_parts_kernel<D, 8>), grid, block, 0, stream, p);
    else
      hipLaunchKernelGGL((merge_parts_kernel<D, 1>), grid, block, 0, stream, p);
    return hipGetLastError();
  };
  return head_dim == 128 ? launch(std::integral_constant<int, 128>{}) : launch(std::integral_constant<int, 64>{});
}

}  // namespace zs
