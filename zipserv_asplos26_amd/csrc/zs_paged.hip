// zs_paged.hip -- the state of an appendable paged KV cache (gfx950): block
// tables and slot maps from the requests' lengths, new keys and values into
// their slots with the bounds of the pages that they fall into, and the pages
// that a query's attention should read, chosen by those bounds.
//
// A pool has num_blocks pages [page][Hkv][D]; token t of sequence b is row
// t % page of page table[b][t / page], its slot that page * page + t % page.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <climits>
#include <cstddef>
#include <type_traits>

#include "../../include/zipserv.h"
#include "zs_device.hpp"

namespace zs {

// ---------------------------------------------------------------------------
// Plan of a step
// ---------------------------------------------------------------------------
// Sequence b has c_b tokens in ceil(c_b / page) pages and brings n_b more; the
// new tokens of all sequences stand one behind another, at most max_tokens of
// them.  Pages are taken in the order of the sequences from the end of the list
// of free ones: the g-th new page is free[F - 1 - g].  So every token's place
// follows from two prefix sums over the sequences, of tokens and of new pages.
//
// One launch: every workgroup makes both sums for itself (8 bytes a sequence,
// from L2) and then places its 512 tokens by a search over the first sum.  A
// table entry is written by the token that opens its page and read only for
// pages that the sequence had before, so no workgroup waits for another.  What it
// takes is latency: loads, two barriers a chunk of sequences, a search in LDS; 3.5 us
// for one sequence, 4.7 for 300 with 24400 places (6.3 with a scan for each of the
// four counts and 256 sequences a chunk).
constexpr int kPlanThreads = 512;
constexpr int kPlanMaxBatch = 4096;

struct PlanParams {
  const int32_t* context;
  const int32_t* fresh;
  const int32_t* free_pages;
  const int32_t* num_free;
  int32_t* table;
  int64_t table_stride;
  int32_t* slots;
  int32_t* sequences;
  int32_t* positions;
  int32_t* seqlens;
  int32_t* cu_new;
  int32_t* counts;
  int batch, width, free_capacity, max_tokens;
  FastDiv page;
};

// Inclusive sum of a value of 0..2^31 - 1 over the lanes of a wave: two sums of
// 16 bits over DPP, which 32 bits hold.
__device__ __forceinline__ int64_t plan_wave_scan(int x) {
  return ((int64_t)wave_inclusive_scan(x >> 16) << 16) + wave_inclusive_scan(x & 0xFFFF);
}

// The same over the workgroup, and the total.  `sums` is one call's own until the
// workgroup's next barrier but one.
__device__ __forceinline__ int64_t plan_scan(int v, int64_t* sums, int64_t& total) {
  const int w = threadIdx.x >> 6;
  int64_t x = plan_wave_scan(v);
  if (lane_id() == 63) sums[w] = x;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int i = 0; i < kPlanThreads / 64; ++i) {
    const int64_t y = sums[i];
    x += i < w ? y : 0;
    total += y;
  }
  return x;
}

__device__ __forceinline__ int32_t plan_saturate(int64_t x) {
  return (int32_t)min(x, (int64_t)INT_MAX);
}

__global__ __launch_bounds__(kPlanThreads) void plan_kernel(PlanParams p) {
  __shared__ int first[kPlanMaxBatch + 1];      // the sequence's first token of the step
  __shared__ int first_page[kPlanMaxBatch];     // how many pages the ones before it take
  __shared__ int held[kPlanMaxBatch];           // pages that it had
  __shared__ int had[kPlanMaxBatch];            // tokens that it had
  __shared__ int64_t sums[4][kPlanThreads / 64];
  const int page = (int)p.page.d;
  const int64_t F = min(max(*p.num_free, 0), p.free_capacity);
  int64_t tokens = 0, taken = 0;    // of the sequences so far
  int64_t asked = 0, wanted = 0;    // of this thread's
  const bool lead = blockIdx.x == 0;
  auto pages_of = [&](uint32_t n) {
    const uint32_t q = p.page.div(n);
    return (int)(q + (q * page != n));
  };
  for (int b0 = 0, i = 0; b0 < p.batch; b0 += kPlanThreads, i ^= 2) {
    const int b = b0 + threadIdx.x;
    const bool live = b < p.batch;
    const int c = live ? max(p.context[b], 0) : 0;
    const int n_asked = live ? max(p.fresh[b], 0) : 0;
    int n = min(n_asked, INT_MAX - c);
    int64_t total;
    const int64_t end = tokens + plan_scan(n, sums[i], total);
    const int start = (int)min(end - n, (int64_t)p.max_tokens);
    n = (int)min((int64_t)n, p.max_tokens - (int64_t)start);
    tokens += total;
    const uint32_t all = (uint32_t)c + (uint32_t)n;
    const int have = pages_of(c), need = pages_of(all);
    const int more = max(min(need, p.width) - have, 0);
    const int64_t before = taken + plan_scan(more, sums[i + 1], total) - more;
    taken += total;
    asked += n_asked;
    wanted += need - have;
    if (live) {
      first[b] = start;
      first_page[b] = plan_saturate(before);
      held[b] = have;
      had[b] = c;
      if (lead) {
        const int given = (int)min((int64_t)more, max(F - before, (int64_t)0));
        const int64_t room = ((int64_t)have + given) * page;
        p.seqlens[b] = (int)min((int64_t)all, room);
        p.cu_new[b] = start;
      }
    }
  }
  const int used = (int)min(tokens, (int64_t)p.max_tokens);
  if (threadIdx.x == 0) first[p.batch] = used;
  if (lead) {  // (uniform)
    int64_t a = 0, m = 0, unused;
    // (each in halves that a scan takes)
    for (int half = 0; half < 2; ++half) {
      __syncthreads();
      plan_scan((int)(asked >> (half ? 31 : 0) & INT_MAX), sums[0], unused);
      a += half ? unused << 31 : unused;
      plan_scan((int)(wanted >> (half ? 31 : 0) & INT_MAX), sums[1], unused);
      m += half ? unused << 31 : unused;
    }
    if (threadIdx.x == 0) {
      const int64_t given = min(taken, F);
      p.cu_new[p.batch] = used;
      p.counts[0] = plan_saturate(a);
      p.counts[1] = (int)given;
      p.counts[2] = plan_saturate(m - given);
      p.counts[3] = (int)(F - given);
    }
  }
  __syncthreads();
  const int t = blockIdx.x * kPlanThreads + threadIdx.x;
  if (t >= p.max_tokens) return;
  int slot = -1, row = -1, pos = -1;
  if (t < used) {
    int lo = 0, hi = p.batch - 1;  // the last sequence that starts at t or before and has tokens
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (first[mid + 1] > t)
        hi = mid;
      else
        lo = mid + 1;
    }
    row = lo;
    pos = had[row] + (t - first[row]);
    const int lp = (int)p.page.div((uint32_t)pos), off = pos - lp * page;
    if (lp < p.width) {
      int32_t* entry = p.table + row * p.table_stride + lp;
      int block = -1;
      if (lp < held[row]) {
        block = *entry;
      } else {
        const int64_t g = (int64_t)first_page[row] + (lp - held[row]);
        if (g < F) {
          block = p.free_pages[F - 1 - g];
          if (off == 0) *entry = block;
        }
      }
      const int64_t s = (int64_t)block * page + off;
      slot = block >= 0 && s <= INT_MAX ? (int)s : -1;
    }
  }
  p.slots[t] = slot;
  p.sequences[t] = row;
  p.positions[t] = pos;
}

// ---------------------------------------------------------------------------
// Append
// ---------------------------------------------------------------------------
// Row i of k / v goes into slot slots[i] of the pool; a slot outside it is left
// out.  bounds[block][h] = the smallest and the largest key of each channel in
// the page: the token at offset 0 starts them anew, the others widen them; NaNs
// are passed over.  The tokens of one page stand next to one another, a run; the
// workgroup that has a run's first token takes the bounds of the whole run.
//
// A workgroup takes 2048 / D tokens of one KV head, 16 bytes a thread, and passes
// the keys through LDS: the threads of a run's first token go through the run's
// other rows there.  Where the last run goes on behind the workgroup's tokens, all
// its threads read the rest of it (from L2, as another workgroup copies it) and
// meet in LDS.  8000 tokens of 8 heads of 128 in pages of 16: 16.9 us, 78% of the
// rate of a copy; 3001 of 16 heads of 64 in pages of 128: 11.9 us, 6.2 without
// bounds, the rest being the chain of a run's rows.  (One thread group reading a
// whole run, row after row: 30 and 102 us.)
constexpr int kAppendThreads = 256;

struct AppendParams {
  const uint16_t* k;
  const uint16_t* v;
  int64_t k_token, k_head, v_token, v_head;  // strides in elements
  const int32_t* slots;
  uint16_t* k_cache;
  uint16_t* v_cache;
  uint16_t* bounds;  // [blocks][Hkv][2][D] or null
  int tokens, heads_k, num_slots;
  FastDiv page, over_heads;
};

// Eight bf16 as unsigned numbers in the order of their values, -inf 0 and +inf
// kMost, with every NaN behind them (flipping the magnitude of negative ones
// makes the bits a signed order, which is then moved by -inf's place): so the
// smallest number is that of the smallest value, NaNs are passed over, and one that
// is alone stays one.  kMost - x turns the order round for the largest value.
typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));
typedef int16_t i16x8 __attribute__((ext_vector_type(8)));
constexpr uint16_t kMinusInf = 0x807F, kMost = 0xFF01;

__device__ __forceinline__ u16x8 bound_order(u32x4 x) {
  const i16x8 u = __builtin_bit_cast(i16x8, x);
  return __builtin_bit_cast(u16x8, u ^ ((u >> 15) & (int16_t)0x7FFF)) - kMinusInf;
}
__device__ __forceinline__ u32x4 bound_value(u16x8 x) {
  const i16x8 u = __builtin_bit_cast(i16x8, x + kMinusInf);
  return __builtin_bit_cast(u32x4, u ^ ((u >> 15) & (int16_t)0x7FFF));
}
__device__ __forceinline__ void bound_widen(u16x8& low, u16x8& high, u16x8 x) {
  low = __builtin_elementwise_min(low, x);
  high = __builtin_elementwise_min(high, kMost - x);
}

template <int D>
__global__ __launch_bounds__(kAppendThreads) void append_kernel(AppendParams p) {
  constexpr int kLanes = D / 8, kRows = kAppendThreads / kLanes;
  __shared__ u16x8 part[2][kRows][kLanes];
  __shared__ int flags[kRows];
  __shared__ int cross, cross_block, cross_anew;  // the row whose run goes on behind the workgroup's
  const int segment = (int)p.over_heads.div(blockIdx.x), h = blockIdx.x - segment * p.heads_k;
  const int r = threadIdx.x / kLanes, c = threadIdx.x % kLanes;
  const int t0 = segment * kRows, t = t0 + r, page = (int)p.page.d;
  auto slot_of = [&](int i) {
    const int s = i >= 0 && i < p.tokens ? p.slots[i] : -1;
    return s < p.num_slots ? s : -1;
  };
  auto block_of = [&](int s) { return s < 0 ? -1 : (int)p.page.div((uint32_t)s); };
  const int slot = slot_of(t), before = slot_of(t - 1), next = slot_of(t0 + kRows);
  const int block = block_of(slot);
  const bool lead = p.bounds && slot >= 0 && block_of(before) != block;
  u32x4* low = reinterpret_cast<u32x4*>(p.bounds + ((int64_t)block * p.heads_k + h) * 2 * D + 8 * c);
  u32x4 k = {0, 0, 0, 0}, old_low = k, old_high = k;
  if (slot >= 0) {
    k = *reinterpret_cast<const u32x4*>(p.k + t * p.k_token + h * p.k_head + 8 * c);
    const u32x4 v = *reinterpret_cast<const u32x4*>(p.v + t * p.v_token + h * p.v_head + 8 * c);
    if (lead) {
      old_low = low[0];
      old_high = low[D / 8];
    }
    const int64_t at = ((int64_t)slot * p.heads_k + h) * D + 8 * c;
    *reinterpret_cast<u32x4*>(p.k_cache + at) = k;
    *reinterpret_cast<u32x4*>(p.v_cache + at) = v;
  }
  if (!p.bounds) return;
  u16x8 lo = bound_order(k), hi = kMost - lo;
  part[0][r][c] = lo;
  // 1: goes on with the run of the row before, 2: starts a page
  bool anew = slot == block * page;
  if (c == 0) flags[r] = (slot >= 0 && !lead ? 1 : 0) | (anew ? 2 : 0);
  if (threadIdx.x == 0) cross = -1, cross_anew = 0;
  __syncthreads();
  {
    const int f = lane_id() < kRows ? flags[lane_id()] : 0;
    const uint64_t goes_on = __builtin_amdgcn_ballot_w64(f & 1), opens = __builtin_amdgcn_ballot_w64(f & 2);
    if (lead) {
      const int end = r + 1 + __builtin_ctzll(~(goes_on >> (r + 1)));
#pragma unroll 4
      for (int e = r + 1; e < end; ++e) bound_widen(lo, hi, part[0][e][c]);
      anew |= (opens & ((1ull << end) - 1)) >> r;
      if (end == kRows && block_of(next) == block && c == 0) cross = r, cross_block = block;
    }
  }
  __syncthreads();
  if (cross >= 0) {  // (uniform)
    u16x8 more_lo = ~(u16x8)(uint16_t)0, more_hi = more_lo;
    // (a run has `page` tokens at most; its rows are read until none is of it, and
    // four ahead of what is known of them)
    const int end = min(t0 + cross + page, p.tokens);
    for (int i = t0 + kRows + r; i < end; i += 4 * kRows) {
      u32x4 x[4];
      int s[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int row = min(i + j * kRows, end - 1);
        s[j] = i + j * kRows < end ? slot_of(row) : -1;
        x[j] = *reinterpret_cast<const u32x4*>(p.k + row * p.k_token + h * p.k_head + 8 * c);
      }
      bool of_run = false;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        of_run = block_of(s[j]) == cross_block;
        if (of_run) {
          bound_widen(more_lo, more_hi, bound_order(x[j]));
          if (s[j] == cross_block * page && c == 0) cross_anew = 1;
        }
      }
      if (!__builtin_amdgcn_ballot_w64(of_run)) break;
    }
    part[0][r][c] = more_lo;
    part[1][r][c] = more_hi;
    __syncthreads();
    if (r == cross) {
      anew |= cross_anew;
#pragma unroll 4
      for (int i = 0; i < kRows; ++i) {
        lo = __builtin_elementwise_min(lo, part[0][i][c]);
        hi = __builtin_elementwise_min(hi, part[1][i][c]);
      }
    }
  }
  if (lead) {
    if (!anew) {
      lo = __builtin_elementwise_min(lo, bound_order(old_low));
      hi = __builtin_elementwise_min(hi, kMost - bound_order(old_high));
    }
    low[0] = bound_value(lo);
    low[D / 8] = bound_value(kMost - hi);
  }
}

// ---------------------------------------------------------------------------
// Selection
// ---------------------------------------------------------------------------
// score[b][h][p] = max over the group's heads of sum_d max(q_d, 0) kmax_d +
// min(q_d, 0) kmin_d, the largest q.k that the bounds of page p allow, with NaN
// as +inf.  The selection is the one of the exact scores:
//
// score_kernel computes them in fp32 on the matrix cores, with a bound of their
// error.  A product of two bf16 is exact there, and the 2D additions are off by
// 2^-22 of the sum of the products' sizes at most (a rounded one by 2^-24; the
// allowance covers sums aligned and cut inside the instruction), so a score is
// off by less than E = kScoreError * sum |terms| (2^-14 of the sizes; 2^-20.8 was the
// most seen, over values of all sizes, sums that cancel and powers of two).  The
// sum of sizes is a second product, of the same operands without their signs.
// pick_kernel finds a narrow window that holds the top_k-th largest fp32 score,
// 3 E wider on both sides (one for each of two scores that are compared and one for
// the rounding of its ends, and 0.01 of a digit for the digits'): scores above it are
// taken and scores below it are not, whatever their errors.  What lies in it, a few pages, is scored again in 64 bits
// and ranked, ties to the lowest page; where it holds hundreds (long rows cut in
// their middle, equal scores) the choice runs over 64-bit keys.  Rows where the
// bound says nothing (scores or operands so large that products or sums leave
// fp32's range, values that are no numbers) are scored in 64 bits as a whole:
// products are exact there and each of D additions is off by 2^-53.
struct SelectParams {
  const uint16_t* q;
  int64_t q_batch, q_head;  // strides in elements
  const uint16_t* bounds;   // [blocks][Hkv][2][D]
  const int32_t* table;
  int64_t table_stride;
  const int32_t* seqlens;
  int32_t* pages;           // [B][Hkv][top_k]
  float2* scores;           // [B][Hkv][width]: the fp32 score and the sum of its terms' sizes
  int num_blocks, width, page, heads_k, group, top_k, sink, local;
  FastDiv over_heads;
};

__device__ __forceinline__ int select_pages(const SelectParams& p, int b) {
  const int len = max(p.seqlens[b], 0);
  return min(len / p.page + (len % p.page != 0), p.width);
}

// 2 D 2^-22 of the sizes, rounded up (D = 128), and an absolute rest for bounds and
// products below the normal range, which an instruction may take as 0.  The rest
// is one for queries of 0 or 2^-126..2^60; pick_kernel looks for others.  (A bound
// that is not finite makes every sum of sizes not finite.)
constexpr float kScoreError = 1.02f / (1 << 14), kScoreRest = 0x1p-50f;
constexpr uint32_t kQuerySmall = 0x0080, kQueryLarge = 0x5D80;  // 2^-126 and 2^60 in bf16

// max over the 16 lanes of a row, in all of them
__device__ __forceinline__ float row_max16(float x) {
  auto step = [&](auto ctrl) {
    x = fmaxf(x, __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), decltype(ctrl)::value, 0xF, 0xF,
                                                             false)));
  };
  step(std::integral_constant<int, 0x128>{});  // row_ror:8
  step(std::integral_constant<int, 0x124>{});
  step(std::integral_constant<int, 0x122>{});
  step(std::integral_constant<int, 0x121>{});
  return x;
}

// The largest of each of v's four values over the 16 lanes of a row, the one of
// value 2 (l & 1) + (l >> 1 & 1) in lane l: two exchanges that halve the values,
// two that keep one (5 maxima where four whole reductions take 16).
template <int kCtrl>
__device__ __forceinline__ float dpp(float x) {
  return __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(x), kCtrl, 0xF, 0xF, true));
}
__device__ __forceinline__ float row_max16x4(f32x4 v, int l) {
  const bool odd = l & 1, up = l & 2;
  const float a = fmaxf(odd ? v[2] : v[0], dpp<0xB1>(odd ? v[0] : v[2]));  // quad_perm:[1,0,3,2]
  const float b = fmaxf(odd ? v[3] : v[1], dpp<0xB1>(odd ? v[1] : v[3]));
  float x = fmaxf(up ? b : a, dpp<0x4E>(up ? a : b));  // quad_perm:[2,3,0,1]
  x = fmaxf(x, dpp<0x124>(x));                         // row_ror:4
  return fmaxf(x, dpp<0x128>(x));
}

// A workgroup of one wave scores 16 pages for one KV head.  The heads of the same
// pages run next to one another, so a page's bounds are read from memory as one
// piece (32 sequences to 64000 tokens, 64 / 8 heads, 271 MB: selection 81.5 -> 71.3
// us; with 16 pages a wave in place of 64 69.5).  Workgroups of four waves took 11.1
// and 64.8 us where these took 10.4 and 65.4 (one sequence of 32000 tokens, the 32 to
// 64000; 9.3 and 64.5 since the choice's last change), 69.5 and 68.3 us with the
// attention of 16 to 40000.
template <int D>
__global__ __launch_bounds__(64) void score_kernel(SelectParams p) {
  constexpr int kC = D / 32;
  const int b = blockIdx.y;
  const int n = select_pages(p, b);
  const int l = lane_id(), g = l & 15, lg = l >> 4;
  const int tile = (int)p.over_heads.div(blockIdx.x), h = blockIdx.x - tile * p.heads_k, p0 = 16 * tile;
  if (n <= p.top_k || p0 >= n) return;
  // lane i: the place of the wave's page i%16, -1 without one
  int block = -1;
  if (p0 + g < n) block = p.table[b * p.table_stride + p0 + g];
  if (block >= p.num_blocks) block = -1;
  // A page's bounds, 2 D bytes each, come as whole rows (an instruction reads 1 KB of
  // them) and pass through LDS into operand order, one after the other (twice the
  // LDS for both together left the CU fewer waves: 66.8 us for 66.0).
  constexpr int kRow = 2 * D, kPitch = kRow + 16, kRows = 1024 / kRow;
  __shared__ __attribute__((aligned(16))) uint8_t lds[16 * kPitch];
  const int lrow = l / (kRow / 16), lcol = 16 * (l % (kRow / 16));
  const uint8_t* from = reinterpret_cast<const uint8_t*>(p.bounds) + (int64_t)h * 2 * kRow + lcol;
  u32x4 x[kC], y[kC], in[2 * kC];
#pragma unroll
  for (int i = 0; i < kC; ++i) {
    const uint8_t* at = from + (int64_t)max(__shfl(block, i * kRows + lrow), 0) * p.heads_k * (2 * kRow);
    in[i] = *reinterpret_cast<const u32x4*>(at);
    in[kC + i] = *reinterpret_cast<const u32x4*>(at + kRow);
  }
  // the B operands (lane l: head l%16, dims 32c + 8*(l/16)..+7): q's positive and
  // negative parts
  u32x4 qp[kC], qn[kC];
  const uint16_t* qrow = p.q + b * p.q_batch + (h * p.group + (g < p.group ? g : 0)) * p.q_head + 8 * lg;
#pragma unroll
  for (int c = 0; c < kC; ++c) {
    const u32x4 q = *reinterpret_cast<const u32x4*>(qrow + 32 * c);
    const u32x4 neg = __builtin_bit_cast(u32x4, __builtin_bit_cast(i16x8, q) >> 15);
    qp[c] = q & ~neg;
    qn[c] = q & neg;
  }
  const uint32_t no_sign = 0x7FFF7FFFu;
#pragma unroll
  for (int i = 0; i < kC; ++i) *reinterpret_cast<u32x4*>(lds + (i * kRows + lrow) * kPitch + lcol) = in[i];
#pragma unroll
  for (int c = 0; c < kC; ++c) x[c] = *reinterpret_cast<const u32x4*>(lds + g * kPitch + 16 * lg + 64 * c);
#pragma unroll
  for (int i = 0; i < kC; ++i) *reinterpret_cast<u32x4*>(lds + (i * kRows + lrow) * kPitch + lcol) = in[kC + i];
#pragma unroll
  for (int c = 0; c < kC; ++c) y[c] = *reinterpret_cast<const u32x4*>(lds + g * kPitch + 16 * lg + 64 * c);
  f32x4 S = {0.f, 0.f, 0.f, 0.f}, A = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int c = 0; c < kC; ++c) {
    S = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(x[c]), as_bf16x8(qn[c]), S, 0, 0, 0);
    S = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(y[c]), as_bf16x8(qp[c]), S, 0, 0, 0);
    A = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(x[c] & no_sign), as_bf16x8(qn[c] & no_sign), A, 0, 0, 0);
    A = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(y[c] & no_sign), as_bf16x8(qp[c]), A, 0, 0, 0);
  }
  // lane l: head l%16, pages 4*(l/16)..+3 of S and A
  const float s = row_max16x4(S, l);
  float a = row_max16x4(A, l);
  const int at = 4 * lg + 2 * (l & 1) + (l >> 1 & 1);
  // an infinite sum of sizes says that the score is not to be gone by
  if (__shfl(block, at) < 0 || !(a < INFINITY && fabsf(s) < INFINITY)) a = INFINITY;
  if (g < 4 && p0 + at < n) p.scores[((int64_t)b * p.heads_k + h) * p.width + p0 + at] = float2{s, a};
}

// An exact score as a number in its order.
__device__ __forceinline__ uint64_t score_key(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);  // -0 is 0
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

template <int kCtrl>
__device__ __forceinline__ double dpp_add(double x) {
  const uint64_t u = (uint64_t)__double_as_longlong(x);
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (uint32_t)u, kCtrl, 0xF, 0xF, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (uint32_t)(u >> 32), kCtrl, 0xF, 0xF, true);
  return x + __longlong_as_double((int64_t)((uint64_t)hi << 32 | lo));
}

// A page's bounds, eight channels in each of its D / 8 lanes.
struct PageBounds {
  u32x4 low, high;
  bool gone, odd;  // outside the pool; some bound of the lane's is not finite
};

template <int D>
__device__ __forceinline__ PageBounds load_bounds(const SelectParams& p, int b, int h, int lp, int c) {
  PageBounds r;
  const int block = p.table[b * p.table_stride + lp];
  r.gone = block < 0 || block >= p.num_blocks;
  const uint16_t* at = p.bounds + ((int64_t)(r.gone ? 0 : block) * p.heads_k + h) * 2 * D + 8 * c;
  r.low = *reinterpret_cast<const u32x4*>(at);
  r.high = *reinterpret_cast<const u32x4*>(at + D);
  r.odd = false;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    auto bad = [](uint32_t x) { return (x & 0x7F80) == 0x7F80 || (x & 0x7F800000) == 0x7F800000; };
    r.odd |= bad(r.low[i]) || bad(r.high[i]);
  }
  return r;
}

// The exact score of a page for one head, in all of its lanes: NaN as +inf, a page
// outside the pool 0.  A channel's other product is 0 times its bound: nothing, or
// NaN where that is not finite.
template <int D>
__device__ __forceinline__ uint64_t exact_key(const SelectParams& p, const PageBounds& k, int b, int h, int g, int c) {
  const u32x4 u = *reinterpret_cast<const u32x4*>(p.q + b * p.q_batch + (h * p.group + g) * p.q_head + 8 * c);
  double s = k.odd ? NAN : 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    auto at = [&](const u32x4& v) { return i & 1 ? v[i / 2] >> 16 : v[i / 2] & 0xFFFF; };
    const uint32_t q = at(u);
    s = fma((double)bf16_bits_to_f32(q), (double)bf16_bits_to_f32(q >> 15 ? at(k.low) : at(k.high)), s);
  }
  s = dpp_add<0xB1>(s);                              // quad_perm:[1,0,3,2]
  s = dpp_add<0x4E>(s);                              // quad_perm:[2,3,0,1]
  s = dpp_add<0x141>(s);                             // row_half_mirror: eight lanes
  if constexpr (D == 128) s = dpp_add<0x140>(s);     // row_mirror
  return k.gone ? 0 : score_key(s != s ? INFINITY : s);
}

// One workgroup a (sequence, KV head).  What it takes is a chain of short steps, each
// ended by a barrier: so scores are loaded before the row's length is known and stay
// in registers (kKeys a thread; the rest of longer rows is read again), sums
// and maxima run over DPP and ballots, and one pass does all that goes by the window.
// 8 rows of 2000 pages 7 us, of 8188 11 us, 256 rows of 125..4000 11 us.  For the
// first, eight scores a thread took 8 us and sixteen 9.7, the same steps in rolled
// loops over scores in LDS 9.6.
constexpr int kPickBins = 2048;
constexpr int kPickFew = 256;      // pages of the window that are ranked among themselves
constexpr int kPickList = 4096;    // that are scored by themselves and chosen from with the row
constexpr int kPickChunk = 65536;  // pages of a bit map

__device__ __forceinline__ float wave_max(float x) { return wave_max16(row_max16(x)); }

template <int NT>
struct alignas(16) PickLds {
  union {  // (first: its digits are read and cleared 16 bytes at a time)
    int hist[kPickBins];
    uint64_t map[kPickChunk / 64];
    int list[kPickList];
  };
  uint64_t few_key[kPickFew];
  int few_page[kPickFew];
  float red[3][16];
  int sum[NT / 64];
  int bin, above, in, count;
  float low, high;
};

// Writes the pages of [c0, c0 + kPickChunk) whose bits are set, in order, from
// place `base` of the list on; returns the next place.
template <int NT>
__device__ __forceinline__ int pick_write(PickLds<NT>& L, int32_t* out, int base, int c0, int n) {
  const int words = (min(n - c0, kPickChunk) + 63) / 64, tid = threadIdx.x, l = lane_id();
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
#pragma unroll 1
  for (int i0 = 0; i0 < words; i0 += NT) {
    uint64_t m = i0 + tid < words ? L.map[i0 + tid] : 0;
    const int incl = wave_inclusive_scan(__builtin_popcountll(m));
    if (l == 63) L.sum[w] = incl;
    __syncthreads();
    const int s = l < NT / 64 ? L.sum[l] : 0;
    const int upto = wave_inclusive_scan(s);
    int at = base + incl - __builtin_popcountll(m) + __builtin_amdgcn_readlane(upto - s, w);
    base += __builtin_amdgcn_readlane(upto, 63);
    for (; m; m &= m - 1) out[at++] = c0 + 64 * (i0 + tid) + __builtin_ctzll(m);
    __syncthreads();  // the sums and the map are read
  }
  return base;
}

// A row by keys of 64 bits: the key of the last page taken found digit by digit, 8
// bits at a time from the top, until a digit's pages are all taken or none is left.
// Keys are the exact scores of the pages whose fp32 scores lie in [low, high], at
// most kPickList of them, and the most or least for those above or below; or of
// all pages (`window` false).
template <int D, int NT>
__device__ void pick_exact(const SelectParams& p, PickLds<NT>& L, int b, int h, int n, float2* scores, int32_t* out,
                           bool window, float low, float high) {
  constexpr int kLanes = D / 8;
  const int tid = threadIdx.x, l = lane_id(), w = tid >> 6;
  uint64_t* keys = reinterpret_cast<uint64_t*>(scores);
  if (tid == 0) L.count = 0;
  __syncthreads();
  if (window) {
    for (int i = tid; i < n; i += NT) {
      const float x = scores[i].x;
      const bool always = i < p.sink || i >= n - p.local;
      if (always || x > high || x < low)
        keys[i] = always || x > high ? ~0ull : 0;
      else
        L.list[min(atomicAdd(&L.count, 1), kPickList - 1)] = i;
    }
    __syncthreads();
  }
  const int count = window ? L.count : n;
  for (int i = tid / kLanes; i < count; i += NT / kLanes) {
    const int lp = window ? L.list[i] : i;
    uint64_t k = lp < p.sink || lp >= n - p.local ? ~0ull : 0;
    if (k == 0) {
      const PageBounds bounds = load_bounds<D>(p, b, h, lp, tid % kLanes);
      for (int g = 0; g < p.group; ++g) k = max(k, exact_key<D>(p, bounds, b, h, g, tid % kLanes));
    }
    if (tid % kLanes == 0) keys[lp] = k;
  }
  __threadfence_block();
  __syncthreads();
  uint64_t prefix = 0;  // of the keys' bits from `shift` on
  int need = p.top_k, shift = 64;
  while (shift > 0) {
    shift -= 8;
    for (int i = tid; i < 256; i += NT) L.hist[i] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += NT) {
      const uint64_t k = keys[i];
      if (shift == 56 || (k >> (shift + 8)) == prefix) atomicAdd(&L.hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid < 64) {  // four digits a lane, the largest first
      int v[4], sum = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += v[i] = L.hist[255 - 4 * tid - i];
      int above = wave_inclusive_scan(sum) - sum;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (above < need && above + v[i] >= need) {
          L.bin = 255 - 4 * tid - i;
          L.above = above;
          L.in = v[i];
        }
        above += v[i];
      }
    }
    __syncthreads();
    prefix = prefix << 8 | (uint64_t)L.bin;
    need -= L.above;
    if (L.in == need) break;  // (uniform)
  }
  // keys above `prefix` are taken, and the first `need` equal to it
  int base = 0, equal = 0;
  for (int c0 = 0; c0 < n; c0 += kPickChunk) {
    __syncthreads();
    for (int i0 = c0; i0 < min(n, c0 + kPickChunk); i0 += NT) {
      const int i = i0 + tid;
      const uint64_t k = i < n ? keys[i] >> shift : 0;
      const bool is = i < n && k == prefix;
      const uint64_t eq = __builtin_amdgcn_ballot_w64(is);
      __syncthreads();
      if (l == 0) L.sum[w] = __builtin_popcountll(eq);
      __syncthreads();
      int rank = equal + __builtin_popcountll(eq & ((1ull << l) - 1));
      for (int j = 0; j < NT / 64; ++j) {
        if (j < w) rank += L.sum[j];
        equal += L.sum[j];
      }
      const uint64_t take = __builtin_amdgcn_ballot_w64(i < n && (k > prefix || (is && rank < need)));
      if (l == 0 && i < n) L.map[(i - c0) / 64] = take;
    }
    __syncthreads();
    base = pick_write<NT>(L, out, base, c0, n);
  }
}

template <int D, int NT, int kKeys>
__global__ __launch_bounds__(NT) void pick_kernel(SelectParams p) {
  constexpr int kWaves = NT / 64;
  __shared__ PickLds<NT> L;
  static_assert(alignof(PickLds<NT>) >= 16 && offsetof(PickLds<NT>, hist) % 16 == 0, "digits in pieces of 16 bytes");
  const int row = blockIdx.x, b = row / p.heads_k, h = row % p.heads_k, tid = threadIdx.x, l = lane_id();
  const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
  float2* scores = p.scores + (int64_t)row * p.width;
  float2 own[kKeys];
#pragma unroll
  for (int j = 0; j < kKeys; ++j)  // (what lies behind the row's end is not looked at)
    own[j] = j * NT + tid < p.width ? scores[j * NT + tid] : float2{0.f, 0.f};
  // (a group has at most 16 heads: 256 pieces of 8 values)
  static_assert(NT >= 256, "a piece a thread");
  u32x4 query = {0, 0, 0, 0};
  if (tid < p.group * (D / 8)) {
    const int g = tid / (D / 8);
    query = *reinterpret_cast<const u32x4*>(p.q + b * p.q_batch + (h * p.group + g) * p.q_head + 8 * (tid % (D / 8)));
  }
  const int n = select_pages(p, b);
  int32_t* out = p.pages + (int64_t)row * p.top_k;
  if (n <= p.top_k) {
    for (int i = tid; i < p.top_k; i += NT) out[i] = i < n ? i : -1;
    return;
  }
  const int first = p.sink, last = n - p.local;  // the pages between are chosen from
  const int need = p.top_k - p.sink - p.local;
  const bool whole = n <= kKeys * NT;
  // A page's score: NaN for one that is always taken, -inf behind the last one.
  auto marked = [&](int i, float x) { return i >= first && i < last ? x : i < n ? NAN : -INFINITY; };
  float key[kKeys], size = 0.f, lo = INFINITY, hi = -INFINITY;
  auto note = [&](int i, float2 x) {  // the first round's range
    const bool in = i >= first && i < last;
    size = fmaxf(size, in ? x.y : 0.f);
    lo = fminf(lo, in ? x.x : INFINITY);
    hi = fmaxf(hi, in ? x.x : -INFINITY);
  };
#pragma unroll
  for (int j = 0; j < kKeys; ++j) {
    note(j * NT + tid, own[j]);
    key[j] = marked(j * NT + tid, own[j].x);
  }
  // The pages past the registers', f(page, its score) for all lanes of a wave that
  // has one: four loads in flight.
  auto rest = [&](auto f) {
    if (whole) return;
    for (int i0 = kKeys * NT + tid; i0 - l < n; i0 += 4 * NT) {
      float2 x[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = scores[min(i0 + j * NT, n - 1)];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        if (i0 + j * NT - l >= n) break;  // (uniform)
        f(i0 + j * NT, x[j]);
      }
    }
  };
  rest(note);
  {
    const u16x8 u = __builtin_bit_cast(u16x8, query) & (uint16_t)0x7FFF;
    bool odd = false;
#pragma unroll
    for (int j = 0; j < 8; ++j) odd |= u[j] >= kQueryLarge || (u[j] != 0 && u[j] < kQuerySmall);
    if (odd) size = INFINITY;
  }
  size = wave_max(size);
  if (l == 0) L.red[2][w] = size;
  auto each = [&](auto f) {
#pragma unroll
    for (int j = 0; j < kKeys; ++j) f(key[j]);
    rest([&](int i, float2 x) { f(marked(i, x.x)); });
  };

  // The window [low, high] that holds the need-th largest score.  A window of too
  // many pages is cut again.
  float low = -FLT_MAX, high = FLT_MAX;
  int page = -1;  // of the window's, if this thread's one is taken
  bool exact = false, window = false;  // by 64-bit keys; of the window's pages alone
  for (int round = 0;; ++round) {
    if (round > 0) {
      lo = INFINITY, hi = -INFINITY;
      each([&](float x) {
        const bool in = x >= low && x <= high;
        lo = fminf(lo, in ? x : INFINITY);
        hi = fmaxf(hi, in ? x : -INFINITY);
      });
      __syncthreads();  // the last round's maxima and map are read
    }
    lo = -wave_max(-lo);
    hi = wave_max(hi);
    if (l == 0) L.red[0][w] = lo, L.red[1][w] = hi;
    if (tid == 0) L.above = L.count = 0;
#pragma unroll
    for (int i = 4 * tid; i < kPickBins; i += 4 * NT) *reinterpret_cast<u32x4*>(&L.hist[i]) = u32x4{0, 0, 0, 0};
    __syncthreads();
    lo = -row_max16(-L.red[0][l % kWaves]);
    hi = row_max16(L.red[1][l % kWaves]);
    size = row_max16(L.red[2][l % kWaves]);
    if (!(size < INFINITY && hi - lo < INFINITY)) {  // (uniform) some page's score is not to be gone by
      exact = true;
      break;
    }
    if (need > 0) {
      const float scale = hi > lo ? kPickBins / (hi - lo) : 0.f;
      each([&](float x) {
        if (x >= lo && x <= hi) atomicAdd(&L.hist[min((int)((x - lo) * scale), kPickBins - 1)], 1);
      });
      // (in a later round: how many lie above the range)
      int above = 0;
      if (round > 0) {
        each([&](float x) { above += x > hi; });
        above = __builtin_amdgcn_readlane(wave_inclusive_scan(above), 63);
        if (l == 0) atomicAdd(&L.above, above);
      }
      __syncthreads();
      above = L.above;
      constexpr int kPer = kPickBins / NT;  // digits a thread, from the largest
      const int mine = kPickBins - kPer * (tid + 1);
      int v[kPer], sum = 0;
      if constexpr (kPer >= 4) {
#pragma unroll
        for (int i = 0; i < kPer; i += 4) {
          const u32x4 x = *reinterpret_cast<const u32x4*>(&L.hist[mine + i]);
#pragma unroll
          for (int j = 0; j < 4; ++j) v[i + j] = (int)x[j];
        }
      } else {
#pragma unroll
        for (int i = 0; i < kPer; ++i) v[i] = L.hist[mine + i];
      }
#pragma unroll
      for (int i = 0; i < kPer; ++i) sum += v[i];
      const int incl = wave_inclusive_scan(sum);
      if (l == 63) L.sum[w] = incl;
      __syncthreads();
      const int s = l < kWaves ? L.sum[l] : 0;
      int over = above + incl - sum + __builtin_amdgcn_readlane(wave_inclusive_scan(s) - s, w);
      if (over < need && over + sum >= need) {
        int at = mine;
#pragma unroll
        for (int i = kPer - 1; i >= 0; --i) {
          if (over < need) at = mine + i;
          over += v[i];
        }
        // the digit's ends, the margin and what the digits' own rounding may be off by
        const float step = scale > 0.f ? 1.f / scale : 0.f;
        const float margin = 3 * (kScoreError * size + kScoreRest) + 0.01f * step;
        L.low = fmaxf(lo, lo + at * step - margin);
        L.high = fminf(hi, lo + (at + 1) * step + margin);
      }
      if (tid == 0) L.above = 0;
      __syncthreads();
      low = L.low;
      high = L.high;
    } else {
      low = high = INFINITY;  // nothing but the pages that are always taken
    }
    // Taken pages into the map, the window's into the list.
    int taken = 0;
    auto put = [&](int i, float x) {  // the wave's taken pages, a bit each
      if (x >= low && x <= high) {
        const int at = atomicAdd(&L.count, 1);
        if (at < kPickFew) {
          L.few_page[at] = i;
          L.few_key[at] = 0;
        }
      }
      const uint64_t m = __builtin_amdgcn_ballot_w64(!(x <= high));
      taken += __builtin_popcountll(m);
      return m;
    };
    uint64_t word = 0;  // lane j: of the wave's j-th 64 pages
#pragma unroll
    for (int j = 0; j < kKeys; ++j) {
      const uint64_t m = put(j * NT + tid, key[j]);
      word = l == j ? m : word;
    }
    if (l < kKeys) L.map[l * kWaves + w] = word;
    rest([&](int i, float2 x) {
      const uint64_t m = put(i, marked(i, x.x));
      if (i < kPickChunk && l == 0) L.map[i / 64] = m;
    });
    if (l == 0) atomicAdd(&L.above, taken);
    __syncthreads();
    const int in = L.count, left = p.top_k - L.above;
    if (in <= kPickFew) {  // (uniform)
      if (in == left) {
        if (tid < in) page = L.few_page[tid];
        break;
      }
      constexpr int kLanes = D / 8;  // of a page and a head
      for (int i = tid / kLanes; i < in * p.group; i += NT / kLanes) {
        const int at = i / p.group;
        const PageBounds bounds = load_bounds<D>(p, b, h, L.few_page[at], tid % kLanes);
        const uint64_t k = exact_key<D>(p, bounds, b, h, i - at * p.group, tid % kLanes);
        if (tid % kLanes == 0) atomicMax((unsigned long long*)&L.few_key[at], k);
      }
      __syncthreads();
      if (tid < in) {
        const uint64_t k = L.few_key[tid];
        page = L.few_page[tid];
        int rank = 0;
#pragma unroll 4
        for (int i = 0; i < in; ++i) {
          const uint64_t o = L.few_key[i];
          rank += o > k || (o == k && L.few_page[i] < page);
        }
        if (rank >= left) page = -1;
      }
      break;
    }
    if (round == 2) {
      exact = true;
      window = in <= kPickList;
      break;
    }
  }
  if (exact) {  // (uniform)
    __syncthreads();
    pick_exact<D, NT>(p, L, b, h, n, scores, out, window, low, high);
    return;
  }
  if (whole) {
    // every wave sums the bits of all words, and writes its own ones' pages
    if (page >= 0) atomicOr((unsigned long long*)&L.map[page / 64], 1ull << (page & 63));
    __syncthreads();
    constexpr int kPer = kKeys * kWaves > 64 ? 2 : 1;  // words a lane
    static_assert(kKeys * kWaves <= 64 * kPer, "");
    uint64_t m[kPer];
    int c[kPer], sum = 0;
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      m[i] = kPer * l + i < kKeys * kWaves ? L.map[kPer * l + i] : 0;
      sum += c[i] = __builtin_popcountll(m[i]);
    }
    const int before = wave_inclusive_scan(sum) - sum;
#pragma unroll
    for (int j = 0; j < kKeys; ++j) {
      const int at = j * kWaves + w, of = at / kPer, i = at % kPer;
      int base = __builtin_amdgcn_readlane(before, of);
      if (kPer == 2 && i) base += __builtin_amdgcn_readlane(c[0], of);
      const uint64_t mine = kPer == 2 && i ? m[kPer - 1] : m[0];
      const uint32_t lo32 = __builtin_amdgcn_readlane((uint32_t)mine, of);
      const uint32_t hi32 = __builtin_amdgcn_readlane((uint32_t)(mine >> 32), of);
      const uint64_t bits = (uint64_t)hi32 << 32 | lo32;
      if (bits >> l & 1) out[base + __builtin_popcountll(bits & ((1ull << l) - 1))] = j * NT + tid;
    }
    return;
  }
  int base = 0;
  for (int c0 = 0; c0 < n; c0 += kPickChunk) {
    const int end = min(n, c0 + kPickChunk);
    if (c0 > 0) {
      for (int i0 = c0; i0 < end; i0 += NT) {
        const int i = i0 + tid;
        const uint64_t m = __builtin_amdgcn_ballot_w64(!(marked(i, scores[min(i, n - 1)].x) <= high));
        if (l == 0 && i < n) L.map[(i - c0) / 64] = m;
      }
      __syncthreads();
    }
    if (page >= c0 && page < end) atomicOr((unsigned long long*)&L.map[(page - c0) / 64], 1ull << (page & 63));
    __syncthreads();
    base = pick_write<NT>(L, out, base, c0, n);
  }
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Page size, pool and heads that every paged entry point asks for.
int paged_checks(int num_blocks, int page, int heads_k, int head_dim) {
  if (num_blocks <= 0 || page <= 0 || heads_k <= 0) return ZS_E_INVAL;
  if (page % 16 || heads_k > 65535) return ZS_E_UNSUPPORTED;
  if (head_dim != 64 && head_dim != 128) return ZS_E_UNSUPPORTED;
  if ((int64_t)num_blocks * page > INT_MAX) return ZS_E_OVERFLOW;
  return ZS_OK;
}

// Whether a launch takes this many workgroups of so many threads: fewer than 2^32
// threads in all.
bool grid_fits(int64_t groups, int threads) { return groups * threads <= UINT32_MAX; }

}  // namespace zs

using namespace zs;

extern "C" int zs_paged_plan(void* stream, const int32_t* context_lens, const int32_t* new_lens, int batch,
                             int32_t* block_table, int64_t table_stride, int max_blocks_per_seq,
                             const int32_t* free_pages, int free_capacity, const int32_t* num_free,
                             int page_block_size, int max_tokens, int32_t* slots, int32_t* sequences,
                             int32_t* positions, int32_t* seqlens, int32_t* cu_new, int32_t* counts) {
  if (!context_lens || !new_lens || !block_table || !num_free || !seqlens || !cu_new || !counts)
    return ZS_E_INVAL;
  if (batch <= 0 || max_blocks_per_seq <= 0 || free_capacity < 0 || page_block_size <= 0 || max_tokens < 0)
    return ZS_E_INVAL;
  if (table_stride < max_blocks_per_seq && batch > 1) return ZS_E_INVAL;
  if (free_capacity > 0 && !free_pages) return ZS_E_INVAL;
  if (max_tokens > 0 && (!slots || !sequences || !positions)) return ZS_E_INVAL;
  if (page_block_size % 16 || batch > kPlanMaxBatch) return ZS_E_UNSUPPORTED;
  PlanParams p{};
  p.context = context_lens;
  p.fresh = new_lens;
  p.free_pages = free_pages;
  p.num_free = num_free;
  p.table = block_table;
  p.table_stride = table_stride;
  p.slots = slots;
  p.sequences = sequences;
  p.positions = positions;
  p.seqlens = seqlens;
  p.cu_new = cu_new;
  p.counts = counts;
  p.batch = batch;
  p.width = max_blocks_per_seq;
  p.free_capacity = free_capacity;
  p.max_tokens = max_tokens;
  p.page = FastDiv::of(page_block_size);
  const int grid = std::max(1, (int)(((int64_t)max_tokens + kPlanThreads - 1) / kPlanThreads));
  hipLaunchKernelGGL(plan_kernel, dim3(grid), dim3(kPlanThreads), 0, (hipStream_t)stream, p);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? ZS_OK : (int)e;
}

extern "C" int zs_paged_append(void* stream, const uint16_t* k, const uint16_t* v, int64_t k_token_stride,
                               int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                               const int32_t* slots, int num_tokens, uint16_t* k_cache, uint16_t* v_cache,
                               uint16_t* page_bounds, int num_blocks, int page_block_size, int num_heads_k,
                               int head_dim) {
  if (num_tokens < 0 || !k_cache || !v_cache) return ZS_E_INVAL;
  const int bad = paged_checks(num_blocks, page_block_size, num_heads_k, head_dim);
  if (bad != ZS_OK) return bad;
  if (num_tokens == 0) return ZS_OK;
  if (!k || !v || !slots) return ZS_E_INVAL;
  if (!aligned16(k) || !aligned16(v) || !aligned16(k_cache) || !aligned16(v_cache) || !aligned16(page_bounds))
    return ZS_E_INVAL;
  if ((k_token_stride | k_head_stride | v_token_stride | v_head_stride) & 7) return ZS_E_INVAL;
  AppendParams p{};
  p.k = k;
  p.v = v;
  p.k_token = k_token_stride;
  p.k_head = k_head_stride;
  p.v_token = v_token_stride;
  p.v_head = v_head_stride;
  p.slots = slots;
  p.k_cache = k_cache;
  p.v_cache = v_cache;
  p.bounds = page_bounds;
  p.tokens = num_tokens;
  p.heads_k = num_heads_k;
  p.num_slots = num_blocks * page_block_size;
  p.page = FastDiv::of(page_block_size);
  p.over_heads = FastDiv::of(num_heads_k);
  const int rows = kAppendThreads * 8 / head_dim;
  const int64_t items = ((int64_t)num_tokens + rows - 1) / rows * num_heads_k;
  if (!grid_fits(items, kAppendThreads)) return ZS_E_OVERFLOW;
  const dim3 grid((unsigned)items);
  if (head_dim == 128)
    hipLaunchKernelGGL(append_kernel<128>, grid, dim3(kAppendThreads), 0, (hipStream_t)stream, p);
  else
    hipLaunchKernelGGL(append_kernel<64>, grid, dim3(kAppendThreads), 0, (hipStream_t)stream, p);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? ZS_OK : (int)e;
}

extern "C" size_t zs_select_kv_pages_workspace_bytes(int batch, int num_heads_k, int max_blocks_per_seq) {
  if (batch <= 0 || num_heads_k <= 0 || max_blocks_per_seq <= 0) return 0;
  return (size_t)batch * num_heads_k * max_blocks_per_seq * sizeof(float2);
}

extern "C" int zs_select_kv_pages(void* stream, const uint16_t* q, int64_t q_batch_stride, int64_t q_head_stride,
                                  const uint16_t* page_bounds, int num_blocks, int page_block_size,
                                  const int32_t* block_table, int64_t table_stride, int max_blocks_per_seq,
                                  const int32_t* cache_seqlens, int batch, int num_heads, int num_heads_k,
                                  int head_dim, int top_k, int sink_pages, int local_pages, int32_t* pages,
                                  void* workspace, size_t workspace_bytes) {
  if (!q || !page_bounds || !block_table || !cache_seqlens || !pages || !workspace) return ZS_E_INVAL;
  const int bad = paged_checks(num_blocks, page_block_size, num_heads_k, head_dim);
  if (bad != ZS_OK) return bad;
  if (batch <= 0 || num_heads <= 0 || num_heads % num_heads_k || max_blocks_per_seq <= 0) return ZS_E_INVAL;
  if (table_stride < max_blocks_per_seq && batch > 1) return ZS_E_INVAL;
  if (top_k <= 0 || sink_pages < 0 || local_pages < 0 || (int64_t)sink_pages + local_pages > top_k) return ZS_E_INVAL;
  if (!aligned16(q) || !aligned16(page_bounds) || ((q_batch_stride | q_head_stride) & 7)) return ZS_E_INVAL;
  if (reinterpret_cast<uintptr_t>(workspace) & 7) return ZS_E_INVAL;
  if (num_heads / num_heads_k > 16 || batch > 65535) return ZS_E_UNSUPPORTED;
  if (workspace_bytes < zs_select_kv_pages_workspace_bytes(batch, num_heads_k, max_blocks_per_seq))
    return ZS_E_INVAL;
  const int64_t score_items = ((int64_t)max_blocks_per_seq + 15) / 16 * num_heads_k;
  const int64_t pick_rows = (int64_t)batch * num_heads_k;
  const int pick_threads = max_blocks_per_seq <= 4 * 256 ? 256 : max_blocks_per_seq <= 4 * 512 ? 512 : 1024;
  if (!grid_fits(score_items, 64) || !grid_fits(pick_rows, pick_threads)) return ZS_E_OVERFLOW;
  SelectParams p{};
  p.q = q;
  p.q_batch = q_batch_stride;
  p.q_head = q_head_stride;
  p.bounds = page_bounds;
  p.table = block_table;
  p.table_stride = table_stride;
  p.seqlens = cache_seqlens;
  p.pages = pages;
  p.scores = static_cast<float2*>(workspace);
  p.num_blocks = num_blocks;
  p.width = max_blocks_per_seq;
  p.page = page_block_size;
  p.heads_k = num_heads_k;
  p.group = num_heads / num_heads_k;
  p.top_k = top_k;
  p.over_heads = FastDiv::of(num_heads_k);
  p.sink = sink_pages;
  p.local = local_pages;
  const hipStream_t st = (hipStream_t)stream;
  auto launch = [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    if (max_blocks_per_seq > top_k) {
      const dim3 grid((unsigned)score_items, batch);
      hipLaunchKernelGGL(score_kernel<D>, grid, dim3(64), 0, st, p);
    }
    const dim3 rows((unsigned)pick_rows);
    auto pick = [&](auto threads, auto keys) {
      constexpr int NT = decltype(threads)::value;
      hipLaunchKernelGGL((pick_kernel<D, NT, decltype(keys)::value>), rows, dim3(NT), 0, st, p);
    };
    using Four = std::integral_constant<int, 4>;
    if (pick_threads == 256)
      pick(std::integral_constant<int, 256>{}, Four{});
    else if (pick_threads == 512)
      pick(std::integral_constant<int, 512>{}, Four{});
    else if (max_blocks_per_seq <= 4 * 1024)
      pick(std::integral_constant<int, 1024>{}, Four{});
    else
      pick(std::integral_constant<int, 1024>{}, std::integral_constant<int, 8>{});
  };
  if (head_dim == 128)
    launch(std::integral_constant<int, 128>{});
  else
    launch(std::integral_constant<int, 64>{});
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? ZS_OK : (int)e;
}
