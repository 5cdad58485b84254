// zs_paged.hip -- the state of an appendable paged KV cache (gfx950): block
// tables and slot maps from the requests' lengths, new keys and values into
// their slots with the bounds of the pages that they fall into, and the pages
// that a query's attention should read, chosen by those bounds.
//
// A pool has num_blocks pages [page][Hkv][D]; token t of sequence b is row
// t % page of page table[b][t / page], its slot that page * page + t % page.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>

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
// from L2) and then places its 256 tokens by a search over the first sum.  A
// table entry is written by the token that opens its page and read only for
// pages that the sequence had before, so no workgroup waits for another.
constexpr int kPlanThreads = 256;
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

// Inclusive sum over the workgroup of one value a thread, and the total.
__device__ __forceinline__ int64_t plan_scan(int64_t x, int64_t* wave_sum, int64_t& total) {
  const int l = lane_id(), w = threadIdx.x >> 6;
#pragma unroll
  for (int off = 1; off < 64; off <<= 1) {
    const int64_t y = __shfl_up(x, off);
    if (l >= off) x += y;
  }
  __syncthreads();  // the last scan's sums are read
  if (l == 63) wave_sum[w] = x;
  __syncthreads();
  total = 0;
#pragma unroll
  for (int i = 0; i < kPlanThreads / 64; ++i) {
    if (i < w) x += wave_sum[i];
    total += wave_sum[i];
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
  __shared__ int64_t sums[kPlanThreads / 64];
  const int page = (int)p.page.d;
  const int64_t F = min(max(*p.num_free, 0), p.free_capacity);
  int64_t asked = 0, tokens = 0, taken = 0, wanted = 0;  // of the sequences so far
  const bool lead = blockIdx.x == 0;
  for (int b0 = 0; b0 < p.batch; b0 += kPlanThreads) {
    const int b = b0 + threadIdx.x;
    const bool live = b < p.batch;
    const int c = live ? max(p.context[b], 0) : 0;
    const int n_asked = live ? max(p.fresh[b], 0) : 0;
    int n = min(n_asked, INT_MAX - c);
    int64_t total;
    const int64_t end = tokens + plan_scan(n, sums, total);
    const int start = (int)min(end - n, (int64_t)p.max_tokens);
    n = (int)min((int64_t)n, p.max_tokens - (int64_t)start);
    tokens += total;
    plan_scan(n_asked, sums, total);
    asked += total;
    const int have = (int)p.page.div((uint32_t)c) + (p.page.div((uint32_t)c) * page != (uint32_t)c);
    const uint32_t all = (uint32_t)c + (uint32_t)n;
    const int need = (int)(p.page.div(all) + (p.page.div(all) * page != all));
    const int more = max(min(need, p.width) - have, 0);
    const int64_t before = taken + plan_scan(more, sums, total) - more;
    taken += total;
    plan_scan(need - have, sums, total);
    wanted += total;
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
  if (threadIdx.x == 0) {
    first[p.batch] = used;
    if (lead) {
      const int64_t given = min(taken, F);
      p.cu_new[p.batch] = used;
      p.counts[0] = plan_saturate(asked);
      p.counts[1] = (int)given;
      p.counts[2] = plan_saturate(wanted - given);
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
// are passed over.  The tokens of one page stand next to one
// another, so the first of such a run takes the bounds of the whole run.
//
// A workgroup takes 2048 / D tokens of one KV head, 16 bytes a thread.
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
  FastDiv page;
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
  const int r = threadIdx.x / kLanes, c = threadIdx.x % kLanes, h = blockIdx.y;
  const int t = blockIdx.x * kRows + r;
  auto slot_of = [&](int i) {
    const int s = i >= 0 && i < p.tokens ? p.slots[i] : -1;
    return s < p.num_slots ? s : -1;
  };
  const int slot = slot_of(t);
  if (slot < 0) return;
  const u32x4 k = *reinterpret_cast<const u32x4*>(p.k + t * p.k_token + h * p.k_head + 8 * c);
  const u32x4 v = *reinterpret_cast<const u32x4*>(p.v + t * p.v_token + h * p.v_head + 8 * c);
  const int64_t at = ((int64_t)slot * p.heads_k + h) * D + 8 * c;
  *reinterpret_cast<u32x4*>(p.k_cache + at) = k;
  *reinterpret_cast<u32x4*>(p.v_cache + at) = v;
  if (!p.bounds) return;
  const int block = (int)p.page.div((uint32_t)slot);
  auto block_of = [&](int s) { return s < 0 ? -1 : (int)p.page.div((uint32_t)s); };
  if (block_of(slot_of(t - 1)) == block) return;
  u32x4* low = reinterpret_cast<u32x4*>(p.bounds + ((int64_t)block * p.heads_k + h) * 2 * D + 8 * c);
  u32x4* high = low + D / 8;
  bool anew = slot == block * (int)p.page.d;
  u16x8 lo = bound_order(k), hi = kMost - lo;
  for (int i = t + 1; i < p.tokens; ++i) {
    const int s = slot_of(i);
    if (block_of(s) != block) break;
    anew |= s == block * (int)p.page.d;
    const u32x4 x = *reinterpret_cast<const u32x4*>(p.k + i * p.k_token + h * p.k_head + 8 * c);
    bound_widen(lo, hi, bound_order(x));
  }
  if (!anew) {
    lo = __builtin_elementwise_min(lo, bound_order(*low));
    hi = __builtin_elementwise_min(hi, kMost - bound_order(*high));
  }
  *low = bound_value(lo);
  *high = bound_value(kMost - hi);
}

// ---------------------------------------------------------------------------
// Selection
// ---------------------------------------------------------------------------
// score[b][h][p] = max over the group's heads of sum_d max(q_d, 0) kmax_d +
// min(q_d, 0) kmin_d, the largest q.k that the bounds of page p allow.  In 64
// bits: products of two bf16 are exact there and a sum is off by 2^-53, so the
// answer is the definition's and not a rounding's.  As 2 score = sum_d q_d (kmax
// + kmin) + |q_d| (kmax - kmin), which needs q once.  NaN (a bound or a query
// that is not finite) counts as +inf.  Keys are the scores' bits in an order of
// unsigned numbers; pages that are always taken have the largest key.
struct SelectParams {
  const uint16_t* q;
  int64_t q_batch, q_head;  // strides in elements
  const uint16_t* bounds;   // [blocks][Hkv][2][D]
  const int32_t* table;
  int64_t table_stride;
  const int32_t* seqlens;
  int32_t* pages;           // [B][Hkv][top_k]
  uint64_t* keys;           // [B][Hkv][width]
  int num_blocks, width, page, batch, heads_k, group, top_k, sink, local;
};

__device__ __forceinline__ int select_pages(const SelectParams& p, int b) {
  const int len = max(p.seqlens[b], 0);
  return min(len / p.page + (len % p.page != 0), p.width);
}

__device__ __forceinline__ uint64_t select_key(double x) {
  if (x != x) x = INFINITY;
  const uint64_t u = (uint64_t)__double_as_longlong(x + 0.0);  // -0 is 0
  return u >> 63 ? ~u : u | 0x8000000000000000ull;
}

constexpr int kScoreThreads = 256;

template <int D>
__global__ __launch_bounds__(kScoreThreads) void score_kernel(SelectParams p) {
  constexpr int kLanes = D / 8, kPages = kScoreThreads / kLanes;
  const int b = blockIdx.y / p.heads_k, h = blockIdx.y % p.heads_k;
  const int n = select_pages(p, b);
  const int lp = blockIdx.x * kPages + threadIdx.x / kLanes, c = threadIdx.x % kLanes;
  if (n <= p.top_k || lp >= n) return;  // (all lanes of a page alike)
  uint64_t key = ~0ull;
  if (lp >= p.sink && lp < n - p.local) {
    const int block = p.table[b * p.table_stride + lp];
    double best = -INFINITY;
    bool odd = true;
    if (block >= 0 && block < p.num_blocks) {
      const uint16_t* lo = p.bounds + ((int64_t)block * p.heads_k + h) * 2 * D + 8 * c;
      const u32x4 x = *reinterpret_cast<const u32x4*>(lo), y = *reinterpret_cast<const u32x4*>(lo + D);
      double mid[8], wide[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const double k0 = bf16_bits_to_f32(i & 1 ? x[i / 2] >> 16 : x[i / 2] & 0xFFFF);
        const double k1 = bf16_bits_to_f32(i & 1 ? y[i / 2] >> 16 : y[i / 2] & 0xFFFF);
        mid[i] = k1 + k0;
        wide[i] = k1 - k0;
      }
      odd = false;
      for (int g = 0; g < p.group; ++g) {
        const u32x4 u = *reinterpret_cast<const u32x4*>(p.q + b * p.q_batch + (h * p.group + g) * p.q_head + 8 * c);
        double s = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const double q = bf16_bits_to_f32(i & 1 ? u[i / 2] >> 16 : u[i / 2] & 0xFFFF);
          s = fma(q, mid[i], s);
          s = fma(fabs(q), wide[i], s);
        }
#pragma unroll
        for (int off = 1; off < kLanes; off <<= 1) s += __shfl_xor(s, off);
        odd |= s != s;
        best = fmax(best, s);
      }
    }
    key = min(select_key(odd ? INFINITY : best), ~0ull - 1);
    if (block < 0 || block >= p.num_blocks) key = 0;  // no such page: taken last
  }
  if (c == 0) p.keys[(int64_t)blockIdx.y * p.width + lp] = key;
}

// The top_k largest keys of one (sequence, KV head), ties to the lowest page, in
// ascending order: the key of the last one taken digit by digit, 8 bits at a
// time from the top, until the pages of a digit are all taken or none is left.
constexpr int kPickThreads = 256;

__global__ __launch_bounds__(kPickThreads) void pick_kernel(SelectParams p) {
  __shared__ int hist[256];
  __shared__ int wave_sum[2][kPickThreads / 64];
  __shared__ int s_bin, s_above, s_in;
  const int row = blockIdx.x, b = row / p.heads_k, tid = threadIdx.x;
  const int n = select_pages(p, b);
  int32_t* out = p.pages + (int64_t)row * p.top_k;
  if (n <= p.top_k) {
    for (int i = tid; i < p.top_k; i += kPickThreads) out[i] = i < n ? i : -1;
    return;
  }
  const uint64_t* keys = p.keys + (int64_t)row * p.width;
  uint64_t prefix = 0;  // of the keys' bits from `shift` on
  int need = p.top_k, shift = 64;
  while (shift > 0) {
    shift -= 8;
    hist[tid] = 0;
    __syncthreads();
    for (int i = tid; i < n; i += kPickThreads) {
      const uint64_t k = keys[i];
      if (shift == 56 || (k >> (shift + 8)) == prefix) atomicAdd(&hist[(k >> shift) & 255], 1);
    }
    __syncthreads();
    if (tid < 64) {  // four digits a lane, the largest first
      int v[4], sum = 0;
#pragma unroll
      for (int i = 0; i < 4; ++i) sum += v[i] = hist[255 - 4 * tid - i];
      int above = wave_inclusive_scan(sum) - sum;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        if (above < need && above + v[i] >= need) {
          s_bin = 255 - 4 * tid - i;
          s_above = above;
          s_in = v[i];
        }
        above += v[i];
      }
    }
    __syncthreads();
    prefix = prefix << 8 | (uint64_t)s_bin;
    need -= s_above;
    if (s_in == need) break;  // (uniform)
  }
  // keys above `prefix` are taken, and the first `need` equal to it
  int at = 0, equal = 0;
  const int w = tid >> 6, l = lane_id();
  for (int i0 = 0; i0 < n; i0 += kPickThreads) {
    const int i = i0 + tid;
    const uint64_t k = i < n ? keys[i] >> shift : 0;
    const bool is = i < n && k == prefix;
    const uint64_t eq = __builtin_amdgcn_ballot_w64(is);
    if (l == 0) wave_sum[0][w] = __builtin_popcountll(eq);
    __syncthreads();
    int rank = equal + __builtin_popcountll(eq & ((1ull << l) - 1));
    for (int j = 0; j < kPickThreads / 64; ++j) {
      if (j < w) rank += wave_sum[0][j];
      equal += wave_sum[0][j];
    }
    const bool take = i < n && (k > prefix || (is && rank < need));
    const uint64_t tk = __builtin_amdgcn_ballot_w64(take);
    if (l == 0) wave_sum[1][w] = __builtin_popcountll(tk);
    __syncthreads();
    int place = at + __builtin_popcountll(tk & ((1ull << l) - 1));
    for (int j = 0; j < kPickThreads / 64; ++j) {
      if (j < w) place += wave_sum[1][j];
      at += wave_sum[1][j];
    }
    if (take) out[place] = i;
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
  const int rows = kAppendThreads * 8 / head_dim;
  const dim3 grid((unsigned)(((int64_t)num_tokens + rows - 1) / rows), num_heads_k);
  if (head_dim == 128)
    hipLaunchKernelGGL(append_kernel<128>, grid, dim3(kAppendThreads), 0, (hipStream_t)stream, p);
  else
    hipLaunchKernelGGL(append_kernel<64>, grid, dim3(kAppendThreads), 0, (hipStream_t)stream, p);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? ZS_OK : (int)e;
}

extern "C" size_t zs_select_kv_pages_workspace_bytes(int batch, int num_heads_k, int max_blocks_per_seq) {
  if (batch <= 0 || num_heads_k <= 0 || max_blocks_per_seq <= 0) return 0;
  return (size_t)batch * num_heads_k * max_blocks_per_seq * sizeof(uint64_t);
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
  if (num_heads / num_heads_k > 16 || (int64_t)batch * num_heads_k > 65535) return ZS_E_UNSUPPORTED;
  if (workspace_bytes < zs_select_kv_pages_workspace_bytes(batch, num_heads_k, max_blocks_per_seq))
    return ZS_E_INVAL;
  SelectParams p{};
  p.q = q;
  p.q_batch = q_batch_stride;
  p.q_head = q_head_stride;
  p.bounds = page_bounds;
  p.table = block_table;
  p.table_stride = table_stride;
  p.seqlens = cache_seqlens;
  p.pages = pages;
  p.keys = static_cast<uint64_t*>(workspace);
  p.num_blocks = num_blocks;
  p.width = max_blocks_per_seq;
  p.page = page_block_size;
  p.batch = batch;
  p.heads_k = num_heads_k;
  p.group = num_heads / num_heads_k;
  p.top_k = top_k;
  p.sink = sink_pages;
  p.local = local_pages;
  const hipStream_t st = (hipStream_t)stream;
  if (max_blocks_per_seq > top_k) {
    const int per = kScoreThreads * 8 / head_dim;
    const dim3 grid((unsigned)(((int64_t)max_blocks_per_seq + per - 1) / per), batch * num_heads_k);
    if (head_dim == 128)
      hipLaunchKernelGGL(score_kernel<128>, grid, dim3(kScoreThreads), 0, st, p);
    else
      hipLaunchKernelGGL(score_kernel<64>, grid, dim3(kScoreThreads), 0, st, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return (int)e;
  }
  hipLaunchKernelGGL(pick_kernel, dim3(batch * num_heads_k), dim3(kPickThreads), 0, st, p);
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? ZS_OK : (int)e;
}
