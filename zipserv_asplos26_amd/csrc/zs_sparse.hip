// zs_sparse.hip -- single-token (decode) GQA attention over chosen pages of a
// paged bf16 KV cache (gfx950): every (sequence, KV head) has a list of logical
// pages, and softmax(scale q K^T) V runs over the tokens in them.
//
// A workgroup of W waves takes one (sequence, KV head, split of the list); a
// wave takes 32 tokens (two 16-token tiles of one or two pages) at a time.
//   Both K and V come as whole rows (16 bytes a lane, 1 KB of consecutive rows an
//   instruction) and pass through the wave's own LDS.  K read straight into
//   operand order asks for half a line at a time, twice the requests: 194 against
//   184 us for 64 sequences' 4096 tokens (64 / 8 heads, head_dim 128, pages of 16,
//   1.07 GB), 31 against 29 us for head_dim 64.
//   S^T = K q^T with v_mfma_f32_16x16x32_bf16: the K fragment (lane l: token
//   l%16, dims 32c + 8*(l/16)..+7) is the A operand, q^T (lane l: head l%16 of the
//   group) the B operand.
//   Online softmax in the log2 domain, fp32, one maximum for the 32 tokens.
//   O^T += V^T P^T with the same instruction over K = 32 tokens: S^T leaves lane
//   l the weights of head l%16 for tokens 4*(l/16)..+3 of both tiles, which is
//   the B operand if k index 8*(l/16) + j stands for token 4*(l/16) + j%4 of
//   tile j/4; V^T in that order are two ds_read_b64_tr_b16 of the V tiles.
// A weight enters the product as the sum of three bf16, all of its 24 bits, so
// the output's rounding to bf16 is the only one that shows.  None of the three is 0
// unless the weight is, or an infinite V would meet it as inf * 0: a part is what
// stands above one step less than the number, which leaves a rest, and 2^-133 (the
// smallest bf16, of a weight of 2^-126 or more) where that is less.
//
// HBM bounds it where there is enough to read: 64 sequences' 4096 tokens at 5.75
// to 6.0 TB/s, and a plain reader of as many random pages gets 6.0.  One pair of tiles
// in flight a wave is enough for that; loading the next pair ahead, more waves a
// workgroup and more splits were slower.  One sequence's 2048 tokens of 8 heads take 6
// us and 2.6 for the merge.
//
// Tokens at or past the sequence's length, pages that are not in the sequence
// and table entries outside the pool count for nothing: their scores are masked
// and their rows are not read (a tile's last valid row is read in their place,
// and V is 0 there, for it may not be finite).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <type_traits>

#include "../../include/zipserv.h"
#include "zs_device.hpp"
#include "zs_splits.hpp"

namespace zs {

int device_cu_count();                                                 // zs_gemm.hip
int paged_checks(int num_blocks, int page, int heads_k, int head_dim);  // zs_paged.hip
bool grid_fits(int64_t groups, int threads);                           // zs_paged.hip

typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef short v8i16 __attribute__((ext_vector_type(8)));

struct SparseParams {
  const uint16_t* q;
  int64_t q_batch, q_head;  // strides in elements
  const uint16_t* k;        // [blocks][page][Hkv][D]
  const uint16_t* v;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* pages;     // [B][Hkv][top_k]
  const int32_t* seqlens;
  uint16_t* out;            // [B][H][D]
  float* lse;               // [B][H] or null
  float* ws_o;              // [B][H][splits][D]  (splits > 1)
  float* ws_ml;             // [B][H][splits][2]
  int num_blocks, width, page, heads, heads_k, group, top_k, splits, chunk;  // chunk: tiles a split
  FastDiv tiles;            // 16-token tiles of a page
  float scale_log2;
};

constexpr uint32_t kLeastPart = 0x00010000;  // 2^-133 in fp32: the smallest bf16

template <int D, int W>
struct SparseLds {
  static constexpr int kPitchK = 2 * D + 16;                // bytes of a row: 16 rows' 16 bytes on all banks
  static constexpr int kPitch = 2 * D + 32;                 // of V, for the transposed reads
  static constexpr int kWave = 2 * 16 * kPitch;             // a wave's two tiles, K then V
  static constexpr int kState = (D / 4 + 2) * 64 * 4;       // a wave's O, maximum and sum
  static constexpr int kBytes = W * (kWave > kState ? kWave : kState);
};

template <int D, int W>
__global__ __launch_bounds__(W * 64) void sparse_attn_kernel(SparseParams p) {
  constexpr int kC = D / 32, kO = D / 16, kPitch = SparseLds<D, W>::kPitch, kPitchK = SparseLds<D, W>::kPitchK;
  __shared__ __attribute__((aligned(16))) uint8_t smem[SparseLds<D, W>::kBytes];
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id();
  const int sp = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
  const int len = max(p.seqlens[b], 0);
  const int t0 = sp * p.chunk, t1 = min(t0 + p.chunk, p.top_k * (int)p.tiles.d);
  const int32_t* list = p.pages + ((int64_t)b * p.heads_k + h) * p.top_k;

  const int g = l & 15, lg = l >> 4;
  bf16x8 Q[kC];
  {
    const uint16_t* qrow = p.q + b * p.q_batch + (h * p.group + (g < p.group ? g : 0)) * p.q_head + 8 * lg;
#pragma unroll
    for (int c = 0; c < kC; ++c) Q[c] = *reinterpret_cast<const bf16x8*>(qrow + 32 * c);
  }
  f32x4 O[kO];
#pragma unroll
  for (int i = 0; i < kO; ++i) O[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY, l_run = 0.f;

  uint8_t* t_lds = smem + w * SparseLds<D, W>::kWave;
  constexpr int kRows = 512 / D;                                        // rows an instruction reads
  const int lrow = l / (D / 8), lcol = 8 * (l % (D / 8));               // this lane's 16 bytes of them
  const int wr = lrow * kPitch + 2 * lcol;
  const int krd = g * kPitchK + 16 * lg;                                // row l%16, dims 8*(l/16)
  const int vrd = (4 * lg + (g >> 2)) * kPitch + 8 * (l & 3);           // transposed read

  // Lane i holds the place of tile i%2 of the wave's (32 c0 + i/2)-th pair: its
  // first row in the pool and how many of its tokens are there.
  for (int c0 = 0; t0 + 2 * (w + W * 32 * c0) < t1; ++c0) {
    int row = 0, live = 0;
    {
      const int pair = w + W * (32 * c0 + (l >> 1));
      const int tile = t0 + 2 * pair + (l & 1);
      if (tile < t1) {
        const int e = (int)p.tiles.div((uint32_t)tile), sub = tile - e * (int)p.tiles.d;
        const int lp = list[e];
        if (lp >= 0 && lp < p.width && lp < INT_MAX / p.page) {
          const int block = p.table[b * p.table_stride + lp];
          if (block >= 0 && block < p.num_blocks) {
            row = block * p.page + 16 * sub;
            live = min(max(len - (lp * p.page + 16 * sub), 0), 16);
          }
        }
      }
    }
    for (int i = 0; i < 32; ++i) {
      if (t0 + 2 * (w + W * (32 * c0 + i)) >= t1) break;
      int r0 = __builtin_amdgcn_readlane(row, 2 * i), n0 = __builtin_amdgcn_readlane(live, 2 * i);
      int r1 = __builtin_amdgcn_readlane(row, 2 * i + 1), n1 = __builtin_amdgcn_readlane(live, 2 * i + 1);
      if (n0 + n1 == 0) continue;
      // a tile without tokens reads the other one's rows
      const int f0 = n0 ? r0 : r1, f1 = n1 ? r1 : r0, m0 = (n0 ? n0 : n1) - 1, m1 = (n1 ? n1 : n0) - 1;
      int64_t o0[kC], o1[kC];
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        o0[c] = ((int64_t)(f0 + min(lrow + c * kRows, m0)) * p.heads_k + h) * D + lcol;
        o1[c] = ((int64_t)(f1 + min(lrow + c * kRows, m1)) * p.heads_k + h) * D + lcol;
      }
      u32x4 K0[kC], K1[kC], V0[kC], V1[kC];
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        K0[c] = *reinterpret_cast<const u32x4*>(p.k + o0[c]);
        K1[c] = *reinterpret_cast<const u32x4*>(p.k + o1[c]);
      }
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        V0[c] = *reinterpret_cast<const u32x4*>(p.v + o0[c]);
        V1[c] = *reinterpret_cast<const u32x4*>(p.v + o1[c]);
      }
      // through LDS into operand order
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        *reinterpret_cast<u32x4*>(t_lds + (lrow + c * kRows) * kPitchK + 2 * lcol) = K0[c];
        *reinterpret_cast<u32x4*>(t_lds + (16 + lrow + c * kRows) * kPitchK + 2 * lcol) = K1[c];
      }
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        K0[c] = *reinterpret_cast<const u32x4*>(t_lds + krd + 64 * c);
        K1[c] = *reinterpret_cast<const u32x4*>(t_lds + 16 * kPitchK + krd + 64 * c);
      }
      f32x4 S0 = {0.f, 0.f, 0.f, 0.f}, S1 = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        S0 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(K0[c]), Q[c], S0, 0, 0, 0);
        S1 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(as_bf16x8(K1[c]), Q[c], S1, 0, 0, 0);
      }
      float s[8];
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[j] = 4 * lg + j < n0 ? S0[j] * p.scale_log2 : -INFINITY;
        s[4 + j] = 4 * lg + j < n1 ? S1[j] * p.scale_log2 : -INFINITY;
      }
      float mx = s[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) mx = fmaxf(mx, s[j]);
      const float m_new = fmaxf(m_run, wave_max16(mx));
      const float m_use = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = __builtin_amdgcn_exp2f(m_run - m_use);
      float e[8], sum = 0.f;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        e[j] = __builtin_amdgcn_exp2f(s[j] - m_use);
        sum += e[j];
      }
      l_run = l_run * alpha + sum;  // this lane's tokens; summed over the lanes at the end
      if (__builtin_amdgcn_ballot_w64(alpha != 1.f)) {
#pragma unroll
        for (int k = 0; k < kO; ++k) O[k] *= alpha;
      }
      m_run = m_new;
      // the weights as a sum of three bf16 each: the upper half of one fp32 step less,
      // the same of the rest, and what is left (eight bits at most, exact)
      u32x4 hi, mid, lo;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        uint32_t a[2], c[2], d[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          const uint32_t u = __float_as_uint(e[2 * j + i]), least = min(u, kLeastPart);
          a[i] = __builtin_elementwise_sub_sat(u, 1u) & 0xFFFF0000u;
          const float r = e[2 * j + i] - __uint_as_float(a[i]);
          c[i] = max(__builtin_elementwise_sub_sat(__float_as_uint(r), 1u), least) & 0xFFFF0000u;
          d[i] = (uint32_t)max((int)__float_as_uint(r - __uint_as_float(c[i])), (int)least);
        }
        hi[j] = __builtin_amdgcn_perm(a[1], a[0], 0x07060302);
        mid[j] = __builtin_amdgcn_perm(c[1], c[0], 0x07060302);
        lo[j] = __builtin_amdgcn_perm(d[1], d[0], 0x07060302);
      }
      if (n0 + n1 < 32) {  // (uniform)
#pragma unroll
        for (int c = 0; c < kC; ++c) {
          if (lrow + c * kRows >= n0) V0[c] = u32x4{0, 0, 0, 0};
          if (lrow + c * kRows >= n1) V1[c] = u32x4{0, 0, 0, 0};
        }
      }
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        *reinterpret_cast<u32x4*>(t_lds + wr + c * kRows * kPitch) = V0[c];
        *reinterpret_cast<u32x4*>(t_lds + (16 + c * kRows) * kPitch + wr) = V1[c];
      }
#pragma unroll
      for (int k = 0; k < kO; ++k) {
        typedef __attribute__((address_space(3))) v4i16* lds_v4;
        const v4i16 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4)(t_lds + vrd + 32 * k));
        const v4i16 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4)(t_lds + 16 * kPitch + vrd + 32 * k));
        const bf16x8 A = __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
        O[k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(A, as_bf16x8(hi), O[k], 0, 0, 0);
        O[k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(A, as_bf16x8(mid), O[k], 0, 0, 0);
        O[k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(A, as_bf16x8(lo), O[k], 0, 0, 0);
      }
    }
  }

  // The waves' states merged by the first one.
  l_run = wave_sum16(l_run);
  __syncthreads();
  float* cb = reinterpret_cast<float*>(smem) + w * (SparseLds<D, W>::kState / 4) + l;
#pragma unroll
  for (int i = 0; i < kO; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) cb[(4 * i + r) * 64] = O[i][r];
  cb[4 * kO * 64] = m_run;
  cb[(4 * kO + 1) * 64] = l_run;
  __syncthreads();
  if (w != 0) return;
  const float* c0 = reinterpret_cast<const float*>(smem) + l;
  constexpr int kStride = SparseLds<D, W>::kState / 4;
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < W; ++i) m = fmaxf(m, c0[i * kStride + 4 * kO * 64]);
  const float m_use = m == -INFINITY ? 0.f : m;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kO; ++i) O[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const float f = __builtin_amdgcn_exp2f(c0[i * kStride + 4 * kO * 64] - m_use);
    sum += c0[i * kStride + (4 * kO + 1) * 64] * f;
#pragma unroll
    for (int k = 0; k < kO; ++k)
#pragma unroll
      for (int r = 0; r < 4; ++r) O[k][r] += c0[i * kStride + (4 * k + r) * 64] * f;
  }
  if (g >= p.group) return;
  const int64_t head = (int64_t)b * p.heads + h * p.group + g;
  if (p.splits == 1) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    uint16_t* o = p.out + head * D + 4 * lg;
#pragma unroll
    for (int k = 0; k < kO; ++k) {
      uint2 x;
      x.x = pack_bf16x2(O[k][0] * inv, O[k][1] * inv);
      x.y = pack_bf16x2(O[k][2] * inv, O[k][3] * inv);
      *reinterpret_cast<uint2*>(o + 16 * k) = x;
    }
    if (p.lse && lg == 0) p.lse[head] = sum == 0.f ? -INFINITY : (m + __log2f(sum)) * 0.6931471805599453f;
  } else {
    const int64_t slot = head * p.splits + sp;
    float* o = p.ws_o + slot * D + 4 * lg;
#pragma unroll
    for (int k = 0; k < kO; ++k) *reinterpret_cast<f32x4*>(o + 16 * k) = O[k];
    if (lg == 0) *reinterpret_cast<float2*>(p.ws_ml + 2 * slot) = float2{m, sum};
  }
}

// How a call is cut: workgroups of four waves, one a CU (256), each list in as
// many splits as that takes; lists of up to 384 tokens whole, whose merge costs
// more than it gives (8 KV heads' 256 tokens: 6.6 us whole, over 8 in two).  More
// splits only add partial results (128 lists of 4096 tokens, head_dim 128: 53.4 us
// in 2, 54.9 and up in 4).  Where that leaves the last round of the CUs part empty,
// workgroups of two waves, up to four a CU, spread better: 320 lists of 1024,
// 2048, 4096 tokens 41.2 -> 39.4, 71.6 -> 68.8, 130 -> 128 us, 800 of 1024 88.8 ->
// 86.2, but 512 of 4096 (two full rounds) 183.8 -> 190.5.
struct SparseCut {
  int waves, splits;
};

static SparseCut sparse_cut(int batch, int heads_k, int64_t tiles, int num_splits) {
  auto at_most = [&](int64_t s, int waves) {  // every wave has a pair of tiles
    return (int)std::max<int64_t>(1, std::min<int64_t>(s, (tiles + 2 * waves - 1) / (2 * waves)));
  };
  if (num_splits > 0) return {4, at_most(num_splits, 4)};
  const int64_t units = (int64_t)batch * heads_k, cus = device_cu_count();
  if (tiles <= 24) return {units > cus ? 2 : 4, 1};
  const int splits = at_most(cus / units, 4);
  const int64_t items = units * splits, rounds = (items + cus - 1) / cus;
  if (100 * items >= 85 * rounds * cus || splits < cus / units) return {4, splits};
  return {2, at_most(4 * cus / units, 2)};
}

static size_t sparse_ws_bytes(int batch, int heads, int head_dim, int splits) {
  return splits <= 1 ? 0 : (size_t)batch * heads * splits * (head_dim + 2) * sizeof(float);
}

}  // namespace zs

using namespace zs;

extern "C" size_t zs_decode_attention_sparse_workspace_bytes(int batch, int num_heads, int num_heads_k, int head_dim,
                                                             int top_k, int page_block_size, int num_splits) {
  if (batch <= 0 || num_heads <= 0 || num_heads_k <= 0 || head_dim <= 0 || top_k <= 0 || page_block_size < 16 ||
      num_splits < 0)
    return 0;
  return sparse_ws_bytes(batch, num_heads, head_dim,
                         sparse_cut(batch, num_heads_k, (int64_t)top_k * (page_block_size / 16), num_splits).splits);
}

extern "C" int zs_decode_attention_sparse_paged(void* stream, const uint16_t* q, int64_t q_batch_stride,
                                                int64_t q_head_stride, const uint16_t* k_cache,
                                                const uint16_t* v_cache, int num_blocks, int page_block_size,
                                                const int32_t* block_table, int64_t table_stride,
                                                int max_blocks_per_seq, const int32_t* pages, int top_k,
                                                const int32_t* cache_seqlens, int batch, int num_heads,
                                                int num_heads_k, int head_dim, float softmax_scale, uint16_t* out,
                                                float* softmax_lse, void* workspace, size_t workspace_bytes,
                                                int num_splits) {
  if (!q || !k_cache || !v_cache || !block_table || !pages || !cache_seqlens || !out) return ZS_E_INVAL;
  const int bad = paged_checks(num_blocks, page_block_size, num_heads_k, head_dim);
  if (bad != ZS_OK) return bad;
  if (batch <= 0 || num_heads <= 0 || num_heads % num_heads_k || max_blocks_per_seq <= 0 || top_k <= 0 ||
      num_splits < 0)
    return ZS_E_INVAL;
  if (table_stride < max_blocks_per_seq && batch > 1) return ZS_E_INVAL;
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(k_cache) | reinterpret_cast<uintptr_t>(v_cache) |
        reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) & 15) ||
      ((q_batch_stride | q_head_stride) & 7))
    return ZS_E_INVAL;
  if (num_heads / num_heads_k > 16 || batch > 65535 || (int64_t)batch * num_heads > INT_MAX)
    return ZS_E_UNSUPPORTED;
  const int64_t tiles = (int64_t)top_k * (page_block_size / 16);
  if (tiles > INT_MAX / 2) return ZS_E_OVERFLOW;
  SparseParams p{};
  const SparseCut cut = sparse_cut(batch, num_heads_k, tiles, num_splits);
  p.splits = cut.splits;
  if (!grid_fits(p.splits, cut.waves * 64) ||
      (p.splits > 1 && !grid_fits((int64_t)batch * num_heads, kMergeWaves * 64)))
    return ZS_E_OVERFLOW;
  if (workspace_bytes < sparse_ws_bytes(batch, num_heads, head_dim, p.splits) || (p.splits > 1 && !workspace))
    return ZS_E_INVAL;
  p.chunk = (int)((tiles + p.splits - 1) / p.splits);
  p.chunk += p.chunk & 1;
  p.q = q;
  p.q_batch = q_batch_stride;
  p.q_head = q_head_stride;
  p.k = k_cache;
  p.v = v_cache;
  p.table = block_table;
  p.table_stride = table_stride;
  p.pages = pages;
  p.seqlens = cache_seqlens;
  p.out = out;
  p.lse = softmax_lse;
  p.ws_o = static_cast<float*>(workspace);
  p.ws_ml = p.ws_o + (size_t)batch * num_heads * p.splits * head_dim;
  p.num_blocks = num_blocks;
  p.width = max_blocks_per_seq;
  p.page = page_block_size;
  p.heads = num_heads;
  p.heads_k = num_heads_k;
  p.group = num_heads / num_heads_k;
  p.top_k = top_k;
  p.tiles = FastDiv::of(page_block_size / 16);
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  const hipStream_t st = (hipStream_t)stream;
  const dim3 grid(p.splits, num_heads_k, batch);
  auto launch = [&](auto dim) {
    constexpr int D = decltype(dim)::value;
    if (cut.waves == 4)
      hipLaunchKernelGGL((sparse_attn_kernel<D, 4>), grid, dim3(4 * 64), 0, st, p);
    else
      hipLaunchKernelGGL((sparse_attn_kernel<D, 2>), grid, dim3(2 * 64), 0, st, p);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || p.splits == 1) return e;
    return merge_splits(st, SplitMerge{p.ws_o, p.ws_ml, p.out, p.lse, p.splits, batch * num_heads}, D);
  };
  const hipError_t e = head_dim == 128 ? launch(std::integral_constant<int, 128>{})
                                       : launch(std::integral_constant<int, 64>{});
  return e == hipSuccess ? ZS_OK : (int)e;
}
