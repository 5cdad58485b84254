// zs_sparse.hip -- single-token (decode) GQA attention over chosen pages of a
// paged bf16 KV cache (gfx950): every (sequence, KV head) has a list of logical
// pages, and softmax(scale q K^T) V runs over the tokens in them.
//
// A workgroup of four waves takes one (sequence, KV head, split of the list); a
// wave takes 32 tokens (two 16-token tiles of one or two pages) at a time.
//   S^T = K q^T with v_mfma_f32_16x16x32_bf16: the K fragment (lane l: token
//   l%16, dims 32c + 8*(l/16)..+7) comes straight from memory and is the A
//   operand, q^T (lane l: head l%16 of the group) the B operand.
//   Online softmax in the log2 domain, fp32, one maximum for the 32 tokens.
//   O^T += V^T P^T with the same instruction over K = 32 tokens: S^T leaves lane
//   l the weights of head l%16 for tokens 4*(l/16)..+3 of both tiles, which is
//   the B operand if k index 8*(l/16) + j stands for token 4*(l/16) + j%4 of
//   tile j/4; V^T in that order are two ds_read_b64_tr_b16 of the V tiles, which
//   pass through the wave's own LDS.
// A weight enters the product as the sum of two bf16, so it keeps 16 bits, and
// the output's rounding to bf16 is the only one that shows.  The second one is
// never 0, or an infinite V would meet it as inf * 0.
//
// Tokens at or past the sequence's length, pages that are not in the sequence
// and table entries outside the pool count for nothing: their scores are masked
// and their rows are not read (a tile's last valid row is read in their place,
// and V is 0 there, for it may not be finite).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
#include <climits>

#include "../../include/zipserv.h"
#include "zs_device.hpp"

namespace zs {

int device_cu_count();                                                 // zs_gemm.hip
int paged_checks(int num_blocks, int page, int heads_k, int head_dim);  // zs_paged.hip

typedef short v4i16 __attribute__((ext_vector_type(4)));
typedef short v8i16 __attribute__((ext_vector_type(8)));

constexpr int kSparseWaves = 4;

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

template <int D>
struct SparseLds {
  static constexpr int kPitch = 2 * D + 32;                 // bytes of a V row
  static constexpr int kWave = 2 * 16 * kPitch;             // a wave's two V tiles
  static constexpr int kState = (D / 4 + 2) * 64 * 4;       // a wave's O, maximum and sum
  static constexpr int kBytes = kSparseWaves * (kWave > kState ? kWave : kState);
};

template <int D>
__global__ __launch_bounds__(kSparseWaves * 64) void sparse_attn_kernel(SparseParams p) {
  constexpr int kC = D / 32, kO = D / 16, kPitch = SparseLds<D>::kPitch;
  __shared__ __attribute__((aligned(16))) uint8_t smem[SparseLds<D>::kBytes];
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

  uint8_t* vt = smem + w * SparseLds<D>::kWave;
  const int vwr = g * kPitch + 16 * lg;                                // row l%16, dims 8*(l/16)
  const int vrd = (4 * lg + (g >> 2)) * kPitch + 8 * (l & 3);          // transposed read

  // Lane i holds the place of tile i%2 of the wave's (32 c0 + i/2)-th pair: its
  // first row in the pool and how many of its tokens are there.
  for (int c0 = 0; t0 + 2 * (w + kSparseWaves * 32 * c0) < t1; ++c0) {
    int row = 0, live = 0;
    {
      const int pair = w + kSparseWaves * (32 * c0 + (l >> 1));
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
      if (t0 + 2 * (w + kSparseWaves * (32 * c0 + i)) >= t1) break;
      int r0 = __builtin_amdgcn_readlane(row, 2 * i), n0 = __builtin_amdgcn_readlane(live, 2 * i);
      int r1 = __builtin_amdgcn_readlane(row, 2 * i + 1), n1 = __builtin_amdgcn_readlane(live, 2 * i + 1);
      if (n0 + n1 == 0) continue;
      // a tile without tokens reads the other one's rows
      const int a0 = (n0 ? r0 : r1) + min(g, (n0 ? n0 : n1) - 1);
      const int a1 = (n1 ? r1 : r0) + min(g, (n1 ? n1 : n0) - 1);
      const int64_t o0 = ((int64_t)a0 * p.heads_k + h) * D + 8 * lg, o1 = ((int64_t)a1 * p.heads_k + h) * D + 8 * lg;
      u32x4 K0[kC], K1[kC], V0[kC], V1[kC];
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        K0[c] = *reinterpret_cast<const u32x4*>(p.k + o0 + 32 * c);
        K1[c] = *reinterpret_cast<const u32x4*>(p.k + o1 + 32 * c);
      }
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        V0[c] = *reinterpret_cast<const u32x4*>(p.v + o0 + 32 * c);
        V1[c] = *reinterpret_cast<const u32x4*>(p.v + o1 + 32 * c);
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
      // the weights as a sum of two bf16 each: the upper half cut off, the rest
      // (exact in fp32) rounded
      u32x4 hi, lo;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const uint32_t x = __float_as_uint(e[2 * j]), y = __float_as_uint(e[2 * j + 1]);
        hi[j] = __builtin_amdgcn_perm(y, x, 0x07060302);
        lo[j] = pack_bf16x2(fmaxf(e[2 * j] - __uint_as_float(x & 0xFFFF0000u), FLT_MIN),
                            fmaxf(e[2 * j + 1] - __uint_as_float(y & 0xFFFF0000u), FLT_MIN));
      }
      if (n0 + n1 < 32) {  // (uniform)
#pragma unroll
        for (int c = 0; c < kC; ++c) {
          if (g >= n0) V0[c] = u32x4{0, 0, 0, 0};
          if (g >= n1) V1[c] = u32x4{0, 0, 0, 0};
        }
      }
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        *reinterpret_cast<u32x4*>(vt + vwr + 64 * c) = V0[c];
        *reinterpret_cast<u32x4*>(vt + 16 * kPitch + vwr + 64 * c) = V1[c];
      }
#pragma unroll
      for (int k = 0; k < kO; ++k) {
        typedef __attribute__((address_space(3))) v4i16* lds_v4;
        const v4i16 x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4)(vt + vrd + 32 * k));
        const v4i16 y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4)(vt + 16 * kPitch + vrd + 32 * k));
        const bf16x8 A = __builtin_bit_cast(bf16x8, __builtin_shufflevector(x, y, 0, 1, 2, 3, 4, 5, 6, 7));
        O[k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(A, as_bf16x8(hi), O[k], 0, 0, 0);
        O[k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(A, as_bf16x8(lo), O[k], 0, 0, 0);
      }
    }
  }

  // The four waves' states merged by the first one.
  l_run = wave_sum16(l_run);
  __syncthreads();
  float* cb = reinterpret_cast<float*>(smem) + w * (SparseLds<D>::kState / 4) + l;
#pragma unroll
  for (int i = 0; i < kO; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) cb[(4 * i + r) * 64] = O[i][r];
  cb[4 * kO * 64] = m_run;
  cb[(4 * kO + 1) * 64] = l_run;
  __syncthreads();
  if (w != 0) return;
  const float* c0 = reinterpret_cast<const float*>(smem) + l;
  constexpr int kStride = SparseLds<D>::kState / 4;
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < kSparseWaves; ++i) m = fmaxf(m, c0[i * kStride + 4 * kO * 64]);
  const float m_use = m == -INFINITY ? 0.f : m;
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kO; ++i) O[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int i = 0; i < kSparseWaves; ++i) {
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

// The splits of one (sequence, head) merged by a wave.
template <int D>
__global__ __launch_bounds__(64) void sparse_merge_kernel(SparseParams p) {
  const int64_t head = blockIdx.x;
  const int l = lane_id();
  const float* ml = p.ws_ml + head * p.splits * 2;
  const float* o = p.ws_o + head * p.splits * D;
  float m = -INFINITY;
  for (int s = 0; s < p.splits; ++s) m = fmaxf(m, ml[2 * s]);
  const float m_use = m == -INFINITY ? 0.f : m;
  float sum = 0.f, acc[D / 64] = {};
  for (int s = 0; s < p.splits; ++s) {
    const float f = __builtin_amdgcn_exp2f(ml[2 * s] - m_use);
    sum += ml[2 * s + 1] * f;
#pragma unroll
    for (int i = 0; i < D / 64; ++i) acc[i] += o[s * D + (D / 64) * l + i] * f;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint16_t* out = p.out + head * D + (D / 64) * l;
#pragma unroll
  for (int i = 0; i < D / 64; ++i) out[i] = (uint16_t)f32_to_bf16_bits(acc[i] * inv);
  if (p.lse && l == 0) p.lse[head] = sum == 0.f ? -INFINITY : (m + __log2f(sum)) * 0.6931471805599453f;
}

// Splits of the list: about two workgroups a CU, at least 8 tiles (one pair a
// wave) each.
static int sparse_splits(int batch, int heads_k, int64_t tiles, int num_splits) {
  const int64_t most = std::max<int64_t>(1, (tiles + 7) / 8);
  if (num_splits > 0) return (int)std::min<int64_t>(num_splits, most);
  const int64_t units = (int64_t)batch * heads_k;
  return (int)std::min(most, std::max<int64_t>(1, 2 * (int64_t)device_cu_count() / units));
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
                         sparse_splits(batch, num_heads_k, (int64_t)top_k * (page_block_size / 16), num_splits));
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
  if (num_heads / num_heads_k > 16 || batch > 65535) return ZS_E_UNSUPPORTED;
  const int64_t tiles = (int64_t)top_k * (page_block_size / 16);
  if (tiles > INT_MAX / 2) return ZS_E_OVERFLOW;
  SparseParams p{};
  p.splits = sparse_splits(batch, num_heads_k, tiles, num_splits);
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
  const dim3 grid(p.splits, num_heads_k, batch), block(kSparseWaves * 64);
  if (head_dim == 128)
    hipLaunchKernelGGL(sparse_attn_kernel<128>, grid, block, 0, st, p);
  else
    hipLaunchKernelGGL(sparse_attn_kernel<64>, grid, block, 0, st, p);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && p.splits > 1) {
    const dim3 rows((unsigned)((int64_t)batch * num_heads));
    if (head_dim == 128)
      hipLaunchKernelGGL(sparse_merge_kernel<128>, rows, dim3(64), 0, st, p);
    else
      hipLaunchKernelGGL(sparse_merge_kernel<64>, rows, dim3(64), 0, st, p);
    e = hipGetLastError();
  }
  return e == hipSuccess ? ZS_OK : (int)e;
}
