// zs_quant_attention.hip -- attention of each sequence's last tokens over a paged
// KV cache held in 4 or 8 bits (gfx950; the layout is in zs_quant.hpp).
//
// With a key k = low_k + s_k c and a value v = low_v + s_v c, c whole numbers of
// 0..15 or 0..255,
//   q.k       = s_k (q.c) + low_k sum(q),
//   sum p v   = sum (p s_v) c + sum p low_v,
// so the codes themselves are the matrix operands, exact in bf16, and a token costs two
// products more a row, not a value each channel.
//
// A column is a (new token, query head) of one KV head's group; a workgroup of
// kWaves waves takes 16 columns of a sequence and a split of its tokens, a wave 32
// tokens (two tiles of 16) at a time, all in registers:
//   S^T = C_k q^T with v_mfma_f32_16x16x32_bf16: lane l holds D / 4 codes of token
//   l%16 (channels D/4 * (l/16) and up, one piece of its row), 8 of them the A operand of a
//   step; q^T (lane l: column l%16, the same channels) is the B operand.
//   Online softmax in the log2 domain, fp32.
//   O^T += C_v^T W^T over K = 32 tokens: S^T leaves lane l the weights of column l%16
//   for tokens 4*(l/16)..+3 of both tiles, the B operand if k index 8*(l/16) + j
//   stands for token 4*(l/16) + j%4 of tile j/4; lane l reads the l%16-th part of those
//   eight rows, D / 16 channels of 8 tokens, which are D / 16 A operands.
// In 4 bits a shift and a mask put two codes into the mantissas of two bf16 of
// exponent 4, that is 16 + c: the 16s are taken off through the sums of q and of the weights.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <type_traits>

#include "../../include/zipserv.h"
#include "zs_device.hpp"
#include "zs_quant.hpp"
#include "zs_splits.hpp"

namespace zs {

int device_cu_count();                                                                             // zs_gemm.hip
bool grid_fits(int64_t groups, int threads);                                                       // zs_paged.hip
int quant_checks(const void* cache, int num_blocks, int page, int heads_k, int head_dim, int bits);  // zs_quant.hip

struct QuantAttnParams {
  const uint16_t* q;
  int64_t q_batch, q_token, q_head;  // strides in elements
  const uint8_t* cache;
  int64_t record;
  const int32_t* table;
  int64_t table_stride;
  const int32_t* seqlens;
  uint16_t* out;  // [B][new][H][D]
  float* lse;     // [B][H][new] or null
  float* ws_o;    // [row][splits][D], rows in the order of lse (splits > 1)
  float* ws_ml;   // [row][splits][2]
  int num_blocks, width, page, heads, heads_k, group, new_tokens, columns, splits;
  FastDiv tiles;        // 16-token tiles of a page
  FastDiv over_group;   // a column's new token
  FastDiv over_heads_k;
  float scale_log2;
};

constexpr int kQaWaves = 4;

template <int D, int kBits>
struct QaShape {
  static constexpr int kC = D / 32;               // steps of q.c
  static constexpr int kO = D / 16;               // tiles of channels of the output
  static constexpr int kKey = D * kBits / 128;    // dwords of a key row a lane takes
  static constexpr int kState = (4 * kO + 2) * 64;  // floats of a wave's O, maximum and sum
};

// N dwords from a place aligned to them (to 16 bytes).
template <int N>
__device__ __forceinline__ void load_words(const uint8_t* at, uint32_t* w) {
  typedef uint32_t Whole __attribute__((ext_vector_type(N)));
  typedef Whole Vec __attribute__((aligned(N < 4 ? 4 * N : 16)));
  const Vec x = *reinterpret_cast<const Vec*>(at);
#pragma unroll
  for (int i = 0; i < N; ++i) w[i] = x[i];
}

// Nibble i of both halves of w as two bf16 of 16 + code.
template <int i>
__device__ __forceinline__ uint32_t nibbles_bf16(uint32_t w) {
  const uint32_t x = 4 * i < 3 ? w << (3 - 4 * i) : w >> (4 * i - 3);
  return (x & 0x00780078u) | 0x41804180u;
}

// Bytes i of a and b as two bf16.
template <int i>
__device__ __forceinline__ uint32_t bytes_bf16(uint32_t a, uint32_t b) {
  const uint32_t x = __float_as_uint((float)(a >> 8 * i & 255u)), y = __float_as_uint((float)(b >> 8 * i & 255u));
  return __builtin_amdgcn_perm(y, x, 0x07060302);
}

// Step c's operand from a lane's piece of a key row.
template <int kBits>
__device__ __forceinline__ bf16x8 key_operand(const uint32_t* w, int c) {
  u32x4 x;
  if constexpr (kBits == 4) {
    x = u32x4{nibbles_bf16<0>(w[c]), nibbles_bf16<1>(w[c]), nibbles_bf16<2>(w[c]), nibbles_bf16<3>(w[c])};
  } else {
    const uint32_t a = w[2 * c], b = w[2 * c + 1];
    x = u32x4{bytes_bf16<0>(a, a >> 8), bytes_bf16<2>(a, a >> 8), bytes_bf16<0>(b, b >> 8), bytes_bf16<2>(b, b >> 8)};
  }
  return as_bf16x8(x);
}

// A lane's parts of eight value rows, and the operand of output tile n from them:
// its channel n (the map from (part, n) to a channel is qa_channel).
template <int D, int kBits>
struct ValuePart;

template <>
struct ValuePart<128, 4> {
  uint32_t w[8];
  __device__ __forceinline__ void load(int j, const uint8_t* row, int g) {
    w[j] = *reinterpret_cast<const uint32_t*>(row + 4 * g);
  }
  template <int n>
  __device__ __forceinline__ bf16x8 operand() const {
    u32x4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x[i] = nibbles_bf16<n / 2>(__builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], n % 2 ? 0x07060302 : 0x05040100));
    return as_bf16x8(x);
  }
};

template <>
struct ValuePart<64, 4> {
  uint16_t w[8];
  __device__ __forceinline__ void load(int j, const uint8_t* row, int g) {
    w[j] = *reinterpret_cast<const uint16_t*>(row + 2 * g);
  }
  template <int n>
  __device__ __forceinline__ bf16x8 operand() const {
    u32x4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = nibbles_bf16<n>((uint32_t)w[2 * i] | (uint32_t)w[2 * i + 1] << 16);
    return as_bf16x8(x);
  }
};

template <int D>
struct ValuePart<D, 8> {
  static constexpr int kW = D / 64;
  uint32_t w[8][kW];
  __device__ __forceinline__ void load(int j, const uint8_t* row, int g) { load_words<kW>(row + 4 * kW * g, w[j]); }
  template <int n>
  __device__ __forceinline__ bf16x8 operand() const {
    u32x4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = bytes_bf16<n % 4>(w[2 * i][n / 4], w[2 * i + 1][n / 4]);
    return as_bf16x8(x);
  }
};

// Output tile n leaves lane l its channels of parts 4 * (l/16) + r; of the lane's
// D / 4 channels, which stand next to one another, this is the one of (r, n).
template <int D, int kBits>
constexpr int qa_channel(int r, int n) {
  if (D == 64 && kBits == 4) return 8 * (r / 2) + r % 2 + 2 * n;
  return D / 16 * r + n;
}

template <int n, int N, class F>
__device__ __forceinline__ void unrolled(F&& f) {
  if constexpr (n < N) {
    f(std::integral_constant<int, n>{});
    unrolled<n + 1, N>(f);
  }
}

template <int D, int kBits>
__global__ __launch_bounds__(kQaWaves * 64) void quant_attn_kernel(QuantAttnParams p) {
  typedef QaShape<D, kBits> Shape;
  typedef QuantRow<D, kBits> Row;
  constexpr int kC = Shape::kC, kO = Shape::kO, W = kQaWaves;
  __shared__ float smem[W * Shape::kState];
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = lane_id();
  const int g = l & 15, lg = l >> 4;
  const int ct = (int)p.over_heads_k.div(blockIdx.y), h = blockIdx.y - ct * p.heads_k, b = blockIdx.z;
  const int len = max(p.seqlens[b], 0);

  // the split's tiles: an equal part of those that the sequence has
  const int all = (int)min(((int64_t)len + 15) / 16, (int64_t)p.width * p.tiles.d);
  const int t0 = (int)((int64_t)all * blockIdx.x / p.splits), t1 = (int)((int64_t)all * (blockIdx.x + 1) / p.splits);

  // this lane's column: new token `fresh` of head h * group + hh; it sees `limit` tokens
  const int column = min(16 * ct + g, p.columns - 1);
  const int fresh = (int)p.over_group.div((uint32_t)column), hh = column - fresh * p.group;
  const int first = len - p.new_tokens + 1, limit = first + fresh;
  bf16x8 Q[kC];
  {
    const uint16_t* row = p.q + b * p.q_batch + fresh * p.q_token + (int64_t)(h * p.group + hh) * p.q_head + D / 4 * lg;
#pragma unroll
    for (int c = 0; c < kC; ++c) Q[c] = *reinterpret_cast<const bf16x8*>(row + 8 * c);
  }
  // the sum of the column's q, and what the 16s of 4-bit codes add to a score
  f32x4 sum_q = {0.f, 0.f, 0.f, 0.f};
  {
    const bf16x8 ones = as_bf16x8(u32x4{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u});
#pragma unroll
    for (int c = 0; c < kC; ++c) sum_q = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, Q[c], sum_q, 0, 0, 0);
  }
  const float qs = sum_q[0] * p.scale_log2;
  const f32x4 start = sum_q * (kBits == 4 ? -16.f : 0.f);

  f32x4 O[kO];
#pragma unroll
  for (int i = 0; i < kO; ++i) O[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  float m_run = -INFINITY, l_run = 0.f, z = 0.f;  // z: sum p low_v, and the 16s

  const int page = p.page;
  const int k_at = 8 * page + g * Row::kBytes + 4 * Shape::kKey * lg;
  const int v_at = (8 + Row::kBytes) * page + 4 * lg * Row::kBytes;

  // Lane i holds the place of tile i%2 of the wave's (32 c0 + i/2)-th pair: its page
  // (-1: none of the pool, or no tile of the split) and its tile there.
  for (int c0 = 0; t0 + 2 * (w + W * 32 * c0) < t1; ++c0) {
    int block = -1, sub = 0;
    {
      const int tile = t0 + 2 * (w + W * (32 * c0 + (l >> 1))) + (l & 1);
      if (tile < t1) {
        const int lp = (int)p.tiles.div((uint32_t)tile);
        sub = tile - lp * (int)p.tiles.d;
        block = p.table[b * p.table_stride + lp];
        if (block >= p.num_blocks) block = -1;
      }
    }
    for (int i = 0; i < 32; ++i) {
      const int tile = t0 + 2 * (w + W * (32 * c0 + i));
      if (tile >= t1) break;
      int b0 = __builtin_amdgcn_readlane(block, 2 * i), s0 = __builtin_amdgcn_readlane(sub, 2 * i);
      int b1 = __builtin_amdgcn_readlane(block, 2 * i + 1), s1 = __builtin_amdgcn_readlane(sub, 2 * i + 1);
      if (b0 < 0 && b1 < 0) continue;
      const bool none0 = b0 < 0, none1 = b1 < 0;  // a tile without a page reads the other's
      if (none0) b0 = b1, s0 = s1;
      if (none1) b1 = b0, s1 = s0;
      const uint8_t* r0 = p.cache + ((int64_t)b0 * p.heads_k + h) * p.record;
      const uint8_t* r1 = p.cache + ((int64_t)b1 * p.heads_k + h) * p.record;
      uint32_t K0[Shape::kKey], K1[Shape::kKey], side[2][8];
      ValuePart<D, kBits> V;
      load_words<Shape::kKey>(r0 + k_at + 16 * s0 * Row::kBytes, K0);
      load_words<Shape::kKey>(r1 + k_at + 16 * s1 * Row::kBytes, K1);
      load_words<8>(r0 + 8 * (16 * s0 + 4 * lg), side[0]);
      load_words<8>(r1 + 8 * (16 * s1 + 4 * lg), side[1]);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        V.load(j, r0 + v_at + (16 * s0 + j) * Row::kBytes, g);
        V.load(4 + j, r1 + v_at + (16 * s1 + j) * Row::kBytes, g);
      }
      f32x4 S0 = start, S1 = start;
#pragma unroll
      for (int c = 0; c < kC; ++c) {
        S0 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(key_operand<kBits>(K0, c), Q[c], S0, 0, 0, 0);
        S1 = __builtin_amdgcn_mfma_f32_16x16x32_bf16(key_operand<kBits>(K1, c), Q[c], S1, 0, 0, 0);
      }
      float s[8], vs[8], vl[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const uint32_t kp = side[j / 4][2 * (j % 4)], vp = side[j / 4][2 * (j % 4) + 1];
        const float ks = __uint_as_float(kp << 16), kl = __uint_as_float(kp & 0xFFFF0000u);
        s[j] = fmaf(ks * p.scale_log2, j < 4 ? S0[j % 4] : S1[j % 4], kl * qs);
        vs[j] = __uint_as_float(vp << 16);
        vl[j] = __uint_as_float(vp & 0xFFFF0000u);
      }
      // Behind a column's limit and where there is no page nothing counts, whatever it holds.
      if (none0 || none1 || first - 16 * tile < 32) {  // (uniform)
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool seen = 16 * (j / 4) + 4 * lg + j % 4 < limit - 16 * tile && !(j < 4 ? none0 : none1);
          s[j] = seen ? s[j] : -INFINITY;
          vs[j] = seen ? vs[j] : 0.f;
          vl[j] = seen ? vl[j] : 0.f;
        }
      }
      float mx = s[0];
#pragma unroll
      for (int j = 1; j < 8; ++j) mx = fmaxf(mx, s[j]);
      const float m_new = fmaxf(m_run, wave_max16(mx));
      const float m_use = m_new == -INFINITY ? 0.f : m_new;
      const float alpha = __builtin_amdgcn_exp2f(m_run - m_use);
      m_run = m_new;
      l_run *= alpha;
      z *= alpha;
      if (__builtin_amdgcn_ballot_w64(alpha != 1.f)) {
#pragma unroll
        for (int k = 0; k < kO; ++k) O[k] *= alpha;
      }
      // weights times scales as sums of three bf16, all of their 24 bits
      u32x4 hi, mid, lo;
#pragma unroll
      for (int i2 = 0; i2 < 4; ++i2) {
        uint32_t a[2], c[2], d[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const int j = 2 * i2 + e;
          const float x = __builtin_amdgcn_exp2f(s[j] - m_use);
          l_run += x;
          const float y = x * vs[j];
          z = fmaf(x, vl[j], z);
          if constexpr (kBits == 4) z = fmaf(y, -16.f, z);
          a[e] = __float_as_uint(y) & 0xFFFF0000u;
          const float r = y - __uint_as_float(a[e]);
          c[e] = __float_as_uint(r) & 0xFFFF0000u;
          d[e] = __float_as_uint(r - __uint_as_float(c[e]));
        }
        hi[i2] = __builtin_amdgcn_perm(a[1], a[0], 0x07060302);
        mid[i2] = __builtin_amdgcn_perm(c[1], c[0], 0x07060302);
        lo[i2] = __builtin_amdgcn_perm(d[1], d[0], 0x07060302);
      }
      unrolled<0, kO>([&](auto n) {
        constexpr int k = decltype(n)::value;
        const bf16x8 A = V.template operand<k>();
        O[k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(A, as_bf16x8(hi), O[k], 0, 0, 0);
        O[k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(A, as_bf16x8(mid), O[k], 0, 0, 0);
        O[k] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(A, as_bf16x8(lo), O[k], 0, 0, 0);
      });
    }
  }

  // The waves' states merged by the first one.
  l_run = wave_sum16(l_run);
  z = wave_sum16(z);
  float* cb = smem + w * Shape::kState + l;
#pragma unroll
  for (int i = 0; i < kO; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r) cb[(4 * i + r) * 64] = O[i][r] + z;
  cb[4 * kO * 64] = m_run;
  cb[(4 * kO + 1) * 64] = l_run;
  __syncthreads();
  if (w != 0) return;
  const float* src = smem + l;
  float m = -INFINITY;
#pragma unroll
  for (int i = 0; i < W; ++i) m = fmaxf(m, src[i * Shape::kState + 4 * kO * 64]);
  const float m_use = m == -INFINITY ? 0.f : m;
  float sum = 0.f, o[4 * kO];
#pragma unroll
  for (int i = 0; i < 4 * kO; ++i) o[i] = 0.f;
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const float f = __builtin_amdgcn_exp2f(src[i * Shape::kState + 4 * kO * 64] - m_use);
    sum += src[i * Shape::kState + (4 * kO + 1) * 64] * f;
#pragma unroll
    for (int k = 0; k < kO; ++k)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[qa_channel<D, kBits>(r, k)] += src[i * Shape::kState + (4 * k + r) * 64] * f;
  }
  if (16 * ct + g >= p.columns) return;
  const int head = h * p.group + hh;
  const int64_t row = ((int64_t)b * p.heads + head) * p.new_tokens + fresh;
  if (p.splits == 1) {
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    uint16_t* out = p.out + (((int64_t)b * p.new_tokens + fresh) * p.heads + head) * D + D / 4 * lg;
#pragma unroll
    for (int i = 0; i < kO / 2; ++i) {
      u32x4 x;
#pragma unroll
      for (int j = 0; j < 4; ++j) x[j] = pack_bf16x2(o[8 * i + 2 * j] * inv, o[8 * i + 2 * j + 1] * inv);
      *reinterpret_cast<u32x4*>(out + 8 * i) = x;
    }
    if (p.lse && lg == 0) p.lse[row] = sum == 0.f ? -INFINITY : (m + __log2f(sum)) * 0.6931471805599453f;
  } else {
    const int64_t slot = row * p.splits + blockIdx.x;
    float* out = p.ws_o + slot * D + D / 4 * lg;
#pragma unroll
    for (int i = 0; i < kO; ++i)
      *reinterpret_cast<f32x4*>(out + 4 * i) = f32x4{o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]};
    if (lg == 0) *reinterpret_cast<float2*>(p.ws_ml + 2 * slot) = float2{m, sum};
  }
}

// How many splits: one workgroup a CU, each wave with a pair of tiles at least.
static int qa_splits(int batch, int units, int64_t tiles, int num_splits) {
  const int64_t most = std::max<int64_t>(1, (tiles + 2 * kQaWaves - 1) / (2 * kQaWaves));
  const int64_t want = num_splits > 0 ? num_splits : std::max<int64_t>(1, device_cu_count() / ((int64_t)batch * units));
  return (int)std::min(want, most);
}

static int qa_column_tiles(int heads, int heads_k, int new_tokens) {
  return (int)(((int64_t)(heads / heads_k) * new_tokens + 15) / 16);
}

static size_t qa_ws_bytes(int64_t rows, int head_dim, int splits) {
  return splits <= 1 ? 0 : (size_t)rows * splits * (head_dim + 2) * sizeof(float);
}

}  // namespace zs

using namespace zs;

extern "C" size_t zs_decode_attention_quant_workspace_bytes(int batch, int new_tokens, int num_heads, int num_heads_k,
                                                            int head_dim, int max_blocks_per_seq,
                                                            int page_block_size, int num_splits) {
  if (batch <= 0 || new_tokens <= 0 || num_heads <= 0 || num_heads_k <= 0 || num_heads % num_heads_k ||
      head_dim <= 0 || max_blocks_per_seq <= 0 || page_block_size < 16 || num_splits < 0)
    return 0;
  const int64_t rows = (int64_t)batch * num_heads * new_tokens, tiles = (int64_t)max_blocks_per_seq * (page_block_size / 16);
  const int64_t units = (int64_t)num_heads_k * qa_column_tiles(num_heads, num_heads_k, new_tokens);
  if (rows > INT_MAX || tiles > INT_MAX || units > 65535) return 0;  // (such a call is refused)
  return qa_ws_bytes(rows, head_dim, qa_splits(batch, (int)units, tiles, num_splits));
}

extern "C" int zs_decode_attention_quant_paged(void* stream, const uint16_t* q, int64_t q_batch_stride,
                                               int64_t q_token_stride, int64_t q_head_stride, const uint8_t* cache,
                                               int num_blocks, int page_block_size, int bits,
                                               const int32_t* block_table, int64_t table_stride,
                                               int max_blocks_per_seq, const int32_t* cache_seqlens, int batch,
                                               int new_tokens, int num_heads, int num_heads_k, int head_dim,
                                               float softmax_scale, uint16_t* out, float* softmax_lse,
                                               void* workspace, size_t workspace_bytes, int num_splits) {
  if (!q || !cache || !block_table || !cache_seqlens || !out) return ZS_E_INVAL;
  const int bad = quant_checks(cache, num_blocks, page_block_size, num_heads_k, head_dim, bits);
  if (bad != ZS_OK) return bad;
  if (batch <= 0 || new_tokens <= 0 || num_heads <= 0 || num_heads % num_heads_k || max_blocks_per_seq <= 0 ||
      num_splits < 0)
    return ZS_E_INVAL;
  if (table_stride < max_blocks_per_seq && batch > 1) return ZS_E_INVAL;
  if (((reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(out) | reinterpret_cast<uintptr_t>(workspace)) &
       15) ||
      ((q_batch_stride | q_token_stride | q_head_stride) & 7))
    return ZS_E_INVAL;
  const int64_t rows = (int64_t)batch * num_heads * new_tokens, tiles = (int64_t)max_blocks_per_seq * (page_block_size / 16);
  const int64_t columns = (int64_t)(num_heads / num_heads_k) * new_tokens, units = num_heads_k * ((columns + 15) / 16);
  if (batch > 65535 || units > 65535) return ZS_E_UNSUPPORTED;
  if (rows > INT_MAX || tiles > INT_MAX) return ZS_E_OVERFLOW;
  QuantAttnParams p{};
  p.splits = qa_splits(batch, (int)units, tiles, num_splits);
  if (!grid_fits(p.splits, kQaWaves * 64) || (p.splits > 1 && !grid_fits(rows, kMergeWaves * 64)))
    return ZS_E_OVERFLOW;
  if (workspace_bytes < qa_ws_bytes(rows, head_dim, p.splits) || (p.splits > 1 && !workspace)) return ZS_E_INVAL;
  p.q = q;
  p.q_batch = q_batch_stride;
  p.q_token = q_token_stride;
  p.q_head = q_head_stride;
  p.cache = cache;
  p.record = (int64_t)page_block_size * quant_token_bytes(head_dim, bits);
  p.table = block_table;
  p.table_stride = table_stride;
  p.seqlens = cache_seqlens;
  p.out = out;
  p.lse = softmax_lse;
  p.ws_o = static_cast<float*>(workspace);
  p.ws_ml = p.ws_o + (size_t)rows * p.splits * head_dim;
  p.num_blocks = num_blocks;
  p.width = max_blocks_per_seq;
  p.page = page_block_size;
  p.heads = num_heads;
  p.heads_k = num_heads_k;
  p.group = num_heads / num_heads_k;
  p.new_tokens = new_tokens;
  p.columns = (int)columns;
  p.tiles = FastDiv::of(page_block_size / 16);
  p.over_group = FastDiv::of(p.group);
  p.over_heads_k = FastDiv::of(num_heads_k);
  p.scale_log2 = softmax_scale * 1.4426950408889634f;
  const hipStream_t st = (hipStream_t)stream;
  const dim3 grid(p.splits, (unsigned)units, batch), block(kQaWaves * 64);
  auto launch = [&](auto d, auto n) {
    hipLaunchKernelGGL((quant_attn_kernel<decltype(d)::value, decltype(n)::value>), grid, block, 0, st, p);
  };
  typedef std::integral_constant<int, 4> Four;
  typedef std::integral_constant<int, 8> Eight;
  typedef std::integral_constant<int, 64> Small;
  typedef std::integral_constant<int, 128> Large;
  if (head_dim == 128)
    bits == 4 ? launch(Large{}, Four{}) : launch(Large{}, Eight{});
  else
    bits == 4 ? launch(Small{}, Four{}) : launch(Small{}, Eight{});
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && p.splits > 1)
    e = merge_splits(st, SplitMerge::of(p.ws_o, p.ws_ml, out, softmax_lse, p.splits, (int)rows, num_heads, new_tokens),
                     head_dim);
  return e == hipSuccess ? ZS_OK : (int)e;
}
