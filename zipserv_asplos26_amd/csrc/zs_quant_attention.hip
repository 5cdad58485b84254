// zs_quant_attention.hip -- attention of each sequence's last tokens over a paged
// KV cache held in 4 or 8 bits (gfx950; the layout is in zs_quant.hpp).
//
// With a key k = low_k + s_k c and a value v = low_v + s_v c, c whole numbers of
// 0..15 or 0..255,
//   q.k       = s_k (q.c) + low_k sum(q),
//   sum p v   = sum (p s_v) c + sum p low_v,
// so the codes themselves are the matrix operands, exactly, and a token costs two
// products more a row, not a value each channel.
//
// A column is a (new token, query head) of one KV head's group; a workgroup of
// kQaWaves waves takes up to 16 columns (of many: 32) and a part of the tokens, a wave 32
// tokens (two tiles of 16) at a time, all in registers, with the next pair's loads on the way:
//   S^T = C_k q^T with v_mfma_f32_16x16x32_bf16: lane l holds D / 4 codes of token
//   l%16 (channels D/4 * (l/16) and up, one piece of its row), 8 of them the A operand of a
//   step; q^T (lane l: column l%16, the same channels) is the B operand.
//   Online softmax in the log2 domain, fp32.
//   O^T += C_v^T W^T over K = 32 tokens with the same instruction: S^T leaves lane l the
//   weights of column l%16 for tokens 4*(l/16)..+3 of both tiles, the B operand if k
//   index 8*(l/16) + j stands for token 4*(l/16) + j%4 of tile j/4; lane l reads the
//   l%16-th part of those eight rows, D / 16 channels of 8 tokens, which are D / 16 A
//   operands.
// A code is a bf16's bits, which the matrix cores take as they are: below 128 a subnormal's,
// and above they go on in the same steps.  That takes an "and" for two codes and a
// shift for four (8 bits of values: a byte permute for two).  What meets them is bf16 as well:
// q itself, times a power of two a column, and the weights times s_v as three bf16 each, all
// of their 24 bits.  A weight is relative to the largest score alone: the size of a value
// needs no reference of its own as long as the sums stay between kLeastSum and kMostSum.  A
// part of a sequence where they do not is done a second time, with a power of two for each
// value and a reference for weights times these beside the one for weights.
// With 8 columns or fewer the tile's other columns repeat them, and a lane does the softmax
// of only a half of its tokens (4 or fewer: a quarter) and gets the other weights from
// the lanes that did them.
//
// What bounds it: 64 sequences' 8000 tokens (64 / 8 heads of 128 in 4 bits, 557 MB) take 107
// us, 5.2 TB/s, with the vector unit at work in half of the cycles; with 16 columns and
// more the vector instructions do (three tiles of columns over 113 MB: 67 us); one
// sequence's 32000 tokens 13.5 us and 4 for the merge, start, loads and merge being a chain
// of latencies.  A part that is done a second time takes 1.5 to 2.3 times as long.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cfloat>
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
  float* ws_o;    // [slot][Hkv][columns of a KV head][D] (where sequences may be cut): results of the slots
  float* ws_ml;   // [slot][Hkv][columns][2]: what weights are relative to (a power of two: its log2) and their sum
  int2* ws_plan;  // [B]: a sequence's first slot and its splits (where they go by the lengths)
  int num_blocks, width, page, heads, heads_k, group, new_tokens, columns, batch;
  int splits;           // of every sequence, or 0: by the lengths
  int parts;            // of all sequences together, where they are cut by the lengths
  FastDiv tiles;        // 16-token tiles of a page
  FastDiv over_group;   // a column's new token
  FastDiv over_heads_k, over_column_tiles, over_splits;
  float scale_log2, flip;  // of the softmax scale: its size, and its sign as 1 or -1
};

constexpr int kQaWaves = 4;
// A column's largest weight so far is 1, or up to 2^4 before the reference moves (small, so that
// the argument of a weight's exponential has few digits before its point).  Scales of values go
// in times kScaleFactor, so that weight * scale times a code in units of 2^kCodeUnit is
// 1 / kSumFactor of what it stands for: 2^-63 for the largest weight and a scale of 2^-30, 63
// bits above the least normal number, while scales up to 2^22 leave sums of 2^31 room.
constexpr float kWeightLag = 4.f;
constexpr float kScaleFactor = 0x1p100f;
constexpr float kSumFactor = 0x1p33f;  // 2^-kCodeUnit / kScaleFactor
// Whether that was enough is seen from a column's largest sum of such products: below the one
// (small scales, or none with the large weights) digits may be lost, above the other (or
// with a sum of lows above kSumFactor times that) a sum may have left fp32.
constexpr float kLeastSum = 0x1p-80f, kMostSum = 0x1p80f;

template <int D, int kBits>
struct QaShape {
  static constexpr int kC = D / 32;               // steps of q.c
  static constexpr int kO = D / 16;               // tiles of channels of the output
  static constexpr int kKey = D * kBits / 128;    // dwords of a key row a lane takes
  static constexpr int kState = (4 * kO + 3) * 64;  // floats of a wave's O, references and sum
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

// Codes as a bf16's bits: code c stands for c 2^kCodeUnit, in nibbles 1 and 3 for 16 times as
// much.  (The matrix cores line sums up by the exponent that an operand could have, and a
// small subnormal's leading zeros are digits lost: 4-bit scores are 2^-24.7 of their
// products' sizes off at most and 2^-28.5 on average here.  As fp16 subnormals at bits 0..3 and
// 4..7 they were 2^-21.2 and 2^-23.8 off, at bits 2..5 and 6..9, with another shift, 2^-24.1 and
// 2^-27.1.)
constexpr int kCodeUnit = -133;

template <int i>
__device__ __forceinline__ uint32_t nibbles_bf16(uint32_t w) {
  return (i >= 2 ? w >> 8 : w) & (i % 2 ? 0x00F000F0u : 0x000F000Fu);
}

// Step c's operand from a lane's piece of a key row.  Nibbles 1 and 3 are 16 times as
// large, and q is 1/16 there.
template <int kBits>
__device__ __forceinline__ bf16x8 key_operand(const uint32_t* w, int c) {
  u32x4 x;
  if constexpr (kBits == 4) {
    x = u32x4{nibbles_bf16<0>(w[c]), nibbles_bf16<1>(w[c]), nibbles_bf16<2>(w[c]), nibbles_bf16<3>(w[c])};
  } else {
    const uint32_t u = w[2 * c], v = w[2 * c + 1];
    x = u32x4{u & 0x00FF00FFu, u >> 8 & 0x00FF00FFu, v & 0x00FF00FFu, v >> 8 & 0x00FF00FFu};
  }
  return __builtin_bit_cast(bf16x8, x);
}

// The same channels of q, 8 bf16 times 2^up (and by, 1 or -1), in the order and with the factors
// of a key operand.
template <int kBits>
__device__ __forceinline__ bf16x8 query_operand(u32x4 in, float by, int up) {
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = ldexpf(__uint_as_float(in[i] << 16) * by, up);
    x[2 * i + 1] = ldexpf(__uint_as_float(in[i] & 0xFFFF0000u) * by, up);
  }
  bf16x8 y;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    y[i] = (__bf16)(kBits == 4 ? x[i] * (i & 2 ? 0.0625f : 1.f) : x[(i & 4) + (i & 1) * 2 + (i >> 1 & 1)]);
  return y;
}

// A lane's parts of eight value rows, and the operand of output tile n from them, its
// channel n of the eight tokens (the map from (part, n) to a channel is qa_channel),
// 16 times as large where sixteenfold(n).
template <int D, int kBits>
struct ValuePart;

template <>
struct ValuePart<128, 4> {
  uint32_t w[8];
  __device__ __forceinline__ void load(int j, const uint8_t* part) {
    w[j] = *reinterpret_cast<const uint32_t*>(part);
  }
  static constexpr bool sixteenfold(int n) { return n / 2 % 2; }
  template <int n>
  __device__ __forceinline__ bf16x8 operand() const {
    u32x4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x[i] = nibbles_bf16<n / 2>(__builtin_amdgcn_perm(w[2 * i + 1], w[2 * i], n % 2 ? 0x07060302 : 0x05040100));
    return __builtin_bit_cast(bf16x8, x);
  }
};

template <>
struct ValuePart<64, 4> {
  uint16_t w[8];
  __device__ __forceinline__ void load(int j, const uint8_t* part) {
    w[j] = *reinterpret_cast<const uint16_t*>(part);
  }
  static constexpr bool sixteenfold(int n) { return n % 2; }
  template <int n>
  __device__ __forceinline__ bf16x8 operand() const {
    u32x4 x;
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = nibbles_bf16<n>((uint32_t)w[2 * i] | (uint32_t)w[2 * i + 1] << 16);
    return __builtin_bit_cast(bf16x8, x);
  }
};

template <int D>
struct ValuePart<D, 8> {
  static constexpr int kW = D / 64;
  uint32_t w[8][kW];
  __device__ __forceinline__ void load(int j, const uint8_t* part) { load_words<kW>(part, w[j]); }
  static constexpr bool sixteenfold(int) { return false; }
  template <int n>
  __device__ __forceinline__ bf16x8 operand() const {
    u32x4 x;  // byte n % 4 of both tokens, zeros above
#pragma unroll
    for (int i = 0; i < 4; ++i)
      x[i] = __builtin_amdgcn_perm(w[2 * i + 1][n / 4], w[2 * i][n / 4], 0x0C040C00u + 0x00010001u * (n % 4));
    return __builtin_bit_cast(bf16x8, x);
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

// How the tokens of a batch are cut.  Either every sequence into the same number of
// splits, or, where that is left open, the tiles of all sequences, one behind another, into
// p.parts equal parts, so that every workgroup has as much to do however the lengths differ:
// a workgroup takes what its part has of each sequence, one after the other.  Part i
// starts at tile floor(i T / P) of the T.  What it has of a sequence that it does not
// have whole goes into slot 2 i, or 2 i + 1 where the sequence starts inside the part (a
// part has one at most that ends, and one that starts, outside it).
constexpr int kLeastChunk = 16;  // tiles of a part (one sequence of 2000 tokens: 14.3 us with 32, 12.5 with 16)

__device__ __forceinline__ int qa_tiles_of(const QuantAttnParams& p, int len) {
  return (int)min(((int64_t)max(len, 0) + 15) / 16, (int64_t)p.width * p.tiles.d);
}

// (Products below 2^53 are exact, and so is the floor of a quotient of them.)
__device__ __forceinline__ int qa_part_start(int i, int parts, int total) {
  return (int)floor((double)i * total / parts);
}
// The part that tile t is in: the last i with floor(i T / P) <= t.
__device__ __forceinline__ int qa_part_of(int t, int parts, int total) {
  return (int)floor(((double)(t + 1) * parts - 1) / total);
}

// The lane, and what is made of it, anew: kept over a loop that it is used in at both ends
// it takes registers.
__device__ __forceinline__ int qa_lane() {
  int l = lane_id();
  asm volatile("" : "+v"(l));
  return l;
}

// The waves' states of a tile of columns merged and written, two output tiles a wave: the
// result, or what goes into a slot (slot >= 0; O divided by the sum as well, so that
// slots are alike whatever their weights were relative to).  kOdd: O is to be
// multiplied by 2^(off_own - 128).
template <int D, int kBits, int kColumns, bool kOdd>
__device__ __forceinline__ void qa_finish(const QuantAttnParams& p, float* smem, const f32x4* O, float m_own,
                                          float l_own, float off_own, int ct, int h, int b, int slot) {
  typedef QaShape<D, kBits> Shape;
  constexpr int kO = Shape::kO, W = kQaWaves;
  static_assert(W >= kO / 2, "");
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), l = qa_lane(), lg = l >> 4;
  float* cb = smem + w * Shape::kState + l;
#pragma unroll
  for (int i = 0; i < kO; ++i)
#pragma unroll
    for (int r = 0; r < 4; ++r)
      cb[(4 * i + r) * 64] = O[i][r];
  cb[4 * kO * 64] = m_own;
  cb[(4 * kO + 1) * 64] = l_own;
  if constexpr (kOdd) cb[(4 * kO + 2) * 64] = off_own;
  __syncthreads();
  if (w >= kO / 2) return;
  const float* src = smem + l;
  float m = -FLT_MAX, off = -FLT_MAX, sum = 0.f, o[2][4] = {};
#pragma unroll
  for (int i = 0; i < W; ++i) m = fmaxf(m, src[i * Shape::kState + 4 * kO * 64]);
  if constexpr (kOdd) {
#pragma unroll
    for (int i = 0; i < W; ++i)
      off = fmaxf(off, src[i * Shape::kState + (4 * kO + 2) * 64] + (src[i * Shape::kState + 4 * kO * 64] - m));
  }
#pragma unroll
  for (int i = 0; i < W; ++i) {
    const float less = src[i * Shape::kState + 4 * kO * 64] - m;
    const float f = __builtin_amdgcn_exp2f(less);
    float fo = f;
    if constexpr (kOdd) fo = __builtin_amdgcn_exp2f(src[i * Shape::kState + (4 * kO + 2) * 64] + less - off);
    sum += src[i * Shape::kState + (4 * kO + 1) * 64] * f;
#pragma unroll
    for (int n = 0; n < 2; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) o[n][r] += src[i * Shape::kState + (4 * (2 * w + n) + r) * 64] * fo;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
  for (int n = 0; n < 2; ++n)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      o[n][r] *= inv;
      if constexpr (kOdd) o[n][r] = ldexpf(o[n][r], (int)fmaxf(off, -1000.f) - 128);
    }
  const int column = kColumns * ct + (l & 15);
  if ((l & 15) >= kColumns || column >= p.columns) return;
  // neighbouring channels: (r, 0), (r, 1), or with two codes of a byte apart (2i, 0),
  // (2i + 1, 0), (2i, 1), (2i + 1, 1)
  constexpr bool kFour = D == 64 && kBits == 4;
  static_assert(qa_channel<D, kBits>(1, 0) == (kFour ? 1 : D / 16), "");
  const int at = D / 4 * lg + (kFour ? 4 : 2) * w;
  const int fresh = (int)p.over_group.div((uint32_t)column), head = h * p.group + column - fresh * p.group;
  if (slot < 0) {
    uint16_t* out = p.out + (((int64_t)b * p.new_tokens + fresh) * p.heads + head) * D + at;
    if constexpr (kFour) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        *reinterpret_cast<uint2*>(out + 8 * i) = uint2{pack_bf16x2(o[0][2 * i], o[0][2 * i + 1]),
                                                       pack_bf16x2(o[1][2 * i], o[1][2 * i + 1])};
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r)
        *reinterpret_cast<uint32_t*>(out + D / 16 * r) = pack_bf16x2(o[0][r], o[1][r]);
    }
    if (p.lse && lg == 0 && w == 0)
      p.lse[((int64_t)b * p.heads + head) * p.new_tokens + fresh] = natural_log_sum(m, sum);
  } else {
    const int64_t row = ((int64_t)slot * p.heads_k + h) * p.columns + column;
    float* out = p.ws_o + row * D + at;
    if constexpr (kFour) {
#pragma unroll
      for (int i = 0; i < 2; ++i)
        *reinterpret_cast<f32x4*>(out + 8 * i) = f32x4{o[0][2 * i], o[0][2 * i + 1], o[1][2 * i], o[1][2 * i + 1]};
    } else {
#pragma unroll
      for (int r = 0; r < 4; ++r) *reinterpret_cast<float2*>(out + D / 16 * r) = float2{o[0][r], o[1][r]};
    }
    if (lg == 0 && w == 0) *reinterpret_cast<float2*>(p.ws_ml + 2 * row) = float2{m, sum};
  }
}

// What a wave has of a pair of tiles: codes, and (scale, low) of the keys and values of
// the lane's kTokens tokens.
template <int D, int kBits, int kTokens>
struct QaPair {
  uint32_t k[2][QaShape<D, kBits>::kKey], side[2 * kTokens];
  ValuePart<D, kBits> v;
  int tile;        // the first one's number in the sequence
  bool none[2];    // no page of the pool
};

// What no kernel writes while this one runs, for scalar loads.
typedef const int32_t __attribute__((address_space(4))) * ConstantInts;
__device__ __forceinline__ ConstantInts as_constant(const int32_t* p) { return (ConstantInts)(uintptr_t)p; }

// Lane l's x from lane l%16 + kBy (of the 16, going round) of its row.
template <int kBy>
__device__ __forceinline__ uint32_t row_from(uint32_t x) {
  return __builtin_amdgcn_update_dpp(0, x, 0x120 + 16 - kBy, 0xF, 0xF, false);  // row_ror
}
__device__ __forceinline__ float row_from8(float x) { return __uint_as_float(row_from<8>(__float_as_uint(x))); }
__device__ __forceinline__ float row_from4(float x) { return __uint_as_float(row_from<4>(__float_as_uint(x))); }

// Waves a SIMD: what the registers of a pair on its way and one in work leave room for.
constexpr int qa_waves(int dim, int bits, int fold, int tiles) {
  return tiles > 1 || (dim == 128 && bits == 8 && fold < 4) ? 2 : 3;
}

// What a workgroup's waves share.
template <int D, int kBits, int kTiles>
struct QaShared {
  float states[kQaWaves * QaShape<D, kBits>::kState];
  __attribute__((aligned(16))) bf16x8 q[kTiles][QaShape<D, kBits>::kC][64];  // (one tile's stays in registers)
  float2 column[kTiles][16];
  int odd[kQaWaves];
};

// Tiles t0 .. t1 of sequence b, into its slot or as its result.  kOdd: value rows may be of any
// size; without, whether sums say that some are too small or too large is returned (for the
// whole workgroup), and then nothing is written.
template <int D, int kBits, int kFold, int kTiles, bool kOdd>
__device__ __forceinline__ bool qa_segment(const QuantAttnParams& p, QaShared<D, kBits, kTiles>& shared, int ct, int h,
                                           int b, int len, int t0, int t1, int slot) {
  static_assert(kTiles == 1 || (kFold == 1 && kTiles <= kQaWaves), "");
  typedef QaShape<D, kBits> Shape;
  typedef QuantRow<D, kBits> Row;
  constexpr int kC = Shape::kC, kO = Shape::kO, W = kQaWaves;
  constexpr int kColumns = 16 / kFold, kTokens = 8 / kFold;  // of a tile of columns; a lane's tokens of a pair
  typedef QaPair<D, kBits, kTokens> Pair;
  const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int l = qa_lane();
  const int g = l & 15, lg = l >> 4;
  const int fold = g / kColumns;
  // the lane's tokens of a pair: kTokens from `token` of tile `mine` (all of both: 4 each)
  const int mine = fold * 2 / kFold, token = 4 * lg + (kFold == 4 ? 2 * (fold & 1) : 0);
  // Where the two tiles of the wave's n-th pair are: the table's entry and the tile in the
  // page.  Scalar loads, which the many vector loads on the way do not have to be waited
  // out for, and looked at only when the pair is fetched.
  struct Place {
    int block[2], sub[2];
  };
  const volatile auto* row = as_constant(p.table + b * p.table_stride);  // (volatile: or the loads move to their use)
  auto places = [&](int n) {
    Place x;
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      const int tile = t0 + 2 * (w + W * n) + t;
      const int lp = (int)p.tiles.div((uint32_t)min(tile, t1 - 1));
      x.sub[t] = tile - lp * (int)p.tiles.d;
      x.block[t] = row[lp];
    }
    return x;
  };
  const uint32_t k_at = g * Row::kBytes + 4 * Shape::kKey * lg, v_at = 4 * lg * Row::kBytes + Row::kBytes / 16 * g;
  // The wave's n-th pair, on its way.  A tile without a page reads page 0.
  auto fetch = [&](Pair& x, const Place& at, int n) {
    x.tile = t0 + 2 * (w + W * n);
    const uint8_t* kr[2];
    const uint8_t* vr[2];
    const uint8_t* sr[2];
#pragma unroll
    for (int t = 0; t < 2; ++t) {
      x.none[t] = (uint32_t)at.block[t] >= (uint32_t)p.num_blocks || x.tile + t >= t1;
      const int bl = x.none[t] ? 0 : at.block[t], su = x.none[t] ? 0 : at.sub[t];
      // (scalar addresses, and a lane's own part in 32 bits)
      const uint8_t* record = p.cache + ((int64_t)bl * p.heads_k + h) * p.record;
      kr[t] = record + 8 * p.page + 16 * su * Row::kBytes;
      vr[t] = kr[t] + p.page * Row::kBytes;
      load_words<Shape::kKey>(kr[t] + k_at, x.k[t]);
      sr[t] = record + 128 * su;
    }
    if constexpr (kFold == 1) {
#pragma unroll
      for (int t = 0; t < 2; ++t) load_words<8>(sr[t] + 32u * lg, x.side + 8 * t);
    } else {
      load_words<2 * kTokens>((mine ? sr[1] : sr[0]) + 8u * token, x.side);
    }
#pragma unroll
    for (int j = 0; j < 8; ++j) x.v.load(j, vr[j / 4] + v_at + j % 4 * Row::kBytes);
  };
  const int pairs = t1 - t0 - 2 * w > 0 ? (t1 - t0 - 2 * w + 2 * W - 1) / (2 * W) : 0;  // of this wave
  Pair pair[kOdd ? 1 : 2];
  Place ahead[2];
  if (!kOdd && pairs > 0) {
    ahead[0] = places(0);
    ahead[1] = places(1);
    fetch(pair[0], ahead[0], 0);
  }

  // This lane's column of a tile: new token `fresh` of head h * group + hh; it sees `limit`
  // tokens.  q goes in times a power of two that takes the largest of a column's to 2^117 or
  // more, so that products with codes of units of 2^kCodeUnit are normal numbers, those of q
  // 2^-100 of the largest among them, and s_k (q.c) is below 2^128 whatever s_k.  Scores are
  // kept without `unit`, which is left to do.
  const int first = len - p.new_tokens + 1;
  bf16x8 Q[kTiles == 1 ? kC : 1];
  float qs[kTiles], qs_rest[kTiles], unit[kTiles];
  int limit[kTiles];
  auto query = [&](int i, bf16x8* to, float& sum_q, float& unit_q) {
    const int column = min(kColumns * (kTiles * ct + i) + g % kColumns, p.columns - 1);
    const int fresh = (int)p.over_group.div((uint32_t)column), hh = column - fresh * p.group;
    const int64_t head = h * p.group + hh;
    const uint16_t* row = p.q + b * p.q_batch + fresh * p.q_token + head * p.q_head + D / 4 * lg;
    u32x4 x[kC];
    float sum = 0.f, most = 0.f;
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      x[c] = *reinterpret_cast<const u32x4*>(row + 8 * c);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const float u = __uint_as_float(x[c][j] << 16), v = __uint_as_float(x[c][j] & 0xFFFF0000u);
        sum += u + v;
        most = fmaxf(most, fmaxf(fabsf(u), fabsf(v)));
      }
    }
    most = wave_max16(most);
    const int e = (int)(__float_as_uint(most) >> 23) - 127;
#pragma unroll
    for (int c = 0; c < kC; ++c) to[c] = query_operand<kBits>(x[c], p.flip, 117 - e);
    sum_q = ldexpf(wave_sum16(sum) * p.flip, 117 - e + kCodeUnit);
    unit_q = ldexpf(p.scale_log2, e - 117 - kCodeUnit);
  };
  if constexpr (kTiles == 1) {
    query(0, Q, qs[0], unit[0]);
  } else {
    // wave i makes tile i's, for all of them
    if (w < kTiles) {
      bf16x8 mine_q[kC];
      float2 x;
      query(w, mine_q, x.x, x.y);
#pragma unroll
      for (int c = 0; c < kC; ++c) shared.q[w][c][l] = mine_q[c];
      if (lg == 0) shared.column[w][g] = x;
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < kTiles; ++i) {
    const int column = min(kColumns * (kTiles * ct + i) + g % kColumns, p.columns - 1);
    limit[i] = first + (int)p.over_group.div((uint32_t)column);
    if constexpr (kTiles > 1) {
      const float2 x = shared.column[i][g];
      qs[i] = x.x;
      unit[i] = x.y;
    }
    // (a low times 16 bits of sum q is exact, so what the two terms of a score cancel takes
    // no digits of their products')
    const float sum_q = qs[i];
    qs[i] = __uint_as_float(__float_as_uint(sum_q) & 0xFFFFFF00u);
    qs_rest[i] = sum_q - qs[i];
  }

  // l_run: sum of weights, weight * 2^-m_run; z: of weights * low_v.  kOdd: O and z are of
  // weights * 2^-off_run, and of values times a power of two each.
  f32x4 O[kTiles][kO];
  float m_run[kTiles], l_run[kTiles], z[kTiles], off_run[kTiles];
#pragma unroll
  for (int i = 0; i < kTiles; ++i) {
#pragma unroll
    for (int k = 0; k < kO; ++k) O[i][k] = f32x4{0.f, 0.f, 0.f, 0.f};
    m_run[i] = -FLT_MAX;
    l_run[i] = z[i] = 0.f;
    off_run[i] = -1000.f;
  }
  auto consume = [&](const Pair& x) {
    f32x4 S[kTiles][2] = {};
#pragma unroll
    for (int c = 0; c < kC; ++c) {
      const bf16x8 K0 = key_operand<kBits>(x.k[0], c), K1 = key_operand<kBits>(x.k[1], c);
#pragma unroll
      for (int i = 0; i < kTiles; ++i) {
        bf16x8 q;
        if constexpr (kTiles == 1)
          q = Q[c];
        else
          q = shared.q[i][c][l];
        S[i][0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(K0, q, S[i][0], 0, 0, 0);
        S[i][1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(K1, q, S[i][1], 0, 0, 0);
      }
    }
    float ks[kTokens], kl[kTokens], vs[kTokens], vl[kTokens], vs_log[kOdd ? kTokens : 1];
#pragma unroll
    for (int j = 0; j < kTokens; ++j) {
      const uint32_t kp = x.side[2 * j], vp = x.side[2 * j + 1];
      ks[j] = __uint_as_float(kp << 16);
      kl[j] = __uint_as_float(kp & 0xFFFF0000u);
      vs[j] = __uint_as_float(vp << 16);
      vl[j] = __uint_as_float(vp & 0xFFFF0000u);
      if constexpr (!kOdd) {
        vs[j] *= kScaleFactor;
      } else {
        // The exponent field f of the scale or, if more, of low 2^-kBits; times 2^(128 - f) the
        // scale is below 4 and low below 2^(kBits + 2).
        const int size = max(max((int)(vp << 16 & 0x7FFF0000u), (int)(vp & 0x7FFF0000u) - (kBits << 23)), 1 << 23);
        const float by = __uint_as_float((255u << 23) - (size & 0x7F800000u));
        vs[j] = vs[j] * by * kScaleFactor;
        vl[j] *= by;
        vs_log[j] = (float)(size >> 23);
      }
    }
    // Behind a column's limit and where there is no page nothing counts, whatever it holds.
    const bool cut = x.none[0] || x.none[1] || first - 16 * x.tile < 32;  // (uniform)
    constexpr int kWords = kTokens / 2;  // packed pairs of a lane's weights
    bf16x8 weights[kTiles][3];
    auto products = [&](int i0, int i1) {
      unrolled<0, kO>([&](auto n) {
        constexpr int o = decltype(n)::value;
        const bf16x8 A = x.v.template operand<o>();
#pragma unroll
        for (int k = 0; k < 3; ++k)
#pragma unroll
          for (int i = i0; i < i1; ++i)
            O[i][o] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(A, weights[i][k], O[i][o], 0, 0, 0);
      });
    };
#pragma unroll
    for (int i = 0; i < kTiles; ++i) {
      float s[kTokens], vs_i[kTokens], vl_i[kTokens];
#pragma unroll
      for (int j = 0; j < kTokens; ++j) {
        float c;
        if constexpr (kFold == 1)
          c = S[i][j / 4][j % 4];
        else if constexpr (kFold == 2)
          c = fold ? S[i][1][j] : S[i][0][j];
        else
          c = fold & 2 ? (fold & 1 ? S[i][1][2 + j] : S[i][1][j]) : (fold & 1 ? S[i][0][2 + j] : S[i][0][j]);
        s[j] = fmaf(kl[j], qs_rest[i], fmaf(ks[j], c, kl[j] * qs[i])) * unit[i];
        vs_i[j] = vs[j];
        vl_i[j] = vl[j];
      }
      if (cut) {
#pragma unroll
        for (int j = 0; j < kTokens; ++j) {
          const int t = kFold == 1 ? j / 4 : mine, at = 16 * t + token + (kFold == 1 ? j % 4 : j);
          const bool seen = at < limit[i] - 16 * x.tile && !(t ? x.none[1] : x.none[0]);
          s[j] = seen ? s[j] : -INFINITY;
          vs_i[j] = seen ? vs[j] : 0.f;
          vl_i[j] = seen ? vl[j] : 0.f;
        }
      }
      // References are whole numbers, so that moving one changes exponents only, and are moved
      // where a weight (kOdd: or one times a value's power of two) would be larger than it may.
      auto column_max = [](float x) {
        if constexpr (kFold >= 2) x = fmaxf(x, row_from8(x));
        if constexpr (kFold == 4) x = fmaxf(x, row_from4(x));
        return wave_max16(x);
      };
      float mx = s[0];
#pragma unroll
      for (int j = 1; j < kTokens; ++j) mx = fmaxf(mx, s[j]);
      bool late = mx > m_run[i] + kWeightLag;
      if constexpr (kOdd) {
#pragma unroll
        for (int j = 0; j < kTokens; ++j)
          late = late || s[j] - m_run[i] + (vs_log[j] - off_run[i]) > kWeightLag;
      }
      if (__builtin_amdgcn_ballot_w64(late)) {
        const float m_new = fmaxf(m_run[i], ceilf(column_max(mx)));
        const float alpha = __builtin_amdgcn_exp2f(m_run[i] - m_new);
        float beta = alpha;
        l_run[i] *= alpha;
        if constexpr (kOdd) {
          float most = s[0] - m_new + vs_log[0];
#pragma unroll
          for (int j = 1; j < kTokens; ++j) most = fmaxf(most, s[j] - m_new + vs_log[j]);
          const float old = off_run[i] + (m_run[i] - m_new);
          off_run[i] = fmaxf(old, ceilf(column_max(most)));
          beta = __builtin_amdgcn_exp2f(old - off_run[i]);
        }
        m_run[i] = m_new;
        z[i] *= beta;
#pragma unroll
        for (int k = 0; k < kO; ++k) O[i][k] *= beta;
      }
      // Weights times scales as sums of three bf16, which is exact: the upper 8 of 24 bits, the
      // upper 8 of the rest, and the rest of that.
      uint32_t own[3][kWords];
#pragma unroll
      for (int j = 0; j < kTokens; j += 2) {
        uint32_t y[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
          const float d = s[j + e] - m_run[i];
          float weight = __builtin_amdgcn_exp2f(d);
          l_run[i] += weight;
          if constexpr (kOdd) weight = __builtin_amdgcn_exp2f(d + (vs_log[j + e] - off_run[i]));
          z[i] = fmaf(weight, vl_i[j + e], z[i]);
          y[e] = __float_as_uint(weight * vs_i[j + e]);
        }
#pragma unroll
        for (int k = 0; k < 3; ++k) {
          own[k][j / 2] = __builtin_amdgcn_perm(y[1], y[0], 0x07060302);
#pragma unroll
          for (int e = 0; e < 2; ++e)
            y[e] = __float_as_uint(__uint_as_float(y[e]) - __uint_as_float(y[e] & 0xFFFF0000u));
        }
      }
      // the other folds' tokens of the column
#pragma unroll
      for (int k = 0; k < 3; ++k) {
        u32x4 y;
        if constexpr (kFold == 1)
          y = u32x4{own[k][0], own[k][1], own[k][kWords - 2], own[k][kWords - 1]};
        else if constexpr (kFold == 2)
          y = u32x4{own[k][0], own[k][kWords - 1], row_from<8>(own[k][0]), row_from<8>(own[k][kWords - 1])};
        else
          y = u32x4{own[k][0], row_from<4>(own[k][0]), row_from<8>(own[k][0]), row_from<12>(own[k][0])};
        weights[i][k] = __builtin_bit_cast(bf16x8, y);
      }
      if constexpr (kOdd) products(i, i + 1);
    }
    if constexpr (!kOdd) products(0, kTiles);
  };

  // A pair's loads go out while the one before is worked on, and its places are read one
  // pair earlier still.  (Past the last pair page 0 is read, so that the number of loads
  // on the way is known.)
  if constexpr (kOdd) {
    for (int n = 0; n < pairs; ++n) {
      fetch(pair[0], places(n), n);
      consume(pair[0]);
    }
  } else {
    for (int n = 0; n < pairs; n += 2) {
      fetch(pair[1], ahead[1], n + 1);
      ahead[0] = places(n + 2);
      consume(pair[0]);
      fetch(pair[0], ahead[0], n + 2);
      ahead[1] = places(n + 3);
      if (n + 1 < pairs) consume(pair[1]);
    }
  }

  auto column_sum = [](float x) {
    x = wave_sum16(x);
    if constexpr (kFold >= 2) x += row_from8(x);
    if constexpr (kFold == 4) x += row_from4(x);
    return x;
  };
#pragma unroll
  for (int i = 0; i < kTiles; ++i) l_run[i] = column_sum(l_run[i]), z[i] = column_sum(z[i]);
  bool small = false, large = false;
#pragma unroll
  for (int i = 0; i < kTiles; ++i) {
    // (fmaxf passes over what is no number: where a sum of a column is that, another of it is
    // infinite, or all are and the largest is 0)
    float most = 0.f;
#pragma unroll
    for (int k = 0; k < kO; ++k)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        most = fmaxf(most, O[i][k][r]);
        O[i][k][r] = fmaf(O[i][k][r], ValuePart<D, kBits>::sixteenfold(k) ? kSumFactor / 16 : kSumFactor, z[i]);
      }
    most = wave_max16(most);
    small = small || (most < kLeastSum && l_run[i] > 0.f);
    large = large || !(most <= kMostSum && fabsf(z[i]) <= kMostSum * kSumFactor);
  }
  if constexpr (!kOdd) {
    uint64_t odd = __builtin_amdgcn_ballot_w64(large);
    if (!odd && __builtin_amdgcn_ballot_w64(small)) {
      // not where no row has a scale (a cache of zeros)
      for (int n = 0; n < pairs && !odd; ++n) {
        const Place at = places(n);
#pragma unroll
        for (int t = 0; t < 2; ++t) {
          if (t0 + 2 * (w + W * n) + t >= t1 || (uint32_t)at.block[t] >= (uint32_t)p.num_blocks) continue;
          const uint8_t* record = p.cache + ((int64_t)at.block[t] * p.heads_k + h) * p.record;
          odd |= __builtin_amdgcn_ballot_w64(
              *reinterpret_cast<const uint16_t*>(record + 128 * at.sub[t] + 8 * (qa_lane() & 15) + 4) != 0);
        }
      }
    }
    if (qa_lane() == 0) shared.odd[w] = odd != 0;
    __syncthreads();
    int any = 0;
#pragma unroll
    for (int i = 0; i < W; ++i) any |= shared.odd[i];
    if (__builtin_amdgcn_readfirstlane(any)) return true;
  }
#pragma unroll
  for (int i = 0; i < kTiles; ++i) {
    if (i) __syncthreads();  // the last tile's states are read
    qa_finish<D, kBits, kColumns, kOdd>(p, shared.states, O[i], m_run[i], l_run[i], off_run[i], kTiles * ct + i, h, b,
                                        slot);
  }
  return false;
}

// Whether the second time is a function of its own.  Where both together need more registers than
// there are it is the main loop that loses them (64 sequences of 8000 tokens: 116 us, 110 with
// a call; five new tokens of 16 sequences 73 and 70); where not, a call's rules cost more (heads
// of 64 in 8 bits, 20 ragged sequences: 30 us, 36 with a call).
constexpr bool qa_calls(int dim, int bits, int fold, int tiles) {
  return dim == 128 && (tiles > 1 || (bits == 4 && fold <= 2));
}
// (Addresses as numbers: of the kernel's arguments and in the workgroup's memory, so
// that both are read as what they are.)
template <int D, int kBits, int kFold, int kTiles>
__device__ __attribute__((noinline)) void qa_segment_odd(uint64_t params, uint32_t shared, int ct, int h, int b,
                                                         int len, int t0, int t1, int slot) {
  typedef const QuantAttnParams __attribute__((address_space(4))) * Params;
  typedef QaShared<D, kBits, kTiles> __attribute__((address_space(3))) * Shared;
  auto uniform = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
  const uint64_t at = (uint64_t)(uint32_t)uniform((int)(params >> 32)) << 32 | (uint32_t)uniform((int)params);
  const Shared states = (Shared)(uintptr_t)uniform(shared);
  qa_segment<D, kBits, kFold, kTiles, true>(*(const QuantAttnParams*)(Params)at, *(QaShared<D, kBits, kTiles>*)states,
                                            uniform(ct), uniform(h), uniform(b), uniform(len), uniform(t0),
                                            uniform(t1), uniform(slot));
}

// kTiles tiles of columns in one workgroup: codes are loaded and widened once for all.  With
// more than one, q is read from LDS for each pair.
template <int D, int kBits, int kFold, int kTiles>
__global__ __launch_bounds__(kQaWaves * 64, qa_waves(D, kBits, kFold, kTiles)) void quant_attn_kernel(
    QuantAttnParams p) {
  __shared__ QaShared<D, kBits, kTiles> shared;
  const int l = lane_id();
  // Column tiles of the same tokens go to one XCD (workgroups are dealt out to the
  // eight in turn), one soon after another.
  const int item = (int)p.over_column_tiles.div(blockIdx.x >> 3);
  const int ct = (int)(blockIdx.x >> 3) - item * (int)p.over_column_tiles.d;
  const int at = 8 * item + (blockIdx.x & 7);
  const int part = (int)p.over_heads_k.div((uint32_t)at), h = at - part * p.heads_k;

  // The range of tiles, and the first sequence that has any of it (one without tiles
  // belongs to the part that its place is in), with its length and first tile.
  int from, to, b, len, start = 0, parts = 0, total = 0;
  const ConstantInts lens = as_constant(p.seqlens);
  if (p.splits) {  // (uniform)
    b = (int)p.over_splits.div((uint32_t)part);
    if (b >= p.batch) return;
    len = lens[b];
    const int tiles = qa_tiles_of(p, len), i = part - b * p.splits;
    from = (int)((int64_t)tiles * i / p.splits);
    to = (int)((int64_t)tiles * (i + 1) / p.splits);
  } else {
    // lane i: sequence s0 + i; one sequence alone by scalars, 1 us sooner
    int s0 = 0, mine = 0, tiles = 0, end = 0;
    auto look = [&](int before) {
      mine = s0 + l < p.batch ? p.seqlens[s0 + l] : 0;
      tiles = qa_tiles_of(p, mine);
      end = before + wave_inclusive_scan(tiles);
      return __builtin_amdgcn_readlane(end, 63);
    };
    if (p.batch == 1)
      total = qa_tiles_of(p, lens[0]);
    else
      for (; s0 < p.batch; s0 += 64) total = look(total);
    parts = min(p.parts, max(1, total / kLeastChunk));
    if (part >= parts) return;
    from = qa_part_start(part, parts, total);
    to = qa_part_start(part + 1, parts, total);
    if (p.batch == 1) {
      b = 0;
      len = lens[0];
    } else {
      uint64_t have = 0;
      for (int before = 0, s1 = 0; s1 < p.batch && !have; s1 += 64) {
        s0 = s1;
        if (p.batch > 64) before = look(before);
        have = __builtin_amdgcn_ballot_w64(s0 + l < p.batch && (tiles ? end > from : end >= from));
      }
      if (!have) return;  // (never: `from` is below `total`, or all are empty)
      const int i = __builtin_ctzll(have);
      b = s0 + i;
      len = __builtin_amdgcn_readlane(mine, i);
      start = __builtin_amdgcn_readlane(end, i) - __builtin_amdgcn_readlane(tiles, i);
    }
  }

  for (;;) {
    const int tiles = qa_tiles_of(p, len);
    const int t0 = max(from - start, 0), t1 = min(to - start, tiles);
    int slot = p.splits == 1 ? -1 : part;
    if (p.splits == 0) {
      const bool whole = t0 == 0 && t1 == tiles;
      slot = 2 * part + (start > from);
      if (t0 == 0 && h == 0 && ct == 0 && threadIdx.x == 0)
        p.ws_plan[b] = int2{slot, whole ? 1 : qa_part_of(start + tiles - 1, parts, total) + 1 - part};
      slot = whole ? -1 : slot;
    }
    const int most = max(len, 0);
    const bool again = qa_segment<D, kBits, kFold, kTiles, false>(p, shared, ct, h, b, most, t0, t1, slot);
    if constexpr (qa_calls(D, kBits, kFold, kTiles)) {
      if (again)
        qa_segment_odd<D, kBits, kFold, kTiles>((uint64_t)__builtin_amdgcn_kernarg_segment_ptr(),
                                                (uint32_t)(uintptr_t)&shared, ct, h, b, most, t0, t1, slot);
    } else {
      if (again) qa_segment<D, kBits, kFold, kTiles, true>(p, shared, ct, h, b, most, t0, t1, slot);
    }
    start += tiles;
    if (++b >= p.batch || p.splits || (start >= to && part != parts - 1)) return;
    len = lens[b];
    __syncthreads();  // the states are read
  }
}

// How a call is cut.  Where num_splits leaves it open: sequences whole where the table
// holds no more than kWholeTiles (the merge costs 4 us: 1000 tokens of one sequence take
// 11.8 us whole, 12.2 in parts, 1500 15.1 and 12.5), or where there are six (sequence, KV
// head, column tile) units a CU; else into parts, as many as registers allow at once, two
// to four workgroups a CU (one less or one more costs up to 30%: 20 ragged sequences of
// 8000 tokens with 64 heads of 128 in 8 bits take 38 us in two a CU, 45 in three), but 64
// a sequence at most (32000 tokens: 19.1 us in 96, 17.1 in 64).
// The six units even out where lengths are spread evenly (256 sequences of 2000 tokens with
// 8 KV heads: 109 us whole, 127 in parts; of 16 to 4000 tokens 108 and 184), but the host
// does not see the lengths, and one sequence much longer than the others is then one
// workgroup's work a KV head: 255 sequences of 500 tokens and one of 64000 take 388 us,
// with num_splits = 8 157; 190 and one, which are cut by their lengths, 59.
constexpr int kWholeTiles = 64;
// Tiles of columns go two to a workgroup where none or few are left over, and in 8 bits
// of 128 channels always.  Sixteen sequences of 8000 tokens, heads of 128, one tile
// against two a workgroup: two tiles 59 and 55 us (8 bits 75 and 63), three 74 and 84 (8
// bits 116 and 93; heads of 64 59 and 67), four 94 and 85 (8 bits 118 and 96), seven 163
// and 143; four sequences of 4000 tokens with 32 tiles 104 and 83.
constexpr int kOddTiles = 7;
struct QaCut {
  int64_t columns, column_tiles;  // the latter: of `tiles` times 16 columns
  int64_t groups, slots;          // groups: workgroups of a KV head and a tile of columns
  int tiles, splits, parts;       // (the last two as in the parameters)

  bool whole() const { return splits == 1; }
  size_t ws_bytes(int batch, int heads_k, int head_dim) const {
    return whole() ? 0 : (size_t)slots * heads_k * columns * (head_dim + 2) * sizeof(float) + batch * sizeof(int2);
  }
};

static QaCut qa_cut(int batch, int new_tokens, int heads, int heads_k, int head_dim, int bits, int64_t tiles,
                    int num_splits) {
  QaCut c{};
  c.columns = (int64_t)(heads / heads_k) * new_tokens;
  const int64_t all = (c.columns + 15) / 16;
  c.tiles = all > 1 && (all % 2 == 0 || all >= kOddTiles || (head_dim == 128 && bits == 8)) ? 2 : 1;
  c.column_tiles = (all + c.tiles - 1) / c.tiles;
  const int64_t units = c.column_tiles * heads_k, cus = device_cu_count();
  const int fit = c.tiles == 2 || (head_dim == 128 && bits == 8 && c.columns > 4) ? 2
                  : head_dim == 64 && c.columns <= 8                               ? 4
                                                                                   : 3;
  if (num_splits > 0)
    c.splits = (int)std::max<int64_t>(1, std::min<int64_t>(num_splits, (tiles + 2 * kQaWaves - 1) / (2 * kQaWaves)));
  else if (tiles <= kWholeTiles || batch * units >= 6 * cus || batch * tiles > INT_MAX)
    c.splits = 1;
  else
    c.parts = (int)std::max<int64_t>(1, std::min<int64_t>(fit * cus / units, 64 * (int64_t)batch));
  if (c.parts > batch) c.parts -= c.parts % batch;  // sequences of one length are cut alike
  c.groups = c.splits ? (int64_t)batch * c.splits : c.parts;
  c.slots = c.splits ? c.groups : 2 * c.groups;
  return c;
}

}  // namespace zs

using namespace zs;

extern "C" size_t zs_decode_attention_quant_workspace_bytes(int batch, int new_tokens, int num_heads, int num_heads_k,
                                                            int head_dim, int max_blocks_per_seq,
                                                            int page_block_size, int num_splits) {
  if (batch <= 0 || new_tokens <= 0 || num_heads <= 0 || num_heads_k <= 0 || num_heads % num_heads_k ||
      head_dim <= 0 || max_blocks_per_seq <= 0 || page_block_size < 16 || num_splits < 0)
    return 0;
  const int64_t rows = (int64_t)batch * num_heads * new_tokens;
  const int64_t tiles = (int64_t)max_blocks_per_seq * (page_block_size / 16);
  if (rows > INT_MAX || tiles > INT_MAX) return 0;  // (such a call is refused)
  size_t most = 0;
  for (int bits = 4; bits <= 8; bits += 4)
    most = std::max(most, qa_cut(batch, new_tokens, num_heads, num_heads_k, head_dim, bits, tiles, num_splits)
                              .ws_bytes(batch, num_heads_k, head_dim));
  return most;
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
  const int64_t rows = (int64_t)batch * num_heads * new_tokens;
  const int64_t tiles = (int64_t)max_blocks_per_seq * (page_block_size / 16);
  if (rows > INT_MAX || tiles > INT_MAX) return ZS_E_OVERFLOW;
  const QaCut cut = qa_cut(batch, new_tokens, num_heads, num_heads_k, head_dim, bits, tiles, num_splits);
  const int64_t groups = (cut.groups * num_heads_k + 7) / 8 * 8 * cut.column_tiles;
  if (cut.groups > INT_MAX / num_heads_k || !grid_fits(groups, kQaWaves * 64) ||
      (!cut.whole() && !grid_fits(merge_parts_groups(batch, num_heads_k, cut.columns), kPartMergeThreads)))
    return ZS_E_OVERFLOW;
  if (workspace_bytes < cut.ws_bytes(batch, num_heads_k, head_dim) || (!cut.whole() && !workspace)) return ZS_E_INVAL;
  QuantAttnParams p{};
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
  if (!cut.whole()) {
    const size_t ws_rows = (size_t)cut.slots * num_heads_k * cut.columns;
    p.ws_o = static_cast<float*>(workspace);
    p.ws_ml = p.ws_o + ws_rows * head_dim;
    p.ws_plan = reinterpret_cast<int2*>(p.ws_ml + 2 * ws_rows);
  }
  p.batch = batch;
  p.splits = cut.splits;
  p.parts = cut.parts;
  p.num_blocks = num_blocks;
  p.width = max_blocks_per_seq;
  p.page = page_block_size;
  p.heads = num_heads;
  p.heads_k = num_heads_k;
  p.group = num_heads / num_heads_k;
  p.new_tokens = new_tokens;
  p.columns = (int)cut.columns;
  p.tiles = FastDiv::of(page_block_size / 16);
  p.over_group = FastDiv::of(p.group);
  p.over_heads_k = FastDiv::of(num_heads_k);
  p.over_column_tiles = FastDiv::of((uint32_t)cut.column_tiles);
  p.over_splits = FastDiv::of(std::max(1, cut.splits));
  p.scale_log2 = (float)(fabs((double)softmax_scale) * 1.4426950408889634);
  p.flip = softmax_scale < 0.f ? -1.f : 1.f;
  const hipStream_t st = (hipStream_t)stream;
  const dim3 grid((unsigned)groups), block(kQaWaves * 64);
  auto launch = [&](auto dim, auto width) {
    constexpr int D = decltype(dim)::value, kBits = decltype(width)::value;
    if (cut.columns <= 4)
      hipLaunchKernelGGL((quant_attn_kernel<D, kBits, 4, 1>), grid, block, 0, st, p);
    else if (cut.columns <= 8)
      hipLaunchKernelGGL((quant_attn_kernel<D, kBits, 2, 1>), grid, block, 0, st, p);
    else if (cut.tiles == 1)
      hipLaunchKernelGGL((quant_attn_kernel<D, kBits, 1, 1>), grid, block, 0, st, p);
    else
      hipLaunchKernelGGL((quant_attn_kernel<D, kBits, 1, 2>), grid, block, 0, st, p);
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
  if (e == hipSuccess && !cut.whole()) {
    PartMerge m{p.ws_o, p.ws_ml, p.splits ? nullptr : p.ws_plan, out, softmax_lse, p.splits, p.columns, new_tokens,
                p.over_group};
    e = merge_parts(st, m, batch, num_heads_k, head_dim);
  }
  return e == hipSuccess ? ZS_OK : (int)e;
}
