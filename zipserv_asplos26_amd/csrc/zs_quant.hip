// zs_quant.hip -- a paged KV cache held in 4 or 8 bits (gfx950): new keys and
// values quantised into their slots, and the values of slots read back.
//
// A row is one token's key or value of one KV head, D channels.  Of a row x
//   low   = min x,
//   scale = the least bf16 with (2^bits - 1) scale >= max x - low,
//   code  = (x - low) / scale to the nearest, the even one of two (0 where scale is 0),
// the differences rounded to fp32; low is one of the row's bf16 values, so nothing
// of it is lost, and no code leaves its bits.  A value comes back as low + code
// scale, half a scale off at most.  A row with a value that is not finite, or whose
// max x - low is not, has NaN for low and scale and codes 0: what is read of it is NaN.
//
// The layout is in zs_quant.hpp.
#include <hip/hip_runtime.h>

#include <climits>
#include <type_traits>

#include "../../include/zipserv.h"
#include "zs_device.hpp"
#include "zs_quant.hpp"

namespace zs {

int paged_checks(int num_blocks, int page, int heads_k, int head_dim);  // zs_paged.hip
bool grid_fits(int64_t groups, int threads);                           // zs_paged.hip

constexpr int kQuantThreads = 256;

struct QuantParams {
  const uint16_t* k;
  const uint16_t* v;
  int64_t k_token, k_head, v_token, v_head;  // strides in elements
  uint16_t* k_out;                           // of a read: [tokens][Hkv][D]
  uint16_t* v_out;
  const int32_t* slots;
  uint8_t* cache;
  int64_t record;
  int tokens, heads_k, num_slots;
  FastDiv page, over_heads;
};

// min and max over the D / 8 lanes of a row (8 or 16 neighbouring lanes), in all of
// them: exchanges with lane ^ 1, ^ 2, 7 - lane and 15 - lane, which integers take in the same
// instruction (of bits that are ordered like the numbers: the magnitude of
// negative ones flipped).
__device__ __forceinline__ int float_order(int bits) { return bits ^ (bits >> 31 & INT_MAX); }

template <int kLanes>
__device__ __forceinline__ void row_min_max(float& lo, float& hi) {
  int x = float_order(__float_as_int(lo)), y = float_order(__float_as_int(hi));
  auto step = [&](auto ctrl) {
    constexpr int kCtrl = decltype(ctrl)::value;
    x = min(x, __builtin_amdgcn_mov_dpp(x, kCtrl, 0xF, 0xF, true));
    y = max(y, __builtin_amdgcn_mov_dpp(y, kCtrl, 0xF, 0xF, true));
  };
  step(std::integral_constant<int, 0xB1>{});   // quad_perm [1, 0, 3, 2]
  step(std::integral_constant<int, 0x4E>{});   // quad_perm [2, 3, 0, 1]
  step(std::integral_constant<int, 0x141>{});  // row_half_mirror
  if constexpr (kLanes == 16) step(std::integral_constant<int, 0x140>{});  // row_mirror
  lo = __int_as_float(float_order(x));
  hi = __int_as_float(float_order(y));
}

// Eight channels of a row, whose lanes work together, to codes (4 bits: in
// words[0], 8 bits: in words[0..1]); returns (scale, low), scale in the lower half.
template <int kLanes, int kBits>
__device__ __forceinline__ uint32_t quantize8(u32x4 in, uint32_t* words) {
  typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
  constexpr float kMost = (1 << kBits) - 1;
  float x[8];
  u16x2 size = {0, 0};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = __uint_as_float(in[i] << 16);
    x[2 * i + 1] = __uint_as_float(in[i] & 0xFFFF0000u);
    size = __builtin_elementwise_max(size, __builtin_bit_cast(u16x2, in[i] & 0x7FFF7FFFu));
  }
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) lo = fminf(lo, x[i]), hi = fmaxf(hi, x[i]);
  if (max(size[0], size[1]) >= 0x7F80) lo = -INFINITY, hi = INFINITY;  // a value that is not finite
  row_min_max<kLanes>(lo, hi);
  const float span = hi - lo;
  // The quotient in fp32 is off by 2^-22 of it, so the least bf16 that reaches the
  // span is the one at or below it or one of the next two; a product of a bf16 and
  // 15 or 255 is exact.
  uint32_t s = __float_as_uint(span * (1.f / kMost)) & 0xFFFF0000u;
  s += kMost * __uint_as_float(s) < span ? 0x10000u : 0u;
  s += kMost * __uint_as_float(s) < span ? 0x10000u : 0u;
  // (x - low) / scale with 1 / scale as a sum of two fp32, off by 2^-45 of it before its
  // one rounding.  That gives the same code as the quotient itself: n + 1/2 times scale has
  // 17 bits, so a difference that is not exactly that, having 24, is 2^-24 (1 + 2^-17) of it
  // away or more, and the quotient's next fp32 are nearer; and n + 1/2 itself stays it.
  float scale = __uint_as_float(s), t[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) t[i] = x[i] - lo;
  if (s < 0x00800000u || s > 0x71800000u) {  // below 2^-126 or past 2^100: a reciprocal loses bits
    const float by = s < 0x00800000u ? 0x1p60f : 0x1p-60f;
    scale *= by;
#pragma unroll
    for (int i = 0; i < 8; ++i) t[i] *= by;
  }
  const float r = __builtin_amdgcn_rcpf(scale), rest = r * fmaf(-scale, r, 1.f);
  // The nearest whole number, the even one of two, is in the lower bits of the sum with
  // 1.5 2^23; the upper ones are taken off all codes at once.
  uint32_t w[kBits / 4] = {}, above[kBits / 4] = {};
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t c = __float_as_uint(fmaf(t[i], r, t[i] * rest) + 12582912.f);
    const int at = kBits == 4 ? 4 * (i / 2) + 16 * (i % 2) : 8 * (i % 4), h = kBits == 4 ? 0 : i / 4;
    w[h] += c << at;
    above[h] += 0x4B400000u << at;
  }
  const bool none = s == 0 || !(span < INFINITY);
#pragma unroll
  for (int h = 0; h < kBits / 4; ++h) words[h] = none ? 0u : w[h] - above[h];
  return span < INFINITY ? s >> 16 | (__float_as_uint(lo) & 0xFFFF0000u) : 0x7FC07FC0u;
}

// Where a slot's page of head h starts, and its token in it.
__device__ __forceinline__ uint8_t* quant_record(const QuantParams& p, int slot, int h, int& off) {
  const int block = (int)p.page.div((uint32_t)slot);
  off = slot - block * (int)p.page.d;
  return p.cache + ((int64_t)block * p.heads_k + h) * p.record;
}

// A workgroup takes 2048 / D tokens of one KV head, 16 bytes of k and of v a thread.
// 8000 tokens of 8 heads of 128 in 4 bits (42 MB): 10.1 us, 80% of the rate of a copy;
// 14.6 with a division a value, of which its 300 vector instructions a thread had 200.
template <int D, int kBits>
__global__ __launch_bounds__(kQuantThreads) void quant_append_kernel(QuantParams p) {
  typedef QuantRow<D, kBits> Row;
  constexpr int kLanes = D / 8, kRows = kQuantThreads / kLanes;
  const int segment = (int)p.over_heads.div(blockIdx.x), h = blockIdx.x - segment * p.heads_k;
  const int t = segment * kRows + threadIdx.x / kLanes, c = threadIdx.x % kLanes;
  const int slot = t < p.tokens ? p.slots[t] : -1;
  if (slot < 0 || slot >= p.num_slots) return;  // (all lanes of a row alike)
  const u32x4 k = *reinterpret_cast<const u32x4*>(p.k + t * p.k_token + h * p.k_head + 8 * c);
  const u32x4 v = *reinterpret_cast<const u32x4*>(p.v + t * p.v_token + h * p.v_head + 8 * c);
  int off;
  uint8_t* record = quant_record(p, slot, h, off);
  const int page = (int)p.page.d;
  uint32_t kw[kBits / 4], vw[kBits / 4];
  const uint32_t ks = quantize8<kLanes, kBits>(k, kw), vs = quantize8<kLanes, kBits>(v, vw);
  uint8_t* kr = record + 8 * page + off * Row::kBytes + kBits * c;
  uint8_t* vr = kr + page * Row::kBytes;
  if constexpr (kBits == 4) {
    *reinterpret_cast<uint32_t*>(kr) = kw[0];
    *reinterpret_cast<uint32_t*>(vr) = vw[0];
  } else {
    *reinterpret_cast<uint2*>(kr) = uint2{kw[0], kw[1]};
    *reinterpret_cast<uint2*>(vr) = uint2{vw[0], vw[1]};
  }
  if (c == 0) *reinterpret_cast<uint2*>(record + 8 * off) = uint2{ks, vs};
}

// Eight channels of a row from their codes and (scale, low).
template <int kBits>
__device__ __forceinline__ u32x4 dequantize8(const uint32_t* words, uint32_t pair) {
  const float scale = __uint_as_float(pair << 16), low = __uint_as_float(pair & 0xFFFF0000u);
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const uint32_t c = kBits == 4 ? words[0] >> (4 * (i / 2) + 16 * (i % 2)) & 15u
                                  : words[kBits == 4 ? 0 : i / 4] >> (8 * (i % 4)) & 255u;
    x[i] = fmaf((float)c, scale, low);
  }
  return u32x4{pack_bf16x2(x[0], x[1]), pack_bf16x2(x[2], x[3]), pack_bf16x2(x[4], x[5]), pack_bf16x2(x[6], x[7])};
}

// The same cut as the append's; a slot outside the pool gives zeros.  Bound by its
// writes, 3.8 times its reads in 4 bits: 60000 tokens of 8 heads of 128 (311 MB) take 46
// us, 6.7 TB/s, with stores past the caches, 67 with ordinary ones.
template <int D, int kBits>
__global__ __launch_bounds__(kQuantThreads) void quant_read_kernel(QuantParams p) {
  typedef QuantRow<D, kBits> Row;
  constexpr int kLanes = D / 8, kRows = kQuantThreads / kLanes;
  const int segment = (int)p.over_heads.div(blockIdx.x), h = blockIdx.x - segment * p.heads_k;
  const int t = segment * kRows + threadIdx.x / kLanes, c = threadIdx.x % kLanes;
  if (t >= p.tokens) return;
  const int slot = p.slots[t], page = (int)p.page.d;
  u32x4 k = {0, 0, 0, 0}, v = k;
  if (slot >= 0 && slot < p.num_slots) {
    int off;
    const uint8_t* record = quant_record(p, slot, h, off);
    const uint2 side = *reinterpret_cast<const uint2*>(record + 8 * off);
    const uint8_t* kr = record + 8 * page + off * Row::kBytes + kBits * c;
    const uint8_t* vr = kr + page * Row::kBytes;
    uint32_t kw[kBits / 4], vw[kBits / 4];
#pragma unroll
    for (int i = 0; i < kBits / 4; ++i) {
      kw[i] = reinterpret_cast<const uint32_t*>(kr)[i];
      vw[i] = reinterpret_cast<const uint32_t*>(vr)[i];
    }
    k = dequantize8<kBits>(kw, side.x);
    v = dequantize8<kBits>(vw, side.y);
  }
  const int64_t at = ((int64_t)t * p.heads_k + h) * D + 8 * c;
  __builtin_nontemporal_store(k, reinterpret_cast<u32x4*>(p.k_out + at));
  __builtin_nontemporal_store(v, reinterpret_cast<u32x4*>(p.v_out + at));
}

static bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Checks of both entry points, and the launch of `kernel<D, bits>`.
int quant_checks(const void* cache, int num_blocks, int page, int heads_k, int head_dim, int bits) {
  if (!cache) return ZS_E_INVAL;
  const int bad = paged_checks(num_blocks, page, heads_k, head_dim);
  if (bad != ZS_OK) return bad;
  if (bits != 4 && bits != 8) return ZS_E_UNSUPPORTED;
  if ((int64_t)page * quant_token_bytes(head_dim, bits) > INT_MAX) return ZS_E_OVERFLOW;
  return aligned16(cache) ? ZS_OK : ZS_E_INVAL;
}

template <class Launch>
static int quant_launch(QuantParams& p, int num_blocks, int page, int head_dim, int bits, Launch launch) {
  p.record = (int64_t)page * quant_token_bytes(head_dim, bits);
  p.num_slots = num_blocks * page;
  p.page = FastDiv::of(page);
  p.over_heads = FastDiv::of(p.heads_k);
  const int rows = kQuantThreads * 8 / head_dim;
  const int64_t items = ((int64_t)p.tokens + rows - 1) / rows * p.heads_k;
  if (!grid_fits(items, kQuantThreads)) return ZS_E_OVERFLOW;
  typedef std::integral_constant<int, 4> Four;
  typedef std::integral_constant<int, 8> Eight;
  typedef std::integral_constant<int, 64> Small;
  typedef std::integral_constant<int, 128> Large;
  const dim3 grid((unsigned)items);
  if (head_dim == 128)
    bits == 4 ? launch(grid, Large{}, Four{}) : launch(grid, Large{}, Eight{});
  else
    bits == 4 ? launch(grid, Small{}, Four{}) : launch(grid, Small{}, Eight{});
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? ZS_OK : (int)e;
}

}  // namespace zs

using namespace zs;

extern "C" int64_t zs_quant_record_bytes(int page_block_size, int head_dim, int bits) {
  if (page_block_size <= 0 || head_dim <= 0 || head_dim % 64 || (bits != 4 && bits != 8)) return -1;
  return (int64_t)page_block_size * (8 + (int64_t)head_dim * bits / 4);
}

extern "C" int zs_paged_append_quant(void* stream, const uint16_t* k, const uint16_t* v, int64_t k_token_stride,
                                     int64_t k_head_stride, int64_t v_token_stride, int64_t v_head_stride,
                                     const int32_t* slots, int num_tokens, uint8_t* cache, int num_blocks,
                                     int page_block_size, int num_heads_k, int head_dim, int bits) {
  if (num_tokens < 0) return ZS_E_INVAL;
  const int bad = quant_checks(cache, num_blocks, page_block_size, num_heads_k, head_dim, bits);
  if (bad != ZS_OK) return bad;
  if (num_tokens == 0) return ZS_OK;
  if (!k || !v || !slots || !aligned16(k) || !aligned16(v)) return ZS_E_INVAL;
  if ((k_token_stride | k_head_stride | v_token_stride | v_head_stride) & 7) return ZS_E_INVAL;
  QuantParams p{};
  p.k = k;
  p.v = v;
  p.k_token = k_token_stride;
  p.k_head = k_head_stride;
  p.v_token = v_token_stride;
  p.v_head = v_head_stride;
  p.slots = slots;
  p.cache = cache;
  p.tokens = num_tokens;
  p.heads_k = num_heads_k;
  return quant_launch(p, num_blocks, page_block_size, head_dim, bits, [&](dim3 grid, auto d, auto b) {
    hipLaunchKernelGGL((quant_append_kernel<decltype(d)::value, decltype(b)::value>), grid, dim3(kQuantThreads), 0,
                       (hipStream_t)stream, p);
  });
}

extern "C" int zs_paged_read_quant(void* stream, const uint8_t* cache, int num_blocks, int page_block_size,
                                   int num_heads_k, int head_dim, int bits, const int32_t* slots, int num_tokens,
                                   uint16_t* k_out, uint16_t* v_out) {
  if (num_tokens < 0) return ZS_E_INVAL;
  const int bad = quant_checks(cache, num_blocks, page_block_size, num_heads_k, head_dim, bits);
  if (bad != ZS_OK) return bad;
  if (num_tokens == 0) return ZS_OK;
  if (!slots || !k_out || !v_out || !aligned16(k_out) || !aligned16(v_out)) return ZS_E_INVAL;
  QuantParams p{};
  p.k_out = k_out;
  p.v_out = v_out;
  p.slots = slots;
  p.cache = const_cast<uint8_t*>(cache);
  p.tokens = num_tokens;
  p.heads_k = num_heads_k;
  return quant_launch(p, num_blocks, page_block_size, head_dim, bits, [&](dim3 grid, auto d, auto b) {
    hipLaunchKernelGGL((quant_read_kernel<decltype(d)::value, decltype(b)::value>), grid, dim3(kQuantThreads), 0,
                       (hipStream_t)stream, p);
  });
}
