// zs_rotary.hip -- rotary positions (gfx950): pairs of a head's first channels
// turned by an angle that grows with the token's position.
//
// Pair i of a token at position t turns by t w_i:
//   y_a = f (x_a cos - x_b sin),  y_b = f (x_b cos + x_a sin)
// with (a, b) = (2i, 2i + 1), or (i, i + n) of 2n rotated channels; the others
// pass.  The angle is made in two numbers of 64 bits (t w_i of a far position has no digits
// left in 32, and of the farthest 2^-21 in 64) and taken into an eighth of a turn there;
// sine and cosine are their Taylor polynomials in 64 bits, rounded once to fp32 (off by
// 2^-37 before, at any position), so no table of positions is read.  They are made once a
// token and shared by its heads through LDS.
//
// A workgroup takes one token, or up to four while they have no more than 64 angles, one
// wave's work; a thread 16 bytes of both members of its pairs (of one, where they are
// neighbours) at a time, written past the caches.  HBM bounds it: 8192 tokens of 40 heads of
// 128 in bf16 take 26.0 us, 168 MB at 6.5 TB/s, some of it from the last-level cache (28.5
// in workgroups of 256 threads and four tokens); one token 3.2 us, launch and latency.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <type_traits>

#include "../../include/zipserv.h"
#include "zs_device.hpp"

namespace zs {

bool grid_fits(int64_t groups, int threads);  // zs_paged.hip

constexpr int kRotaryThreads = 512;
constexpr int kRotaryPairs = 512;  // angles a workgroup holds

struct RotaryTensor {
  const void* in;
  void* out;
  int64_t in_token, in_head, out_token, out_head;  // strides in elements
};

struct RotaryParams {
  RotaryTensor q, k;
  const int32_t* positions;
  const double* frequencies;
  double factor;
  int tokens, heads_q, pairs, group;  // group: tokens of a workgroup
  int items, per_token;               // items of a head, of a token
  int rotated_items;                  // of a head's items the ones that turn; the rest are copied
  FastDiv over_items, over_token, over_pairs;
};

// cos and sin of t w, times the factor.
__device__ __forceinline__ float2 rotary_turn(int t, double w, double factor) {
#pragma clang fp contract(off)  // (a product taken twice has to be the same number)
  // t w / 2 pi, of a whole turn, with what its product and 1 / 2 pi's rounding leave out: far
  // positions have turned 2^30 times and more, and the whole turns are taken off exactly.
  constexpr double kTurn = 0.15915494309189535, kTurnRest = -9.839338337591243e-18;
  const double angle = t * w, angle_rest = fma((double)t, w, -angle);
  const double turns = angle * kTurn;
  const double turns_rest = fma(angle, kTurn, -turns) + fma(angle, kTurnRest, angle_rest * kTurn);
  const double frac = (turns - rint(turns)) + turns_rest;
  const double quarter = rint(4.0 * frac);
  const double x = (4.0 * frac - quarter) * 1.57079632679489661923, y = x * x;
  double s = fma(y, -1.0 / 39916800, 1.0 / 362880);
  s = fma(y, s, -1.0 / 5040);
  s = fma(y, s, 1.0 / 120);
  s = fma(y, s, -1.0 / 6);
  s = fma(x * y, s, x);
  double c = fma(y, 1.0 / 479001600, -1.0 / 3628800);
  c = fma(y, c, 1.0 / 40320);
  c = fma(y, c, -1.0 / 720);
  c = fma(y, c, 1.0 / 24);
  c = fma(y, c, -0.5);
  c = fma(y, c, 1.0);
  const int q = (int)quarter & 3;
  double cs = q & 1 ? s : c, sn = q & 1 ? c : s;
  if (q == 1 || q == 2) cs = -cs;
  if (q >= 2) sn = -sn;
  return float2{(float)(cs * factor), (float)(sn * factor)};
}

// E elements of type T at a time: two pieces of a head with E pairs, or with
// kNeighbours one piece with E / 2.  kWide: 16 bytes, aligned; otherwise the
// smallest piece, and what is not turned is copied by the element.
template <class T, int E, bool kNeighbours, bool kWide>
__global__ __launch_bounds__(kRotaryThreads) void rotary_kernel(RotaryParams p) {
  typedef T Whole __attribute__((ext_vector_type(E)));
  typedef Whole Vec __attribute__((aligned(kWide ? 16 : sizeof(T))));
  auto store = [](T* at, Whole x) { __builtin_nontemporal_store(x, reinterpret_cast<Vec*>(at)); };
  __shared__ float2 turn[kRotaryPairs];
  const int t0 = blockIdx.x * p.group, n = min(p.group, p.tokens - t0);
  for (int i = threadIdx.x; i < n * p.pairs; i += kRotaryThreads) {
    const int t = (int)p.over_pairs.div((uint32_t)i);
    turn[i] = rotary_turn(p.positions[t0 + t], p.frequencies[i - t * p.pairs], p.factor);
  }
  __syncthreads();
  const int all = n * p.per_token;
  for (int i = threadIdx.x; i < all; i += kRotaryThreads) {
    const int t = (int)p.over_token.div((uint32_t)i), in_token = i - t * p.per_token;
    int h = (int)p.over_items.div((uint32_t)in_token);
    const int c = in_token - h * p.items;
    const bool of_k = h >= p.heads_q;
    h -= of_k ? p.heads_q : 0;
    const RotaryTensor& x = of_k ? p.k : p.q;
    const T* in = static_cast<const T*>(x.in) + (t0 + t) * x.in_token + h * x.in_head;
    T* out = static_cast<T*>(x.out) + (t0 + t) * x.out_token + h * x.out_head;
    const float2* cs = turn + t * p.pairs;
    const bool placed = p.positions[t0 + t] >= 0;
    if (c >= p.rotated_items) {  // behind the rotated channels
      const int at = 2 * p.pairs + (c - p.rotated_items) * (kWide ? E : 1);
      if constexpr (kWide)
        store(out + at, *reinterpret_cast<const Vec*>(in + at));
      else
        out[at] = in[at];
    } else if constexpr (kNeighbours) {
      Vec a = *reinterpret_cast<const Vec*>(in + c * E), y = a;
#pragma unroll
      for (int j = 0; j < E; j += 2) {
        const float2 r = cs[(c * E + j) / 2];
        const float u = (float)a[j], v = (float)a[j + 1];
        y[j] = (T)(u * r.x - v * r.y);
        y[j + 1] = (T)(v * r.x + u * r.y);
      }
      store(out + c * E, placed ? y : a);
    } else {
      const Vec a = *reinterpret_cast<const Vec*>(in + c * E);
      const Vec b = *reinterpret_cast<const Vec*>(in + p.pairs + c * E);
      Vec y = a, z = b;
#pragma unroll
      for (int j = 0; j < E; ++j) {
        const float2 r = cs[c * E + j];
        const float u = (float)a[j], v = (float)b[j];
        y[j] = (T)(u * r.x - v * r.y);
        z[j] = (T)(v * r.x + u * r.y);
      }
      store(out + c * E, placed ? y : a);
      store(out + p.pairs + c * E, placed ? z : b);
    }
  }
}

}  // namespace zs

using namespace zs;

extern "C" int zs_rotary(void* stream, const void* q, int64_t q_token_stride, int64_t q_head_stride, void* q_out,
                         int64_t q_out_token_stride, int64_t q_out_head_stride, int num_heads, const void* k,
                         int64_t k_token_stride, int64_t k_head_stride, void* k_out, int64_t k_out_token_stride,
                         int64_t k_out_head_stride, int num_heads_k, int type, const int32_t* positions,
                         int num_tokens, int head_dim, const double* frequencies, int num_pairs, double factor,
                         int interleaved) {
  if (num_tokens < 0 || num_heads < 0 || num_heads_k < 0 || head_dim <= 0 || num_pairs <= 0 ||
      num_pairs > head_dim / 2)
    return ZS_E_INVAL;
  if (type != ZS_TYPE_BF16 && type != ZS_TYPE_FP16 && type != ZS_TYPE_FP32) return ZS_E_INVAL;
  if (num_pairs > kRotaryPairs) return ZS_E_UNSUPPORTED;
  if (num_tokens == 0 || (num_heads == 0 && num_heads_k == 0)) return ZS_OK;
  if (!positions || !frequencies || (num_heads && (!q || !q_out)) || (num_heads_k && (!k || !k_out)))
    return ZS_E_INVAL;
  const int size = type == ZS_TYPE_FP32 ? 4 : 2;
  if (reinterpret_cast<uintptr_t>(positions) & 3 || reinterpret_cast<uintptr_t>(frequencies) & 7) return ZS_E_INVAL;
  uintptr_t at = 0;
  int64_t strides = 0;
  if (num_heads) {
    at |= reinterpret_cast<uintptr_t>(q) | reinterpret_cast<uintptr_t>(q_out);
    strides |= q_token_stride | q_head_stride | q_out_token_stride | q_out_head_stride;
  }
  if (num_heads_k) {
    at |= reinterpret_cast<uintptr_t>(k) | reinterpret_cast<uintptr_t>(k_out);
    strides |= k_token_stride | k_head_stride | k_out_token_stride | k_out_head_stride;
  }
  if (at & (size - 1)) return ZS_E_INVAL;
  RotaryParams p{};
  p.q = RotaryTensor{q, q_out, q_token_stride, q_head_stride, q_out_token_stride, q_out_head_stride};
  p.k = RotaryTensor{k, k_out, k_token_stride, k_head_stride, k_out_token_stride, k_out_head_stride};
  p.positions = positions;
  p.frequencies = frequencies;
  p.factor = factor;
  p.tokens = num_tokens;
  p.heads_q = num_heads;
  p.pairs = num_pairs;
  // 16 bytes at a time where every piece is aligned to them and none is cut, and the
  // smallest piece otherwise
  const int whole = 16 / size, least = interleaved ? 2 : 1;
  const int cut = interleaved ? 2 * num_pairs : num_pairs;
  const bool wide = (at & 15) == 0 && strides % whole == 0 && cut % whole == 0 && head_dim % whole == 0;
  const int e = wide ? whole : least;
  p.rotated_items = cut / e;
  const bool in_place = (!num_heads || q == q_out) && (!num_heads_k || k == k_out);
  p.items = p.rotated_items + (in_place ? 0 : (head_dim - 2 * num_pairs) / (wide ? whole : 1));
  const int64_t per_token = (int64_t)p.items * (num_heads + (int64_t)num_heads_k);
  if (per_token > INT_MAX / 8) return ZS_E_OVERFLOW;
  p.per_token = (int)per_token;
  p.group = std::max(1, std::min(4, 64 / num_pairs));
  p.over_items = FastDiv::of(p.items);
  p.over_token = FastDiv::of(p.per_token);
  p.over_pairs = FastDiv::of(num_pairs);
  const int groups = (int)(((int64_t)num_tokens + p.group - 1) / p.group);
  if (!grid_fits(groups, kRotaryThreads)) return ZS_E_OVERFLOW;
  auto launch = [&](auto type_tag, auto neighbours, auto wide_tag) {
    typedef decltype(type_tag) T;
    constexpr bool kN = decltype(neighbours)::value, kW = decltype(wide_tag)::value;
    constexpr int kE = kW ? 16 / sizeof(T) : kN ? 2 : 1;
    hipLaunchKernelGGL((rotary_kernel<T, kE, kN, kW>), dim3(groups), dim3(kRotaryThreads), 0, (hipStream_t)stream, p);
    const hipError_t err = hipGetLastError();
    return err == hipSuccess ? ZS_OK : (int)err;
  };
  auto with_type = [&](auto type_tag) {
    if (interleaved)
      return wide ? launch(type_tag, std::true_type{}, std::true_type{})
                  : launch(type_tag, std::true_type{}, std::false_type{});
    return wide ? launch(type_tag, std::false_type{}, std::true_type{})
                : launch(type_tag, std::false_type{}, std::false_type{});
  };
  if (type == ZS_TYPE_BF16) return with_type(__bf16{});
  if (type == ZS_TYPE_FP16) return with_type(_Float16{});
  return with_type(float{});
}
