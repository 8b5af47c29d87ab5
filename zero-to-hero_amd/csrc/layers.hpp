// Shared pieces of the layer operators (libppo_layers.so): element types,
// activations, the dropout generator and the host-side launch helpers.
#pragma once

#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>
#include <hip/hip_runtime.h>
#include <math.h>
#include <stdint.h>

#include "ppo_amd.h"
#include "ppo_layers.h"

namespace ppo {

using bf16 = __hip_bfloat16;
using fp16 = __half;

typedef float v4f __attribute__((ext_vector_type(4)));
typedef int v4i __attribute__((ext_vector_type(4)));
// Sixteen bytes at any address: rows of an odd width start anywhere.
typedef v4i v4i_any __attribute__((aligned(1)));

inline int hip_status(hipError_t e) { return e == hipSuccess ? PPO_OK : PPO_ERR_HIP_BASE + (int)e; }
inline int last_launch_status() { return hip_status(hipGetLastError()); }

__host__ __device__ constexpr int64_t round_up(int64_t x, int64_t a) { return (x + a - 1) / a * a; }
__host__ __device__ constexpr int64_t div_up(int64_t x, int64_t a) { return (x + a - 1) / a; }
inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

inline int dtype_size(int dtype) { return dtype == PPO_DTYPE_F32 ? 4 : 2; }
inline bool dtype_ok(int dtype) { return dtype >= PPO_DTYPE_F32 && dtype <= PPO_DTYPE_F16; }

// Takes PPO_LAYER_ALIGNED off an argument; whether it was there.
template <class I>
bool take_aligned(I& arg) {
  const bool there = arg >= 0 && (arg & PPO_LAYER_ALIGNED);
  if (there) arg &= ~PPO_LAYER_ALIGNED;
  return there;
}

// Elements that 16 bytes hold.
template <class T>
constexpr int kPer16 = 16 / (int)sizeof(T);

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(bf16 x) { return __bfloat162float(x); }
__device__ __forceinline__ float to_f32(fp16 x) { return __half2float(x); }
// Rounds to nearest even, as torch's casts do.
template <class T>
__device__ __forceinline__ T from_f32(float x);
template <>
__device__ __forceinline__ float from_f32<float>(float x) { return x; }
template <>
__device__ __forceinline__ bf16 from_f32<bf16>(float x) { return __float2bfloat16(x); }
template <>
__device__ __forceinline__ fp16 from_f32<fp16>(float x) { return __float2half_rn(x); }

// Calls f with a value of the C++ type of `dtype` (checked by the caller).
template <class F>
int with_dtype(int dtype, F&& f) {
  if (dtype == PPO_DTYPE_F32) return f(float{});
  if (dtype == PPO_DTYPE_BF16) return f(bf16{});
  return f(fp16{});
}

// Sixteen bytes from any address, as the five aligned words that hold them
// (none of which lies outside), shifted together: loads that start off 4 bytes
// take three to four times as long.
__device__ __forceinline__ v4i load16_shifted(const char* p) {
  const int off = (int)((uintptr_t)p & 3);
  typedef int v4i_words __attribute__((ext_vector_type(4), aligned(4)));
  const char* words = p - off;
  const v4i lo = *reinterpret_cast<const v4i_words*>(words);
  const int hi = *reinterpret_cast<const int*>(words + (off ? 16 : 12));
  v4i r;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    r[i] = (int)__builtin_amdgcn_alignbit(i < 3 ? lo[i + 1] : hi, lo[i], off * 8);
  return r;
}

// Whether rows of `width` elements from p on start at multiples of four elements.
template <class T>
__host__ __device__ __forceinline__ bool rows_of_fours(const T* p, int width) {
  return (width & 3) == 0 && ((uintptr_t)p & (4 * sizeof(T) - 1)) == 0;
}

// Four consecutive elements, stored together where p allows it (`vec`:
// rows_of_fours), else those in range.
// kStream: results that this kernel and the next do not read again leave the
// L2 to the operands (int8 8192 x 8192 x 4096 267 -> 252 us, gated
// 8192 x 4096 -> 8192 with g and u saved 971 -> 904).
template <bool kStream = false, class T>
__device__ __forceinline__ void store4(T* p, const float (&v)[4], int count, bool vec) {
  struct __attribute__((aligned(4 * sizeof(T)))) Four { T x[4]; } q;
  typedef int Words __attribute__((ext_vector_type(sizeof(T))));
#pragma unroll
  for (int i = 0; i < 4; ++i) q.x[i] = from_f32<T>(v[i]);
  if (vec && count >= 4) {
    if (kStream)
      __builtin_nontemporal_store(__builtin_bit_cast(Words, q), reinterpret_cast<Words*>(p));
    else
      *reinterpret_cast<Four*>(p) = q;
  } else if (count >= 4) {  // (a start off its size takes the same instruction)
    typedef Words __attribute__((aligned(1))) WordsAny;
    *reinterpret_cast<WordsAny*>(p) = __builtin_bit_cast(Words, q);
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (i < count) p[i] = q.x[i];
  }
}

// ---------------------------------------------------------------------------
// Activations: a = act(g), and da = act'(g) for the backward pass, in 32 bits
// and without branches, so that several elements' arithmetic overlaps (an
// epilogue runs on one wave per SIMD; a call per element of the library's
// tanhf and erff took 14 of the 64 us of 4096 x 1024 -> 2048).
// ---------------------------------------------------------------------------

// e^x as 2^(x log2 e), 0 below the smallest normal number.  The product's
// rounding error, up to |x| 2^-24 in the result, is carried along for fp32
// (kFine; within the bounds there: e^-150 is 0, as gelu's density needs, which is
// multiplied by g, and 1 / (1 + e^88) comes out as 0) and below a 16-bit type's own
// rounding by far otherwise.  `below` is what x lost in a rounding of its own.
template <bool kFine>
__device__ __forceinline__ float exponential(float x, float below = 0.0f) {
  if (!kFine) return __builtin_amdgcn_exp2f(x * 1.44269504f);
  x = fminf(fmaxf(x, -150.0f), 88.0f);
  const float t = x * 1.44269504f;
  const float e = __builtin_amdgcn_exp2f(t);
  // x log2 e - t, with log2 e = 1.44269504 + 1.9259630e-8
  const float rest =
      fmaf(below, 1.44269504f, fmaf(x, 1.44269504f, -t) + x * 1.9259630e-8f);
  return fmaf(e, rest * 0.69314718f, e);
}

// Reciprocal within one unit in the last place; 0 where it is subnormal.
__device__ __forceinline__ float reciprocal(float x) { return __builtin_amdgcn_rcpf(x); }

// The normal CDF and its density: with z = |g| / sqrt(2) and t = 1 / (1 + 0.38 z),
// erfc z = t P(t) e^(-z^2), P the polynomial of degree 8 that comes relatively
// closest to e^(z^2) erfc(z) / t over 0 <= z <= 9.6 (within 2e-8; e^(-z^2) is 0
// beyond), so the smaller tail keeps its leading digits however small it is.  For
// fp32 what g^2 / 2 loses in its rounding goes into the exponential as well.  (The
// five terms of Abramowitz and Stegun 7.1.26, 1.5e-7 of 1, are off by 5e-5 of the
// tail at g = -3 and 4e-3 at -6; 4096 x 1024 -> 2048 with dropout 48.6 -> 49.7 us.)
template <bool kFine>
__device__ __forceinline__ void normal_cdf(float g, float& cdf, float& density) {
  const float m = fminf(fabsf(g), 20.0f);  // (e is 0 from 13.3 on)
  const float square = -0.5f * m * m;
  const float e = exponential<kFine>(square, kFine ? fmaf(-0.5f * m, m, -square) : 0.0f);
  const float t = reciprocal(fmaf(0.38f * 0.70710678f, fabsf(g), 1.0f));
  float q = fmaf(t, 0.05889616f, -0.26192135f);
  q = fmaf(t, q, 0.36308f);
  q = fmaf(t, q, -0.16051474f);
  q = fmaf(t, q, 0.22933216f);
  q = fmaf(t, q, 0.13896517f);
  q = fmaf(t, q, 0.20382008f);
  q = fmaf(t, q, 0.21393241f);
  q = fmaf(t, q, 0.21441014f);
  const float tail = 0.5f * t * q * e;
  cdf = g > 0.0f ? 1.0f - tail : tail;
  density = e * 0.39894228f;
}

// tanh: its series near zero, where 1 - 2 / (1 + e^2g) would cancel.
template <bool kFine>
__device__ __forceinline__ float hyperbolic_tangent(float g) {
  const float g2 = g * g;
  float q = fmaf(g2, -8.8632356e-3f, 2.1869489e-2f);  // -1382/155925, 62/2835
  q = fmaf(g2, q, -5.3968254e-2f);                    // -17/315
  q = fmaf(g2, q, 0.13333333f);
  q = fmaf(g2, q, -0.33333333f);
  const float near = fmaf(g * g2, q, g);
  const float far = fmaf(-2.0f, reciprocal(1.0f + exponential<kFine>(2.0f * g)), 1.0f);
  return fabsf(g) > 0.4f ? far : near;  // (a NaN takes `near`, which keeps it)
}

// kN elements; T is the type that the results are for.
template <class T, int kN>
__device__ __forceinline__ void activate(int act, const float (&g)[kN], float (&a)[kN]) {
  constexpr bool kFine = sizeof(T) == 4;
  if (act == PPO_LAYER_SILU) {
#pragma unroll
    for (int i = 0; i < kN; ++i) a[i] = g[i] * reciprocal(1.0f + exponential<kFine>(-g[i]));
  } else if (act == PPO_LAYER_GELU) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      float cdf, density;
      normal_cdf<kFine>(g[i], cdf, density);
      a[i] = g[i] * cdf;
    }
  } else if (act == PPO_LAYER_TANH) {
#pragma unroll
    for (int i = 0; i < kN; ++i) a[i] = hyperbolic_tangent<kFine>(g[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kN; ++i) a[i] = g[i] < 0.0f ? 0.0f : g[i];
  }
}

template <class T, int kN>
__device__ __forceinline__ void activate_grad(int act, const float (&g)[kN], float (&a)[kN],
                                              float (&da)[kN]) {
  constexpr bool kFine = sizeof(T) == 4;
  if (act == PPO_LAYER_SILU) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const float s = reciprocal(1.0f + exponential<kFine>(-g[i]));
      a[i] = g[i] * s;
      da[i] = s * fmaf(g[i], 1.0f - s, 1.0f);
    }
  } else if (act == PPO_LAYER_GELU) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      float cdf, density;
      normal_cdf<kFine>(g[i], cdf, density);
      a[i] = g[i] * cdf;
      da[i] = fmaf(g[i], density, cdf);
    }
  } else if (act == PPO_LAYER_TANH) {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      a[i] = hyperbolic_tangent<kFine>(g[i]);
      da[i] = fmaf(-a[i], a[i], 1.0f);
    }
  } else {
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      a[i] = g[i] < 0.0f ? 0.0f : g[i];
      da[i] = g[i] > 0.0f ? 1.0f : 0.0f;
    }
  }
}

// ---------------------------------------------------------------------------
// Dropout.  Element (row, column) is kept if word (column mod 4) of
// Philox4x32 at the counter (column / 4, row id, 0) under the 64-bit seed is
// below keep = round((1 - p) 2^32), and is then multiplied by 1 / (1 - p).
// The mask is a function of (seed, row id, column) alone, so the backward
// pass, or an update that meets the row again in another minibatch, forms it
// anew instead of reading it.  Seven rounds: the fewest that its authors
// (Salmon, Moraes, Dror, Shaw, SC 2011) found to pass every test of
// BigCrush; each round is two 32x32-bit products.
// ---------------------------------------------------------------------------
struct Dropout {
  const int64_t* rows;      // row ids, or null: 0, 1, ...
  const uint64_t* seed_at;  // seed in device memory, or null: `seed`
  uint64_t seed;
  uint32_t keep;            // kept: word < keep (all: every word)
  int mode;                 // 0 no dropout, 1 a random mask, 2 nothing is kept
  float scale;              // 1 / (1 - p)
};

inline Dropout make_dropout(double p, uint64_t seed, const uint64_t* seed_at, const int64_t* rows) {
  Dropout d = {rows, seed_at, seed, 0, 0, 1.0f};
  if (!(p > 0.0)) return d;
  d.scale = p < 1.0 ? (float)(1.0 / (1.0 - p)) : 0.0f;
  // nearbyint rounds ties to even; 2^32 (p below 2^-33) keeps every word
  const double keep = nearbyint((1.0 - p) * 4294967296.0);
  if (keep >= 4294967296.0) return d;  // (and then scale rounds to 1)
  d.keep = (uint32_t)keep;
  d.mode = d.keep ? 1 : 2;
  return d;
}

__device__ __forceinline__ uint4 philox(uint64_t seed, uint32_t c0, uint64_t row) {
  uint32_t x0 = c0, x1 = (uint32_t)row, x2 = (uint32_t)(row >> 32), x3 = 0;
  uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#pragma unroll
  for (int r = 0; r < 7; ++r) {
    const uint64_t p0 = (uint64_t)x0 * 0xD2511F53u, p1 = (uint64_t)x2 * 0xCD9E8D57u;
    x0 = (uint32_t)(p1 >> 32) ^ x1 ^ k0;
    x1 = (uint32_t)p1;
    x2 = (uint32_t)(p0 >> 32) ^ x3 ^ k1;
    x3 = (uint32_t)p0;
    k0 += 0x9E3779B9u;
    k1 += 0xBB67AE85u;
  }
  return make_uint4(x0, x1, x2, x3);
}

__device__ __forceinline__ uint64_t dropout_seed(const Dropout& d) {
  return d.seed_at ? *d.seed_at : d.seed;
}

// Which of the four columns from 4 * group on are kept.
__device__ __forceinline__ void keep4(const Dropout& d, uint64_t seed, uint64_t row, uint32_t group,
                                      bool (&keep)[4]) {
  uint4 w = make_uint4(0, 0, 0, 0);
  if (d.mode == 1) w = philox(seed, group, row);
  keep[0] = d.mode == 0 || w.x < d.keep;  // (mode 2: below 0)
  keep[1] = d.mode == 0 || w.y < d.keep;
  keep[2] = d.mode == 0 || w.z < d.keep;
  keep[3] = d.mode == 0 || w.w < d.keep;
}

// Dropout of those columns: dropped elements are selected away, not multiplied
// by zero, so an infinity or a NaN there goes.
__device__ __forceinline__ void drop4(const Dropout& d, uint64_t seed, uint64_t row,
                                      uint32_t group, float (&v)[4]) {
  if (d.mode == 0) return;
  bool keep[4];
  keep4(d, seed, row, group, keep);
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = keep[i] ? v[i] * d.scale : 0.0f;
}

}  // namespace ppo
