// Shared pieces of the token-policy operators (libppo_tokens.so): a row of
// logits held by a group of lanes, its softmax statistics, and the reductions
// over lanes, waves and rows.
//
// A group of G lanes holds a row (G = 16: four rows to a wave; 64: a wave;
// 256 to 1024: a workgroup).  A row starts at any address that its type
// allows, so it is cut into `head` elements up to the first multiple of 16
// bytes, `nvec` chunks of 16 bytes, and `tail` elements: chunk i G + t is lane
// t's i-th, and the up to 14 elements at the two ends are one more to a lane.
// Every access to chunks is aligned, whatever the width.
//
// Statistics are relative to m = max l, in powers of two: e_j = 2^(c (l_j - m)),
// c = log2(e) / temperature: a subtraction, a product and a v_exp_f32 each.  (One
// fma of c l_j - c m would save an operation; it overflows in rows of a type's
// lowest values, which masks leave behind.)  The taken action a is kept out of the
// sums (`rest`): 1 - p_a = rest / s and, where a outweighs the others, log p_a =
// -log1p(rest / e_a) keep their leading digits as p_a goes to 1.
#pragma once

#include "layers.hpp"
#include "ppo_tokens.h"

namespace ppo {

constexpr int kWave = 64;
constexpr float kLn2 = 0.69314718056f;
constexpr double kLn2d = 0.693147180559945309417;
constexpr float kNegInf = -__builtin_inff();
#define PPO_NAN __builtin_nanf("")

// Workgroups of a launch that leaves partial sums behind, and partial counts.
constexpr int kMaxPartials = 8192;
constexpr int kCountBlocks = 256;
constexpr int kSums = 5;  // policy, KL, entropy, approximate KL, clipped

typedef unsigned v4u __attribute__((ext_vector_type(4)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// ---------------------------------------------------------------------------
// Reductions
// ---------------------------------------------------------------------------

// Orders LDS only; a wave's global loads and stores stay in flight.
__device__ __forceinline__ void lds_barrier() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "workgroup", "local");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "workgroup", "local");
}

template <int kCtrl>
__device__ __forceinline__ float dpp(float x) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, x), kCtrl,
                                                               0xF, 0xF, false));
}
template <int kCtrl>
__device__ __forceinline__ double dpp(double x) {
  const int2 v = __builtin_bit_cast(int2, x);
  int2 r;
  r.x = __builtin_amdgcn_update_dpp(0, v.x, kCtrl, 0xF, 0xF, false);
  r.y = __builtin_amdgcn_update_dpp(0, v.y, kCtrl, 0xF, 0xF, false);
  return __builtin_bit_cast(double, r);
}
__device__ __forceinline__ float lane_of(float x, int lane) {
  return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
}
__device__ __forceinline__ double lane_of(double x, int lane) {
  const int2 v = __builtin_bit_cast(int2, x);
  int2 r;
  r.x = __builtin_amdgcn_readlane(v.x, lane);
  r.y = __builtin_amdgcn_readlane(v.y, lane);
  return __builtin_bit_cast(double, r);
}

// f over 16 lanes (quad_perm [1,0,3,2], [2,3,0,1], row_half_mirror, row_mirror),
// or over the wave, the same value in every lane, in a fixed order.
template <int G, class T, class F>
__device__ __forceinline__ T lanes_reduce(T x, F f) {
  x = f(x, dpp<0xB1>(x));
  x = f(x, dpp<0x4E>(x));
  x = f(x, dpp<0x141>(x));
  x = f(x, dpp<0x140>(x));
  if (G == 16) return x;
  return f(f(lane_of(x, 0), lane_of(x, 16)), f(lane_of(x, 32), lane_of(x, 48)));
}
template <int G, class T>
__device__ __forceinline__ T lanes_sum(T x) {
  return lanes_reduce<G>(x, [](T a, T b) { return a + b; });
}
template <int G>
__device__ __forceinline__ float lanes_max(float x) {
  return lanes_reduce<G>(x, [](float a, float b) { return fmaxf(a, b); });
}

// ---------------------------------------------------------------------------
// Elements
// ---------------------------------------------------------------------------

// Element j of 16 bytes.
template <class T>
__device__ __forceinline__ float unpack(v4i w, int j);
template <>
__device__ __forceinline__ float unpack<float>(v4i w, int j) {
  const int x = w[j];  // (a bit cast of the element itself takes the vector's first)
  return __builtin_bit_cast(float, x);
}
template <>
__device__ __forceinline__ float unpack<bf16>(v4i w, int j) {
  return __builtin_bit_cast(float, j & 1 ? w[j >> 1] & (int)0xFFFF0000 : w[j >> 1] << 16);
}
template <>
__device__ __forceinline__ float unpack<fp16>(v4i w, int j) {
  const int x = w[j >> 1];
  return (float)__builtin_bit_cast(v2h, x)[j & 1];
}

// Sixteen bytes of -inf: what stands in for a chunk behind the last.
template <class T>
__device__ __forceinline__ v4i no_chunk() {
  const int w = sizeof(T) == 4 ? (int)0xFF800000
                               : __is_same(T, bf16) ? (int)0xFF80FF80 : (int)0xFC00FC00;
  return v4i{w, w, w, w};
}

// Element j of 16 bytes becomes -inf.
template <class T>
__device__ __forceinline__ void knock_out(v4i& w, int j) {
  constexpr int kInf = __is_same(T, bf16) ? 0xFF80 : 0xFC00;
#pragma unroll
  for (int k = 0; k < 4; ++k)
    if (sizeof(T) == 4) {
      if (k == j) w[k] = (int)0xFF800000;
    } else if (k == j >> 1) {
      w[k] = j & 1 ? (w[k] & 0xFFFF) | (kInf << 16) : (w[k] & (int)0xFFFF0000) | kInf;
    }
}

// Two floats to the two halves of a word, to nearest even.
template <class T>
__device__ __forceinline__ int pack2(float a, float b) {
  const v2f v = {a, b};
  if constexpr (__is_same(T, bf16))
    return __builtin_bit_cast(int, __builtin_convertvector(v, v2bf));
  else
    return __builtin_bit_cast(int, __builtin_convertvector(v, v2h));
}
template <class T, int kN>
__device__ __forceinline__ v4i pack(const float (&x)[kN]) {
  static_assert(kN == kPer16<T>, "");
  v4i w;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if constexpr (kN == 4)
      w[i] = __builtin_bit_cast(int, x[i]);
    else
      w[i] = pack2<T>(x[2 * i], x[2 * i + 1]);
  return w;
}

// Sixteen bytes of gradients: past the caches, at any address of the type (rows
// of the result may start elsewhere in 16 bytes than the logits' do).
__device__ __forceinline__ void store16(void* p, v4i w, bool aligned) {
  if (aligned)
    __builtin_nontemporal_store(w, reinterpret_cast<v4i*>(p));
  else
    *reinterpret_cast<v4i_any*>(p) = w;
}

// How a row is cut into chunks and ends.
template <class T>
struct Cut {
  int head = 0, nvec = 0, ends = 0;
  Cut() = default;
  __device__ __forceinline__ Cut(const T* row, int A) {
    const int off = (int)(((uintptr_t)row & 15) / sizeof(T));
    head = min(off ? kPer16<T> - off : 0, A);
    nvec = (A - head) / kPer16<T>;
    ends = A - nvec * kPer16<T>;
  }
  // Column of the e-th element at the ends.
  __device__ __forceinline__ int end_column(int e) const {
    return e < head ? e : e + nvec * kPer16<T>;
  }
};

// ---------------------------------------------------------------------------
// Rows of a call, as kernels take them
// ---------------------------------------------------------------------------
struct Rows {
  const void* logits;
  const void* actions;
  const uint8_t* mask;
  int64_t n, T;  // rows; rows a sequence
  int64_t S;
  int A, actions64;
  float c;       // log2(e) / temperature
  float inv_tau;
  float c_down, c_left;  // the same rounded down, and what that left of it (above 0)

  __device__ __forceinline__ bool live(int64_t r) const { return !mask || mask[r]; }
  // The row's action, -1 where it lies outside the row.
  __device__ __forceinline__ int action(int64_t r) const {
    const int64_t a = actions64 ? static_cast<const int64_t*>(actions)[r]
                                : (int64_t) static_cast<const int32_t*>(actions)[r];
    return a >= 0 && a < A ? (int)a : -1;
  }
};

// Sums of a row's e_j (all but the action's) and of e_j c (l_j - m), relative to
// the row's largest logit m.
struct Stat {
  static constexpr bool kFine = false;
  float m, s, u;
};
// The same for log-probabilities of which another policy's are taken away: their own
// rounding, and that of c, which all of a row's exponents share, would be what is left of a
// small difference.  Sums in 64 bits, exponents with all of c; two instructions more an
// element (the preference loss of 4096 x 50304 bf16 and its gradient 220 -> 224 us).
struct FineStat {
  static constexpr bool kFine = true;
  float m, u;
  double s;
};

// c times a difference of logits, as a kind of sums takes it.  (Both parts of a fine c are
// above 0, so that -inf stays that.)
template <class S>
struct Scale {
  float c, left;
  __device__ __forceinline__ explicit Scale(const Rows& rows)
      : c(S::kFine ? rows.c_down : rows.c), left(rows.c_left) {}
  __device__ __forceinline__ float operator()(float d) const {
    return S::kFine ? fmaf(d, c, d * left) : d * c;  // (rounded once)
  }
  __device__ __forceinline__ double exact(double d) const {
    return d * (S::kFine ? (double)c + (double)left : (double)c);
  }
};

// x relative to m, no smaller than its own; parts without elements have m = -inf,
// s = u = 0.
__device__ __forceinline__ float fused(float a, float b, float c) { return fmaf(a, b, c); }
__device__ __forceinline__ double fused(double a, float b, double c) { return fma(a, (double)b, c); }
template <bool kEntropy, class X, class S>
__device__ __forceinline__ void rebase(X& x, float m, const Scale<S>& c) {
  using U = decltype(x.u);
  const bool none = x.m == kNegInf;
  const float d = c(x.m - m);
  const float f = none ? 0.0f : exp2_fast(d);
  if (kEntropy) x.u = none || f == 0.0f ? (U)0.0f : f * fused((U)x.s, d, x.u);
  x.s *= f;
  x.m = m;
}
template <int G, bool kEntropy, class S>
__device__ __forceinline__ S lanes_join(S x, const Scale<S>& c) {
  rebase<kEntropy>(x, lanes_max<G>(x.m), c);
  x.s = lanes_sum<G>(x.s);
  if (kEntropy) x.u = lanes_sum<G>(x.u);
  return x;
}

// The parts of a workgroup's waves as one, the same in every lane of wave 0 (other
// lanes: not defined).  One barrier; `part` may be written again once wave 0 has
// passed another.
template <bool kEntropy, class S>
__device__ __forceinline__ S block_join(S x, const Scale<S>& c, S* part) {
  x = lanes_join<kWave, kEntropy>(x, c);
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  const int waves = blockDim.x / kWave;
  if (lane == 0) part[wave] = x;
  lds_barrier();
  if (wave == 0) {
    const int k = lane & 15;
    x = k < waves ? part[k] : S{kNegInf, 0.0f, 0.0f};
    x = lanes_join<16, kEntropy>(x, c);
  }
  return x;
}

// 2 atanh(num / den) = log((den + num) / (den - num)) for |num / den| <= 1/3, in 64
// bits: its series, whose next term is below 2^-44 of the first.
__device__ __forceinline__ double twice_atanh(double num, double den) {
  double r = __builtin_amdgcn_rcp(den);
  r = fma(fma(-den, r, 1.0), r, r);
  const double z = num * r, q = z * z;
  double x = 1.0 / 23.0;
#pragma unroll
  for (int k = 21; k >= 1; k -= 2) x = fma(x, q, 1.0 / k);
  return 2.0 * z * x;
}

// What a row comes to, given the action's logit: log p_a in 64 bits and the
// pieces that the gradient needs.  (The library's log and log1p in 64 bits would take
// more registers than the row's own chunks leave.)
struct RowTerms {
  double lp;                        // log p_a
  float m, inv_s, lns, H, omp, pa;  // lns = log s, omp = 1 - p_a
};
template <bool kEntropy, class S>
__device__ __forceinline__ RowTerms row_terms(S x, float la, const Scale<S>& c) {
  RowTerms o;
  // (a NaN passes through: fmaxf drops it, e_a keeps it)
  rebase<kEntropy>(x, fmaxf(x.m, la), c);
  const float ta = c(la - x.m);
  const float ea = exp2_fast(ta);
  const auto whole = x.s + ea;  // (in the sums' own type)
  const float s = (float)whole;
  o.m = x.m;
  o.inv_s = 1.0f / s;
  // where a outweighs the others log s = log e_a + log(s / e_a), whose last term is
  // -log p_a; else s = 2^n f with f in [0.7, 1.4).  (Below the others the difference of
  // logarithms loses nothing, and holds where e_a has underflowed.)
  const bool most = ea >= x.s;
  int n = __builtin_amdgcn_frexp_expf(s);
  if (__builtin_amdgcn_frexp_mantf(s) < 0.70710678f) n -= 1;
  const double f = __builtin_ldexp((double)whole, -n);
  const double L = twice_atanh(most ? (double)x.s : f - 1.0,
                               most ? (double)whole + (double)ea : f + 1.0);
  const double lns = fma(most ? (double)ta : (double)n, kLn2d, L);
  o.lns = (float)lns;
  o.lp = most ? -L : c.exact((double)la - (double)x.m) * kLn2d - lns;
  o.omp = (float)x.s * o.inv_s;
  o.pa = ea * o.inv_s;
  o.H = 0.0f;
  if (kEntropy) {
    const float u = x.u + (ea == 0.0f ? 0.0f : ea * ta);
    o.H = fmaf(-kLn2 * u, o.inv_s, o.lns);
  }
  return o;
}

// One row of `saved`.
struct __attribute__((aligned(16))) Saved {
  float m, inv_s, lns, H, omp, pa, lp, weight;
};
static_assert(sizeof(Saved) == PPO_TOKEN_SAVED * sizeof(float), "");
__device__ __forceinline__ Saved saved_of(const RowTerms& t, float weight) {
  return {t.m, t.inv_s, t.lns, t.H, t.omp, t.pa, (float)t.lp, weight};
}

// A row's gradient: dlogits_j = e_j (B + C c (l_j - m)), and da at the action
// (-1: none).  From G = dloss/dlog p_a and E = dloss/dH:
//   G ([j = a] - p_j) - E p_j (log p_j + H), over the temperature.
struct Grad {
  float m, B, C, da;
  int a;
};
__device__ __forceinline__ Grad row_grad(const Saved& t, float G, float E, float inv_tau, int a) {
  Grad g;
  g.m = t.m;
  g.a = a;
  g.B = inv_tau * t.inv_s * (-G - E * (t.H - t.lns));
  g.C = -inv_tau * t.inv_s * kLn2 * E;
  g.da = inv_tau * (G * t.omp - (t.pa == 0.0f ? 0.0f : E * t.pa * (t.lp + t.H)));
  return g;
}
// (kC: C is not 0.  An e of 0 has an exponent of -inf, or one that times C may become that:
// it is held where e has long been 0, and its product with any C of use finite.)
constexpr float kLeastExponent = -256.0f;
template <bool kC>
__device__ __forceinline__ float grad_at(const Grad& g, float c, float l) {
  const float t = (l - g.m) * c;
  const float e = exp2_fast(t);
  return kC ? e * fmaf(g.C, fmaxf(t, kLeastExponent), g.B) : e * g.B;
}

// ---------------------------------------------------------------------------
// A row in registers
// ---------------------------------------------------------------------------
// A value that all lanes of a row's group share: in a scalar register where the group is
// whole waves.
template <int G>
__device__ __forceinline__ float shared_by(float x) {
  if (G < kWave) return x;
  return __builtin_bit_cast(float, __builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, x)));
}
template <int G>
__device__ __forceinline__ int shared_by(int x) {
  return G < kWave ? x : __builtin_amdgcn_readfirstlane(x);
}
template <int G>
__device__ __forceinline__ Grad shared_by(const Grad& g) {
  return {shared_by<G>(g.m), shared_by<G>(g.B), shared_by<G>(g.C), shared_by<G>(g.da),
          shared_by<G>(g.a)};
}

// The workgroup's group that this lane is in; of a wave's or a workgroup's the
// compiler is told that it is one.
template <int G>
__device__ __forceinline__ int group_of() {
  if (G > kWave) return 0;
  const int g = threadIdx.x / G;
  return G == kWave ? __builtin_amdgcn_readfirstlane(g) : g;
}

// A wave of one row addresses its chunks through a buffer descriptor, which ends
// them: loads behind the last give 0, stores there write nothing, and one offset
// a lane serves all of them.  (Rows of 16 lanes, four to a wave, have addresses of
// their own.)
// The descriptor starts at the round's own first chunk: the lane's offset is then the same
// in every round, and no register holds one for each.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t chunk_buffer(const v4i* chunks, int count,
                                                               int round) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<v4i*>(chunks) + round, 0,
                                           max(count - round, 0) * 16, 0x00027000);
}
constexpr int kPastCaches = 2;  // the buffer instructions' nt bit

// A row, V chunks a lane: between V G / 2 and V G of them hold it.  The loads go
// straight through; a pass over the chunks leaves out the rounds of G that lie behind
// the last, of which there may be some in the second half (`reaches`).
template <class T, int G, int V>
struct RowRegs {
  static constexpr int kN = kPer16<T>;
  static constexpr bool kBuffer = G >= kWave;
  v4i raw[V];
  float end;   // the lane's element at the ends (-inf: none)
  Cut<T> cut;
  int end_col; // its column, -1: none

  // No row: nothing is read.
  static __device__ __forceinline__ Cut<T> cut_of(const T* row, int A) {
    return row ? Cut<T>(row, A) : Cut<T>();
  }
  __device__ __forceinline__ void load_end(const T* row, int t) {
    end_col = t < cut.ends ? cut.end_column(t) : -1;
    end = end_col >= 0 ? to_f32(row[end_col]) : kNegInf;
  }
  __device__ __forceinline__ RowRegs(const T* row, int A, int t) : cut(cut_of(row, A)) {
    const v4i* body = reinterpret_cast<const v4i*>(row + cut.head);
#pragma unroll
    for (int i = 0; i < V; ++i)
      if constexpr (kBuffer)
        raw[i] = __builtin_bit_cast(
            v4i, __builtin_amdgcn_raw_buffer_load_b128(chunk_buffer(body, cut.nvec, i * G), t * 16, 0,
                                                       kPastCaches));
      else if (i * G + t < cut.nvec)
        raw[i] = __builtin_nontemporal_load(body + i * G + t);
    load_end(row, t);
  }

  // (at 128 registers to a lane the branches spill; those layouts come in finer steps)
  __device__ __forceinline__ bool reaches(int i) const {
    return G >= 512 || i < V / 2 || i * G < cut.nvec;
  }

  // The compiler would unpack 16-bit chunks once and keep them so, in twice the
  // registers, and take many chunks at a time (a row of 256 KB spills half of itself; 512 x
  // 65536 fp32 69 us, 61 so): for each pass over a chunk it is to take it for changed, and
  // its turn for coming after `sum`.
  __device__ __forceinline__ void turn(int i, float& sum) {
    if (sizeof(T) == 2 || G >= 512) asm volatile("" : "+v"(raw[i]), "+v"(sum));
  }

  // Chunks behind the last take no part in the sums, nor does column a.
  __device__ __forceinline__ void take_out(int a, int t) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i * G + t >= cut.nvec) raw[i] = no_chunk<T>();
    if (a < 0) return;
    if (end_col == a) end = kNegInf;
    const int b = a - cut.head, v = b >= 0 ? b / kN : -1;
    if (v < 0 || v >= cut.nvec || v % G != t) return;
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i == v / G) knock_out<T>(raw[i], b - v * kN);
  }

  template <bool kEntropy>
  __device__ __forceinline__ Stat stat(const Scale<Stat>& c) {
    float m = end;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (!reaches(i)) continue;
      turn(i, m);
#pragma unroll
      for (int j = 0; j < kN; ++j) m = fmaxf(m, unpack<T>(raw[i], j));
    }
    Stat x = {m, 0.0f, 0.0f};
    // (a lane without a finite element: exponents of -inf rather than NaN)
    if (m == kNegInf) m = 0.0f;
    float s2 = 0.0f;
    auto add = [&](float l, float& s) {
      const float p = c(l - m), e = exp2_fast(p);
      s += e;
      if (kEntropy) x.u = fmaf(e, fmaxf(p, -1e30f), x.u);
    };
    add(end, x.s);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (!reaches(i)) continue;
      turn(i, x.s);
#pragma unroll
      for (int j = 0; j < kN; j += 2) {
        add(unpack<T>(raw[i], j), x.s);
        add(unpack<T>(raw[i], j + 1), s2);
      }
    }
    x.s += s2;
    return x;
  }

  // `out` lies in 16 bytes as the logits' row does.  With a `next` row (null: none) each
  // chunk's registers take that row's as soon as its own gradient is on its way, so that
  // reads and writes overlap however few rows a CU holds.
  template <bool kC>
  __device__ __forceinline__ void write(const Grad& g, float c, T* out, int A, int t,
                                        const T* next = nullptr) {
    v4i* body = reinterpret_cast<v4i*>(out + cut.head);
    const Cut<T> now = cut;
    const int now_col = end_col;
    const float now_end = end;
    cut = cut_of(next, A);
    const v4i* from = reinterpret_cast<const v4i*>(next + cut.head);
    float last = 0.0f;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (G >= 512 || i < V / 2 || i * G < now.nvec) {
        float d[kN];
        turn(i, last);
#pragma unroll
        for (int j = 0; j < kN; ++j) d[j] = grad_at<kC>(g, c, unpack<T>(raw[i], j));
        const v4i w = pack<T>(d);
        last = d[0];
        if constexpr (kBuffer)
          __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(v4u, w),
                                                 chunk_buffer(body, now.nvec, i * G), t * 16, 0,
                                                 kPastCaches);
        else if (i * G + t < now.nvec)
          __builtin_nontemporal_store(w, body + i * G + t);
      }
      if constexpr (kBuffer)
        raw[i] = __builtin_bit_cast(
            v4i, __builtin_amdgcn_raw_buffer_load_b128(chunk_buffer(from, cut.nvec, i * G), t * 16, 0,
                                                       kPastCaches));
    }
    load_end(next, t);
    if (now_col >= 0) out[now_col] = from_f32<T>(grad_at<kC>(g, c, now_end));
    // the action's own element, by the lane that wrote its place
    const int b = g.a - now.head;
    const bool inside = g.a >= 0 && b >= 0 && b < now.nvec * kN;
    if (inside ? (b / kN) % G == t : (g.a >= 0 && g.a == now_col)) out[g.a] = from_f32<T>(g.da);
  }
};

// Zeros over a row of gradients, by G lanes.
template <class T, int G>
__device__ __forceinline__ void write_zeros(T* out, int A, int t) {
  const Cut<T> cut(out, A);
  v4i* body = reinterpret_cast<v4i*>(out + cut.head);
  const v4i zero = {0, 0, 0, 0};
  for (int i = t; i < cut.nvec; i += G) __builtin_nontemporal_store(zero, body + i);
  if (t < cut.ends) out[cut.end_column(t)] = from_f32<T>(0.0f);
}

// ---------------------------------------------------------------------------
// The rows' weights
// ---------------------------------------------------------------------------

// counts: what a counting launch left (null: every row counts, `inverse` is the
// weight).  With lengths [S] the mean is over sequences, else over rows.
struct Weights {
  const int* counts;
  const int* lengths;
  int partials;
  float inverse;  // > 0: 1 / denominator in place of the count's
};
// 1 / denominator, for every lane of the wave.
__device__ __forceinline__ float inverse_count(const Weights& w) {
  if (w.inverse > 0.0f) return w.inverse;
  double n = 0.0;
  for (int i = threadIdx.x & (kWave - 1); i < w.partials; i += kWave) n += w.counts[i];
  n = lanes_sum<kWave>(n);
  return n > 0.0 ? (float)(1.0 / n) : 0.0f;
}
__device__ __forceinline__ float row_weight(const Weights& w, float inverse, int64_t seq) {
  return w.lengths ? inverse / (float)w.lengths[seq] : inverse;
}

// The rows in the order in which a launch takes them: those that count, then the others
// from the last on (null: as they lie, and whether one counts is looked up).  Where a
// workgroup has a handful of long rows, taking every so many of the first kind gives
// all of them as many.
struct Order {
  const int* rows;
  const int* live;  // how many count
};

// Scratch: counts, lengths, the order, partial sums, then the split statistics.
struct Scratch {
  int* counts;
  int* lengths;
  int* order;
  double* sums;   // [kSums][kMaxPartials]
  Stat* parts;    // [rows][splits], or FineStat
  size_t bytes;
};

// Partial sums of a launch's workgroups, [kSums][kMaxPartials]; every lane's own
// sums are given, lanes without any give zeros.
template <int kN>
__device__ __forceinline__ void leave_sums(double (&x)[kN], double* sums) {
  __shared__ double part[16][kN];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
#pragma unroll
  for (int k = 0; k < kN; ++k) {
    x[k] = lanes_sum<kWave>(x[k]);
    if (lane == 0) part[wave][k] = x[k];
  }
  __syncthreads();
  if ((int)threadIdx.x < kN) {
    double v = 0.0;
    for (int w = 0; w < (int)blockDim.x / kWave; ++w) v += part[w][threadIdx.x];
    sums[(int64_t)threadIdx.x * kMaxPartials + blockIdx.x] = v;
  }
}

// Host side (tokens.hip) -----------------------------------------------------------

constexpr int kMaxSplits = 64;
// Workgroups that share a row's statistics where one to a row would leave the chip
// empty, or where a row does not fit a workgroup's registers.
int row_splits(int64_t rows, int64_t A, int dtype);
Scratch scratch_of(void* workspace, int64_t S, int64_t T, int64_t A, int dtype);
// Checks rows; fills what kernels take.
int take_rows(const ppo_token_rows* r, bool actions, Rows& out);
// Checks a loss's weights; what they need counted.
int take_weights(const Rows& rows, const ppo_token_loss* loss, const Scratch& s, Weights& w);
// Enqueues the counting, or the ordering of rows (mask given) and the counting.
void count_weights(const Rows& rows, const Weights& w, const Scratch& s, hipStream_t stream);
Order take_order(const Rows& rows, Weights& w, const Scratch& s, hipStream_t stream);

// A launch has fewer than 2^32 lanes.
inline bool fits_launch(int64_t blocks, int lanes) { return blocks < ((int64_t)1 << 32) / lanes; }
inline int launch_blocks(int64_t groups, int64_t most) {
  return (int)(groups < most ? groups : most);
}
inline int64_t chunks_of(int64_t A, int dtype) { return div_up(A * dtype_size(dtype), 16); }

}  // namespace ppo
