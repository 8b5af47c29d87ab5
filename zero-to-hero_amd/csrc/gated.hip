// The gated feed-forward block and its backward pass:
//   g = x wg^T + bg,  u = x wu^T + bu,  h = dropout(act(g) * u)
//   dh' = dropout(dh),  du = dh' act(g),  dg = dh' u act'(g)
//   dx = dg wg + du wu,  dwg = dg^T x,  dwu = du^T x,  dbg = sum dg, dbu = sum du
// Forward: one product over both weight matrices (gemm_tile.hpp; a wave holds
// the gate's and the up projection's sums of the same elements, so g and u
// never leave registers unless the backward pass wants them).  Backward: one
// elementwise pass forms dg and du, then two products read them, x and the
// weights as they lie.
#include "gemm_tile.hpp"

namespace ppo {
namespace {

template <class T>
struct GatedEpi {
  static constexpr bool kGated = true;
  static constexpr int kBatch = 2;
  const T* bg;
  const T* bu;
  T* h;
  float* saved;   // [2][M][F4] or null
  int64_t half;   // M * F4
  int F, F4, act;
  Dropout drop;

  static constexpr bool kRows = true;
  struct Cols {
    float g[4], u[4];
    __device__ __forceinline__ void arrived() {
#pragma unroll
      for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(g[i]), "+v"(u[i]));
    }
  };
  typedef long Row;
  __device__ __forceinline__ Cols columns(int n) const {
    Cols c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = min(n + i, F - 1);
      c.g[i] = bg ? to_f32(bg[at]) : 0.0f;
      c.u[i] = bg ? to_f32(bu[at]) : 0.0f;
    }
    return c;
  }
  __device__ __forceinline__ Row row(int m) const {
    return drop.mode && drop.rows ? drop.rows[m] : m;
  }
  template <int B>
  __device__ __forceinline__ void apply(int n, const Cols& cols, const int (&m)[B],
                                        const bool (&live)[B], const Row (&id)[B],
                                        const v4f (&cg)[B], const v4f (&cu)[B]) const {
    float g[4 * B], u[4 * B], a[4 * B];
#pragma unroll
    for (int k = 0; k < 4 * B; ++k) {
      g[k] = cg[k / 4][k % 4] + cols.g[k % 4];
      u[k] = cu[k / 4][k % 4] + cols.u[k % 4];
    }
    if (saved) {
#pragma unroll
      for (int b = 0; b < B; ++b) {
        float* s = saved + (int64_t)m[b] * F4 + n;
        const v4f vg = {g[4 * b], g[4 * b + 1], g[4 * b + 2], g[4 * b + 3]};
        const v4f vu = {u[4 * b], u[4 * b + 1], u[4 * b + 2], u[4 * b + 3]};
        if (live[b]) {
          __builtin_nontemporal_store(vg, reinterpret_cast<v4f*>(s));
          __builtin_nontemporal_store(vu, reinterpret_cast<v4f*>(s + half));
        }
      }
    }
    activate<T>(act, g, a);
#pragma unroll
    for (int b = 0; b < B; ++b) {
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = a[4 * b + i] * u[4 * b + i];
      if (drop.mode) drop4(drop, dropout_seed(drop), (uint64_t)id[b], (uint32_t)n >> 2, v);
      if (live[b]) store4<true>(h + (int64_t)m[b] * F + n, v, F - n, rows_of_fours(h, F));
    }
  }
};

// Plain store of the sums.  Rows from `second` on go to a second output;
// `rows` of each are stored (the rest belongs to padding).
template <class T>
struct StoreEpi {
  static constexpr bool kGated = false;
  static constexpr int kBatch = 4;
  T* out0;
  T* out1;
  int rows, second, N;
  static constexpr bool kRows = false;
  struct Cols {
    __device__ __forceinline__ void arrived() {}
  };
  struct Row {};
  __device__ __forceinline__ Cols columns(int) const { return {}; }
  __device__ __forceinline__ Row row(int) const { return {}; }
  template <int B>
  __device__ __forceinline__ void apply(int n, Cols, const int (&m)[B], const bool (&live)[B],
                                        const Row (&)[B], const v4f (&c)[B]) const {
#pragma unroll
    for (int b = 0; b < B; ++b) {
      const bool other = m[b] >= second;
      const int at = other ? m[b] - second : m[b];
      const float v[4] = {c[b][0], c[b][1], c[b][2], c[b][3]};
      T* out = other ? out1 : out0;
      if (live[b] && at < rows)
        store4<true>(out + (int64_t)at * N + n, v, N - n, rows_of_fours(out, N));
    }
  }
};

// What rounding x to T leaves (nothing where the rounded value is not finite).
template <class T>
__device__ __forceinline__ float rounding_rest(float x) {
  const float left = x - to_f32(from_f32<T>(x));
  return fabsf(left) <= fabsf(x) ? left : 0.0f;
}

// Rows and columns that a workgroup of the next kernel takes: whole kilobytes
// of the saved rows (tiles of 64 x 64 took 291 us for 8192 x 8192 in bf16, whose
// 0.94 GB need 178 at a large copy's rate).
constexpr int kTileM = 16;
constexpr int kTileF = 256;

// dg and du from dh and the saved g and u, as rows [dg | du] of `pitch` elements
// (each of fp: F rounded up to 16 bytes, zeros behind F), the operand of both
// products; with `rest`, what their rounding to T left follows in the row.
// With `sums`, a tile's column sums for the biases ([row tiles][2 F], joined in
// order by BiasJoin).
template <class T>
__global__ void __launch_bounds__(256) gated_grad_kernel(const T* dh, const float* saved, int64_t M,
                                                         int F, int F4, int act, Dropout drop,
                                                         T* dgu, int64_t fp, int64_t pitch,
                                                         bool rest, float* sums) {
  __shared__ float part[4][2 * kTileF];
  // neighbouring workgroups take neighbouring columns
  const uint32_t across = (uint32_t)((fp + kTileF - 1) / kTileF);
  const uint32_t row_tile = blockIdx.x / across;
  const int64_t r0 = (int64_t)row_tile * kTileM;
  const int c0 = (int)(blockIdx.x % across) * kTileF;
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;  // four columns, rows ty + 4 i
  const int n = c0 + tx * 4;
  const uint64_t seed = drop.mode ? dropout_seed(drop) : 0;
  const bool vec = rows_of_fours(dh, F);
  constexpr int kRows = kTileM / 4;
  struct __attribute__((aligned(4 * sizeof(T)))) Four { T x[4]; };
  v4f g[kRows], u[kRows];
  Four d[kRows];
  int64_t id[kRows];
  // (every row's loads are under way before the first is used)
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int64_t m = min(r0 + ty + 4 * i, M - 1);
    const int c = min(n, F4 - 4);
    g[i] = *reinterpret_cast<const v4f*>(saved + m * F4 + c);
    u[i] = *reinterpret_cast<const v4f*>(saved + (M + m) * F4 + c);
    id[i] = drop.mode && drop.rows ? drop.rows[m] : m;
    const T* dp = dh + m * F;
    if (vec) {
      d[i] = *reinterpret_cast<const Four*>(dp + c);
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) d[i].x[k] = dp[min(n + k, F - 1)];
    }
  }
  float sg[4] = {0, 0, 0, 0}, su[4] = {0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < kRows; ++i) {
    const int64_t m = r0 + ty + 4 * i;
    float v[4], dg[4], du[4], a[4], da[4];
    const float gs[4] = {g[i][0], g[i][1], g[i][2], g[i][3]};
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = to_f32(d[i].x[k]) * drop.scale;
    // (a dropped element has no gradient, also where g or u is not finite)
    bool keep[4];
    keep4(drop, seed, (uint64_t)id[i], (uint32_t)n >> 2, keep);
    activate_grad<T>(act, gs, a, da);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const bool live = keep[k] && m < M && n + k < F;  // (behind F lies nothing that was saved)
      du[k] = live ? v[k] * a[k] : 0.0f;
      dg[k] = live ? v[k] * u[i][k] * da[k] : 0.0f;
      su[k] += du[k];
      sg[k] += dg[k];
    }
    if (m < M && n < fp) {
      T* row = dgu + m * pitch + n;
      store4(row, dg, 4, true);
      store4(row + fp, du, 4, true);
      if (rest) {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          dg[k] = rounding_rest<T>(dg[k]);
          du[k] = rounding_rest<T>(du[k]);
        }
        store4(row + 2 * fp, dg, 4, true);
        store4(row + 3 * fp, du, 4, true);
      }
    }
  }
  if (!sums) return;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    part[ty][tx * 4 + k] = sg[k];
    part[ty][kTileF + tx * 4 + k] = su[k];
  }
  __syncthreads();
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const int c = threadIdx.x;
    if (c0 + c >= F) continue;
    float s = 0.0f;
#pragma unroll
    for (int r = 0; r < 4; ++r) s += part[r][half * kTileF + c];
    sums[(int64_t)row_tile * 2 * F + half * F + c0 + c] = s;
  }
}

// Column sums over the row tiles: kJoinRows sums of every kJoinRows-th tile, and
// then those, each in order.  64 columns a workgroup.
constexpr int kJoinRows = 16;
template <class T>
struct BiasJoin {
  const float* sums;
  int64_t parts;
  T* dbg;
  T* dbu;
  int F, blocks;
  template <int kThreads>
  __device__ __forceinline__ void run(int block, char* lds) const {
    constexpr int kLanes = kThreads / 64, kEach = kJoinRows / kLanes;
    double (*part)[64] = reinterpret_cast<double (*)[64]>(lds);
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
    const int c = block * 64 + tx;
    double s[kEach] = {};
    if (c < 2 * F)
      for (int64_t k = ty; k < parts; k += kJoinRows)
#pragma unroll
        for (int j = 0; j < kEach; ++j)
          if (k + j * kLanes < parts) s[j] += sums[(k + j * kLanes) * 2 * F + c];
#pragma unroll
    for (int j = 0; j < kEach; ++j) part[ty + j * kLanes][tx] = s[j];
    __syncthreads();
    if (ty || c >= 2 * F) return;
    double all = s[0];
    for (int r = 1; r < kJoinRows; ++r) all += part[r][tx];
    (c < F ? dbg[c] : dbu[c - F]) = from_f32<T>((float)all);
  }
};
template <class T>
__global__ void __launch_bounds__(64 * kJoinRows) bias_join_kernel(const BiasJoin<T> join) {
  __shared__ __align__(16) char lds[kJoinRows * 64 * 8];
  join.template run<64 * kJoinRows>(blockIdx.x, lds);
}

// A bump allocator over the caller's workspace (or, with a null base, its size).
struct Scratch {
  char* base;
  size_t used = 0;
  char* take(int64_t bytes) {
    char* p = base ? base + used : nullptr;
    used += (size_t)round_up(bytes, 256);
    return p;
  }
};

// Scratch of the forward pass: operands whose rows do not start at multiples
// of 16 bytes get a padded copy, except for the rows kernel, which takes any.
// Room for it is asked for where the length of a row or the operands' addresses
// need it (8192 x 4096 -> 8192 in bf16: 201 MB, and none for aligned operands).
struct ForwardPlan {
  int64_t pitch;  // bytes of a padded row
  bool pad;
  GemmPlan gemm;
  char *x, *wg, *wu, *partial;
  size_t bytes;
};

ForwardPlan plan_forward(int dtype, int64_t M, int64_t D, int64_t F, bool aligned, char* ws) {
  const int64_t size = dtype_size(dtype);
  ForwardPlan f = {};
  f.pitch = round_up(D * size, 16);
  const bool odd = f.pitch != D * size;
  const GemmPlan& g = f.gemm = plan_gemm(M, 2 * F, D * size, size == 4, kTwoMatrices);
  f.pad = g.tile != 0 && (!aligned || odd);
  Scratch s{ws};
  if (f.pad) {
    f.x = s.take(M * f.pitch);
    f.wg = s.take(F * f.pitch);
    f.wu = s.take(F * f.pitch);
  }
  f.partial = s.take((int64_t)g.partial_bytes);
  f.bytes = s.used;
  return f;
}

// The products take dg and du in `dtype`, the matrix cores' operand type.  Their
// roundings are independent, so in a sum they grow as the sum itself does: at any
// size a 16-bit gradient is off by 2.35e-3 (bf16, 2-norm) where its own rounding
// makes 1.66e-3, and by less than 1% more than that when the products take what
// the rounding left as well, as two more ranges of K.  That is done where the
// backward pass takes little longer than its launches (M, D, F: us without and
// with, bf16 in a replayed graph: 64 x 512 -> 512 12.4 and 14.1, 256 x 64 -> 128 9.7
// and 12.6, 32 x 512 -> 2048 16.7 and 19.7); elsewhere it would cost up to two thirds
// of the products (1024 x 512 -> 512 19.3 and 25.4, 1024 x 4096 -> 512 29 and 48,
// and of long sums to dx 1 x 512 -> 8192 22.5 and 31.9).  D past 2^14 counts as that:
// few rows' passes are then bound by reading the weights.
constexpr int64_t kRestWork = (int64_t)1 << 26;
constexpr int64_t kRestColumns = 4096;
bool takes_rest(int64_t size, int64_t M, int64_t D, int64_t F) {
  constexpr int64_t kLongest = (int64_t)1 << 14;
  return size == 2 && F <= kRestColumns && M * F <= kRestWork / (D < kLongest ? D : kLongest);
}

struct BackwardPlan {
  int64_t fp;     // F rounded up to 16 bytes of elements
  bool rest;      // dg and du in two parts each
  int64_t pitch;  // bytes of a row of x and the weights
  bool pad;
  GemmPlan gx, gw;  // of the products to dx and to the weights' gradients
  PairPlan pair;    // and of both together
  char *dgu, *x, *wg, *wu, *sums, *partial;
  size_t partial_w;  // where the second of both has its partial sums
  size_t bytes;
};

BackwardPlan plan_backward(int dtype, int64_t M, int64_t D, int64_t F, bool aligned, char* ws) {
  const int64_t size = dtype_size(dtype);
  BackwardPlan b = {};
  b.fp = round_up(F, 16 / size);
  b.pitch = round_up(D * size, 16);
  b.pad = !aligned || b.pitch != D * size;
  Scratch s{ws};
  b.rest = takes_rest(size, M, D, F);
  const int64_t parts = b.rest ? 4 : 2;
  b.dgu = s.take(M * parts * b.fp * size);
  if (b.pad) {
    b.x = s.take(M * b.pitch);
    b.wg = s.take(F * b.pitch);
    b.wu = s.take(F * b.pitch);
  }
  b.sums = s.take(div_up(M, kTileM) * 2 * F * 4);
  const int64_t kx = parts * b.fp * size, kw = parts / 2 * M * size;
  b.gx = plan_gemm(M, D, kx, size == 4, kByKRows);
  b.gw = plan_gemm(2 * b.fp, D, kw, size == 4, kByKRows);
  b.pair = plan_pair(M, D, kx, 2 * b.fp, D, kw, size == 4, b.gx.us + b.gw.us);
  const size_t apart = b.gx.partial_bytes > b.gw.partial_bytes ? b.gx.partial_bytes
                                                               : b.gw.partial_bytes;
  b.partial_w = (size_t)round_up((int64_t)b.pair.partial_x, 256);
  const size_t both = b.partial_w + b.pair.partial_w;
  b.partial = s.take((int64_t)(apart > both ? apart : both));
  b.bytes = s.used;
  return b;
}

bool sizes_ok(int64_t M, int64_t D, int64_t F) { return M >= 0 && D > 0 && F > 0; }
// The products' operands within what the kernels index.
bool forward_fits(int dtype, int64_t M, int64_t D, int64_t F) {
  return M <= kMaxRows && D <= kMaxRows && F <= kMaxRows &&
         gemm_fits(M, 2 * F, round_up(D * dtype_size(dtype), 16));
}
bool backward_fits(int dtype, int64_t M, int64_t D, int64_t F) {
  const int64_t size = dtype_size(dtype), pitch = 2 * round_up(F, 16) * size;
  return forward_fits(dtype, M, D, F) && gemm_fits(M, D, pitch) && gemm_fits(2 * F, D, pitch) &&
         div_up(M, kTileM) * div_up(F + 8, kTileF) < ((int64_t)1 << 24);  // 2^32 threads
}

// Padded copies of x [M,D] and of the weights [F,D] (those that are not NULL).
int pad_operands(const void* x, const void* wg, const void* wu, char* xp, char* wgp, char* wup,
                 int64_t M, int64_t F, int64_t bytes, int64_t pitch, hipStream_t stream) {
  const PadArgs a = {{(const char*)x, (const char*)wg, (const char*)wu},
                     {xp, wgp, wup},
                     {x ? M : 0, wg ? F : 0, wu ? F : 0}};
  return pad_rows(a, bytes, pitch, stream);
}

bool drop_ok(const ppo_dropout* d) { return !d || (d->p >= 0.0 && d->p <= 1.0); }
Dropout drop_of(const ppo_dropout* d) {
  return d ? make_dropout(d->p, d->seed, d->seed_at, d->row_ids) : make_dropout(0.0, 0, nullptr, nullptr);
}

}  // namespace
}  // namespace ppo

using namespace ppo;

extern "C" size_t ppo_layer_gated_workspace_bytes(int dtype, int64_t M, int64_t D, int64_t F) {
  const bool aligned = take_aligned(dtype);
  if (!dtype_ok(dtype) || !sizes_ok(M, D, F) || !forward_fits(dtype, M, D, F) || M == 0) return 0;
  return plan_forward(dtype, M, D, F, aligned, nullptr).bytes;
}

extern "C" int ppo_layer_gated_forward(const void* x, const void* wg, const void* wu,
                                       const void* bg, const void* bu, int dtype, int64_t M,
                                       int64_t D, int64_t F, int activation,
                                       const ppo_dropout* drop, void* h, float* saved,
                                       void* workspace, size_t workspace_bytes,
                                       void* stream_ptr) {
  const bool promised = take_aligned(dtype);
  if (!dtype_ok(dtype) || !sizes_ok(M, D, F) || !drop_ok(drop) || activation < 0 ||
      activation > PPO_LAYER_GELU || !bg != !bu)
    return PPO_ERR_INVALID_ARG;
  if (M == 0) return PPO_OK;
  if (!x || !wg || !wu || !h || !aligned16(saved)) return PPO_ERR_INVALID_ARG;
  if (!forward_fits(dtype, M, D, F)) return PPO_ERR_TOO_LARGE;
  const bool aligned = aligned16(x) && aligned16(wg) && aligned16(wu);
  if (promised && !aligned) return PPO_ERR_INVALID_ARG;
  const ForwardPlan f = plan_forward(dtype, M, D, F, aligned, (char*)workspace);
  const size_t need = plan_forward(dtype, M, D, F, promised, nullptr).bytes;
  if (need && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return PPO_ERR_WORKSPACE;
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_ptr);
  return with_dtype(dtype, [&](auto zero) {
    using T = decltype(zero);
    GemmArgs a = {};
    a.x = (const char*)x;
    a.w0 = (const char*)wg;
    a.w1 = (const char*)wu;
    a.xpitch = a.wpitch = a.kbytes = D * (int64_t)sizeof(T);
    a.M = (int)M;
    a.N = (int)F;
    if (f.pad) {
      const int st = pad_operands(x, wg, wu, f.x, f.wg, f.wu, M, F, D * (int64_t)sizeof(T), f.pitch,
                                  stream);
      if (st) return st;
      a.x = f.x;
      a.w0 = f.wg;
      a.w1 = f.wu;
      a.xpitch = a.wpitch = a.kbytes = f.pitch;
    }
    const int F4 = (int)round_up(F, 4);
    const GatedEpi<T> epi = {(const T*)bg, (const T*)bu, (T*)h, saved, M * F4, (int)F, F4,
                             activation, drop_of(drop)};
    return launch_gemm<T>(a, epi, f.gemm, f.partial, stream);
  });
}

extern "C" size_t ppo_layer_gated_backward_workspace_bytes(int dtype, int64_t M, int64_t D,
                                                           int64_t F) {
  const bool aligned = take_aligned(dtype);
  if (!dtype_ok(dtype) || !sizes_ok(M, D, F) || !backward_fits(dtype, M, D, F)) return 0;
  return plan_backward(dtype, M, D, F, aligned, nullptr).bytes;
}

extern "C" int ppo_layer_gated_backward(const void* dh, const void* x, const void* wg,
                                        const void* wu, const float* saved, int dtype, int64_t M,
                                        int64_t D, int64_t F, int activation,
                                        const ppo_dropout* drop, void* dx, void* dwg, void* dwu,
                                        void* dbg, void* dbu, void* workspace,
                                        size_t workspace_bytes, void* stream_ptr) {
  const bool promised = take_aligned(dtype);
  if (!dtype_ok(dtype) || !sizes_ok(M, D, F) || !drop_ok(drop) || activation < 0 ||
      activation > PPO_LAYER_GELU || !dwg != !dwu || !dbg != !dbu)
    return PPO_ERR_INVALID_ARG;
  if (M == 0) return PPO_ERR_INVALID_ARG;  // (the sums over no rows are the caller's zeros)
  if (!dh || !saved || !aligned16(saved) || (dwg && !x) || (dx && (!wg || !wu)))
    return PPO_ERR_INVALID_ARG;
  if (!backward_fits(dtype, M, D, F)) return PPO_ERR_TOO_LARGE;
  const bool aligned = aligned16(x) && aligned16(wg) && aligned16(wu);
  if (promised && !aligned) return PPO_ERR_INVALID_ARG;
  const BackwardPlan b = plan_backward(dtype, M, D, F, aligned, (char*)workspace);
  if (!workspace || workspace_bytes < plan_backward(dtype, M, D, F, promised, nullptr).bytes ||
      !aligned16(workspace))
    return PPO_ERR_WORKSPACE;
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_ptr);
  return with_dtype(dtype, [&](auto zero) {
    using T = decltype(zero);
    const int64_t size = sizeof(T), F4 = round_up(F, 4);
    int st;
    if (!dx && !dwg && !dbg) return (int)PPO_OK;
    hipLaunchKernelGGL((gated_grad_kernel<T>),
                       dim3((unsigned)(div_up(M, kTileM) * div_up(b.fp, kTileF))), dim3(256), 0,
                       stream, (const T*)dh, saved, M, (int)F, (int)F4, activation,
                       drop_of(drop), (T*)b.dgu, b.fp, (b.rest ? 4 : 2) * b.fp, b.rest,
                       dbg ? (float*)b.sums : nullptr);
    if ((st = last_launch_status())) return st;
    const bool pair = dx && dwg && b.pair.tile;
    // The join of few row tiles rides along with the pair (a step of 256 x 128 -> 256
    // 25.9 -> 24.5 us, 1000 x 1023 -> 1365 70 -> 67, 2048 x 4096 -> 256 71 -> 65); of many, it
    // would be the last to end (4096 x 1024 -> 2048 156 -> 166).
    const bool along = pair && div_up(M, kTileM) <= 128;
    BiasJoin<T> join = {(const float*)b.sums, div_up(M, kTileM), (T*)dbg, (T*)dbu, (int)F,
                              dbg ? (int)div_up(2 * F, 64) : 0};
    if (dbg && !along) {
      hipLaunchKernelGGL((bias_join_kernel<T>), dim3((unsigned)join.blocks), dim3(64 * kJoinRows),
                         0, stream, join);
      if ((st = last_launch_status())) return st;
      join.blocks = 0;
    }
    if (!dx && !dwg) return (int)PPO_OK;  // (the biases' gradients alone: nothing to multiply)
    if (b.pad) {
      st = pad_operands(dwg ? x : nullptr, dx ? wg : nullptr, dx ? wu : nullptr, b.x, b.wg, b.wu, M,
                        F, D * size, b.pitch, stream);
      if (st) return st;
    }
    GemmArgs ax = {};
    ax.N = (int)D;
    ax.wpitch = b.pad ? b.pitch : D * size;
    ax.x = b.dgu;
    ax.xpitch = (b.rest ? 4 : 2) * b.fp * size;
    GemmArgs aw = ax;
    // dx = [dg | du] [wg; wu], the weights as they lie: k-rows of D columns
    ax.w0 = b.pad ? b.wg : (const char*)wg;
    ax.w1 = b.pad ? b.wu : (const char*)wu;
    ax.M = (int)M;
    ax.kbytes = ax.x_range = b.fp * size;
    ax.k = F;
    ax.ranges = b.rest ? 4 : 2;
    const StoreEpi<T> ex = {(T*)dx, nullptr, (int)M, (int)M, (int)D};
    // [dwg; dwu] = [dg | du]^T x: both operands by their rows m
    aw.w0 = aw.w1 = b.pad ? b.x : (const char*)x;
    aw.M = (int)(2 * b.fp);
    aw.k = M;
    aw.ranges = b.rest ? 2 : 1;
    aw.x_range = 2 * b.fp * size;
    const StoreEpi<T> ew = {(T*)dwg, (T*)dwu, (int)F, (int)b.fp, (int)D};
    if (pair) {
      ax.partial = b.pair.splits_x > 1 ? b.partial : nullptr;
      aw.partial = b.pair.splits_w > 1 ? b.partial + b.partial_w : nullptr;
      return launch_pair<T>(ax, aw, ex, ew, b.pair, join, stream);
    }
    if (dx && (st = launch_gemm<T, false, true>(ax, ex, b.gx, b.partial, stream))) return st;
    if (dwg && (st = launch_gemm<T, true, true>(aw, ew, b.gw, b.partial, stream))) return st;
    return (int)PPO_OK;
  });
}
