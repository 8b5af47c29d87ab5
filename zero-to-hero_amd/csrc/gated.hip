// The gated feed-forward block and its backward pass:
//   g = x wg^T + bg,  u = x wu^T + bu,  h = dropout(act(g) * u)
//   dh' = dropout(dh),  du = dh' act(g),  dg = dh' u act'(g)
//   dx = dg wg + du wu,  dwg = dg^T x,  dwu = du^T x,  dbg = sum dg, dbu = sum du
// Forward: one product over both weight matrices (gemm_tile.hpp; a wave holds
// the gate's and the up projection's sums of the same elements, so g and u
// never leave registers unless the backward pass wants them).  Backward: one
// elementwise pass forms dg and du in both orders, then two products.
#include "gemm_tile.hpp"

namespace ppo {
namespace {

template <class T>
struct GatedEpi {
  static constexpr bool kGated = true;
  static constexpr int kBatch = 1;
  const T* bg;
  const T* bu;
  T* h;
  float* saved;   // [2][M][F4] or null
  int64_t half;   // M * F4
  int F, F4, act;
  Dropout drop;

  struct Cols { float g[4], u[4]; };
  typedef int64_t Row;
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
  __device__ __forceinline__ void operator()(int m, int n, const Cols& cols, Row id, v4f g,
                                             v4f u) const {
    const int count = F - n;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      g[i] += cols.g[i];
      u[i] += cols.u[i];
    }
    if (saved) {
      float* s = saved + (int64_t)m * F4 + n;
      *reinterpret_cast<v4f*>(s) = g;
      *reinterpret_cast<v4f*>(s + half) = u;
    }
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = activate(act, g[i]) * u[i];
    if (drop.mode)
      drop4(drop, dropout_seed(drop), (uint64_t)id, (uint32_t)n >> 2, v);
    store4(h + (int64_t)m * F + n, v, count, (F & 3) == 0);
  }
};

// Plain store of the sums, rows from `split` on to a second output.
template <class T>
struct StoreEpi {
  static constexpr bool kGated = false;
  static constexpr int kBatch = 4;
  T* out0;
  T* out1;
  int split, N;
  struct Cols {};
  struct Row {};
  __device__ __forceinline__ Cols columns(int) const { return {}; }
  __device__ __forceinline__ Row row(int) const { return {}; }
  __device__ __forceinline__ void operator()(int m, int n, Cols, Row, v4f c) const {
    T* row = m < split ? out0 + (int64_t)m * N : out1 + (int64_t)(m - split) * N;
    const float v[4] = {c[0], c[1], c[2], c[3]};
    store4(row + n, v, N - n, (N & 3) == 0);
  }
};

// [rows][cols] -> the same rows at a pitch, zeros behind each row.
template <class T>
__global__ void __launch_bounds__(256) pad_rows_kernel(const T* in, int64_t rows, int cols, T* out,
                                                       int pitch) {
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x)
    for (int c = threadIdx.x; c < pitch; c += 256)
      out[r * pitch + c] = c < cols ? in[r * cols + c] : from_f32<T>(0.0f);
}

constexpr int kTr = 64;  // edge of the tiles that are transposed through LDS

// in [rows][cols] -> out[c][r] at out + c * pitch + r, zeros for r in
// [rows, rows4): the k-contiguous form of an operand whose rows are k.
template <class T>
__global__ void __launch_bounds__(256) transpose_kernel(const T* in, int64_t rows, int cols, T* out,
                                                        int64_t pitch, int64_t padded) {
  __shared__ T tile[kTr][kTr + 16 / sizeof(T) / 2 + 1];
  const int64_t r0 = (int64_t)blockIdx.x * kTr;
  const int c0 = blockIdx.y * kTr;
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
  for (int i = ty; i < kTr; i += 4)
    tile[i][tx] = r0 + i < rows && c0 + tx < cols ? in[(r0 + i) * cols + c0 + tx] : from_f32<T>(0.0f);
  __syncthreads();
  for (int i = ty; i < kTr; i += 4)
    if (c0 + i < cols && r0 + tx < padded) out[(c0 + i) * pitch + r0 + tx] = tile[tx][i];
}

// dg and du of a 64 x 64 tile, from dh and the saved g and u: rows for dx
// (dgu [M][2 Fp], dg then du) and, transposed, rows for the weights' gradients
// (dgu_t [2 F][Mp]); with `sums`, the tile's column sums for the biases
// ([row tiles][2 F], joined in order by bias_join_kernel).
template <class T>
__global__ void __launch_bounds__(256) gated_grad_kernel(const T* dh, const float* saved, int64_t M,
                                                         int F, int F4, int act, Dropout drop,
                                                         T* dgu, int64_t fp, T* dgu_t, int64_t mp,
                                                         float* sums) {
  __shared__ float tile[2][kTr][kTr + 1];
  const int64_t r0 = (int64_t)blockIdx.x * kTr;
  const int c0 = blockIdx.y * kTr;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;  // four columns, rows ty + 16 i
  const int n = c0 + tx * 4;
  const uint64_t seed = drop.mode ? dropout_seed(drop) : 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = ty + 16 * i;
    const int64_t m = r0 + r;
    float dg[4] = {0, 0, 0, 0}, du[4] = {0, 0, 0, 0};
    if (m < M && n < F) {
      const v4f g = *reinterpret_cast<const v4f*>(saved + m * F4 + n);
      const v4f u = *reinterpret_cast<const v4f*>(saved + (M + m) * F4 + n);
      float d[4] = {0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (n + k < F) d[k] = to_f32(dh[m * F + n + k]);
      if (drop.mode) drop4(drop, seed, drop.rows ? drop.rows[m] : m, (uint32_t)n >> 2, d);
#pragma unroll
      for (int k = 0; k < 4; ++k)
        if (n + k < F) {
          float a, da;
          activate_grad(act, g[k], a, da);
          du[k] = d[k] * a;
          dg[k] = d[k] * u[k] * da;
        }
    }
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      tile[0][r][tx * 4 + k] = dg[k];
      tile[1][r][tx * 4 + k] = du[k];
    }
    if (dgu && m < M && n < fp) {  // (columns F..fp are zeros)
      store4(dgu + m * 2 * fp + n, dg, 4, true);
      store4(dgu + m * 2 * fp + fp + n, du, 4, true);
    }
  }
  __syncthreads();
  if (dgu_t) {
    const int cx = threadIdx.x & 15, cy = threadIdx.x >> 4;  // four rows m, columns cy + 16 i
    const int64_t m = r0 + cx * 4;
    for (int i = 0; i < 8; ++i) {
      const int half = i >> 2, c = cy + 16 * (i & 3);
      if (c0 + c >= F || m >= mp) continue;
      const float v[4] = {tile[half][cx * 4][c], tile[half][cx * 4 + 1][c],
                          tile[half][cx * 4 + 2][c], tile[half][cx * 4 + 3][c]};
      store4(dgu_t + ((int64_t)half * F + c0 + c) * mp + m, v, 4, true);
    }
  }
  if (sums && threadIdx.x < 2 * kTr) {
    const int half = threadIdx.x / kTr, c = threadIdx.x % kTr;
    if (c0 + c < F) {
      float s = 0.0f;
      for (int r = 0; r < kTr; ++r) s += tile[half][r][c];
      sums[(int64_t)blockIdx.x * 2 * F + half * F + c0 + c] = s;
    }
  }
}

// Column sums over the row tiles, in order.
template <class T>
__global__ void __launch_bounds__(256) bias_join_kernel(const float* sums, int64_t parts, int F,
                                                        T* dbg, T* dbu) {
  __shared__ double part[4][64];
  const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
  const int c = blockIdx.x * 64 + tx;
  double s = 0.0;
  if (c < 2 * F)
    for (int64_t k = ty; k < parts; k += 4) s += sums[k * 2 * F + c];
  part[ty][tx] = s;
  __syncthreads();
  if (ty || c >= 2 * F) return;
  const float v = (float)((part[0][tx] + part[1][tx]) + (part[2][tx] + part[3][tx]));
  (c < F ? dbg[c] : dbu[c - F]) = from_f32<T>(v);
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
struct ForwardPlan {
  int64_t pitch;  // bytes of a padded row
  bool pad;
  char *x, *wg, *wu, *partial;
  size_t bytes;
};

ForwardPlan plan_forward(int dtype, int64_t M, int64_t D, int64_t F, bool aligned, char* ws) {
  const int64_t size = dtype_size(dtype);
  ForwardPlan f = {};
  f.pitch = round_up(D * size, 16);
  const GemmPlan g = plan_gemm(M, 2 * F, f.pitch);
  f.pad = g.tile != 0 && (!aligned || f.pitch != D * size);
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

struct BackwardPlan {
  int64_t fp, mp;  // F and M rounded up to 16 bytes of elements
  char *dgu, *dgu_t, *w_t, *x_t, *sums, *partial;
  size_t bytes;
};

BackwardPlan plan_backward(int dtype, int64_t M, int64_t D, int64_t F, char* ws) {
  const int64_t size = dtype_size(dtype);
  BackwardPlan b = {};
  b.fp = round_up(F, 16 / size);
  b.mp = round_up(M, 16 / size);
  Scratch s{ws};
  b.dgu = s.take(M * 2 * b.fp * size);
  b.dgu_t = s.take(2 * F * b.mp * size);
  b.w_t = s.take(D * 2 * b.fp * size);
  b.x_t = s.take(D * b.mp * size);
  b.sums = s.take(div_up(M, kTr) * 2 * F * 4);
  const GemmPlan gx = plan_gemm(M, D, 2 * b.fp * size), gw = plan_gemm(2 * F, D, b.mp * size);
  b.partial = s.take((int64_t)(gx.partial_bytes > gw.partial_bytes ? gx.partial_bytes
                                                                   : gw.partial_bytes));
  b.bytes = s.used;
  return b;
}

bool sizes_ok(int64_t M, int64_t D, int64_t F) { return M >= 0 && D > 0 && F > 0; }
// The products' operands within what the kernels index.
bool forward_fits(int dtype, int64_t M, int64_t D, int64_t F) {
  const int64_t lim = (int64_t)1 << 28;
  return M < lim && D < lim && F < lim && gemm_fits(M, 2 * F, round_up(D * dtype_size(dtype), 16));
}
bool backward_fits(int dtype, int64_t M, int64_t D, int64_t F) {
  const int64_t size = dtype_size(dtype);
  return forward_fits(dtype, M, D, F) && gemm_fits(M, D, 2 * round_up(F, 16) * size) &&
         gemm_fits(2 * F, D, round_up(M, 16) * size);
}

template <class T>
void pad_rows(const void* in, int64_t rows, int64_t cols, char* out, int64_t pitch,
              hipStream_t stream) {
  hipLaunchKernelGGL((pad_rows_kernel<T>), dim3((unsigned)(rows < 65536 ? rows : 65536)), dim3(256),
                     0, stream, (const T*)in, rows, (int)cols, (T*)out, (int)(pitch / sizeof(T)));
}

template <class T>
void transpose(const void* in, int64_t rows, int64_t cols, char* out, int64_t pitch,
               int64_t padded, hipStream_t stream) {
  hipLaunchKernelGGL((transpose_kernel<T>),
                     dim3((unsigned)div_up(padded, kTr), (unsigned)div_up(cols, kTr)), dim3(256), 0,
                     stream, (const T*)in, rows, (int)cols, (T*)out, pitch, padded);
}

bool drop_ok(const ppo_dropout* d) { return !d || (d->p >= 0.0 && d->p <= 1.0); }
Dropout drop_of(const ppo_dropout* d) {
  return d ? make_dropout(d->p, d->seed, d->seed_at, d->row_ids) : make_dropout(0.0, 0, nullptr, nullptr);
}

}  // namespace
}  // namespace ppo

using namespace ppo;

extern "C" size_t ppo_layer_gated_workspace_bytes(int dtype, int64_t M, int64_t D, int64_t F) {
  if (!dtype_ok(dtype) || !sizes_ok(M, D, F) || !forward_fits(dtype, M, D, F) || M == 0) return 0;
  return plan_forward(dtype, M, D, F, false, nullptr).bytes;
}

extern "C" int ppo_layer_gated_forward(const void* x, const void* wg, const void* wu,
                                       const void* bg, const void* bu, int dtype, int64_t M,
                                       int64_t D, int64_t F, int activation,
                                       const ppo_dropout* drop, void* h, float* saved,
                                       void* workspace, size_t workspace_bytes,
                                       void* stream_ptr) {
  if (!dtype_ok(dtype) || !sizes_ok(M, D, F) || !drop_ok(drop) || activation < 0 ||
      activation > PPO_LAYER_GELU || !bg != !bu)
    return PPO_ERR_INVALID_ARG;
  if (M == 0) return PPO_OK;
  if (!x || !wg || !wu || !h) return PPO_ERR_INVALID_ARG;
  if (!forward_fits(dtype, M, D, F)) return PPO_ERR_TOO_LARGE;
  const bool aligned = aligned16(x) && aligned16(wg) && aligned16(wu);
  const ForwardPlan f = plan_forward(dtype, M, D, F, aligned, (char*)workspace);
  const size_t need = ppo_layer_gated_workspace_bytes(dtype, M, D, F);
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
      pad_rows<T>(x, M, D, f.x, f.pitch, stream);
      pad_rows<T>(wg, F, D, f.wg, f.pitch, stream);
      pad_rows<T>(wu, F, D, f.wu, f.pitch, stream);
      a.x = f.x;
      a.w0 = f.wg;
      a.w1 = f.wu;
      a.xpitch = a.wpitch = a.kbytes = f.pitch;
    }
    const int F4 = (int)round_up(F, 4);
    const GatedEpi<T> epi = {(const T*)bg, (const T*)bu, (T*)h, saved, M * F4, (int)F, F4,
                             activation, drop_of(drop)};
    return launch_gemm<T>(a, epi, f.partial, stream);
  });
}

extern "C" size_t ppo_layer_gated_backward_workspace_bytes(int dtype, int64_t M, int64_t D,
                                                           int64_t F) {
  if (!dtype_ok(dtype) || !sizes_ok(M, D, F) || !backward_fits(dtype, M, D, F)) return 0;
  return plan_backward(dtype, M, D, F, nullptr).bytes;
}

extern "C" int ppo_layer_gated_backward(const void* dh, const void* x, const void* wg,
                                        const void* wu, const float* saved, int dtype, int64_t M,
                                        int64_t D, int64_t F, int activation,
                                        const ppo_dropout* drop, void* dx, void* dwg, void* dwu,
                                        void* dbg, void* dbu, void* workspace,
                                        size_t workspace_bytes, void* stream_ptr) {
  if (!dtype_ok(dtype) || !sizes_ok(M, D, F) || !drop_ok(drop) || activation < 0 ||
      activation > PPO_LAYER_GELU || !dwg != !dwu || !dbg != !dbu)
    return PPO_ERR_INVALID_ARG;
  if (M == 0) return PPO_ERR_INVALID_ARG;  // (the sums over no rows are the caller's zeros)
  if (!dh || !saved || (dwg && !x) || (dx && (!wg || !wu))) return PPO_ERR_INVALID_ARG;
  if (!backward_fits(dtype, M, D, F)) return PPO_ERR_TOO_LARGE;
  const BackwardPlan b = plan_backward(dtype, M, D, F, (char*)workspace);
  if (!workspace || workspace_bytes < b.bytes || !aligned16(workspace)) return PPO_ERR_WORKSPACE;
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_ptr);
  return with_dtype(dtype, [&](auto zero) {
    using T = decltype(zero);
    const int64_t size = sizeof(T), F4 = round_up(F, 4);
    int st;
    if (!dx && !dwg && !dbg) return (int)PPO_OK;
    hipLaunchKernelGGL((gated_grad_kernel<T>),
                       dim3((unsigned)div_up(M, kTr), (unsigned)div_up(F, kTr)), dim3(256), 0,
                       stream, (const T*)dh, saved, M, (int)F, (int)F4, activation, drop_of(drop),
                       dx ? (T*)b.dgu : nullptr, b.fp, dwg ? (T*)b.dgu_t : nullptr, b.mp,
                       dbg ? (float*)b.sums : nullptr);
    if ((st = last_launch_status())) return st;
    if (dbg) {
      hipLaunchKernelGGL((bias_join_kernel<T>), dim3((unsigned)div_up(2 * F, 64)), dim3(256), 0,
                         stream, (const float*)b.sums, div_up(M, kTr), (int)F, (T*)dbg, (T*)dbu);
      if ((st = last_launch_status())) return st;
    }
    if (dx) {
      transpose<T>(wg, F, D, b.w_t, 2 * b.fp, b.fp, stream);
      transpose<T>(wu, F, D, b.w_t + b.fp * size, 2 * b.fp, b.fp, stream);
      GemmArgs a = {};
      a.x = b.dgu;
      a.w0 = b.w_t;
      a.xpitch = a.wpitch = a.kbytes = 2 * b.fp * size;
      a.M = (int)M;
      a.N = (int)D;
      const StoreEpi<T> epi = {(T*)dx, nullptr, (int)M, (int)D};
      if ((st = launch_gemm<T>(a, epi, b.partial, stream))) return st;
    }
    if (dwg) {
      transpose<T>(x, M, D, b.x_t, b.mp, b.mp, stream);
      GemmArgs a = {};
      a.x = b.dgu_t;
      a.w0 = b.x_t;
      a.xpitch = a.wpitch = a.kbytes = b.mp * size;
      a.M = (int)(2 * F);
      a.N = (int)D;
      const StoreEpi<T> epi = {(T*)dwg, (T*)dwu, (int)F, (int)D};
      if ((st = launch_gemm<T>(a, epi, b.partial, stream))) return st;
    }
    return (int)PPO_OK;
  });
}
