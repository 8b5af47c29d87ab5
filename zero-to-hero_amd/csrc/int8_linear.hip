// 8-bit products: rows quantised with one scale each, and
//   out[m,n] = (sum_k xq[m,k] wq[n,k]) xs[m] ws[n] + bias[n]
// with the sum in int32 on the matrix cores (gemm_tile.hpp).
#include "gemm_tile.hpp"

namespace ppo {
namespace {

template <class T>
struct Int8Epi {
  static constexpr bool kGated = false;
  static constexpr int kBatch = 4;
  const float* xs;
  const float* ws;
  const T* bias;
  T* out;
  int N;
  struct Cols { float scale[4], bias[4]; };
  typedef float Row;
  __device__ __forceinline__ Cols columns(int n) const {
    Cols c;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int at = min(n + i, N - 1);
      c.scale[i] = ws[at];
      c.bias[i] = bias ? to_f32(bias[at]) : 0.0f;
    }
    return c;
  }
  __device__ __forceinline__ Row row(int m) const { return xs[m]; }
  __device__ __forceinline__ void operator()(int m, int n, const Cols& cols, Row s, v4i c) const {
    float v[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      v[i] = (float)c[i] * s * cols.scale[i];
      if (bias) v[i] += cols.bias[i];  // (without one, a zero keeps its sign)
    }
    store4(out + (int64_t)m * N + n, v, N - n, (N & 3) == 0);
  }
};

// Rows of int8 at a pitch, zeros behind each row.
__global__ void __launch_bounds__(256) pad_int8_kernel(const int8_t* in, int64_t rows, int64_t cols,
                                                       int8_t* out, int64_t pitch) {
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x)
    for (int64_t c = threadIdx.x; c < pitch; c += 256)
      out[r * pitch + c] = c < cols ? in[r * cols + c] : 0;
}

// max |x| as its bits: ordered as integers, an infinity above every finite
// value and a NaN above that, so a row that is not finite shows.
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

__device__ __forceinline__ float row_scale(uint32_t top) {
  return top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __uint_as_float(top) / 127.0f;
}

// (a scale that is subnormal leaves quotients past 127: they stay within)
__device__ __forceinline__ int quantize(float x, float scale, bool live) {
  return live ? (int)fminf(fmaxf(rintf(x / scale), -127.0f), 127.0f) : 0;
}

// One workgroup of kThreads a row: its maximum, then its values from a second
// read (in cache).
template <class T, int kThreads>
__global__ void __launch_bounds__(kThreads) quantize_rows_kernel(const T* x, int64_t rows,
                                                                 int64_t cols, int8_t* q,
                                                                 int64_t pitch, float* scale) {
  __shared__ uint32_t tops[kThreads / 64];
  const int64_t r = blockIdx.x;
  const T* xr = x + r * cols;
  uint32_t top = 0;
  for (int64_t c = threadIdx.x; c < cols; c += kThreads) top = max(top, magnitude(to_f32(xr[c])));
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
  if constexpr (kThreads > 64) {
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) top = max(top, tops[i]);
  }
  const float s = row_scale(top);
  const bool live = s > 0.0f;
  for (int64_t c = threadIdx.x; c < pitch; c += kThreads)
    q[r * pitch + c] = (int8_t)(c < cols ? quantize(to_f32(xr[c]), s, live) : 0);
  if (threadIdx.x == 0) scale[r] = s;
}

template <class T>
int launch_quantize(const void* x, int64_t rows, int64_t cols, int8_t* q, int64_t pitch,
                    float* scale, hipStream_t stream) {
  hipLaunchKernelGGL((quantize_rows_kernel<T, 256>), dim3((unsigned)rows), dim3(256), 0, stream,
                     (const T*)x, rows, cols, q, pitch, scale);
  return last_launch_status();
}

struct Int8Plan {
  int64_t pitch;
  bool pad_x, pad_w;
  char *xq, *xs, *wq, *partial;
  size_t bytes;
};

Int8Plan plan_int8(int64_t M, int64_t N, int64_t K, bool quantize, bool ax, bool aw, char* ws) {
  Int8Plan p = {};
  p.pitch = round_up(K, 16);
  const GemmPlan g = plan_gemm(M, N, p.pitch);
  const bool odd = p.pitch != K;
  p.pad_x = !quantize && g.tile != 0 && (odd || !ax);
  p.pad_w = g.tile != 0 && (odd || !aw);
  size_t used = 0;
  auto take = [&](int64_t bytes) {
    char* at = ws ? ws + used : nullptr;
    used += (size_t)round_up(bytes, 256);
    return at;
  };
  if (quantize) p.xs = take(M * 4);
  if (quantize || p.pad_x) p.xq = take(M * p.pitch);
  if (p.pad_w) p.wq = take(N * p.pitch);
  p.partial = take((int64_t)g.partial_bytes);
  p.bytes = used;
  return p;
}

constexpr int64_t kMaxInt8K = (int64_t)1 << 17;  // 127 * 127 * K stays below 2^31

}  // namespace
}  // namespace ppo

using namespace ppo;

extern "C" int ppo_layer_quantize_rows(const void* x, int dtype, int64_t rows, int64_t cols,
                                       int8_t* q, float* scale, void* stream_ptr) {
  if (!dtype_ok(dtype) || rows < 0 || cols <= 0) return PPO_ERR_INVALID_ARG;
  if (rows == 0) return PPO_OK;
  if (!x || !q || !scale) return PPO_ERR_INVALID_ARG;
  if (rows >= ((int64_t)1 << 31) || cols > ((int64_t)1 << 40)) return PPO_ERR_TOO_LARGE;
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_ptr);
  return with_dtype(dtype, [&](auto zero) {
    return launch_quantize<decltype(zero)>(x, rows, cols, q, cols, scale, stream);
  });
}

extern "C" size_t ppo_layer_int8_linear_workspace_bytes(int64_t M, int64_t N, int64_t K,
                                                        int quantize) {
  if (M <= 0 || N <= 0 || K <= 0 || K > kMaxInt8K || !gemm_fits(M, N, round_up(K, 16))) return 0;
  return plan_int8(M, N, K, quantize != 0, false, false, nullptr).bytes;
}

extern "C" int ppo_layer_int8_linear(const void* x, const int8_t* xq, const float* xs,
                                     const int8_t* wq, const float* ws, const void* bias,
                                     int dtype, int64_t M, int64_t N, int64_t K, void* out,
                                     void* workspace, size_t workspace_bytes, void* stream_ptr) {
  if (!dtype_ok(dtype) || M < 0 || N <= 0 || K <= 0) return PPO_ERR_INVALID_ARG;
  if (M == 0) return PPO_OK;
  if (!wq || !ws || !out || (!x && (!xq || !xs))) return PPO_ERR_INVALID_ARG;
  if (K > kMaxInt8K || !gemm_fits(M, N, round_up(K, 16))) return PPO_ERR_TOO_LARGE;
  const Int8Plan p =
      plan_int8(M, N, K, x != nullptr, aligned16(xq), aligned16(wq), (char*)workspace);
  const size_t need = ppo_layer_int8_linear_workspace_bytes(M, N, K, x != nullptr);
  if (need && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return PPO_ERR_WORKSPACE;
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_ptr);
  return with_dtype(dtype, [&](auto zero) {
    using T = decltype(zero);
    GemmArgs a = {};
    a.x = (const char*)xq;
    a.w0 = (const char*)wq;
    a.xpitch = a.wpitch = a.kbytes = K;
    a.M = (int)M;
    a.N = (int)N;
    int st = PPO_OK;
    if (x) {
      st = launch_quantize<T>(x, M, K, (int8_t*)p.xq, p.pitch, (float*)p.xs, stream);
      a.x = p.xq;
      a.xpitch = p.pitch;
    } else if (p.pad_x) {
      hipLaunchKernelGGL(pad_int8_kernel, dim3((unsigned)(M < 65536 ? M : 65536)), dim3(256), 0,
                         stream, xq, M, K, (int8_t*)p.xq, p.pitch);
      a.x = p.xq;
      a.xpitch = p.pitch;
      st = last_launch_status();
    }
    if (st) return st;
    if (p.pad_w) {
      hipLaunchKernelGGL(pad_int8_kernel, dim3((unsigned)(N < 65536 ? N : 65536)), dim3(256), 0,
                         stream, wq, N, K, (int8_t*)p.wq, p.pitch);
      a.w0 = p.wq;
      a.wpitch = p.pitch;
      if ((st = last_launch_status())) return st;
    }
    // the tile kernel's rows end on 16 bytes (zeros behind K), the rows kernel's on K
    if (plan_gemm(M, N, p.pitch).tile) a.kbytes = p.pitch;
    const Int8Epi<T> epi = {x ? (const float*)p.xs : xs, ws, (const T*)bias, (T*)out, (int)N};
    return launch_gemm<int8_t>(a, epi, p.partial, stream);
  });
}
