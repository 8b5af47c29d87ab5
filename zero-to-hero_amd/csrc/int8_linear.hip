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
  static constexpr bool kRows = true;
  struct Cols {
    float scale[4], bias[4];
    __device__ __forceinline__ void arrived() {
#pragma unroll
      for (int i = 0; i < 4; ++i) asm volatile("" : "+v"(scale[i]), "+v"(bias[i]));
    }
  };
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
  template <int B>
  __device__ __forceinline__ void apply(int n, const Cols& cols, const int (&m)[B],
                                        const bool (&live)[B], const Row (&s)[B],
                                        const v4i (&c)[B]) const {
#pragma unroll
    for (int b = 0; b < B; ++b) {
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[i] = (float)c[b][i] * s[b] * cols.scale[i];
        if (bias) v[i] += cols.bias[i];  // (without one, a zero keeps its sign)
      }
      if (live[b]) store4<true>(out + (int64_t)m[b] * N + n, v, N - n, rows_of_fours(out, N));
    }
  }
};

// max |x| as its bits: ordered as integers, an infinity above every finite
// value and a NaN above that, so a row that is not finite shows.
__device__ __forceinline__ uint32_t magnitude(float x) { return __float_as_uint(x) & 0x7fffffffu; }

__device__ __forceinline__ float row_scale(uint32_t top) {
  return top >= 0x7f800000u ? __uint_as_float(0x7fc00000u) : __uint_as_float(top) * (1.0f / 127.0f);
}

// x / scale to the nearest integer.  The product with 1 / scale is off by at
// most 1.5e-5 (two roundings of a value up to 127), so it settles all but the
// quotients within 4e-5 of a tie, one in 12000, which are divided.
struct Quantizer {
  float scale, inverse;
  bool live, direct;  // direct: 1 / scale is no number to multiply by
  __device__ __forceinline__ explicit Quantizer(float s)
      : scale(s), inverse(1.0f / s), live(s > 0.0f), direct(s < 1e-36f) {}
  __device__ __forceinline__ int operator()(float x) const {
    if (!live) return 0;
    const float t = x * inverse;
    float k = rintf(t);
    // (a scale that is subnormal leaves quotients past 127: they stay within)
    if (direct || fabsf(t - k) > 0.49996f) k = fminf(fmaxf(rintf(x / scale), -127.0f), 127.0f);
    return (int)k;
  }
};

// The 16 / sizeof(T) elements of a chunk, zeros behind the row's end.
template <class T>
struct Chunk {
  static constexpr int kN = kPer16<T>;
  T v[kN];
  __device__ __forceinline__ void load(const T* row, int64_t c, int64_t cols) {
    const int64_t left = cols - c * kN;
    if (left >= kN) {
      *reinterpret_cast<v4i*>(v) = *reinterpret_cast<const v4i_any*>(row + c * kN);
    } else {
#pragma unroll
      for (int i = 0; i < kN; ++i) v[i] = i < left ? row[c * kN + i] : from_f32<T>(0.0f);
    }
  }
  __device__ __forceinline__ uint32_t top() const {
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kN; ++i) m = max(m, magnitude(to_f32(v[i])));
    return m;
  }
  // (`pitch` - columns of the padded row, zeros behind cols - is reached by
  // chunks of zeros)
  __device__ __forceinline__ void store(int8_t* row, int64_t c, int64_t pitch,
                                        const Quantizer& q) const {
    struct __attribute__((aligned(1))) Bytes { int8_t b[kN]; } out;
#pragma unroll
    for (int i = 0; i < kN; ++i) out.b[i] = (int8_t)q(to_f32(v[i]));
    const int64_t left = pitch - c * kN;
    if (left >= kN) {
      typedef int __attribute__((aligned(1), may_alias)) int_any;
#pragma unroll
      for (int i = 0; i < kN / 4; ++i)
        reinterpret_cast<int_any*>(row + c * kN)[i] = reinterpret_cast<const int_any*>(out.b)[i];
    } else {
#pragma unroll
      for (int i = 0; i < kN; ++i)
        if (i < left) row[c * kN + i] = out.b[i];
    }
  }
};

template <int kThreads>
__device__ __forceinline__ uint32_t row_max(uint32_t top) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
  if constexpr (kThreads > 64) {
    __shared__ uint32_t tops[kThreads / 64];
    if ((threadIdx.x & 63) == 0) tops[threadIdx.x >> 6] = top;
    __syncthreads();
#pragma unroll
    for (int i = 0; i < kThreads / 64; ++i) top = max(top, tops[i]);
  }
  return top;
}

// Rows that kThreads threads hold in registers, kChunks chunks of 16 bytes
// each: one read, one write.  A workgroup is 256 threads; rows start at any
// address.  Bound by memory: 16384 x 8192 in bf16 72 us, 5.6 TB/s (a copy of
// 1 GB reaches 5.3); 271 us with a second read and element loads.
template <class T, int kThreads, int kChunks>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T* x, int64_t rows, int64_t cols,
                                                            int8_t* q, int64_t pitch,
                                                            float* scale) {
  const int t = threadIdx.x % kThreads;
  const int64_t r = (int64_t)blockIdx.x * (256 / kThreads) + threadIdx.x / kThreads;
  if (r >= rows) return;  // (whole waves, and no barrier behind for kThreads = 64)
  const T* xr = x + r * cols;
  Chunk<T> c[kChunks];
  uint32_t top = 0;
#pragma unroll
  for (int i = 0; i < kChunks; ++i) c[i].load(xr, t + i * kThreads, cols);
#pragma unroll
  for (int i = 0; i < kChunks; ++i) top = max(top, c[i].top());
  const float s = row_scale(row_max<kThreads>(top));
  const Quantizer quantize(s);
#pragma unroll
  for (int i = 0; i < kChunks; ++i) {
    const int64_t at = t + i * kThreads;
    if (at * Chunk<T>::kN < pitch) c[i].store(q + r * pitch, at, pitch, quantize);
  }
  if (t == 0) scale[r] = s;
}

// Longer rows: a workgroup reads its row twice.
template <class T>
__global__ void __launch_bounds__(1024) quantize_long_kernel(const T* x, int64_t cols, int8_t* q,
                                                             int64_t pitch, float* scale) {
  const int64_t r = blockIdx.x;
  const T* xr = x + r * cols;
  uint32_t top = 0;
  Chunk<T> c;
  for (int64_t i = threadIdx.x; i * Chunk<T>::kN < cols; i += 1024) {
    c.load(xr, i, cols);
    top = max(top, c.top());
  }
  const float s = row_scale(row_max<1024>(top));
  const Quantizer quantize(s);
  for (int64_t i = threadIdx.x; i * Chunk<T>::kN < pitch; i += 1024) {
    c.load(xr, i, cols);
    c.store(q + r * pitch, i, pitch, quantize);
  }
  if (threadIdx.x == 0) scale[r] = s;
}

// Rows of one launch: a grid's threads (at most 1024 a row) are counted in 32 bits.
constexpr int64_t kLaunchRows = (int64_t)1 << 21;

template <class T>
int launch_quantize(const void* x, int64_t rows, int64_t cols, int8_t* q, int64_t pitch,
                    float* scale, hipStream_t stream) {
  if (rows > kLaunchRows) {
    for (int64_t r = 0; r < rows; r += kLaunchRows) {
      const int64_t n = rows - r < kLaunchRows ? rows - r : kLaunchRows;
      const int st = launch_quantize<T>((const T*)x + r * cols, n, cols, q + r * pitch, pitch,
                                        scale + r, stream);
      if (st) return st;
    }
    return PPO_OK;
  }
  const int64_t chunks = div_up(pitch, kPer16<T>);
  auto go = [&](auto threads, auto each) {
    constexpr int kT = decltype(threads)::value, kC = decltype(each)::value;
    hipLaunchKernelGGL((quantize_rows_kernel<T, kT, kC>),
                       dim3((unsigned)div_up(rows, 256 / kT)), dim3(256), 0, stream, (const T*)x,
                       rows, cols, q, pitch, scale);
  };
  using std::integral_constant;
  typedef integral_constant<int, 64> Wave;
  typedef integral_constant<int, 256> Group;
  if (chunks <= 64) go(Wave{}, integral_constant<int, 1>{});
  else if (chunks <= 128) go(Wave{}, integral_constant<int, 2>{});
  else if (chunks <= 256) go(Wave{}, integral_constant<int, 4>{});
  else if (chunks <= 512) go(Group{}, integral_constant<int, 2>{});
  else if (chunks <= 1024) go(Group{}, integral_constant<int, 4>{});
  else if (chunks <= 2048) go(Group{}, integral_constant<int, 8>{});
  else
    hipLaunchKernelGGL((quantize_long_kernel<T>), dim3((unsigned)rows), dim3(1024), 0, stream,
                       (const T*)x, cols, q, pitch, scale);
  return last_launch_status();
}

// The product of a few rows of floating x, in one launch: every workgroup
// quantises the rows for itself (into LDS, by 256 / rows threads each), which
// for up to kFewBytes costs it less than a launch of its own would the call (in
// two kernels and here, us in a replayed graph: one row of bf16 1024 -> 1024 5.7 and
// 4.3, 4096 -> 4096 8.1 and 6.9, 8192 -> 4096 11.6 and 11.2; 8 rows of 1024 -> 1024 6.3 and
// 6.9, of fp32 6.2 and 8.2; 4 of bf16 4096 -> 4096 8.8 and 12.9; the second launch costs
// the host 3 more), then takes 16 columns as the rows kernel does.  kOdd: rows of w
// that start off 4 bytes.
constexpr int kFewRows = 16;
constexpr int64_t kFewBytes = 16384;  // of x

template <class T, bool kOdd>
__global__ void __launch_bounds__(256) int8_few_kernel(const T* x, const int8_t* w, int M, int N,
                                                       int K, const float* ws, const T* bias,
                                                       T* out) {
  __shared__ __align__(16) int8_t xq[kFewBytes / sizeof(T) + kFewRows * 32];
  __shared__ uint32_t tops[kFewRows];
  __shared__ float scales[kFewRows];
  __shared__ v4i red[4][64];
  const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int per_row = 256;
  while (per_row * M > 256) per_row >>= 1;  // threads of a row: 256 to 16
  const int row = tid / per_row, t = tid & (per_row - 1);
  const int pitch = (K + 15) / 16 * 16 + 16;  // (16 bytes more spread the rows over the banks)
  // the wave's first runs of W are on their way meanwhile
  const int r16 = lane & 15, kq = lane >> 4, n0 = blockIdx.x * 16;
  const char* wr = (const char*)w + (int64_t)min(n0 + r16, N - 1) * K + kq * 16;
  constexpr int kRuns = 4;
  const int full = K / kRunBytes;
  const bool ahead = wave + (kRuns - 1) * 4 < full;
  v4i early[kRuns][2];
  auto fetch = [&](int s, auto& wf) {
#pragma unroll
    for (int r = 0; r < (int)(sizeof(wf) / sizeof(wf[0])); ++r)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
        if constexpr (kOdd)
          wf[r][ks] = load16_shifted(wr + (s + r * 4) * kRunBytes + ks * 64);
        else
          wf[r][ks] = *reinterpret_cast<const v4i_any*>(wr + (s + r * 4) * kRunBytes + ks * 64);
  };
  if (ahead) fetch(wave, early);
  if (tid < kFewRows) tops[tid] = 0;
  __syncthreads();
  if (row < M) {
    const T* xr = x + (int64_t)row * K;
    uint32_t top = 0;
    Chunk<T> c;
    for (int i = t; i * Chunk<T>::kN < K; i += per_row) {
      c.load(xr, i, K);
      top = max(top, c.top());
    }
    for (int o = 1; o < (per_row < 64 ? per_row : 64); o <<= 1)
      top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
    if ((t & 63) == 0) atomicMax(&tops[row], top);
  }
  __syncthreads();
  if (row < M) {
    const T* xr = x + (int64_t)row * K;
    const float s = row_scale(tops[row]);
    const Quantizer quantize(s);
    Chunk<T> c;
    for (int i = t; i * Chunk<T>::kN < pitch - 16; i += per_row) {
      c.load(xr, i, K);
      c.store(xq + row * pitch, i, pitch - 16, quantize);
    }
    if (t == 0) scales[row] = s;
  }
  __syncthreads();

  const int8_t* xr = xq + min(r16, M - 1) * pitch + kq * 16;
  v4i acc = {0, 0, 0, 0};
  auto take = [&](int s, const auto& wf) {
#pragma unroll
    for (int r = 0; r < (int)(sizeof(wf) / sizeof(wf[0])); ++r)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
        acc = mfma<int8_t, 16>(
            wf[r][ks], *reinterpret_cast<const v4i*>(xr + (s + r * 4) * kRunBytes + ks * 64), acc);
  };
  int s = wave;
  if (ahead) {
    take(s, early);
    s += kRuns * 4;
  }
  for (; s + (kRuns - 1) * 4 < full; s += kRuns * 4) {
    v4i wf[kRuns][2];
    fetch(s, wf);
    take(s, wf);
  }
  for (; s < full; s += 4) {
    v4i wf[1][2];
    fetch(s, wf);
    take(s, wf);
  }
  if (full * kRunBytes < K && wave == full % 4) {
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const int at = full * kRunBytes + ks * 64, left = K - at - kq * 16;
      v4i xf = {0, 0, 0, 0};
      if (left > 0) xf = *reinterpret_cast<const v4i*>(xr + at);  // (zeros behind K)
      acc = mfma<int8_t, 16>(load16_upto(wr + at, left), xf, acc);
    }
  }
  red[wave][lane] = acc;
  __syncthreads();
  if (wave) return;
  const int n = n0 + kq * 4;
  if (r16 >= M || n >= N) return;
  v4i sum = red[0][lane];
#pragma unroll
  for (int v = 1; v < 4; ++v) sum += red[v][lane];
  const Int8Epi<T> epi = {scales, ws, bias, out, N};
  const v4i sums[1] = {sum};
  apply_one<int8_t>(epi, r16, n, epi.columns(n), true, sums);
}

struct Int8Plan {
  int64_t pitch;
  bool pad_x, pad_w;
  GemmPlan gemm;
  char *xq, *xs, *wq, *partial;
  size_t bytes;
};

Int8Plan plan_int8(int64_t M, int64_t N, int64_t K, bool quantize, bool ax, bool aw, char* ws) {
  Int8Plan p = {};
  p.pitch = round_up(K, 16);
  const bool odd = p.pitch != K;
  const GemmPlan& g = p.gemm = plan_gemm(M, N, K, false, kOneMatrix);
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
  const bool aligned = take_aligned(quantize);
  if (M <= 0 || N <= 0 || K <= 0 || K > kMaxInt8K || !gemm_fits(M, N, round_up(K, 16))) return 0;
  return plan_int8(M, N, K, quantize != 0, aligned, aligned, nullptr).bytes;
}

extern "C" int ppo_layer_int8_linear(const void* x, const int8_t* xq, const float* xs,
                                     const int8_t* wq, const float* ws, const void* bias,
                                     int dtype, int64_t M, int64_t N, int64_t K, void* out,
                                     void* workspace, size_t workspace_bytes, void* stream_ptr) {
  const bool promised = take_aligned(dtype);
  if (!dtype_ok(dtype) || M < 0 || N <= 0 || K <= 0) return PPO_ERR_INVALID_ARG;
  if (M == 0) return PPO_OK;
  if (!wq || !ws || !out || (!x && (!xq || !xs))) return PPO_ERR_INVALID_ARG;
  if (K > kMaxInt8K || !gemm_fits(M, N, round_up(K, 16))) return PPO_ERR_TOO_LARGE;
  const bool ax = x || aligned16(xq), aw = aligned16(wq);
  if (promised && !(ax && aw)) return PPO_ERR_INVALID_ARG;
  const Int8Plan p = plan_int8(M, N, K, x != nullptr, ax, aw, (char*)workspace);
  const size_t need = plan_int8(M, N, K, x != nullptr, promised, promised, nullptr).bytes;
  if (need && (!workspace || workspace_bytes < need || !aligned16(workspace)))
    return PPO_ERR_WORKSPACE;
  hipStream_t stream = reinterpret_cast<hipStream_t>(stream_ptr);
  return with_dtype(dtype, [&](auto zero) {
    using T = decltype(zero);
    if (x && M <= kFewRows && M * K <= kFewBytes / (int64_t)sizeof(T)) {
      auto go = [&](auto odd) {
        hipLaunchKernelGGL((int8_few_kernel<T, decltype(odd)::value>), dim3((unsigned)div_up(N, 16)),
                           dim3(256), 0, stream, (const T*)x, wq, (int)M, (int)N, (int)K, ws,
                           (const T*)bias, (T*)out);
      };
      if (((uintptr_t)wq | (uintptr_t)K) & 3) go(std::true_type{});
      else go(std::false_type{});
      return last_launch_status();
    }
    GemmArgs a = {};
    a.x = (const char*)xq;
    a.w0 = (const char*)wq;
    a.xpitch = a.wpitch = a.kbytes = K;
    a.M = (int)M;
    a.N = (int)N;
    int st = PPO_OK;
    if (x) {
      st = launch_quantize<T>(x, M, K, (int8_t*)p.xq, p.pitch, (float*)p.xs, stream);
      if (st) return st;
    }
    if (x || p.pad_x) {
      a.x = p.xq;
      a.xpitch = p.pitch;
    }
    if (p.pad_w) {
      a.w0 = p.wq;
      a.wpitch = p.pitch;
    }
    if (p.pad_x || p.pad_w) {
      const PadArgs pad = {{(const char*)xq, (const char*)wq, nullptr},
                           {p.xq, p.wq, nullptr},
                           {p.pad_x ? M : 0, p.pad_w ? N : 0, 0}};
      if ((st = pad_rows(pad, K, p.pitch, stream))) return st;
    }
    // the tile kernel's rows end on 16 bytes (zeros behind K), the rows kernel's on K
    if (p.gemm.tile) a.kbytes = p.pitch;
    const Int8Epi<T> epi = {x ? (const float*)p.xs : xs, ws, (const T*)bias, (T*)out, (int)N};
    return launch_gemm<int8_t>(a, epi, p.gemm, p.partial, stream);
  });
}
