// The matrix product under the layer operators: C[m,n] = sum_k X[m,k] W[n,k]
// on the matrix cores, for rows of fp32, bf16, fp16 or int8 that are
// contiguous along k, with the operator's epilogue applied to the sums while
// they are still in registers.
//
// Everything is laid out in 16-byte chunks of a row: 4 fp32, 8 16-bit or 16
// int8 elements.  A lane of the matrix instructions below holds one chunk of
// row lane % 16 (16x16x32 on 16-bit types and 16x16x64 on int8 take the whole
// chunk; fp32 takes four 16x16x4 steps, one element each: the order of k
// inside a step is free as long as both operands share it).  So one kernel
// serves all types.  W is the instruction's first operand, so a lane ends up
// with four consecutive columns n of one row m: a vector store, and one call
// of the dropout generator.
//
// A workgroup computes a BM x BN tile over K steps of 128 bytes.  Both tiles
// go from memory to LDS without passing through registers (buffer loads with
// the LDS bit: 64 lanes, 16 bytes each, to consecutive LDS addresses), two
// buffers in turn.  A row's chunk c sits in slot c ^ (row % 8), which spreads
// the sixteen rows that a fragment read touches over all banks; since the LDS
// side of the load is fixed, the lanes permute the addresses they load from
// instead.  The buffer descriptor ends with the operand's last row and lanes
// past the end of a row ask for an offset behind it: the hardware gives zero
// for both, so partial tiles need no other path.
#pragma once

#include <type_traits>

#include "layers.hpp"

namespace ppo {

struct GemmArgs {
  const char* x;    // [M] rows
  const char* w0;   // [N] rows
  const char* w1;   // second matrix of a gated product, [N] rows
  int64_t xpitch, wpitch;  // bytes, multiples of 16
  int64_t kbytes;   // of a row, a multiple of 16
  int M, N;         // N: output columns
  int tiles_m, tiles_n;
  int steps_per_split;     // K steps of 128 bytes that one split takes
  char* partial;    // [splits][1 or 2][M][N4] 32-bit sums, or null: no split
};

constexpr int kStepBytes = 128;

template <class T>
struct AccOf { using type = v4f; };
template <>
struct AccOf<int8_t> { using type = v4i; };
template <class T>
using Acc = typename AccOf<T>::type;

template <class T>
__device__ __forceinline__ Acc<T> mfma16(v4i w, v4i x, Acc<T> c) {
  if constexpr (sizeof(T) == 4) {
    const v4f a = __builtin_bit_cast(v4f, w), b = __builtin_bit_cast(v4f, x);
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
  } else if constexpr (sizeof(T) == 1) {
    return __builtin_amdgcn_mfma_i32_16x16x64_i8(w, x, c, 0, 0, 0);
  } else if constexpr (__is_same(T, fp16)) {
    typedef _Float16 v8h __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, w),
                                                  __builtin_bit_cast(v8h, x), c, 0, 0, 0);
  } else {
    typedef __bf16 v8b __attribute__((ext_vector_type(8)));
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8b, w),
                                                   __builtin_bit_cast(v8b, x), c, 0, 0, 0);
  }
}

// Descriptor of `bytes` (below 2^31) from p on; loads behind it give zero.
__device__ __forceinline__ v4i buffer_of(const char* p, uint32_t bytes) {
  const uint64_t a = (uint64_t)p;
  v4i r;
  r[0] = __builtin_amdgcn_readfirstlane((int)(uint32_t)a);
  r[1] = __builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32) & 0xffff);
  r[2] = __builtin_amdgcn_readfirstlane((int)bytes);
  r[3] = 0x00020000;
  return r;
}

// 64 lanes, 16 bytes each from buffer + offset, to LDS at lds + 16 * lane
// (`lds` is the same in all lanes).  Nothing in registers is written; the
// data has arrived after lds_loads_wait_barrier().
__device__ __forceinline__ void load_to_lds(uint32_t lds, v4i buffer, uint32_t offset) {
  asm volatile(
      "s_mov_b32 m0, %0\n\t"
      "s_nop 0\n\t"
      "buffer_load_dwordx4 %1, %2, 0 offen lds" ::"s"(lds), "v"(offset), "s"(buffer));
}

// Waits for this wave's loads (to LDS too) and LDS reads, then for the whole
// workgroup: what every wave loaded may be read, what it read overwritten.
__device__ __forceinline__ void lds_loads_wait_barrier() {
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" ::: "memory");
}

constexpr uint32_t kBehind = 0x80000000u;  // an offset that no descriptor reaches

// Workgroup -> tile.  Workgroups go round-robin over the eight XCDs, each
// with an L2 of its own: an XCD takes a run of consecutive tiles, and a run
// walks blocks of kGroup row tiles by columns, so that the tiles in flight on
// one XCD share rows and columns.
__device__ __forceinline__ void tile_of(const GemmArgs& a, int& tm, int& tn) {
  constexpr int kXcds = 8, kGroup = 8;
  const int n = a.tiles_m * a.tiles_n, id = blockIdx.x;
  const int xcd = id % kXcds, q = n / kXcds, r = n % kXcds;
  const int t = xcd * q + min(xcd, r) + id / kXcds;
  const int per = kGroup * a.tiles_n, first = t / per * kGroup;
  const int rows = min(kGroup, a.tiles_m - first);
  tm = first + t % per % rows;
  tn = t % per / rows;
}

// One 32-bit sum block to its place among the partial sums of a split.
template <class A>
__device__ __forceinline__ void store_partial(const GemmArgs& a, int split, int half, int halves,
                                              int m, int n, A v) {
  const int64_t n4 = round_up(a.N, 4);
  const int64_t at = ((((int64_t)split * halves + half) * a.M + m) * n4 + n) * 4;
  *reinterpret_cast<A*>(a.partial + at) = v;
}

// Epi: kGated (two W matrices, one output), and
//   void operator()(int m, int n, Acc<T> c [, Acc<T> second]) for columns
// n..n+3 of row m < M, n < N (columns past N - 1 are the callee's to skip).
template <class T, int BM, int BN, int kWavesM, int kWavesN, class Epi>
__global__ void __launch_bounds__(kWavesM* kWavesN * 64)
    gemm_tile_kernel(const GemmArgs a, const Epi epi) {
  constexpr int kWaves = kWavesM * kWavesN;
  constexpr int TM = BM / kWavesM / 16, TN = BN / kWavesN / 16;
  constexpr int XL = BM / 8 / kWaves, WL = BN / 8 / kWaves;  // loads of a wave per step
  constexpr bool kGated = Epi::kGated;
  constexpr int kCols = kGated ? BN / 2 : BN;  // output columns of a tile
  static_assert(BM % (8 * kWaves) == 0 && BN % (8 * kWaves) == 0 && (!kGated || TN % 2 == 0), "");
  __shared__ __align__(1024) char lds[2][(BM + BN) * kStepBytes];

  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wm = wave / kWavesN, wn = wave % kWavesN;
  int tm, tn;
  tile_of(a, tm, tn);
  const int m0 = tm * BM, n0 = tn * kCols;
  const int steps = (int)div_up(a.kbytes, kStepBytes);
  const int first = blockIdx.y * a.steps_per_split;
  const int last = min(steps, first + a.steps_per_split);

  // --- addresses of this wave's loads -----------------------------------------------
  const int row8 = lane >> 3;
  const uint32_t chunk = ((lane & 7) ^ row8) * 16;
  const v4i bx = buffer_of(a.x + m0 * a.xpitch, (uint32_t)min(BM, a.M - m0) * (uint32_t)a.xpitch);
  const uint32_t w_bytes = (uint32_t)min(kCols, a.N - n0) * (uint32_t)a.wpitch;
  const v4i bw0 = buffer_of(a.w0 + n0 * a.wpitch, w_bytes);
  const v4i bw1 = kGated ? buffer_of(a.w1 + n0 * a.wpitch, w_bytes) : bw0;
  uint32_t x_off[XL], w_off[WL];
  bool second[WL];  // of the gated pair, the same in all lanes
#pragma unroll
  for (int i = 0; i < XL; ++i)
    x_off[i] = (uint32_t)((wave * XL + i) * 8 + row8) * (uint32_t)a.xpitch;
#pragma unroll
  for (int i = 0; i < WL; ++i) {
    const int j = (wave * WL + i) * 8;  // first of the eight LDS rows
    int col = j;
    second[i] = false;
    if (kGated) {  // a wave's columns: half from the first matrix, half from the second
      constexpr int kSpan = TN * 16, kHalf = kSpan / 2;
      second[i] = j % kSpan >= kHalf;
      col = j / kSpan * kHalf + j % kHalf;
    }
    w_off[i] = (uint32_t)(col + row8) * (uint32_t)a.wpitch;
  }
  const uint32_t lds0 =
      (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)&lds[0][0];
  auto load_step = [&](int step, int buf) {
    const uint32_t kb = (uint32_t)step * kStepBytes + chunk;
    const uint32_t k_off = kb < (uint32_t)a.kbytes ? kb : kBehind;
    const uint32_t to = lds0 + buf * (BM + BN) * kStepBytes;
#pragma unroll
    for (int i = 0; i < XL; ++i) load_to_lds(to + (wave * XL + i) * 1024, bx, x_off[i] + k_off);
#pragma unroll
    for (int i = 0; i < WL; ++i)
      load_to_lds(to + BM * kStepBytes + (wave * WL + i) * 1024, second[i] ? bw1 : bw0,
                  w_off[i] + k_off);
  };

  // --- sums -------------------------------------------------------------------------
  Acc<T> acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j) acc[i][j] = Acc<T>{0, 0, 0, 0};

  const int r16 = lane & 15, kq = lane >> 4;
  const int x_at = (wm * TM * 16 + r16) * kStepBytes;
  const int w_at = (BM + wn * TN * 16 + r16) * kStepBytes;
  if (first < last) load_step(first, 0);
  lds_loads_wait_barrier();
  for (int step = first; step < last; ++step) {
    const int buf = (step - first) & 1;
    if (step + 1 < last) load_step(step + 1, buf ^ 1);
    const char* s = lds[buf];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const int slot = ((ks * 4 + kq) ^ (r16 & 7)) * 16;
      v4i xf[TM], wf[TN];
#pragma unroll
      for (int j = 0; j < TN; ++j)
        wf[j] = *reinterpret_cast<const v4i*>(s + w_at + j * 16 * kStepBytes + slot);
#pragma unroll
      for (int i = 0; i < TM; ++i)
        xf[i] = *reinterpret_cast<const v4i*>(s + x_at + i * 16 * kStepBytes + slot);
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = mfma16<T>(wf[j], xf[i], acc[i][j]);
    }
    lds_loads_wait_barrier();
  }

  // --- epilogue ---------------------------------------------------------------------
#pragma unroll
  for (int i = 0; i < TM; ++i) {
    const int m = m0 + (wm * TM + i) * 16 + r16;
    if (m >= a.M) continue;
#pragma unroll
    for (int j = 0; j < (kGated ? TN / 2 : TN); ++j) {
      const int n = n0 + wn * (kGated ? TN * 8 : TN * 16) + j * 16 + kq * 4;
      if (n >= a.N) continue;
      if constexpr (kGated) {
        if (a.partial) {
          store_partial(a, blockIdx.y, 0, 2, m, n, acc[i][j]);
          store_partial(a, blockIdx.y, 1, 2, m, n, acc[i][j + TN / 2]);
        } else {
          epi(m, n, acc[i][j], acc[i][j + TN / 2]);
        }
      } else {
        if (a.partial)
          store_partial(a, blockIdx.y, 0, 1, m, n, acc[i][j]);
        else
          epi(m, n, acc[i][j]);
      }
    }
  }
}

// Joins the splits of K in their order and applies the epilogue.
template <class T, class Epi>
__global__ void __launch_bounds__(256) gemm_join_kernel(const GemmArgs a, const Epi epi,
                                                        int splits) {
  constexpr int kHalves = Epi::kGated ? 2 : 1;
  const int64_t groups = div_up(a.N, 4), n4 = groups * 4;
  const int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (id >= a.M * groups) return;
  const int m = (int)(id / groups), n = (int)(id % groups) * 4;
  Acc<T> sum[kHalves];
  for (int s = 0; s < splits; ++s)
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      const int64_t at = ((((int64_t)s * kHalves + h) * a.M + m) * n4 + n) * 4;
      const Acc<T> v = *reinterpret_cast<const Acc<T>*>(a.partial + at);
      sum[h] = s ? sum[h] + v : v;
    }
  if constexpr (kHalves == 2)
    epi(m, n, sum[0], sum[1]);
  else
    epi(m, n, sum[0]);
}

// Sixteen bytes of a row that ends `left` bytes from p on; zeros behind.
__device__ __forceinline__ v4i load16_upto(const char* p, int left) {
  if (left >= 16) return *reinterpret_cast<const v4i_any*>(p);
  union { v4i v; char c[16]; } r;
  r.v = v4i{0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < 16; ++i)
    if (i < left) r.c[i] = p[i];
  return r.v;
}

// Few rows of X (at most 16 * MT): every weight is read once, so the time is
// that of reading W.  A workgroup takes 16 columns and its waves share K in
// runs of 128 bytes; W goes straight to registers (no reuse for LDS to serve)
// from rows of any alignment, and the waves' sums meet in LDS.  Rows of X
// beyond M repeat the last one and are not stored.
template <class T, int MT, int kWaves, class Epi>
__global__ void __launch_bounds__(kWaves * 64) gemm_rows_kernel(const GemmArgs a, const Epi epi) {
  constexpr int kHalves = Epi::kGated ? 2 : 1;
  __shared__ Acc<T> red[kWaves][MT * kHalves][64];
  const int lane = threadIdx.x & 63;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r16 = lane & 15, kq = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const int64_t wrow = min(n0 + r16, a.N - 1);
  const char* w[2] = {a.w0 + wrow * a.wpitch + kq * 16,
                      kHalves == 2 ? a.w1 + wrow * a.wpitch + kq * 16 : nullptr};
  const char* x[MT];
#pragma unroll
  for (int i = 0; i < MT; ++i) x[i] = a.x + (int64_t)min(i * 16 + r16, a.M - 1) * a.xpitch + kq * 16;
  Acc<T> acc[MT][kHalves];
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int h = 0; h < kHalves; ++h) acc[i][h] = Acc<T>{0, 0, 0, 0};

  const int kbytes = (int)a.kbytes;
  const int full = kbytes / kStepBytes;  // whole runs
  // kRuns runs' loads are under way before the first is used
  constexpr int kRuns = MT == 1 ? 4 : MT == 2 ? 3 : 2;
  auto take = [&](int s, auto runs) {
    constexpr int R = decltype(runs)::value;
    v4i wf[R][kHalves][2], xf[R][MT][2];
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int64_t k = (int64_t)(s + r * kWaves) * kStepBytes;
#pragma unroll
      for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
        for (int h = 0; h < kHalves; ++h)
          wf[r][h][ks] = *reinterpret_cast<const v4i_any*>(w[h] + k + ks * 64);
#pragma unroll
        for (int i = 0; i < MT; ++i)
          xf[r][i][ks] = *reinterpret_cast<const v4i_any*>(x[i] + k + ks * 64);
      }
    }
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int ks = 0; ks < 2; ++ks)
#pragma unroll
        for (int i = 0; i < MT; ++i)
#pragma unroll
          for (int h = 0; h < kHalves; ++h)
            acc[i][h] = mfma16<T>(wf[r][h][ks], xf[r][i][ks], acc[i][h]);
  };
  int s = wave;
  for (; s + (kRuns - 1) * kWaves < full; s += kRuns * kWaves)
    take(s, std::integral_constant<int, kRuns>{});
  for (; s < full; s += kWaves) take(s, std::integral_constant<int, 1>{});
  if (full * kStepBytes < kbytes && wave == full % kWaves) {  // the run that ends inside
    const int64_t k = (int64_t)full * kStepBytes;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      const int left = kbytes - (int)k - ks * 64 - kq * 16;
#pragma unroll
      for (int i = 0; i < MT; ++i) {
        const v4i xf = load16_upto(x[i] + k + ks * 64, left);
#pragma unroll
        for (int h = 0; h < kHalves; ++h)
          acc[i][h] = mfma16<T>(load16_upto(w[h] + k + ks * 64, left), xf, acc[i][h]);
      }
    }
  }
#pragma unroll
  for (int i = 0; i < MT; ++i)
#pragma unroll
    for (int h = 0; h < kHalves; ++h) red[wave][i * kHalves + h][lane] = acc[i][h];
  __syncthreads();
#pragma unroll
  for (int i = 0; i < MT; ++i) {
    if (wave != i % kWaves) continue;
    Acc<T> sum[kHalves];
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      sum[h] = red[0][i * kHalves + h][lane];
#pragma unroll
      for (int v = 1; v < kWaves; ++v) sum[h] += red[v][i * kHalves + h][lane];
    }
    const int m = i * 16 + r16, n = n0 + kq * 4;
    if (m >= a.M || n >= a.N) continue;
    if constexpr (kHalves == 2)
      epi(m, n, sum[0], sum[1]);
    else
      epi(m, n, sum[0]);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
struct GemmPlan {
  int tile;     // 0: rows kernel, else the tile's edge
  int splits;
  size_t partial_bytes;
};

constexpr int kRowsMax = 64;       // rows that the rows kernel takes
constexpr int64_t kMaxPitch = (int64_t)1 << 22;  // 256 rows of a tile stay below 2^31 bytes

// How a product of M rows and `wrows` rows of W (both matrices of a gated one
// together) over `kbytes` is cut.
inline GemmPlan plan_gemm(int64_t M, int64_t wrows, int64_t kbytes) {
  GemmPlan p = {0, 1, 0};
  if (M <= kRowsMax) return p;
  const int64_t steps = div_up(kbytes, kStepBytes);
  auto tiles = [&](int64_t b) { return div_up(M, b) * div_up(wrows, b); };
  if (tiles(256) >= 200) {
    p.tile = 256;
  } else if (tiles(128) >= 200) {
    p.tile = 128;
  } else {
    p.tile = 64;
    while (tiles(64) * p.splits < 512 && steps / (p.splits * 2) >= 8 && p.splits < 16)
      p.splits *= 2;
  }
  if (p.splits > 1) p.partial_bytes = (size_t)p.splits * M * round_up(wrows, 8) * 4;
  return p;
}

// Checks what the kernels assume of sizes.
inline bool gemm_fits(int64_t M, int64_t N, int64_t pitch_bytes) {
  return M < ((int64_t)1 << 30) && N < ((int64_t)1 << 30) && pitch_bytes < kMaxPitch &&
         div_up(M, 64) * div_up(N, 32) < ((int64_t)1 << 30);
}

template <class T, class Epi>
int launch_gemm(GemmArgs a, const Epi& epi, char* partial, hipStream_t stream) {
  const int64_t wrows = (int64_t)a.N * (Epi::kGated ? 2 : 1);
  const GemmPlan p = plan_gemm(a.M, wrows, a.kbytes);
  a.partial = p.splits > 1 ? partial : nullptr;
  if (p.tile == 0) {
    const dim3 grid((unsigned)div_up(a.N, 16));
    if (a.M <= 16)
      hipLaunchKernelGGL((gemm_rows_kernel<T, 1, 4, Epi>), grid, dim3(256), 0, stream, a, epi);
    else if (a.M <= 32)
      hipLaunchKernelGGL((gemm_rows_kernel<T, 2, 4, Epi>), grid, dim3(256), 0, stream, a, epi);
    else
      hipLaunchKernelGGL((gemm_rows_kernel<T, 4, 4, Epi>), grid, dim3(256), 0, stream, a, epi);
    return last_launch_status();
  }
  const int steps = (int)div_up(a.kbytes, kStepBytes);
  a.steps_per_split = (int)div_up(steps, p.splits);
  const int cols = Epi::kGated ? p.tile / 2 : p.tile;
  a.tiles_m = (int)div_up(a.M, p.tile);
  a.tiles_n = (int)div_up(a.N, cols);
  const dim3 grid((unsigned)(a.tiles_m * a.tiles_n), (unsigned)p.splits);
  if (p.tile == 256)
    hipLaunchKernelGGL((gemm_tile_kernel<T, 256, 256, 2, 4, Epi>), grid, dim3(512), 0, stream, a,
                       epi);
  else if (p.tile == 128)
    hipLaunchKernelGGL((gemm_tile_kernel<T, 128, 128, 2, 2, Epi>), grid, dim3(256), 0, stream, a,
                       epi);
  else
    hipLaunchKernelGGL((gemm_tile_kernel<T, 64, 64, 2, 2, Epi>), grid, dim3(256), 0, stream, a,
                       epi);
  if (p.splits > 1) {
    const int64_t n = (int64_t)a.M * div_up(a.N, 4);
    hipLaunchKernelGGL((gemm_join_kernel<T, Epi>), dim3((unsigned)div_up(n, 256)), dim3(256), 0,
                       stream, a, epi, p.splits);
  }
  return last_launch_status();
}

}  // namespace ppo
