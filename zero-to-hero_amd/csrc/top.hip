// The K largest logits of each row, in order.  A logit and its column make one
// 64-bit whole number (the logit's order above, the column's complement below), by
// which no two of a row are alike: ties need no care of their own.
//
// A workgroup holds a row, or a part of one, in registers.  The K-th largest of its
// lanes' own maxima bounds the K-th largest element from below, so the few elements
// from there on (about K of them) are all there is to sort, by counting for each
// how many precede it.  Rows of many equal logits, where too many reach the bound,
// are settled by searching for the threshold itself.  What bounds it: HBM reads.
#include "tokens_rows.hpp"

namespace ppo {
namespace {

constexpr int kMaxK = PPO_TOKEN_MAX_K;
// Elements that are sorted at most: about what fewer than kMaxK lanes of one chunk each
// hold together.
constexpr int kSorted = 8 * kMaxK;

typedef unsigned long long u64;

// A logit's order as an unsigned number above 0; -0 is 0, NaN is before everything.
__device__ __forceinline__ unsigned order_of(float l) {
  const unsigned b = __builtin_bit_cast(unsigned, l + 0.0f);
  const unsigned k = b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
  return l != l ? 0xFFFFFFFFu : k;
}
__device__ __forceinline__ u64 place(unsigned order, int col) {
  return (u64)order << 32 | (unsigned)~col;
}
__device__ __forceinline__ int column_of(u64 x) { return (int)~(unsigned)x; }

template <int G>
struct Board {
  u64 list[kSorted];
  unsigned best[G];
  unsigned bound;
  int count, total;
  int part[G / kWave];
};

// The sum of a whole number over the workgroup, for every lane.  Two barriers.
template <int G>
__device__ __forceinline__ int block_count(int x, Board<G>& b) {
  x = (int)lanes_sum<kWave>((float)x);  // (below 2^24)
  if ((threadIdx.x & (kWave - 1)) == 0) b.part[threadIdx.x / kWave] = x;
  lds_barrier();
  int n = 0;
#pragma unroll
  for (int w = 0; w < G / kWave; ++w) n += b.part[w];
  lds_barrier();
  return n;
}

// Leaves in b.list the workgroup's elements among which its K largest are, and in
// b.count how many (at most kSorted).  each(f) calls f(order, column) for every element
// of the lane; `best` is the largest order among them, 0 without any.
template <int G, class Each>
__device__ __forceinline__ void gather(Board<G>& b, int K, int columns, unsigned best, Each&& each) {
  b.best[threadIdx.x] = best;
  if (threadIdx.x == 0) b.count = 0;
  lds_barrier();
  if (threadIdx.x < kWave) {
    // the largest 16-bit prefix that K lanes' best reach (0 if fewer have any)
    unsigned v[G / kWave];
#pragma unroll
    for (int i = 0; i < G / kWave; ++i) v[i] = b.best[i * kWave + threadIdx.x];
    unsigned bound = 0;
    for (unsigned bit = 1u << 31; bit >= 1u << 16; bit >>= 1) {
      int n = 0;
#pragma unroll
      for (int i = 0; i < G / kWave; ++i) n += __builtin_popcountll(__ballot(v[i] >= (bound | bit)));
      if (n >= K) bound |= bit;
    }
    if (threadIdx.x == 0) b.bound = bound > 1 ? bound : 1;  // (order 0 is no element)
  }
  lds_barrier();
  const unsigned bound = b.bound;
  auto collect = [&](auto&& takes) {
    each([&](unsigned order, int col) {
      if (!takes(order, col)) return;
      const int at = atomicAdd(&b.count, 1);
      if (at < kSorted) b.list[at] = place(order, col);
    });
  };
  if (best >= bound) collect([&](unsigned order, int) { return order >= bound; });
  lds_barrier();
  if (b.count <= kSorted) return;
  // Too many equal ones: the K-th largest order exactly, then the column up to which
  // elements of that order are among the K.
  lds_barrier();
  unsigned kth = 0;
  for (unsigned bit = 1u << 31; bit; bit >>= 1) {
    int n = 0;
    each([&](unsigned order, int) { n += order >= (kth | bit); });
    if (block_count(n, b) >= K) kth |= bit;
  }
  int above = 0;
  each([&](unsigned order, int) { above += order > kth; });
  const int ties = K - block_count(above, b);
  int last = 0;  // the smallest column with `ties` elements of order kth up to it
  for (int step = 1 << 30; step; step >>= 1) {
    if (last + step > columns) continue;
    int n = 0;
    each([&](unsigned order, int col) { n += order == kth && col < last + step; });
    if (block_count(n, b) < ties) last += step;
  }
  if (threadIdx.x == 0) b.count = 0;
  lds_barrier();
  collect([&](unsigned order, int col) { return order > kth || (order == kth && col <= last); });
  lds_barrier();
}

// Calls out(rank, element) for each of the listed elements among the K largest.
template <int G, class Out>
__device__ __forceinline__ void ranked(const Board<G>& b, int K, Out&& out) {
  const int n = b.count;
  for (int i = threadIdx.x; i < n; i += G) {
    const u64 x = b.list[i];
    int rank = 0;
    for (int k = 0; k < n; ++k) rank += b.list[k] > x;
    if (rank < K) out(rank, x);
  }
}

// Part `p` of `parts` of each row; one part: the row's results, else its largest
// elements to `found` [rows][parts][K], 0 behind the last.
template <class T, int G, int V>
__global__ void __launch_bounds__(G) top_kernel(const T* logits, int64_t rows, int A, int K,
                                                int parts, int per, T* values, int64_t* ids,
                                                u64* found) {
  constexpr int kN = kPer16<T>;
  __shared__ Board<G> b;
  const int t = threadIdx.x;
  const int64_t r = (int64_t)blockIdx.x / parts;
  const int p = (int)((int64_t)blockIdx.x - r * parts);
  const T* row = logits + r * A;
  const int from = p * per, width = min(per, A - from);
  RowRegs<T, G, V> x(row + from, width, t);
  auto each = [&](auto&& f) {
    if (x.end_col >= 0) f(order_of(x.end), from + x.end_col);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      float none = 0.0f;
      x.turn(i, none);
      if (i * G + t >= x.cut.nvec) continue;
      const int col = from + x.cut.head + (i * G + t) * kN;
#pragma unroll
      for (int j = 0; j < kN; ++j) f(order_of(unpack<T>(x.raw[i], j)), col + j);
    }
  };
  unsigned best = 0;
  each([&](unsigned order, int) { best = order > best ? order : best; });
  gather<G>(b, min(K, width), A, best, each);
  if (parts == 1) {
    ranked<G>(b, K, [&](int rank, u64 e) {
      const int col = column_of(e);
      values[r * K + rank] = row[col];
      ids[r * K + rank] = col;
    });
  } else {
    u64* to = found + (int64_t)blockIdx.x * K;
    ranked<G>(b, K, [&](int rank, u64 e) { to[rank] = e; });
    for (int k = width + t; k < K; k += G) to[k] = 0;
  }
}

// The K largest of a row's parts' (at most kMaxParts of them, K each).
constexpr int kMaxParts = 64, kMergeV = kMaxParts * kMaxK / 1024;
template <class T>
__global__ void __launch_bounds__(1024) top_merge_kernel(const T* logits, int A, int K, int parts,
                                                         T* values, int64_t* ids,
                                                         const u64* found) {
  __shared__ Board<1024> b;
  const int64_t r = blockIdx.x;
  const u64* from = found + r * parts * K;
  const int n = parts * K;
  u64 x[kMergeV];
  unsigned best = 0;
#pragma unroll
  for (int i = 0; i < kMergeV; ++i) {
    const int k = i * 1024 + threadIdx.x;
    x[i] = k < n ? from[k] : 0;
    const unsigned order = (unsigned)(x[i] >> 32);
    best = order > best ? order : best;
  }
  gather<1024>(b, K, A, best, [&](auto&& f) {
#pragma unroll
    for (int i = 0; i < kMergeV; ++i)
      if (x[i]) f((unsigned)(x[i] >> 32), column_of(x[i]));
  });
  ranked<1024>(b, K, [&](int rank, u64 e) {
    const int col = column_of(e);
    values[r * K + rank] = logits[r * A + col];
    ids[r * K + rank] = col;
  });
}

// Parts of a row: what a workgroup can hold, and so many that few rows fill the chip.
struct TopPlan {
  int parts, per;
};
TopPlan plan_of(int64_t rows, int64_t A, int dtype) {
  const int64_t size = dtype_size(dtype), most = (int64_t)1024 * 16 * (16 / size);
  int64_t parts = div_up(A, most);
  if (rows < 128 && A * size > 32768) {
    const int64_t fill = div_up(256, rows), small = div_up(A * size, 16384);
    const int64_t more = fill < small ? fill : small;
    if (more > parts) parts = more;
  }
  if (parts > kMaxParts) parts = kMaxParts;  // (2^22 elements: 64 of 2^16)
  // (parts start at multiples of 16 bytes of the row)
  const int64_t per = round_up(div_up(A, parts), 16 / size);
  return {(int)div_up(A, per), (int)per};
}

}  // namespace
}  // namespace ppo

extern "C" size_t ppo_token_top_workspace_bytes(int64_t rows, int64_t A, int64_t K, int dtype) {
  using namespace ppo;
  if (rows <= 0 || A <= 0 || K <= 0 || !dtype_ok(dtype) || A > ((int64_t)1 << 22)) return 0;
  const TopPlan plan = plan_of(rows, A, dtype);
  return plan.parts == 1 ? 0 : (size_t)(rows * plan.parts * K) * sizeof(u64);
}

extern "C" int ppo_token_top(const void* logits, int dtype, int64_t rows, int64_t A, int64_t K,
                             void* values, int64_t* ids, void* workspace, size_t workspace_bytes,
                             void* stream_ptr) {
  using namespace ppo;
  if (!dtype_ok(dtype) || rows < 0 || A <= 0 || K <= 0 || K > A) return PPO_ERR_INVALID_ARG;
  if (rows == 0) return PPO_OK;
  if (!logits || !values || !ids || (uintptr_t)logits % dtype_size(dtype) ||
      (uintptr_t)values % dtype_size(dtype))
    return PPO_ERR_INVALID_ARG;
  if (K > kMaxK || A > ((int64_t)1 << 22)) return PPO_ERR_TOO_LARGE;
  const TopPlan plan = plan_of(rows, A, dtype);
  if (rows > (((int64_t)1 << 31) - 1) / plan.parts)
    return PPO_ERR_TOO_LARGE;
  if (plan.parts > 1 && (!workspace || !aligned16(workspace) ||
                         workspace_bytes < ppo_token_top_workspace_bytes(rows, A, K, dtype)))
    return PPO_ERR_WORKSPACE;
  hipStream_t stream = (hipStream_t)stream_ptr;
  u64* found = static_cast<u64*>(workspace);
  return with_dtype(dtype, [&](auto zero) {
    using T = decltype(zero);
    const T* in = static_cast<const T*>(logits);
    T* out = static_cast<T*>(values);
    auto go = [&](auto lanes, auto held) {
      constexpr int G = decltype(lanes)::value, V = decltype(held)::value;
      hipLaunchKernelGGL((top_kernel<T, G, V>), dim3((unsigned)(rows * plan.parts)), dim3(G), 0,
                         stream, in, rows, (int)A, (int)K, plan.parts, plan.per, out, ids, found);
      return last_launch_status();
    };
    const int64_t chunks = chunks_of(plan.per, dtype);
    const int code = chunks <= 256 * 1    ? go(Int<256>{}, Int<1>{})
                     : chunks <= 256 * 2  ? go(Int<256>{}, Int<2>{})
                     : chunks <= 256 * 4  ? go(Int<256>{}, Int<4>{})
                     : chunks <= 256 * 8  ? go(Int<256>{}, Int<8>{})
                     : chunks <= 512 * 8  ? go(Int<512>{}, Int<8>{})
                     : chunks <= 1024 * 8 ? go(Int<1024>{}, Int<8>{})
                                          : go(Int<1024>{}, Int<16>{});
    if (code || plan.parts == 1) return code;
    hipLaunchKernelGGL((top_merge_kernel<T>), dim3((unsigned)rows), dim3(1024), 0, stream, in,
                       (int)A, (int)K, plan.parts, out, ids, found);
    return last_launch_status();
  });
}
