// The K largest logits of each row, in order.  A logit and its column make one
// 64-bit whole number (the logit's order above, the column's complement below), by
// which no two of a row are alike: ties need no care of their own.
//
// A workgroup takes a row, or a part of one.  Its lanes keep the largest of what they
// read, in up to sixteen segments each; the K-th largest of the lanes' own maxima bounds the K-th
// largest element from below, so the few segments that reach it (about K of them) are
// all that is looked at again, and the few elements there that do are sorted, by
// counting for each how many precede it.  Rows in which too many reach the bound (many
// equal logits) are settled by a radix search for the threshold itself.  What bounds
// it: HBM reads; a row is in the caches when parts of it are read again (4096 x 32001
// fp32, K = 64, 94 us, 5.5 TB/s, while a workgroup waits for its bound another one
// reads; with segments of eight rounds for two 120, since each one's chunks are lines of
// their own); a single row two launches of 8 and 4 us.
#include "tokens_rows.hpp"

namespace ppo {
namespace {

constexpr int kMaxK = PPO_TOKEN_MAX_K;
// Elements that are sorted at most.
template <int G>
constexpr int kSorted = G == kWave ? 512 : 2048;
constexpr int kSegments = 16;
constexpr int kAgain = 4;  // segments a lane to look at again at most

typedef unsigned long long u64;

// A logit's order as an unsigned number above 0; -0 is 0, NaN is before everything.
constexpr unsigned kNanOrder = 0xFFFFFFFFu;
__device__ __forceinline__ unsigned order_of(float l) {
  const unsigned b = __builtin_bit_cast(unsigned, l + 0.0f);
  const unsigned k = b ^ ((unsigned)((int)b >> 31) | 0x80000000u);
  return l != l ? kNanOrder : k;
}
__device__ __forceinline__ u64 place(unsigned order, int col) {
  return (u64)order << 32 | (unsigned)~col;
}
__device__ __forceinline__ int column_of(u64 x) { return (int)~(unsigned)x; }

template <int G>
struct Board {
  u64 list[kSorted<G>];
  union {
    unsigned best[G];
    unsigned short again[kAgain * G];  // lane + G segment of segments to look at again
    int bins[256];
  };
  unsigned bound;
  int count, items;
  int part[G / kWave];
};

template <int G>
__device__ __forceinline__ void append(Board<G>& b, unsigned order, int col) {
  const int at = atomicAdd(&b.count, 1);
  if (at < kSorted<G>) b.list[at] = place(order, col);
}

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

// The largest 16-bit prefix that K lanes' best reach (1 if fewer lanes have any), for
// every lane; b.count and b.items are 0 afterwards.
template <int G>
__device__ __forceinline__ unsigned bound_of(Board<G>& b, int K, unsigned best) {
  b.best[threadIdx.x] = best;
  if (threadIdx.x == 0) b.count = b.items = 0;
  lds_barrier();
  if (threadIdx.x < kWave) {
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
  return b.bound;
}

// Calls out(rank, element) for each of the listed elements among the K largest, and for
// ranks that none has with element 0.  (There are such only where the logits change
// between the looks at them; no address may then come from what was never found.)
template <int G, class Out>
__device__ __forceinline__ void ranked(const Board<G>& b, int K, Out&& out) {
  const int n = min(b.count, kSorted<G>);
  for (int i = threadIdx.x; i < n; i += G) {
    const u64 x = b.list[i];
    int rank = 0;
    for (int k = 0; k < n; ++k) rank += b.list[k] > x;
    if (rank < K) out(rank, x);
  }
  for (int k = n + threadIdx.x; k < K; k += G) out(k, 0);
}

// A row's result of one rank.
template <class T>
__device__ __forceinline__ void leave(const T* row, u64 x, T* value, int64_t* id) {
  const int col = x ? column_of(x) : 0;
  *value = x ? row[col] : from_f32<T>(PPO_NAN);
  *id = col;
}

// A row, or a part of one from column `from` on.
template <class T, int G>
struct Part {
  static constexpr int kN = kPer16<T>;
  const T* row;
  const v4i* body;
  int from;
  Cut<T> cut;
  int rounds;  // of G chunks a segment: 1, 2, or a multiple of 4

  __device__ __forceinline__ Part(const T* row_, int from_, int width)
      : row(row_), from(from_), cut(row_ + from_, width) {
    body = reinterpret_cast<const v4i*>(row + from + cut.head);
    const int all = (cut.nvec + G - 1) / G;
    rounds = all <= kSegments       ? 1
             : all <= 2 * kSegments ? 2
                                    : (all + 4 * kSegments - 1) / (4 * kSegments) * 4;
  }
  __device__ __forceinline__ int end_column(int e) const { return from + cut.end_column(e); }
  __device__ __forceinline__ int column(int chunk) const { return from + cut.head + chunk * kN; }

  // f(order, column) for each element of the lane.
  template <class F>
  __device__ __forceinline__ void each(F&& f) const {
    const int t = threadIdx.x;
    if (t < cut.ends) f(order_of(to_f32(row[end_column(t)])), end_column(t));
    for (int i = t; i < cut.nvec; i += G) {
      const v4i w = body[i];
#pragma unroll
      for (int j = 0; j < kN; ++j) f(order_of(unpack<T>(w, j)), column(i) + j);
    }
  }
};

// Too many elements reach the bound: the K-th largest order, byte by byte, the elements
// above it, and of those equal to it the first ones by column.
template <class T, int G>
__device__ void settle(const Part<T, G>& p, Board<G>& b, int K) {
  const int t = threadIdx.x;
  unsigned kth = 0;
  int left = K;  // elements of the K among those that share kth's leading bytes
  for (int shift = 24; shift >= 0; shift -= 8) {
    lds_barrier();
    for (int i = t; i < 256; i += G) b.bins[i] = 0;
    lds_barrier();
    p.each([&](unsigned order, int) {
      if (shift < 24 && (order ^ kth) >> (shift + 8)) return;
      const int bin = order >> shift & 255;
      // (equal logits: one lane counts for the others)
      const u64 active = __ballot(1), alike = __ballot(bin == __builtin_amdgcn_readfirstlane(bin));
      if (alike == active) {
        if ((t & (kWave - 1)) == __builtin_ctzll(active))
          atomicAdd(&b.bins[bin], __builtin_popcountll(active));
      } else {
        atomicAdd(&b.bins[bin], 1);
      }
    });
    lds_barrier();
    int bin = 255;
    for (; bin > 0 && b.bins[bin] < left; --bin) left -= b.bins[bin];
    kth |= (unsigned)bin << shift;
  }
  lds_barrier();
  if (t == 0) b.count = 0;
  lds_barrier();
  p.each([&](unsigned order, int col) {
    if (order > kth) append(b, order, col);
  });
  lds_barrier();
  // `left` of the equal ones: the head's elements, the chunks round by round, the tail's
  auto ends = [&](int e, int last) {
    if (t == 0)
      for (; e < last && left > 0; ++e)
        if (order_of(to_f32(p.row[p.end_column(e)])) == kth) {
          append(b, kth, p.end_column(e));
          --left;
        }
    if (t == 0) b.items = left;
    lds_barrier();
    left = b.items;
    lds_barrier();
  };
  ends(0, p.cut.head);
  for (int base = 0; base < p.cut.nvec && left > 0; base += G) {
    const int i = base + t;
    unsigned mine = 0;
    if (i < p.cut.nvec) {
      const v4i w = p.body[i];
#pragma unroll
      for (int j = 0; j < Part<T, G>::kN; ++j)
        mine |= (unsigned)(order_of(unpack<T>(w, j)) == kth) << j;
    }
    // how many lie before this lane's: by its wave's bits, and the waves before
    int n = 0;
#pragma unroll
    for (int j = 0; j < Part<T, G>::kN; ++j)
      n += __builtin_popcountll(__ballot(mine >> j & 1) & ((1ull << (t & (kWave - 1))) - 1));
    const int all = __builtin_amdgcn_readlane(n + __builtin_popcount(mine), kWave - 1);
    if ((t & (kWave - 1)) == 0) b.part[t / kWave] = all;
    lds_barrier();
    int total = 0;
    for (int w = 0; w < G / kWave; ++w) {
      if (w < t / kWave) n += b.part[w];
      total += b.part[w];
    }
    for (int j = 0; j < Part<T, G>::kN; ++j)
      if (mine >> j & 1) {
        if (n < left) append(b, kth, p.column(i) + j);
        ++n;
      }
    left = total < left ? left - total : 0;
    lds_barrier();
  }
  ends(p.cut.head, p.cut.ends);
}

// Part `q` of `parts` of each row; one part: the row's results, else its largest
// elements to `found` [rows][parts][K], 0 behind the last.
template <class T, int G, bool kPast>
__global__ void __launch_bounds__(G) top_kernel(const T* logits, int A, int K, int parts, int per,
                                                T* values, int64_t* ids, u64* found) {
  constexpr int kN = kPer16<T>;
  __shared__ Board<G> b;
  const int t = threadIdx.x;
  const int64_t r = (int64_t)blockIdx.x / parts;
  const int q = (int)((int64_t)blockIdx.x - r * parts);
  const int from = q * per, width = min(per, A - from), want = min(K, width);
  const Part<T, G> p(logits + r * A, from, width);

  // (the largest of a segment as a float, and whether a NaN was among them)
  unsigned best[kSegments] = {}, most = 0;
  const float end = t < p.cut.ends ? to_f32(p.row[p.end_column(t)]) : kNegInf;
  const int nvec = p.cut.nvec;
  // Four chunks of a lane at a time: 4 / kRounds segments, or a quarter of rounds / 4 of one.
  auto look = [&](auto of_segment) {
    constexpr int kRounds = decltype(of_segment)::value, kOf = 4 / kRounds;
#pragma unroll
    for (int s = 0; s < kSegments; s += kOf) {
      if (s * p.rounds * G >= nvec) break;
      float m[kOf];
      bool nan[kOf];
#pragma unroll
      for (int c = 0; c < kOf; ++c) {
        m[c] = kNegInf;
        nan[c] = false;
      }
      const int to = min(nvec, (s + kOf) * p.rounds * G);
      for (int at = s * p.rounds * G; at < to; at += 4 * G) {
        v4i w[4];
#pragma unroll
        for (int k = 0; k < 4; ++k)
          w[k] = at + k * G + t >= nvec ? no_chunk<T>()
                 : kPast ? __builtin_nontemporal_load(p.body + at + k * G + t)
                         : p.body[at + k * G + t];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          if (at + k * G >= nvec) break;
#pragma unroll
          for (int j = 0; j < kN; ++j) {
            const float l = unpack<T>(w[k], j);
            m[k / kRounds] = fmaxf(m[k / kRounds], l);
            nan[k / kRounds] |= l != l;
          }
        }
      }
#pragma unroll
      for (int c = 0; c < kOf; ++c)
        if ((s + c) * p.rounds * G + t < nvec) {
          best[s + c] = nan[c] ? kNanOrder : order_of(m[c]);
          most = max(most, best[s + c]);
        }
    }
  };
  if (p.rounds == 1)
    look(Int<1>{});
  else if (p.rounds == 2)
    look(Int<2>{});
  else
    look(Int<4>{});
  const unsigned end_order = t < p.cut.ends ? order_of(end) : 0;
  const unsigned bound = bound_of(b, want, max(most, end_order));
  if (end_order >= bound) append(b, end_order, p.end_column(t));
#pragma unroll
  for (int s = 0; s < kSegments; ++s) {
    if (s * p.rounds * G >= nvec) break;
    if (best[s] >= bound) {
      const int at = atomicAdd(&b.items, 1);
      if (at < kAgain * G) b.again[at] = (unsigned short)(s * G + t);
    }
  }
  lds_barrier();
  const bool many = b.items > kAgain * G;
  const int items = many ? 0 : b.items * p.rounds;
  for (int i = t; i < items; i += G) {
    const int item = i / p.rounds, who = b.again[item], s = who / G;
    const int chunk = (s * p.rounds + i - item * p.rounds) * G + who % G;
    if (chunk >= nvec) continue;
    const v4i w = p.body[chunk];
#pragma unroll
    for (int j = 0; j < kN; ++j) {
      const unsigned order = order_of(unpack<T>(w, j));
      if (order >= bound) append(b, order, p.column(chunk) + j);
    }
  }
  lds_barrier();
  if (many || b.count > kSorted<G>) settle(p, b, want);
  if (parts == 1) {
    ranked<G>(b, K, [&](int rank, u64 e) {
      leave(p.row, e, values + r * K + rank, ids + r * K + rank);
    });
  } else {
    u64* to = found + (int64_t)blockIdx.x * K;
    ranked<G>(b, K, [&](int rank, u64 e) { to[rank] = e; });
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
    best = max(best, (unsigned)(x[i] >> 32));
  }
  // A bound of the K-th largest: where each part gives its share of the K, the least of the
  // last ones (it lets about three times K by of random rows, and is there 2 us before
  // the closer one); of many candidates the closer one.
  unsigned bound;
  if (n <= kSorted<1024>) {
    if (threadIdx.x == 0) b.count = 0;
    const int lane = threadIdx.x & (kWave - 1), share = (K + parts - 1) / parts;
    bound = lane < parts ? (unsigned)(from[lane * K + share - 1] >> 32) : ~0u;
    for (int d = 1; d < kWave; d <<= 1) bound = min(bound, (unsigned)__shfl_xor((int)bound, d));
    bound = max(bound, 1u);
    lds_barrier();
  } else {
    bound = bound_of(b, K, best);
  }
#pragma unroll
  for (int i = 0; i < kMergeV; ++i)
    if ((unsigned)(x[i] >> 32) >= bound)  // (above 0)
      append(b, (unsigned)(x[i] >> 32), column_of(x[i]));
  lds_barrier();
  if (b.count > kSorted<1024>) {  // (no two are alike: the K-th by its bits)
    lds_barrier();
    u64 kth = 0;
    for (u64 bit = 1ull << 63; bit; bit >>= 1) {
      int above = 0;
#pragma unroll
      for (int i = 0; i < kMergeV; ++i) above += x[i] >= (kth | bit);
      if (block_count(above, b) >= K) kth |= bit;
    }
    if (threadIdx.x == 0) b.count = 0;
    lds_barrier();
#pragma unroll
    for (int i = 0; i < kMergeV; ++i)
      if (x[i] && x[i] >= kth) append(b, (unsigned)(x[i] >> 32), column_of(x[i]));
    lds_barrier();
  }
  ranked<1024>(b, K, [&](int rank, u64 e) {
    leave(logits + r * A, e, values + r * K + rank, ids + r * K + rank);
  });
}

// Parts of a row, so many that few rows fill the chip, of 16 KB at least, and below 512
// rows of about 2^16 elements at most; of more rows one.
struct TopPlan {
  int parts, per;
};
constexpr int64_t kPartElements = 1 << 16;
// Logits of more than the last-level cache holds are read past it (1024 x 200000 bf16, K = 32,
// 85 -> 76 us; 147 MB of them that lie there 24 -> 27).
constexpr int64_t kCacheBytes = (int64_t)256 << 20;
// Bytes of a row that a wave takes by itself (16384 x 2000 bf16 49 -> 25 us; 4096 x 4000
// fp32 20 -> 22).
constexpr int64_t kWaveRow = 8192;
TopPlan plan_of(int64_t rows, int64_t A, int dtype) {
  const int64_t size = dtype_size(dtype);
  int64_t parts = div_up(A, kPartElements);
  if (rows >= 512) parts = 1;
  if (rows < 256 && A * size > 32768)
    parts = std::max(parts, std::min(div_up(512, rows), div_up(A * size, 16384)));
  if (parts > kMaxParts) parts = kMaxParts;
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
      (uintptr_t)values % dtype_size(dtype) || (uintptr_t)ids % 8)
    return PPO_ERR_INVALID_ARG;
  if (K > kMaxK || A > ((int64_t)1 << 22)) return PPO_ERR_TOO_LARGE;
  const TopPlan plan = plan_of(rows, A, dtype);
  // (K of the lanes' maxima: the bound lies close to the K-th element, and few reach it,
  // with more lanes than K)
  const int lanes = plan.parts == 1 && A * dtype_size(dtype) <= kWaveRow && (K <= 48 || A <= 512)
                        ? kWave
                    : K <= 96  ? 256
                    : K <= 192 ? 512
                               : 1024;
  if (!fits_launch(rows * plan.parts, lanes)) return PPO_ERR_TOO_LARGE;  // (parts: of few rows)
  if (plan.parts > 1 && (!workspace || !aligned16(workspace) ||
                         workspace_bytes < ppo_token_top_workspace_bytes(rows, A, K, dtype)))
    return PPO_ERR_WORKSPACE;
  hipStream_t stream = (hipStream_t)stream_ptr;
  u64* found = static_cast<u64*>(workspace);
  return with_dtype(dtype, [&](auto zero) {
    using T = decltype(zero);
    const T* in = static_cast<const T*>(logits);
    T* out = static_cast<T*>(values);
    const bool past = rows * A * dtype_size(dtype) > kCacheBytes;
    auto go = [&](auto group) {
      constexpr int G = decltype(group)::value;
      const auto kernel = past ? top_kernel<T, G, true> : top_kernel<T, G, false>;
      hipLaunchKernelGGL(kernel, dim3((unsigned)(rows * plan.parts)), dim3(G), 0, stream, in, (int)A,
                         (int)K, plan.parts, plan.per, out, ids, found);
      return last_launch_status();
    };
    const int code = lanes == kWave ? go(Int<kWave>{})
                     : lanes == 256 ? go(Int<256>{})
                     : lanes == 512 ? go(Int<512>{})
                                    : go(Int<1024>{});
    if (code || plan.parts == 1) return code;
    hipLaunchKernelGGL((top_merge_kernel<T>), dim3((unsigned)rows), dim3(1024), 0, stream, in,
                       (int)A, (int)K, plan.parts, out, ids, found);
    return last_launch_status();
  });
}
