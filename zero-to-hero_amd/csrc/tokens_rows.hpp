// Passes over rows of logits by any number of workgroups to a row: the statistics
// (read once, nothing kept) and a gradient from them (read once, written once).
#pragma once

#include <algorithm>
#include <type_traits>

#include "tokens.hpp"

namespace ppo {

template <int N>
using Int = std::integral_constant<int, N>;

// What a lane has of a row that it walks, whose length has no bound: the sums of kWalk rounds
// are formed in 32 bits, those of more in 64 (in 32 alone, 2^27 columns of a weight of
// 1/2 + 2^-13 are off by 4e-5; log p and the entropy of 4096 x 50304 bf16 take 65.3 us there,
// 66.3 so, 67.7 with 64 bits in every round).
struct Walked {
  float m;
  double s, u;
};
constexpr int kWalk = 8;

// Statistics of chunks [part / splits) of a row, by G lanes, two chunks of each lane at
// a time (four and eight are slower: 50304 bf16 69, 72 and 76 us of 4096 rows; of short
// rows one); the sums follow the running maximum.  `again`: the rows are read again
// soon, and stay in the caches.
template <class T, int G, bool kEntropy, class S>
__device__ __forceinline__ S stream_stat(const T* row, int A, int a, const Scale<S>& c, int t,
                                         int part, int splits, bool again) {
  constexpr int kN = kPer16<T>, kU = G == 16 ? 1 : 2;
  constexpr bool kLong = G > kWave;  // (smaller groups have rows of a few rounds)
  const Cut<T> cut(row, A);
  const v4i* body = reinterpret_cast<const v4i*>(row + cut.head);
  const int per = (cut.nvec + splits - 1) / splits;
  const int end = min(cut.nvec, (part + 1) * per);
  const int b = a - cut.head, va = a >= 0 && b >= 0 ? b / kN : -1;  // the action's chunk
  S x = {kNegInf, 0.0f, 0.0f};
  if (part == 0 && t < cut.ends) {
    const int col = cut.end_column(t);
    const float l = col == a ? kNegInf : to_f32(row[col]);
    x.m = l;
    const float d = l == kNegInf ? l : l - l;  // (NaN and +inf give NaN)
    x.s = exp2_fast(d);
  }
  Walked all = {kNegInf, 0.0, 0.0};
  for (int i = part * per + t; i < end;) {
    const int stop = kLong ? min(end, i + kWalk * kU * G) : end;
    for (; i < stop; i += kU * G) {
      v4i w[kU];
#pragma unroll
      for (int k = 0; k < kU; ++k)
        w[k] = i + k * G >= end ? no_chunk<T>()
               : again          ? body[i + k * G]
                                : __builtin_nontemporal_load(body + i + k * G);
      float m = x.m;
#pragma unroll
      for (int k = 0; k < kU; ++k) {
        if (i + k * G == va) knock_out<T>(w[k], b - va * kN);
#pragma unroll
        for (int j = 0; j < kN; ++j) m = fmaxf(m, unpack<T>(w[k], j));
      }
      rebase<kEntropy>(x, m, c);
      if (m == kNegInf) m = 0.0f;
      decltype(x.s) s2 = 0.0f;
#pragma unroll
      for (int k = 0; k < kU; ++k)
#pragma unroll
        for (int j = 0; j < kN; ++j) {
          const float d = c(unpack<T>(w[k], j) - m), e = exp2_fast(d);
          (j & 1 ? s2 : x.s) += e;
          if (kEntropy) x.u = fmaf(e, fmaxf(d, -1e30f), x.u);
        }
      x.s += s2;
    }
    if (kLong && i < end) {
      rebase<kEntropy>(all, x.m, c);
      all.s += x.s;
      if (kEntropy) all.u += x.u;
      x.s = x.u = 0.0f;
    }
  }
  if (kLong && all.s != 0.0) {  // (or NaN)
    rebase<kEntropy>(all, x.m, c);
    x.s = (decltype(x.s))(all.s + x.s);
    if (kEntropy) x.u = (float)(all.u + x.u);
  }
  return x;
}

template <class T>
__device__ __forceinline__ float action_logit(const T* row, int a) {
  return a >= 0 ? to_f32(row[a]) : PPO_NAN;
}

// One group to a row and the row finished by it (kDirect), or `splits` workgroups to
// a row that leave their parts.  What bounds it: HBM reads.
template <class T, int G, bool kEntropy, bool kDirect, class Emit>
__global__ void __launch_bounds__(256) statistics_kernel(Rows rows, Emit emit,
                                                         typename Emit::Sums* parts, int splits,
                                                         bool again) {
  using S = typename Emit::Sums;
  __shared__ S s_part[4];
  const Scale<S> c(rows);
  const int t = threadIdx.x % G;
  const int64_t group = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
  const int64_t r = kDirect ? group : group / splits;
  if (r >= rows.n) return;  // (with G = 256 the whole workgroup)
  const int part = kDirect ? 0 : (int)(group - r * splits);
  if (!rows.live(r)) {
    if (kDirect && t == 0) emit.masked(r);
    return;
  }
  const T* row = static_cast<const T*>(rows.logits) + r * rows.A;
  const int a = rows.actions ? rows.action(r) : -1;
  const float la = kDirect ? action_logit(row, a) : 0.0f;
  S x = stream_stat<T, G, kEntropy>(row, rows.A, a, c, t, part, splits, again);
  if (G > kWave) {
    x = block_join<kEntropy>(x, c, s_part);
    if (threadIdx.x >= kWave) return;
  } else {
    x = lanes_join<G <= kWave ? G : kWave, kEntropy>(x, c);
  }
  if constexpr (kDirect)
    emit.template row<kEntropy>(rows, r, x, la, t == 0);
  else if (t == 0)
    parts[group] = x;
}

// The parts of row r as one, by every group of lanes that asks for them (groups smaller
// than a wave have rows of one part).
template <int G, bool kEntropy, class S>
__device__ __forceinline__ S join_parts(const S* parts, int64_t r, int splits, const Scale<S>& c) {
  if (G < kWave) return parts[r];
  const int lane = threadIdx.x & (kWave - 1);
  const S x = lane < splits ? parts[r * splits + lane] : S{kNegInf, 0.0f, 0.0f};
  return lanes_join<kWave, kEntropy>(x, c);
}

// A wave to a row: its parts joined in the order of their lanes, and the row
// finished by its lane 0, or by the wave (kWholeWave).
template <class T, bool kEntropy, class Emit>
__global__ void __launch_bounds__(64) join_kernel(Rows rows, Emit emit,
                                                  const typename Emit::Sums* parts, int splits) {
  const int lane = threadIdx.x;
  for (int64_t r = blockIdx.x; r < rows.n; r += gridDim.x) {
    if (!rows.live(r)) {
      if (lane == 0) emit.masked(r);
      continue;
    }
    const T* row = static_cast<const T*>(rows.logits) + r * rows.A;
    const int a = rows.actions ? rows.action(r) : -1;
    const float la = action_logit(row, a);
    const auto x = join_parts<kWave, kEntropy>(parts, r, splits, Scale<typename Emit::Sums>(rows));
    if constexpr (Emit::kWholeWave)
      emit.row(rows, r, row, x, lane);
    else
      emit.template row<kEntropy>(rows, r, x, la, lane == 0);
  }
  emit.end();
}

// Logits that the last-level cache holds from the forward to the backward pass (at 412 MB
// of them 208 -> 200 us for both, at 537 as much as without).
constexpr int64_t kReadAgain = (int64_t)512 << 20;

// Enqueues the parts of every row's statistics; their number.
template <class T, bool kEntropy, class Emit>
int launch_parts(const Rows& rows, const Scratch& s, const Emit& emit, bool again,
                 hipStream_t stream, int& splits) {
  splits = row_splits(rows.n, rows.A, sizeof(T) == 4 ? PPO_DTYPE_F32 : PPO_DTYPE_BF16);
  if (!fits_launch(rows.n * splits, 256)) return PPO_ERR_TOO_LARGE;
  hipLaunchKernelGGL((statistics_kernel<T, 256, kEntropy, false, Emit>),
                     dim3((unsigned)(rows.n * splits)), dim3(256), 0, stream, rows, emit,
                     reinterpret_cast<typename Emit::Sums*>(s.parts), splits, again);
  return last_launch_status();
}

template <class T, bool kEntropy, bool kMayDirect, class Emit>
int launch_statistics(const Rows& rows, const Scratch& s, const Emit& emit, bool again,
                      hipStream_t stream) {
  const int dtype = sizeof(T) == 4 ? PPO_DTYPE_F32 : PPO_DTYPE_BF16;  // (sizes alike)
  const int splits = row_splits(rows.n, rows.A, dtype);
  if constexpr (kMayDirect)
    if (splits == 1) {
      const int64_t chunks = chunks_of(rows.A, dtype);
      auto go = [&](auto lanes) {
        constexpr int G = decltype(lanes)::value;
        const int64_t blocks = div_up(rows.n, 256 / G);
        if (!fits_launch(blocks, 256)) return (int)PPO_ERR_TOO_LARGE;
        hipLaunchKernelGGL((statistics_kernel<T, G, kEntropy, true, Emit>), dim3((unsigned)blocks),
                           dim3(256), 0, stream, rows, emit, nullptr, 1, again);
        return last_launch_status();
      };
      if (chunks <= 64) return go(Int<16>{});
      if (chunks <= 512) return go(Int<64>{});
      return go(Int<256>{});
    }
  int parts;
  if (const int code = launch_parts<T, kEntropy>(rows, s, emit, again, stream, parts)) return code;
  hipLaunchKernelGGL((join_kernel<T, kEntropy, Emit>), dim3(launch_blocks(rows.n, kMaxPartials)),
                     dim3(64), 0, stream, rows, emit,
                     reinterpret_cast<const typename Emit::Sums*>(s.parts), splits);
  return last_launch_status();
}

// What a gradient pass asks of a row, by the G lanes of one of its pieces: begin() comes
// before the first, with all lanes of every wave; row() gives its terms (called by whole
// groups, so lanes may work together; `first`: the row's first piece, t the lane in its
// group, board the group's or the wave's share of LDS), masked() is called for a row that
// does not count, after() when the piece is written (kAfter).
struct GradientTerms {
  static constexpr bool kAfter = false;
  __device__ __forceinline__ void begin() {}
  __device__ __forceinline__ void masked(const Rows&, int64_t, bool) const {}
};

// Columns of a piece of a row: [from, to) of its body, and its ends where it is the first.
struct PieceColumns {
  int from, to, body, body_end;
  bool first;
  __device__ __forceinline__ bool has(int col) const {
    return col >= body && col < body_end ? col >= from && col < to : first;
  }
};

// dlogits from the logits and the rows' terms: G lanes to a piece of a row, four
// chunks to a lane.  What bounds it: HBM, one read and one write of the rows.
constexpr int kGradU = 4;
template <class T, int G, bool kC, class Terms>
__global__ void __launch_bounds__(256) gradient_kernel(Rows rows, Terms terms, const float* scale,
                                                       float held, T* dlogits, int64_t pieces,
                                                       int board_ints) {
  constexpr int kN = kPer16<T>;
  extern __shared__ __attribute__((aligned(16))) int s_boards[];
  const float up = scale ? *scale : 1.0f;
  if (held != 0.0f && up == held) return;
  terms.begin();
  const int t = threadIdx.x % G;
  int* board = s_boards + threadIdx.x / (G < kWave ? G : kWave) * board_ints;
  const int64_t groups = rows.n * pieces, step = (int64_t)gridDim.x * (256 / G);
  for (int64_t group = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G; group < groups;
       group += step) {
    const int64_t r = group / pieces;
    const int piece = (int)(group - r * pieces);
    const T* row = static_cast<const T*>(rows.logits) + r * rows.A;
    T* out = dlogits + r * rows.A;
    const bool live = rows.live(r);
    const Cut<T> cut(live ? row : out, rows.A);
    const int first = piece * (G * kGradU) + t;
    T* to = out + cut.head;
    const int64_t per = (int64_t)G * kN;
    const bool ends = piece == 0 && t < cut.ends;
    const int end_col = ends ? cut.end_column(t) : 0;
    if (!live) {
      const v4i none = {0, 0, 0, 0};
#pragma unroll
      for (int k = 0; k < kGradU; ++k)
        if (first + k * G < cut.nvec) store16(to + (int64_t)first * kN + k * per, none, true);
      if (ends) out[end_col] = from_f32<T>(0.0f);
      terms.masked(rows, r, piece == 0 && t == 0);
      continue;
    }
    const v4i* body = reinterpret_cast<const v4i*>(row + cut.head);
    v4i w[kGradU];
#pragma unroll
    for (int k = 0; k < kGradU; ++k)
      if (first + k * G < cut.nvec) w[k] = __builtin_nontemporal_load(body + first + k * G);
    const float end = ends ? to_f32(row[end_col]) : kNegInf;
    const Grad g = terms.template row<T, G>(rows, r, row, up, rows.actions ? rows.action(r) : -1, t,
                                            piece == 0, board);
    const bool vec = ((uintptr_t)to & 15) == 0;
    const int b = g.a - cut.head;
    const int va = g.a >= 0 && b >= 0 ? b / kN : -1;
#pragma unroll
    for (int k = 0; k < kGradU; ++k) {
      const int v = first + k * G;
      if (v >= cut.nvec) continue;
      float d[kN];
#pragma unroll
      for (int j = 0; j < kN; ++j) {
        d[j] = grad_at<kC>(g, rows.c, unpack<T>(w[k], j));
        if (v == va && j == b - va * kN) d[j] = g.da;
      }
      store16(to + (int64_t)v * kN, pack<T>(d), vec);
    }
    if (ends) out[end_col] = from_f32<T>(end_col == g.a ? g.da : grad_at<kC>(g, rows.c, end));
    if constexpr (Terms::kAfter) {
      if (G > kWave)
        __syncthreads();  // (the piece is written, by all its waves)
      else
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      const int from = cut.head + piece * (G * kGradU) * kN;
      const PieceColumns cols = {from, from + G * kGradU * kN, cut.head, cut.head + cut.nvec * kN,
                                 piece == 0};
      if (G <= kWave || threadIdx.x < kWave)
        terms.template after<T, G>(rows, g, out, cols, t, board);
      if (G > kWave) lds_barrier();
    }
  }
}

// A pass that may find nothing to do has workgroups enough to fill the chip, and few
// enough to end in 2 us (131072 of them took 29); one that has work one to a piece.
constexpr int64_t kHeldBlocks = 2048;
// Words of LDS that each of a workgroup's sixteen groups of 16 lanes may have; with more,
// rows go one to a wave.
constexpr int kQuadBoard = 640;
template <class T, bool kC, class Terms>
int launch_gradient(const Rows& rows, const Terms& terms, const float* scale, float held,
                    T* dlogits, int board_ints, hipStream_t stream) {
  const int dtype = sizeof(T) == 4 ? PPO_DTYPE_F32 : PPO_DTYPE_BF16;
  const int64_t chunks = chunks_of(rows.A, dtype);
  auto go = [&](auto lanes) {
    constexpr int G = decltype(lanes)::value;
    const int64_t pieces = div_up(chunks, G * kGradU);
    const int64_t most = held != 0.0f ? kHeldBlocks : ((int64_t)1 << 24) - 1;  // (2^32 lanes)
    hipLaunchKernelGGL((gradient_kernel<T, G, kC, Terms>),
                       dim3((unsigned)std::min(div_up(rows.n * pieces, 256 / G), most)), dim3(256),
                       (size_t)board_ints * (256 / std::min(G, kWave)) * sizeof(int), stream, rows,
                       terms, scale, held, dlogits, pieces, board_ints);
    return last_launch_status();
  };
  if (chunks <= 64 && board_ints <= kQuadBoard) return go(Int<16>{});
  if (chunks <= 512) return go(Int<64>{});
  return go(Int<256>{});
}

// A pass's workgroup, and the waves a SIMD is to hold at least: two workgroups of 512
// lanes (65536 bf16 218 -> 214 us, 50304 198 -> 187); smaller ones do better with the
// registers (32768 191 us, 211 with four waves to a SIMD).
template <int G>
constexpr int kRowBlock = G < 256 ? 256 : G;
template <int G>
constexpr int kRowWaves = G >= 512 ? 4 : 1;

// Workgroups of 512 and 1024 lanes, of which a CU holds two or one, take row after row
// and read the next one while they write (131072 bf16 909 -> 851 us of 8192 rows); so
// there are as many as run at once, and the rows are ordered for them.  Smaller ones
// overlap by their number, and come as the rows do (32768 85 us, 93 the other way).
template <int G>
constexpr bool kRowAfterRow = G >= 512;
template <int G>
constexpr int kRowBlocks = G == 1024 ? 256 : G == 512 ? 512 : kMaxPartials;

// The rows of a group: every step-th from its first on.
template <int G>
struct Walk {
  const Rows& rows;
  Order order;
  int64_t step;
  int live;

  __device__ __forceinline__ Walk(const Rows& rows_, const Order& order_, int64_t step_)
      : rows(rows_), order(order_), step(step_),
        live(kRowAfterRow<G> && order.rows ? *order.live : (int)rows.n) {}
  __device__ __forceinline__ int64_t row(int64_t i) const {
    return kRowAfterRow<G> && order.rows ? order.rows[i] : i;
  }
  // From place i on the next one whose row counts (rows.n: none); dead(row) for those
  // before it that do not.
  template <class Dead>
  __device__ __forceinline__ int64_t from(int64_t i, Dead&& dead) const {
    if (kRowAfterRow<G>) {
      if (i < live) return i;
      for (; i < rows.n; i += step) dead(row(i));
      return rows.n;
    }
    for (; i < rows.n && !rows.live(i); i += step) dead(i);
    return i;
  }
};

// Whether gradients lie in 16 bytes as the logits do.  (Without gradients: as if they
// started at a multiple of 16, as a caller's allocation does, so that such a loss takes
// the same layout and has the same bits with and without them.)
inline bool lies_alike(const void* logits, const void* dlogits) {
  return ((uintptr_t)logits - (uintptr_t)dlogits) % 16 == 0;
}
// How a pass that keeps its rows in registers is laid out: held(lanes, chunks a lane) for
// the smallest group that holds a row, or split() where a row does not fit, where the
// gradients lie otherwise in 16 bytes than the logits (not `alike`), or where rows are so few
// that one workgroup to each takes longer, the more so the larger it is (a row of 131072
// bf16 24 us by itself; 32 of them 14 split, 64 17, 128 27 either way; of 50304 100 rows 15
// and 16; of 30000 40 rows 13 either way).  The two largest spill (of 320 bytes a lane the
// policy's 80 and the distillation's 156 to 160, of 384 160 to 172 and 236; the policy's in
// fp16 with the entropy's gradient 348) and are faster all the same (1024 x 163840 bf16 196 us
// read twice, 171; 196608 228, 209; 196000 fp16 207, 261 with that gradient).  Of 208 and 256
// bytes the policy's have 12 in scratch, the distillation's 16 and 76.
// Many rows of up to 128 chunks go four to a wave, which then takes their sums' ends together
// (16384 x 1000 bf16 24 us, 31 one to a wave); none do (`least` 64) that need more LDS than
// that leaves, and of more than 64 chunks none that take entries (kSingle).
template <bool kSingle, class Held, class Split>
int with_row_shape(int64_t rows, int64_t chunks, bool alike, int least, Held&& held,
                   Split&& split) {
  if (!alike) return split();
  if (least <= 16) {
    if (chunks <= 16 * 1) return held(Int<16>{}, Int<1>{});
    if (chunks <= 16 * 2) return held(Int<16>{}, Int<2>{});
    if (chunks <= 16 * 4) return held(Int<16>{}, Int<4>{});
  }
  if constexpr (!kSingle)
    if (chunks <= 16 * 8 && rows >= 4096) return held(Int<16>{}, Int<8>{});
  if (chunks <= 64 * 4) return held(Int<64>{}, Int<4>{});
  if (chunks <= 64 * 8) return held(Int<64>{}, Int<8>{});
  if (chunks <= 64 * 16) return held(Int<64>{}, Int<16>{});
  if (chunks <= 256 * 8) return held(Int<256>{}, Int<8>{});
  if (rows < (chunks <= 256 * 16 ? 40 : 65)) return split();
  if (chunks <= 256 * 16) return held(Int<256>{}, Int<16>{});
  if (chunks <= 512 * 10) return held(Int<512>{}, Int<10>{});
  if (chunks <= 512 * 13) return held(Int<512>{}, Int<13>{});
  if (chunks <= 512 * 16) return held(Int<512>{}, Int<16>{});
  if (chunks <= 1024 * 10) return held(Int<1024>{}, Int<10>{});
  if (chunks <= 1024 * 13) return held(Int<1024>{}, Int<13>{});
  if (chunks <= 1024 * 16) return held(Int<1024>{}, Int<16>{});
  if (chunks <= 1024 * 20) return held(Int<1024>{}, Int<20>{});
  if (chunks <= 1024 * 24) return held(Int<1024>{}, Int<24>{});
  return split();
}

}  // namespace ppo
