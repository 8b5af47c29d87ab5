// Distillation from a teacher's K top logits over wide rows of the student's,
// forward and gradient in one pass: dlogits_j = tau w (p_j - q_j), dense in p and
// with at most K columns of q.  Those are written over the dense row afterwards, from
// LDS, so that no element of the row asks whether it is one.  What bounds it: HBM, one
// read and one write of the student's logits (4096 x 65536 bf16 with a mask 194 us, 4.8
// TB/s); few rows the chain of launches (24 x 262144 21 in a graph).
#include "tokens_rows.hpp"

namespace ppo {
namespace {

constexpr int kMaxK = PPO_TOKEN_MAX_K;

struct Teacher {
  const void *logits, *ids;
  int dtype, ids64, K;

  __device__ __forceinline__ float logit(int64_t r, int k) const {
    const int64_t at = r * K + k;
    if (dtype == PPO_DTYPE_F32) return static_cast<const float*>(logits)[at];
    if (dtype == PPO_DTYPE_BF16) return to_f32(static_cast<const bf16*>(logits)[at]);
    return to_f32(static_cast<const fp16*>(logits)[at]);
  }
  // The entry's column; -1: no entry, -2: outside the row.
  __device__ __forceinline__ int column(int64_t r, int k, int A) const {
    const int64_t at = r * K + k;
    const int64_t c = ids64 ? static_cast<const int64_t*>(ids)[at]
                            : (int64_t) static_cast<const int32_t*>(ids)[at];
    return c < 0 ? -1 : c < A ? (int)c : -2;
  }
};

// A row's entries in LDS, K of each: column, q, the sum of q over the column's entries,
// and the student's logit there; and marks of the columns met, 32 kMarkWords bits by a hash.
constexpr int kMarkWords = 128;
struct Board {
  int* col;
  float *q, *sum, *l;
  unsigned* marks;
  __device__ __forceinline__ Board(int* p, int K, int place) {
    const int per = (K + 3) & ~3;
    col = p + place * (4 * per + kMarkWords);
    q = reinterpret_cast<float*>(col) + per;
    sum = q + per;
    l = sum + per;
    marks = reinterpret_cast<unsigned*>(l) + per;
  }
};
int board_ints(int K) { return 4 * (int)round_up(K, 4) + kMarkWords; }

// What the entries come to: sum q (1; 0 without entries; NaN with one that is not finite)
// and the loss but for the student's m and log s:
//   sum_k q_k (log q_k - log p_k) = c ln 2 (gap + total (m - top)) + log s - log_s.
// (Without entries 0 times the row's own terms: a row that gives NaN gives it here as in its
// gradient.)
struct Entries {
  float total, gap, top, log_s;
  __device__ __forceinline__ float loss(float m, float s_log, float c) const {
    return total == 0.0f ? 0.0f * (m + s_log) : fmaf(c * kLn2, gap + (m - top), s_log - log_s);
  }
};

// log s, in 64 bits up to its rounding.
__device__ __forceinline__ float log_of(float s) {
  float f = __builtin_amdgcn_frexp_mantf(s);
  int n = __builtin_amdgcn_frexp_expf(s);
  if (f < 0.70710678f) {
    f *= 2.0f;
    n -= 1;
  }
  return (float)fma((double)n, kLn2d, twice_atanh((double)f - 1.0, (double)f + 1.0));
}

// The entries of row r, by G lanes of one wave (whose LDS accesses are in order), while
// the row itself is on its way.
template <class T, int G>
__device__ __forceinline__ Entries take_entries(const Teacher& teacher, int64_t r, const T* row,
                                                int A, float c, int lane, const Board& b) {
  const int K = teacher.K;
  float m = kNegInf, top = kNegInf;
  for (int k = lane; k < K; k += G) {
    const int col = teacher.column(r, k, A);
    const float t = col >= 0 ? teacher.logit(r, k) : col == -1 ? kNegInf : PPO_NAN;
    const float l = col >= 0 ? to_f32(row[col]) : kNegInf;
    b.col[k] = col;
    b.q[k] = t;
    b.l[k] = l;
    m = fmaxf(m, t);
    if (t != kNegInf) top = fmaxf(top, l);  // (an entry that weighs nothing has no part)
  }
  for (int k = K + lane; k < ((K + 3) & ~3); k += G) b.col[k] = -1;
  for (int k = lane; k < kMarkWords; k += G) b.marks[k] = 0;
  m = lanes_max<G>(m);
  top = lanes_max<G>(top);
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  // (no entries, or none but -inf: all q are 0)
  const float base = m == kNegInf ? 0.0f : m;
  if (top == kNegInf) top = 0.0f;
  float s = 0.0f, gap = 0.0f;
  for (int k = lane; k < K; k += G) {
    const float t = b.q[k] - base, q = exp2_fast(t * c);
    s += q;
    // (an entry that weighs nothing adds nothing, whatever its logits)
    if (q != 0.0f) gap = fmaf(q, t - (b.l[k] - top), gap);
    b.q[k] = q;
  }
  s = lanes_sum<G>(s);
  gap = lanes_sum<G>(gap);
  const float inv = s == 0.0f ? 0.0f : 1.0f / s;
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  for (int k = lane; k < K; k += G) {
    b.q[k] *= inv;
    if (s == 0.0f) b.col[k] = -1;  // (entries that all weigh nothing are none)
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  // Entries of one column write its sum, all of them.  Such are rare: only where a column's
  // mark is there already are they looked for, four at a time, and summed.
  int met = 0;
  for (int k = lane; k < K; k += G)
    if (b.col[k] >= 0) {
      const unsigned h = (unsigned)b.col[k] * 0x9E3779B1u >> 20;  // 12 bits
      met |= atomicOr(&b.marks[h >> 5], 1u << (h & 31)) >> (h & 31) & 1;
    }
  const bool twice = lanes_max<G>((float)met) != 0.0f;
  for (int k = lane; k < K; k += G) {
    const int col = b.col[k];
    float q = b.q[k];
    if (twice && col >= 0) {
      int same = 0;
      for (int i = 0; i < K; i += 4) {
        const v4i four = *reinterpret_cast<const v4i*>(b.col + i);
        same += (four[0] == col) + (four[1] == col) + (four[2] == col) + (four[3] == col);
      }
      if (same > 1) {
        q = 0.0f;
        for (int i = 0; i < K; ++i) q += b.col[i] == col ? b.q[i] : 0.0f;
      }
    }
    b.sum[k] = q;
  }
  return {s == 0.0f ? 0.0f : s / s, gap * inv, top, s == 0.0f ? 0.0f : log_of(s)};
}

// The entries' columns, those that `in` has: tau w (p - q).
struct AllColumns {
  __device__ __forceinline__ bool has(int) const { return true; }
};
template <class T, class In = AllColumns>
__device__ __forceinline__ void write_entries(const Board& b, int K, float m, float inv_s, float c,
                                              float W, T* out, int t, int lanes,
                                              const In& in = In{}) {
  for (int k = t; k < K; k += lanes) {
    const int col = b.col[k];
    if (col < 0 || !in.has(col)) continue;
    const float p = exp2_fast((b.l[k] - m) * c) * inv_s;
    out[col] = from_f32<T>(W * (p - b.sum[k]));
  }
}

struct Distill {
  Teacher teacher;
  Weights weights;
  float tau, grad_scale;
  Saved* saved;
  double* sums;

  // weight = tau w, pa = the sum of q
  __device__ __forceinline__ void leave(int64_t r, float m, float s, float weight, float q) const {
    if (saved) saved[r] = {m, 1.0f / s, 0.0f, 0.0f, 0.0f, q, 0.0f, weight};
  }
};

// A row's scalars, from its first wave to the others.
struct RowShare {
  Grad g;
  float inv_s, W;
};

// The columns of a row's entries come after the whole row is written.  A workgroup's
// first wave puts them off until the next row's barrier, before which every wave has
// waited for its stores (its loads of that row, which follow them, are in by then), so
// that no wave waits for memory between two rows; there are two boards for that.
template <class T, int G, int V>
__global__ void __launch_bounds__(kRowBlock<G>, kRowWaves<G>)
    distill_kernel(Rows rows, Distill d, Order order, T* dlogits) {
  constexpr int kBlock = kRowBlock<G>, kGroups = kBlock / G;
  constexpr int kTeam = G < kWave ? G : kWave;  // the lanes that take the entries
  extern __shared__ __attribute__((aligned(16))) int s_board[];
  __shared__ Stat s_part[kBlock / kWave];
  __shared__ RowShare s_row;
  const int t = threadIdx.x % G, group = group_of<G>(), K = d.teacher.K;
  int place = group;
  const T* before = nullptr;  // the row whose entries are still to be written, and its terms
  RowShare of_before;
  double sums[1] = {};
  const float inverse = inverse_count(d.weights);
  const T* logits = static_cast<const T*>(rows.logits);
  const Scale<Stat> scale(rows);
  const Walk<G> walk(rows, order, (int64_t)gridDim.x * kGroups);
  auto dead = [&](int64_t r) {
    if (dlogits) write_zeros<T, G>(dlogits + r * rows.A, rows.A, t);
  };
  int64_t i = walk.from((int64_t)blockIdx.x * kGroups + group, dead);
  int64_t r = i < rows.n ? walk.row(i) : -1;
  auto row_at = [&](int64_t k) { return k >= 0 ? logits + k * rows.A : nullptr; };
  auto flush = [&](const T* row, const RowShare& s, int at) {
    write_entries<T>(Board(s_board, K, at), K, s.g.m, s.inv_s, rows.c, s.W,
                     dlogits + (row - logits), t, kTeam);
  };
  RowRegs<T, G, V> x(row_at(r), rows.A, t);
  while (r >= 0) {
    T* out = dlogits + r * rows.A;
    const T* row = logits + r * rows.A;
    const Board board(s_board, K, place);
    Entries e = {};
    if (G <= kWave || threadIdx.x < kWave)
      e = take_entries<T, kTeam>(d.teacher, r, row, rows.A, rows.c, t, board);
    const float W = d.tau * row_weight(d.weights, inverse, r / rows.T);
    i = walk.from(i + walk.step, dead);
    const int64_t next = i < rows.n ? walk.row(i) : -1;
    x.take_out(-1, t);
    Stat st = x.template stat<false>(scale);
    RowShare share;
    auto finish = [&] {
      const float inv_s = 1.0f / st.s;
      share = {{st.m, W * d.grad_scale * e.total * inv_s, 0.0f, 0.0f, -1}, inv_s, W * d.grad_scale};
      if (t == 0) {
        sums[0] += (double)W * e.loss(st.m, log_of(st.s), rows.c);
        d.leave(r, st.m, st.s, W, e.total);
      }
    };
    if (G > kWave) {
      asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      st = block_join<false>(st, scale, s_part);
      if (threadIdx.x < kWave) {
        finish();
        if (t == 0) s_row = share;
        if (before) flush(before, of_before, 1 - place);
      }
      lds_barrier();
      share = s_row;
    } else {
      st = lanes_join<kTeam, false>(st, scale);
      finish();
    }
    share = {shared_by<G>(share.g), shared_by<G>(share.inv_s), shared_by<G>(share.W)};
    if (dlogits) {
      if (kRowAfterRow<G>)
        x.template write<false>(share.g, rows.c, out, rows.A, t, row_at(next));
      else
        x.template write<false>(share.g, rows.c, out, rows.A, t);
      if (G > kWave) {
        before = row;
        of_before = share;
        place = 1 - place;
      } else {
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        flush(row, share, place);
      }
    }
    if (!dlogits || !kRowAfterRow<G>) x = RowRegs<T, G, V>(row_at(next), rows.A, t);
    r = next;
  }
  if (G > kWave) {
    __syncthreads();
    if (before && threadIdx.x < kWave) flush(before, of_before, 1 - place);
  }
  leave_sums(sums, d.sums);
}

struct DistillJoin {
  using Sums = Stat;
  static constexpr bool kWholeWave = true;
  Distill d;
  double sums[1];
  __device__ __forceinline__ void masked(int64_t) const {}
  template <class T>
  __device__ __forceinline__ void row(const Rows& rows, int64_t r, const T* row, Stat x, int lane) {
    __shared__ __attribute__((aligned(16))) int s_board[4 * kMaxK + kMarkWords];
    const Entries e = take_entries<T, kWave>(d.teacher, r, row, rows.A, rows.c, lane,
                                             Board(s_board, d.teacher.K, 0));
    const float W = d.tau * row_weight(d.weights, inverse_count(d.weights), r / rows.T);
    if (lane != 0) return;
    sums[0] += (double)W * e.loss(x.m, log_of(x.s), rows.c);
    d.leave(r, x.m, x.s, W, e.total);
  }
  __device__ __forceinline__ void end() { leave_sums(sums, d.sums); }
};

// Where the pieces of a row are written apart: each takes the row's entries for itself and
// writes those among its own columns.
struct DistillTerms : GradientTerms {
  static constexpr bool kAfter = true;
  Teacher teacher;
  float inv_s, W;  // of the row at hand

  template <class T, int G>
  __device__ __forceinline__ Entries take(const Rows& rows, int64_t r, const T* row, int* board) {
    constexpr int kTeam = G < kWave ? G : kWave;
    return take_entries<T, kTeam>(teacher, r, row, rows.A, rows.c, threadIdx.x % kTeam,
                                  Board(board, teacher.K, 0));
  }
  template <class T, int G>
  __device__ __forceinline__ void after(const Rows& rows, const Grad& g, T* out,
                                        const PieceColumns& cols, int t, int* board) const {
    write_entries<T>(Board(board, teacher.K, 0), teacher.K, g.m, inv_s, rows.c, W, out, t,
                     G < kWave ? G : kWave, cols);
  }
};

// From what the forward pass saved.
struct DistillGrad : DistillTerms {
  const Saved* saved;
  float grad_scale;
  template <class T, int G>
  __device__ __forceinline__ Grad row(const Rows& rows, int64_t r, const T* row, float up, int, int,
                                      bool, int* board) {
    take<T, G>(rows, r, row, board);
    const Saved s = saved[r];
    inv_s = s.inv_s;
    W = up * grad_scale * s.weight;
    return {s.m, W * s.pa * s.inv_s, 0.0f, 0.0f, -1};
  }
};

// From the parts of the rows' statistics, in the forward pass of few rows.
struct DistillSplit : DistillTerms {
  Distill d;
  const Stat* parts;
  int splits;
  float inverse;

  __device__ __forceinline__ void begin() { inverse = inverse_count(d.weights); }
  __device__ __forceinline__ void masked(const Rows&, int64_t r, bool first) const {
    if (first) d.sums[r] = 0.0;
  }
  template <class T, int G>
  __device__ __forceinline__ Grad row(const Rows& rows, int64_t r, const T* row, float, int, int t,
                                      bool first, int* board) {
    const Entries e = take<T, G>(rows, r, row, board);
    const Stat x = join_parts<G, false>(parts, r, splits, Scale<Stat>(rows));
    const float weight = d.tau * row_weight(d.weights, inverse, r / rows.T);
    inv_s = 1.0f / x.s;
    W = weight * d.grad_scale;
    if (first && t == 0) {
      d.sums[r] = (double)weight * e.loss(x.m, log_of(x.s), rows.c);
      d.leave(r, x.m, x.s, weight, e.total);
    }
    return {x.m, W * e.total * inv_s, 0.0f, 0.0f, -1};
  }
};

__global__ void __launch_bounds__(256) distill_scalar_kernel(const double* sums, int n, double tau,
                                                             float* scalar) {
  __shared__ double part[4];
  double v = 0.0;
  for (int i = threadIdx.x; i < n; i += 256) v += sums[i];
  v = lanes_sum<kWave>(v);
  if ((threadIdx.x & (kWave - 1)) == 0) part[threadIdx.x / kWave] = v;
  __syncthreads();
  if (threadIdx.x == 0) *scalar = (float)(tau * ((part[0] + part[1]) + (part[2] + part[3])));
}

template <class T>
int dense_gradient(const Rows& rows, const Teacher& teacher, const Saved* saved, const float* scale,
                   float held, float grad_scale, T* dlogits, hipStream_t stream) {
  const DistillGrad grad = {{{}, teacher, 0.0f, 0.0f}, saved, grad_scale};
  return launch_gradient<T, false>(rows, grad, scale, held, dlogits, board_ints(teacher.K), stream);
}

template <class T>
int run_distill(const Rows& rows, Distill& d, const Scratch& s, T* dlogits, int& partials,
                hipStream_t stream) {
  const int dtype = sizeof(T) == 4 ? PPO_DTYPE_F32 : PPO_DTYPE_BF16;
  const int64_t chunks = chunks_of(rows.A, dtype);
  auto go = [&](auto lanes, auto held) {
    constexpr int G = decltype(lanes)::value, V = decltype(held)::value;
    constexpr int kBlock = kRowBlock<G>;
    partials = launch_blocks(div_up(rows.n, kBlock / G), kRowBlocks<G>);
    Order order = {};
    if (kRowAfterRow<G> && rows.mask)
      order = take_order(rows, d.weights, s, stream);
    else
      count_weights(rows, d.weights, s, stream);
    hipLaunchKernelGGL((distill_kernel<T, G, V>), dim3(partials), dim3(kBlock),
                       (size_t)board_ints(d.teacher.K) * std::max(2, kBlock / G) * sizeof(int), stream,
                       rows, d, order, dlogits);
    return last_launch_status();
  };
  const int least = board_ints(d.teacher.K) <= kQuadBoard ? 16 : 64;
  return with_row_shape<true>(rows.n, chunks, lies_alike(rows.logits, dlogits), least, go, [&] {
    if (!fits_launch(rows.n * row_splits(rows.n, rows.A, dtype), 256))
      return (int)PPO_ERR_TOO_LARGE;
    count_weights(rows, d.weights, s, stream);
    const DistillJoin join = {d, {}};
    if (dlogits && rows.n <= kMaxPartials) {
      DistillSplit split = {{{}, d.teacher, 0.0f, 0.0f}, d, s.parts, 1, 0.0f};
      partials = (int)rows.n;
      if (const int code = launch_parts<T, false>(rows, s, join, true, stream, split.splits))
        return code;
      return launch_gradient<T, false>(rows, split, nullptr, 0.0f, dlogits,
                                       board_ints(d.teacher.K), stream);
    }
    partials = launch_blocks(rows.n, kMaxPartials);
    if (const int code = launch_statistics<T, false, false>(rows, s, join, true, stream))
      return code;
    if (!dlogits) return (int)PPO_OK;
    return dense_gradient<T>(rows, d.teacher, d.saved, nullptr, 0.0f, d.grad_scale, dlogits, stream);
  });
}

bool teacher_ok(const Rows& rows, const void* teacher, int dtype, const void* ids, int64_t K) {
  return dtype_ok(dtype) && K > 0 && (rows.n == 0 || (teacher && ids));
}

}  // namespace
}  // namespace ppo

extern "C" int ppo_token_distillation(const ppo_token_rows* r, const void* teacher,
                                      int teacher_dtype, const void* ids, int ids_are_int64,
                                      int64_t K, const ppo_token_loss* loss, float* scalar,
                                      float* saved, void* dlogits, void* workspace,
                                      size_t workspace_bytes, void* stream_ptr) {
  using namespace ppo;
  Rows rows;
  if (const int code = take_rows(r, false, rows)) return code;
  rows.actions = nullptr;
  if (!loss || !scalar || !teacher_ok(rows, teacher, teacher_dtype, ids, K) ||
      (dlogits && !saved && rows.n) || (saved && !aligned16(saved)) ||
      (uintptr_t)dlogits % dtype_size(r->dtype))
    return PPO_ERR_INVALID_ARG;
  if (K > kMaxK) return PPO_ERR_TOO_LARGE;
  const Scratch s = scratch_of(workspace, rows.S, rows.T, rows.A, r->dtype);
  if (!workspace || !aligned16(workspace) || workspace_bytes < s.bytes) return PPO_ERR_WORKSPACE;
  hipStream_t stream = (hipStream_t)stream_ptr;
  Weights weights;
  if (const int code = take_weights(rows, loss, s, weights)) return code;
  Distill d = {{teacher, ids, teacher_dtype, ids_are_int64, (int)K}, weights,
               (float)r->temperature, (float)loss->grad_scale, reinterpret_cast<Saved*>(saved),
               s.sums};
  int partials = 0;
  if (rows.n)
    if (const int code = with_dtype(r->dtype, [&](auto zero) {
          return run_distill<decltype(zero)>(rows, d, s, (decltype(zero)*)dlogits, partials, stream);
        }))
      return code;
  // (the sums carry one of the two factors of the temperature already)
  hipLaunchKernelGGL(distill_scalar_kernel, dim3(1), dim3(256), 0, stream, s.sums, partials,
                     r->temperature, scalar);
  return last_launch_status();
}

extern "C" int ppo_token_distillation_backward(const ppo_token_rows* r, const void* teacher,
                                               int teacher_dtype, const void* ids,
                                               int ids_are_int64, int64_t K, const float* saved,
                                               const float* scale, double held, void* dlogits,
                                               void* stream_ptr) {
  using namespace ppo;
  Rows rows;
  if (const int code = take_rows(r, false, rows)) return code;
  rows.actions = nullptr;
  if (!teacher_ok(rows, teacher, teacher_dtype, ids, K)) return PPO_ERR_INVALID_ARG;
  if (K > kMaxK) return PPO_ERR_TOO_LARGE;
  if (rows.n == 0) return PPO_OK;
  if (!saved || !aligned16(saved) || !dlogits || (held != 0.0 && !scale) ||
      (uintptr_t)dlogits % dtype_size(r->dtype))
    return PPO_ERR_INVALID_ARG;
  const Teacher top = {teacher, ids, teacher_dtype, ids_are_int64, (int)K};
  return with_dtype(r->dtype, [&](auto zero) {
    using T = decltype(zero);
    return dense_gradient<T>(rows, top, reinterpret_cast<const Saved*>(saved), scale, (float)held,
                             1.0f, (T*)dlogits, (hipStream_t)stream_ptr);
  });
}
