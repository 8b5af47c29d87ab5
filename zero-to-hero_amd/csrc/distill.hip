// Distillation from a teacher's K top logits over wide rows of the student's,
// forward and gradient in one pass: dlogits_j = tau w (p_j - q_j), dense in p and
// with at most K columns of q.
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

// The K entries of a row over G lanes (16, or a wave).
template <int G>
struct Entries {
  static constexpr int kN = kMaxK / G;
  int col[kN];
  float t[kN];     // the teacher's logits
  float m, s;      // their largest, and the sum of 2^(c (t - m))
  float q[kN];

  __device__ __forceinline__ Entries(const Teacher& teacher, int64_t r, int A, float c, int lane) {
    m = kNegInf;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      const int k = i * G + lane;
      col[i] = k < teacher.K ? teacher.column(r, k, A) : -1;
      t[i] = col[i] >= 0 ? teacher.logit(r, k) : col[i] == -1 ? kNegInf : PPO_NAN;
      m = fmaxf(m, t[i]);
    }
    m = lanes_max<G>(m);
    // (no entries, or none but -inf: all q are 0)
    const float base = m == kNegInf ? 0.0f : m;
    s = 0.0f;
#pragma unroll
    for (int i = 0; i < kN; ++i) {
      q[i] = exp2_fast((t[i] - base) * c);
      s += q[i];
    }
    s = lanes_sum<G>(s);
    const float inv = s == 0.0f ? 0.0f : 1.0f / s;
#pragma unroll
    for (int i = 0; i < kN; ++i) q[i] *= inv;
  }
  // 1, 0 without entries, NaN with one that is not finite.
  __device__ __forceinline__ float total() const { return s == 0.0f ? 0.0f : s / s; }
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

// sum_k q_k (log q_k - log p_k) of the row, in every lane.
template <class T, int G>
__device__ __forceinline__ float row_loss(const Entries<G>& e, const T* row, float m, float s,
                                          float c) {
  float x = 0.0f;
#pragma unroll
  for (int i = 0; i < Entries<G>::kN; ++i)
    if (e.col[i] != -1 && e.q[i] != 0.0f) {
      const float l = e.col[i] >= 0 ? to_f32(row[e.col[i]]) : PPO_NAN;
      x = fmaf(e.q[i], (e.t[i] - e.m) - (l - m), x);
    }
  x = lanes_sum<G>(x);
  return e.s == 0.0f ? 0.0f : fmaf(c * kLn2, x, log_of(s) - log_of(e.s));
}

// Writes the entries' columns: tau w (p - q), q summed over entries of one column
// (each of them writes the same value).
template <class T, int G>
__device__ __forceinline__ void write_entries(const Entries<G>& e, const T* row, T* out, int K,
                                              float m, float inv_s, float c, float W, int lane,
                                              float* s_q, int* s_col) {
#pragma unroll
  for (int i = 0; i < Entries<G>::kN; ++i) {
    const int k = i * G + lane;
    if (k < K) {
      s_q[k] = e.q[i];
      s_col[k] = e.col[i];
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // (one wave's LDS is in order)
#pragma unroll
  for (int i = 0; i < Entries<G>::kN; ++i) {
    if (i * G >= K || e.col[i] < 0) continue;
    float q = 0.0f;
    for (int k = 0; k < K; ++k) q += s_col[k] == e.col[i] ? s_q[k] : 0.0f;
    const float p = exp2_fast((to_f32(row[e.col[i]]) - m) * c) * inv_s;
    out[e.col[i]] = from_f32<T>(W * (p - q));
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

template <class T, int G, int V>
__global__ void __launch_bounds__(G < 256 ? 256 : G) distill_kernel(Rows rows, Distill d, T* dlogits) {
  constexpr int kBlock = G < 256 ? 256 : G, kGroups = kBlock / G;
  constexpr int kTeam = G < kWave ? G : kWave;
  __shared__ Stat s_part[kBlock / kWave];
  __shared__ Grad s_grad;
  __shared__ float s_q[kGroups][kMaxK];
  __shared__ int s_col[kGroups][kMaxK];
  const int t = threadIdx.x % G, group = group_of<G>();
  double sums[1] = {};
  const float inverse = inverse_count(d.weights);
  for (int64_t r = (int64_t)blockIdx.x * kGroups + group; r < rows.n;
       r += (int64_t)gridDim.x * kGroups) {
    T* out = dlogits + r * rows.A;
    if (!rows.live(r)) {
      if (dlogits) write_zeros<T, G>(out, rows.A, t);
      continue;
    }
    const T* row = static_cast<const T*>(rows.logits) + r * rows.A;
    RowRegs<T, G, V> x(row, rows.A, t);
    x.take_out(-1, t);
    Stat st = x.template stat<false>(rows.c);
    Grad g;
    // (the first wave of the row's lanes takes the entries)
    const float W = d.tau * row_weight(d.weights, inverse, r / rows.T);
    auto finish = [&](const Entries<kTeam>& e) {
      const float loss = row_loss<T, kTeam>(e, row, st.m, st.s, rows.c);
      g = {st.m, W * d.grad_scale * e.total() * (1.0f / st.s), 0.0f, 0.0f, -1};
      if (t == 0) {
        sums[0] += (double)W * loss;
        d.leave(r, st.m, st.s, W, e.total());
      }
    };
    auto fix = [&](const Entries<kTeam>& e) {
      write_entries<T, kTeam>(e, row, out, d.teacher.K, st.m, 1.0f / st.s, rows.c, W * d.grad_scale,
                              t, s_q[group], s_col[group]);
    };
    if constexpr (G > kWave) {
      st = block_join<false>(st, rows.c, s_part);
      if (threadIdx.x < kWave) {
        const Entries<kTeam> e(d.teacher, r, rows.A, rows.c, t);
        finish(e);
        if (t == 0) s_grad = g;
      }
      lds_barrier();
      g = s_grad;
      if (dlogits) {
        x.template write<false>(g, rows.c, out, t);
        __syncthreads();  // (the whole row is written before the entries' columns)
        if (threadIdx.x < kWave) fix(Entries<kTeam>(d.teacher, r, rows.A, rows.c, t));
      }
    } else {
      st = lanes_join<kTeam, false>(st, rows.c);
      const Entries<kTeam> e(d.teacher, r, rows.A, rows.c, t);
      finish(e);
      if (dlogits) {
        x.template write<false>(g, rows.c, out, t);
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        fix(e);
      }
    }
  }
  leave_sums(sums, d.sums);
}

struct DistillJoin {
  static constexpr bool kWholeWave = true;
  Distill d;
  double sums[1];
  __device__ __forceinline__ void masked(int64_t) const {}
  template <class T>
  __device__ __forceinline__ void row(const Rows& rows, int64_t r, const T* row, Stat x,
                                      int lane) {
    const Entries<kWave> e(d.teacher, r, rows.A, rows.c, lane);
    const float W = d.tau * row_weight(d.weights, inverse_count(d.weights), r / rows.T);
    const float loss = row_loss<T, kWave>(e, row, x.m, x.s, rows.c);
    if (lane != 0) return;
    sums[0] += (double)W * loss;
    d.leave(r, x.m, x.s, W, e.total());
  }
  __device__ __forceinline__ void end() { leave_sums(sums, d.sums); }
};

struct DistillGrad {
  const Saved* saved;
  float grad_scale;
  __device__ __forceinline__ Grad row(const Rows&, int64_t r, float up, int) const {
    const Saved s = saved[r];
    return {s.m, up * grad_scale * s.weight * s.pa * s.inv_s, 0.0f, 0.0f, -1};
  }
};

// The entries' columns after a dense pass over the rows, a wave to a row.
template <class T>
__global__ void __launch_bounds__(64) entries_kernel(Rows rows, Teacher teacher, const Saved* saved,
                                                     const float* scale, float held,
                                                     float grad_scale, T* dlogits) {
  __shared__ float s_q[kMaxK];
  __shared__ int s_col[kMaxK];
  const float up = scale ? *scale : 1.0f;
  if (held != 0.0f && up == held) return;
  const int lane = threadIdx.x;
  for (int64_t r = blockIdx.x; r < rows.n; r += gridDim.x) {
    if (!rows.live(r)) continue;
    const T* row = static_cast<const T*>(rows.logits) + r * rows.A;
    const Saved s = saved[r];
    const Entries<kWave> e(teacher, r, rows.A, rows.c, lane);
    write_entries<T, kWave>(e, row, dlogits + r * rows.A, teacher.K, s.m, s.inv_s, rows.c,
                            up * grad_scale * s.weight, lane, s_q, s_col);
  }
}

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
  const DistillGrad grad = {saved, grad_scale};
  if (const int code = launch_gradient<T, false>(rows, grad, scale, held, dlogits, stream))
    return code;
  hipLaunchKernelGGL((entries_kernel<T>),
                     dim3(launch_blocks(rows.n, held != 0.0f ? kHeldBlocks : kMaxPartials)), dim3(64),
                     0, stream, rows, teacher, saved, scale, held, grad_scale, dlogits);
  return last_launch_status();
}

template <class T>
int run_distill(const Rows& rows, const Distill& d, const Scratch& s, T* dlogits, int& partials,
                hipStream_t stream) {
  const int dtype = sizeof(T) == 4 ? PPO_DTYPE_F32 : PPO_DTYPE_BF16;
  const int64_t chunks = chunks_of(rows.A, dtype);
  auto go = [&](auto lanes, auto held) {
    constexpr int G = decltype(lanes)::value, V = decltype(held)::value;
    constexpr int kBlock = G < 256 ? 256 : G;
    partials = launch_blocks(div_up(rows.n, kBlock / G), kMaxPartials);
    hipLaunchKernelGGL((distill_kernel<T, G, V>), dim3(partials), dim3(kBlock), 0, stream, rows, d,
                       dlogits);
    return last_launch_status();
  };
  return with_row_shape(rows.n, chunks, lies_alike(rows.logits, dlogits), go, [&] {
    const DistillJoin join = {d, {}};
    partials = launch_blocks(rows.n, kMaxPartials);
    if (const int code = launch_statistics<T, false, false>(rows, s, join, stream)) return code;
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
  if (const int code = take_weights(rows, loss, s, stream, weights)) return code;
  const Distill d = {{teacher, ids, teacher_dtype, ids_are_int64, (int)K}, weights,
                     (float)r->temperature, (float)loss->grad_scale,
                     reinterpret_cast<Saved*>(saved), s.sums};
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
