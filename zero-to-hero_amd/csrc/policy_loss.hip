// The clipped policy loss with a KL term over wide rows of logits, forward and
// gradient in one pass: a row stays in the registers of its group of lanes from
// the read to the write.  With G and E the row's dloss/dlog p_a and dloss/dH,
//   dlogits_j = (G ([j = a] - p_j) - E p_j (log p_j + H)) / temperature,
// which needs the whole row's sums before its first element: hence registers, or the
// caches for rows that do not fit.  What bounds it: HBM, one read and one write of the
// logits (8192 x 131072 bf16 839-851 us, 5.1 TB/s; 4096 x 32768 with a mask 86, 5.2);
// few rows the chain of launches (528 x 500 fp32 16 in a graph).
#include "tokens_rows.hpp"

namespace ppo {
namespace {

struct Policy {
  const float *old, *adv, *ref;
  Weights weights;
  float lo, hi, kl_coef, entropy_coef, grad_scale;
  int per_sequence;
  Saved* saved;
  float* coef;   // [2][n]
  double* sums;
};

// What a row adds to the sums.
struct RowLoss {
  float w, policy, kl, H, approx_kl, clipped;
  __device__ __forceinline__ void add_to(double (&sums)[kSums]) const {
    sums[0] += (double)w * policy;
    sums[1] += (double)w * kl;
    sums[2] += (double)w * H;
    sums[3] += (double)w * approx_kl;
    sums[4] += (double)w * clipped;
  }
};

// e^d - d - 1 and its derivative e^d - 1: the first's series where the differences would
// cancel (to |d| = 1, where the next term is below 2^-28 of the sum), and from e^d beyond (a
// derivative of value + d would lose its 1 in a large -d, and be NaN at d = -inf).
struct KlEstimate {
  float value, slope;
};
__device__ __forceinline__ KlEstimate kl_estimate(float d) {
  if (!(fabsf(d) <= 1.0f)) {
    const float e = expf(d);
    return {e - d - 1.0f, e - 1.0f};
  }
  float q = 1.0f / 479001600.0f;
  constexpr float kInv[] = {1.0f / 39916800, 1.0f / 3628800, 1.0f / 362880, 1.0f / 40320,
                            1.0f / 5040,     1.0f / 720,     1.0f / 120,    1.0f / 24,
                            1.0f / 6,        0.5f};
#pragma unroll
  for (float k : kInv) q = fmaf(d, q, k);
  const float v = d * d * q;
  return {v, v + d};
}

// A row's inputs beside its logits.
struct RowIn {
  float old, adv, ref, w;
};
__device__ __forceinline__ RowIn row_in(const Policy& p, const Rows& rows, int64_t r,
                                        float inverse) {
  const int64_t seq = r / rows.T;
  return {p.old[r], p.adv[p.per_sequence ? seq : r], p.ref ? p.ref[r] : 0.0f,
          row_weight(p.weights, inverse, seq)};
}

// The row's loss, its gradient's terms G and E for an incoming gradient of 1.
__device__ __forceinline__ RowLoss policy_row(const Policy& p, const RowIn& in, const RowTerms& t,
                                              float& G, float& E) {
  const float ratio = expf((float)(t.lp - (double)in.old));
  const float clipped = ratio < p.lo ? p.lo : ratio > p.hi ? p.hi : ratio;
  const float u = ratio * in.adv, v = clipped * in.adv;
  RowLoss o = {in.w, -(u > v ? v : u), 0.0f, t.H, (float)((double)in.old - t.lp),
               ratio < p.lo || ratio > p.hi ? 1.0f : 0.0f};
  G = u > v ? 0.0f : -u;
  if (p.ref) {
    const KlEstimate kl = kl_estimate((float)((double)in.ref - t.lp));
    o.kl = kl.value;
    if (p.kl_coef != 0.0f) G -= p.kl_coef * kl.slope;
  }
  G *= in.w;
  E = -p.entropy_coef * in.w;
  return o;
}

__device__ __forceinline__ void leave_row(const Policy& p, const Rows& rows, int64_t r,
                                          const RowTerms& t, float G, float E) {
  if (p.saved) p.saved[r] = saved_of(t, 0.0f);
  if (p.coef) {
    p.coef[r] = G;
    p.coef[rows.n + r] = E;
  }
}
// (a masked row's terms are never read again but for its zero coefficients)
__device__ __forceinline__ void leave_masked(const Policy& p, const Rows& rows, int64_t r) {
  if (p.coef) p.coef[r] = p.coef[rows.n + r] = 0.0f;
}

template <class T, int G, int V, bool kC>
__global__ void __launch_bounds__(kRowBlock<G>, kRowWaves<G>)
    policy_kernel(Rows rows, Policy p, Order order, T* dlogits) {
  constexpr int kBlock = kRowBlock<G>, kGroups = kBlock / G;
  __shared__ Stat s_part[kBlock / kWave];
  __shared__ Grad s_grad;
  __shared__ double s_sums[kSums];
  const int t = threadIdx.x % G;
  double sums[kSums] = {};
  const float inverse = inverse_count(p.weights);
  if (G > kWave && threadIdx.x < kSums) s_sums[threadIdx.x] = 0.0;
  const T* logits = static_cast<const T*>(rows.logits);
  const Scale<Stat> scale(rows);
  const Walk<G> walk(rows, order, (int64_t)gridDim.x * kGroups);
  auto dead = [&](int64_t r) {
    if (dlogits) write_zeros<T, G>(dlogits + r * rows.A, rows.A, t);
    if (t == 0) leave_masked(p, rows, r);
  };
  int64_t i = walk.from((int64_t)blockIdx.x * kGroups + group_of<G>(), dead);
  int64_t r = i < rows.n ? walk.row(i) : -1;
  auto row_at = [&](int64_t k) { return k >= 0 ? logits + k * rows.A : nullptr; };
  RowRegs<T, G, V> x(row_at(r), rows.A, t);
  int a = r >= 0 ? rows.action(r) : -1;
  while (r >= 0) {
    const float la = action_logit(logits + r * rows.A, a);
    const RowIn in = row_in(p, rows, r, inverse);
    i = walk.from(i + walk.step, dead);
    const int64_t next = i < rows.n ? walk.row(i) : -1;
    const int next_a = next >= 0 ? rows.action(next) : -1;
    x.take_out(a, t);
    Stat st = x.template stat<true>(scale);
    Grad g;
    auto finish = [&](double(&to)[kSums]) {
      const RowTerms terms = row_terms<true>(st, la, scale);
      float gl, ge;
      const RowLoss loss = policy_row(p, in, terms, gl, ge);
      if (t == 0) {
        loss.add_to(to);
        leave_row(p, rows, r, terms, gl, ge);
      }
      g = row_grad(saved_of(terms, 0.0f), gl * p.grad_scale, ge * p.grad_scale, rows.inv_tau, a);
    };
    if (G > kWave) {
      st = block_join<true>(st, scale, s_part);
      if (threadIdx.x < kWave) {
        finish(s_sums);
        if (t == 0) s_grad = g;
      }
      lds_barrier();
      g = s_grad;
    } else {
      st = lanes_join<G <= kWave ? G : kWave, true>(st, scale);
      finish(sums);
    }
    g = shared_by<G>(g);
    if (dlogits && kRowAfterRow<G>)
      x.template write<kC>(g, rows.c, dlogits + r * rows.A, rows.A, t, row_at(next));
    else {
      if (dlogits) x.template write<kC>(g, rows.c, dlogits + r * rows.A, rows.A, t);
      x = RowRegs<T, G, V>(row_at(next), rows.A, t);
    }
    r = next;
    a = next_a;
  }
  if (G <= kWave) {
    leave_sums(sums, p.sums);
    return;
  }
  lds_barrier();
  if (threadIdx.x < kSums)
    p.sums[(int64_t)threadIdx.x * kMaxPartials + blockIdx.x] = s_sums[threadIdx.x];
}

// The same from rows' parts (join_kernel), where a row has several workgroups.
struct PolicyJoin {
  using Sums = Stat;
  static constexpr bool kWholeWave = false;
  Policy p;
  double sums[kSums];
  int64_t n;

  __device__ __forceinline__ void masked(int64_t r) const {
    if (p.coef) p.coef[r] = p.coef[n + r] = 0.0f;
  }
  template <bool kEntropy>
  __device__ __forceinline__ void row(const Rows& rows, int64_t r, Stat x, float la, bool first) {
    const RowTerms t = row_terms<kEntropy>(x, la, Scale<Stat>(rows));
    float G, E;
    const RowLoss loss =
        policy_row(p, row_in(p, rows, r, inverse_count(p.weights)), t, G, E);
    if (!first) return;
    loss.add_to(sums);
    leave_row(p, rows, r, t, G, E);
  }
  __device__ __forceinline__ void end() { leave_sums(sums, p.sums); }
};

struct PolicyGrad : GradientTerms {
  const Saved* saved;
  const float* coef;
  float grad_scale;
  template <class T, int G>
  __device__ __forceinline__ Grad row(const Rows& rows, int64_t r, const T*, float, int a, int, bool,
                                      int*) const {
    return row_grad(saved[r], grad_scale * coef[r], grad_scale * coef[rows.n + r], rows.inv_tau, a);
  }
};

// Rows' parts joined where the gradient is formed, by each piece of a row for itself: a
// launch less.  A row's own sums stand in the place of a workgroup's.
struct PolicySplit : GradientTerms {
  Policy p;
  const Stat* parts;
  int splits;
  float inverse;

  __device__ __forceinline__ void begin() { inverse = inverse_count(p.weights); }
  __device__ __forceinline__ void leave(const Rows& rows, int64_t r, const RowLoss& loss) const {
    double sums[kSums] = {};
    loss.add_to(sums);
#pragma unroll
    for (int k = 0; k < kSums; ++k) p.sums[(int64_t)k * kMaxPartials + r] = sums[k];
  }
  __device__ __forceinline__ void masked(const Rows& rows, int64_t r, bool first) const {
    if (!first) return;
    leave_masked(p, rows, r);
    leave(rows, r, RowLoss{});
  }
  template <class T, int G>
  __device__ __forceinline__ Grad row(const Rows& rows, int64_t r, const T* row, float, int a, int t,
                                      bool first, int*) const {
    const Scale<Stat> scale(rows);
    const RowTerms terms = row_terms<true>(join_parts<G, true>(parts, r, splits, scale),
                                           action_logit(row, a), scale);
    float gl, ge;
    const RowLoss loss = policy_row(p, row_in(p, rows, r, inverse), terms, gl, ge);
    if (first && t == 0) {
      leave(rows, r, loss);
      leave_row(p, rows, r, terms, gl, ge);
    }
    return row_grad(saved_of(terms, 0.0f), gl * p.grad_scale, ge * p.grad_scale, rows.inv_tau, a);
  }
};

// The scalars from the workgroups' sums, in their order.
__global__ void __launch_bounds__(1024) policy_scalars_kernel(const double* sums, int n,
                                                              double kl_coef, double entropy_coef,
                                                              float* scalars) {
  __shared__ double part[16][kSums];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  // (four of each sum's in flight: one at a time took 14 us of 8192 workgroups' sums)
  double v[kSums] = {};
  for (int base = threadIdx.x; base < n; base += 4 * 1024) {
    double x[4][kSums];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int k = 0; k < kSums; ++k)
        x[j][k] = base + j * 1024 < n ? sums[(int64_t)k * kMaxPartials + base + j * 1024] : 0.0;
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
      for (int k = 0; k < kSums; ++k) v[k] += x[j][k];
  }
#pragma unroll
  for (int k = 0; k < kSums; ++k) {
    v[k] = lanes_sum<kWave>(v[k]);
    if (lane == 0) part[wave][k] = v[k];
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  double all[kSums] = {};
  for (int w = 0; w < 16; ++w)
#pragma unroll
    for (int k = 0; k < kSums; ++k) all[k] += part[w][k];
  // (a term of coefficient 0 has no part in the loss, whatever it comes to)
  double loss = all[0];
  if (kl_coef != 0.0) loss += kl_coef * all[1];
  if (entropy_coef != 0.0) loss -= entropy_coef * all[2];
  scalars[PPO_TOKEN_SCALAR_LOSS] = (float)loss;
  scalars[PPO_TOKEN_SCALAR_POLICY] = (float)all[0];
  scalars[PPO_TOKEN_SCALAR_KL] = (float)all[1];
  scalars[PPO_TOKEN_SCALAR_ENTROPY] = (float)all[2];
  scalars[PPO_TOKEN_SCALAR_APPROX_KL] = (float)all[3];
  scalars[PPO_TOKEN_SCALAR_CLIPFRAC] = (float)all[4];
}

template <class T>
int run_policy(const Rows& rows, Policy& p, const Scratch& s, T* dlogits, int& partials,
               hipStream_t stream) {
  const int dtype = sizeof(T) == 4 ? PPO_DTYPE_F32 : PPO_DTYPE_BF16;
  const int64_t chunks = chunks_of(rows.A, dtype);
  const bool grad_entropy = p.entropy_coef != 0.0f;
  auto go = [&](auto lanes, auto held) {
    constexpr int G = decltype(lanes)::value, V = decltype(held)::value;
    constexpr int kBlock = kRowBlock<G>;
    partials = launch_blocks(div_up(rows.n, kBlock / G), kRowBlocks<G>);
    Order order = {};
    if (kRowAfterRow<G> && rows.mask)
      order = take_order(rows, p.weights, s, stream);
    else
      count_weights(rows, p.weights, s, stream);
    if (grad_entropy)
      hipLaunchKernelGGL((policy_kernel<T, G, V, true>), dim3(partials), dim3(kBlock), 0, stream,
                         rows, p, order, dlogits);
    else
      hipLaunchKernelGGL((policy_kernel<T, G, V, false>), dim3(partials), dim3(kBlock), 0, stream,
                         rows, p, order, dlogits);
    return last_launch_status();
  };
  return with_row_shape<false>(rows.n, chunks, lies_alike(rows.logits, dlogits), 16, go, [&] {
    if (!fits_launch(rows.n * row_splits(rows.n, rows.A, dtype), 256))
      return (int)PPO_ERR_TOO_LARGE;
    count_weights(rows, p.weights, s, stream);
    PolicyJoin join = {p, {}, rows.n};
    if (dlogits && rows.n <= kMaxPartials) {
      PolicySplit split = {{}, p, s.parts, 1, 0.0f};
      partials = (int)rows.n;
      if (const int code =
              launch_parts<T, true>(rows, s, join, true, stream, split.splits))
        return code;
      return grad_entropy
                 ? launch_gradient<T, true>(rows, split, nullptr, 0.0f, dlogits, 0, stream)
                 : launch_gradient<T, false>(rows, split, nullptr, 0.0f, dlogits, 0, stream);
    }
    partials = launch_blocks(rows.n, kMaxPartials);
    if (const int code = launch_statistics<T, true, false>(rows, s, join, true, stream))
      return code;
    if (!dlogits) return (int)PPO_OK;
    const PolicyGrad grad = {{}, p.saved, p.coef, p.grad_scale};
    return grad_entropy ? launch_gradient<T, true>(rows, grad, nullptr, 0.0f, dlogits, 0, stream)
                        : launch_gradient<T, false>(rows, grad, nullptr, 0.0f, dlogits, 0, stream);
  });
}

}  // namespace
}  // namespace ppo

extern "C" int ppo_token_policy_loss(const ppo_token_rows* r, const float* old_log_probs,
                                     const float* advantages, const float* ref_log_probs,
                                     const ppo_token_loss* loss, float* scalars, float* saved,
                                     float* coef, void* dlogits, void* workspace,
                                     size_t workspace_bytes, void* stream_ptr) {
  using namespace ppo;
  Rows rows;
  if (const int code = take_rows(r, true, rows)) return code;
  if (!loss || !scalars || !(loss->clip_low >= 0.0) || !(loss->clip_high >= 0.0) ||
      !isfinite((float)loss->kl_coef) || !isfinite((float)loss->entropy_coef))
    return PPO_ERR_INVALID_ARG;
  if (loss->kl_coef != 0.0 && !ref_log_probs && rows.n) return PPO_ERR_INVALID_ARG;
  if (rows.n && (!old_log_probs || !advantages)) return PPO_ERR_INVALID_ARG;
  if ((saved == nullptr) != (coef == nullptr) || (dlogits && !saved && rows.n) ||
      (saved && !aligned16(saved)) || (uintptr_t)dlogits % dtype_size(r->dtype))
    return PPO_ERR_INVALID_ARG;
  const Scratch s = scratch_of(workspace, rows.S, rows.T, rows.A, r->dtype);
  if (!workspace || !aligned16(workspace) || workspace_bytes < s.bytes) return PPO_ERR_WORKSPACE;
  hipStream_t stream = (hipStream_t)stream_ptr;
  Weights weights;
  if (const int code = take_weights(rows, loss, s, weights)) return code;
  Policy p = {old_log_probs, advantages, ref_log_probs, weights, (float)(1.0 - loss->clip_low),
              (float)(1.0 + loss->clip_high), (float)loss->kl_coef, (float)loss->entropy_coef,
              (float)loss->grad_scale, loss->advantages_per_sequence,
              reinterpret_cast<Saved*>(saved), coef, s.sums};
  int partials = 0;
  if (rows.n)
    if (const int code = with_dtype(r->dtype, [&](auto zero) {
          return run_policy<decltype(zero)>(rows, p, s, (decltype(zero)*)dlogits, partials, stream);
        }))
      return code;
  hipLaunchKernelGGL(policy_scalars_kernel, dim3(1), dim3(1024), 0, stream, s.sums, partials,
                     loss->kl_coef, loss->entropy_coef, scalars);
  return last_launch_status();
}
