// Token policies: log-probabilities and entropies of the taken actions, their
// gradient, the preference loss over them, and what all of these operators
// share on the host: checks, weights, scratch.  What bounds them: HBM, a read of the
// logits forward (4096 x 50304 bf16, 65% of its rows counting, 58 us, 4.6 TB/s), a read
// and a write backward (95, 7.2 TB/s with part of the read from the caches); few rows
// the launches (256 x 18 fp32 3.1).
#include "tokens_rows.hpp"

namespace ppo {

// ---------------------------------------------------------------------------
// Host
// ---------------------------------------------------------------------------

// A row's statistics by several workgroups: down to 512 chunks (8 KB) each, as
// many as fill the chip four times over.
int row_splits(int64_t rows, int64_t A, int dtype) {
  if (rows <= 0) return 1;
  int64_t s = div_up(1024, rows);
  const int64_t most = chunks_of(A, dtype) / 512;
  if (s > most) s = most;
  if (s > kMaxSplits) s = kMaxSplits;
  return s < 1 ? 1 : (int)s;
}

Scratch scratch_of(void* workspace, int64_t S, int64_t T, int64_t A, int dtype) {
  char* p = static_cast<char*>(workspace);
  size_t at = 0;
  auto take = [&](size_t bytes) {
    char* here = p ? p + at : nullptr;
    at += (size_t)round_up((int64_t)bytes, 256);
    return here;
  };
  Scratch s;
  s.counts = reinterpret_cast<int*>(take((kCountBlocks + 1) * sizeof(int)));
  s.order = reinterpret_cast<int*>(take((size_t)(S * T) * sizeof(int)));
  s.lengths = reinterpret_cast<int*>(take((size_t)S * sizeof(int)));
  s.sums = reinterpret_cast<double*>(take(sizeof(double) * kSums * kMaxPartials));
  s.parts = reinterpret_cast<Stat*>(take((size_t)(S * T) * row_splits(S * T, A, dtype) *
                                         sizeof(FineStat)));
  s.bytes = at;
  return s;
}

static bool sizes_ok(int64_t S, int64_t T, int64_t A) {
  return A <= ((int64_t)1 << 30) && (T == 0 || S < ((int64_t)1 << 31) / T) && S < ((int64_t)1 << 31) &&
         T < ((int64_t)1 << 31) && S * T <= ((int64_t)1 << 46) / A;
}

int take_rows(const ppo_token_rows* r, bool actions, Rows& out) {
  if (!r || !dtype_ok(r->dtype) || r->sequences < 0 || r->tokens < 0 || r->A <= 0 ||
      !(r->temperature > 0.0))
    return PPO_ERR_INVALID_ARG;
  const double exact = 1.44269504088896340736 / r->temperature;
  const float c = (float)exact, c_down = (double)c < exact ? c : nextafterf(c, 0.0f);
  // (what is left underflows at temperatures near the type's largest value)
  const float c_left = fmaxf((float)(exact - (double)c_down), __FLT_DENORM_MIN__);
  const float inv_tau = (float)(1.0 / r->temperature);
  if (!(c > 0.0f) || !(c < INFINITY)) return PPO_ERR_INVALID_ARG;
  if (!sizes_ok(r->sequences, r->tokens, r->A)) return PPO_ERR_TOO_LARGE;
  out = {r->logits, r->actions, r->mask, r->sequences * r->tokens, r->tokens, r->sequences,
         (int)r->A, r->actions_are_int64, c, inv_tau, c_down, c_left};
  if (out.n == 0) return PPO_OK;
  const uintptr_t size = dtype_size(r->dtype);
  if (!r->logits || (uintptr_t)r->logits % size || (actions && !r->actions))
    return PPO_ERR_INVALID_ARG;
  return PPO_OK;
}

namespace {

// Rows that count, by workgroup.
__global__ void __launch_bounds__(256) count_rows_kernel(const uint8_t* mask, int64_t n, int* counts) {
  __shared__ int part[4];
  int k = 0;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256)
    k += mask[i] != 0;
  const int lane = threadIdx.x & (kWave - 1);
  k = (int)lanes_sum<kWave>((float)k);  // (a lane's few hundred: exact)
  if (lane == 0) part[threadIdx.x / kWave] = k;
  __syncthreads();
  if (threadIdx.x == 0) counts[blockIdx.x] = part[0] + part[1] + part[2] + part[3];
}

// Rows that count in each sequence, a wave to a sequence, and by workgroup the
// sequences that have any.
__global__ void __launch_bounds__(256) count_sequences_kernel(const uint8_t* mask, int64_t S,
                                                              int64_t T, int* lengths, int* counts) {
  __shared__ int part[4];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  int some = 0;
  for (int64_t s = (int64_t)blockIdx.x * 4 + wave; s < S; s += (int64_t)gridDim.x * 4) {
    int k = 0;
    for (int64_t i = lane; i < T; i += kWave) k += mask[s * T + i] != 0;
    const double all = lanes_sum<kWave>((double)k);
    if (lane == 0) lengths[s] = (int)all;
    some += all > 0.0;
  }
  if (lane == 0) part[wave] = some;
  __syncthreads();
  if (threadIdx.x == 0) counts[blockIdx.x] = part[0] + part[1] + part[2] + part[3];
}

// Rows that count, ascending, then the others, descending, by one workgroup: 1024 rows a
// round, a wave's by ballot, the waves' by their sums.  (The others are placed from the end,
// so that neither kind needs the other's number.)
__global__ void __launch_bounds__(1024) order_kernel(const uint8_t* mask, int n, int* order,
                                                     int* live) {
  __shared__ int part[2][16];
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  int done = 0;  // rows that count before this round
  for (int base = 0, k = 0; base < n; base += 1024, k ^= 1) {
    const int r = base + threadIdx.x;
    const bool in = r < n && mask[r] != 0;
    const unsigned long long votes = __ballot(in);
    if (lane == 0) part[k][wave] = __builtin_popcountll(votes);
    __syncthreads();  // (two sets of sums: one barrier a round)
    int before = 0, all = 0;
    for (int w = 0; w < 16; ++w) {
      if (w < wave) before += part[k][w];
      all += part[k][w];
    }
    const int mine = done + before + __builtin_popcountll(votes & ((1ull << lane) - 1));
    if (r < n) order[in ? mine : n - 1 - (r - mine)] = r;
    done += all;
  }
  if (threadIdx.x == 0) *live = done;
}

}  // namespace

void count_weights(const Rows& rows, const Weights& w, const Scratch& s, hipStream_t stream) {
  if (w.lengths)
    hipLaunchKernelGGL(count_sequences_kernel, dim3(w.partials), dim3(256), 0, stream, rows.mask,
                       rows.S, rows.T, s.lengths, s.counts);
  else if (w.counts)
    hipLaunchKernelGGL(count_rows_kernel, dim3(w.partials), dim3(256), 0, stream, rows.mask, rows.n,
                       s.counts);
}

Order take_order(const Rows& rows, Weights& w, const Scratch& s, hipStream_t stream) {
  int* live = s.counts + kCountBlocks;
  if (w.counts && !w.lengths) {  // (the order counts the rows, 4 us less)
    w.counts = live;
    w.partials = 1;
  } else {
    count_weights(rows, w, s, stream);
  }
  hipLaunchKernelGGL(order_kernel, dim3(1), dim3(1024), 0, stream, rows.mask, (int)rows.n, s.order,
                     live);
  return {s.order, live};
}

int take_weights(const Rows& rows, const ppo_token_loss* loss, const Scratch& s, Weights& w) {
  const bool sequences = loss->reduction == PPO_SEQUENCE_MEAN;
  const auto held = [](double x) { return x >= PPO_TOKEN_LEAST && x <= PPO_TOKEN_MOST; };
  if ((loss->reduction != PPO_TOKEN_MEAN && !sequences) ||
      (loss->denominator != 0.0 && !held(loss->denominator)) || !held(loss->grad_scale))
    return PPO_ERR_INVALID_ARG;
  w = {nullptr, nullptr, 0, 0.0f};
  if (loss->denominator > 0.0) w.inverse = (float)(1.0 / loss->denominator);
  if (!rows.mask) {
    // every sequence is as long as the others
    if (loss->denominator > 0.0)
      w.inverse = (float)(1.0 / (sequences ? loss->denominator * (double)rows.T : loss->denominator));
    else
      w.inverse = rows.n ? (float)(1.0 / (double)rows.n) : 0.0f;
    return PPO_OK;
  }
  if (rows.n == 0) return PPO_OK;
  if (sequences) {
    w.partials = launch_blocks(div_up(rows.S, 4), kCountBlocks);
    w.counts = s.counts;
    w.lengths = s.lengths;
  } else if (!(w.inverse > 0.0f)) {
    w.partials = launch_blocks(div_up(rows.n, 1024), kCountBlocks);
    w.counts = s.counts;
  }
  return PPO_OK;
}

namespace {

// What ppo_token_log_probs leaves of a row.
template <class S>
struct LogProbs {
  using Sums = S;
  static constexpr bool kWholeWave = false;
  const float* minus;
  float *log_probs, *entropy;
  Saved* saved;

  __device__ __forceinline__ void masked(int64_t r) const {
    log_probs[r] = 0.0f;
    if (entropy) entropy[r] = 0.0f;
  }
  template <bool kEntropy>
  __device__ __forceinline__ void row(const Rows& rows, int64_t r, S x, float la, bool first) {
    const RowTerms t = row_terms<kEntropy>(x, la, Scale<S>(rows));
    if (!first) return;
    log_probs[r] = (float)(minus ? t.lp - (double)minus[r] : t.lp);
    if (entropy) entropy[r] = t.H;
    if (saved) saved[r] = saved_of(t, 0.0f);
  }
  __device__ __forceinline__ void end() const {}
};

// The gradient of a row's log-probability and entropy.
struct LogProbsGrad : GradientTerms {
  const Saved* saved;
  const float *dlp, *dent;

  template <class T, int G>
  __device__ __forceinline__ Grad row(const Rows& rows, int64_t r, const T*, float up, int a, int,
                                      bool, int*) const {
    return row_grad(saved[r], dlp ? up * dlp[r] : 0.0f, dent ? up * dent[r] : 0.0f, rows.inv_tau, a);
  }
};

struct Preferences {
  const float* rel;
  const uint8_t* mask;
  int64_t pairs, T;
  double beta, margin, smoothing;
  int average;
  double* losses;
  float *rewards, *coef;
};

// Pair i by `lanes` lanes (t: this one), a wave or a team of waves that all come here,
// with i behind the last pair too: the two sequences' sums in 64 bits, the loss, and the
// coefficient of each of their rows.  The sums are over differences to the reference's
// log-probabilities, so they are small where the policies are alike.  Returns the loss.
template <bool kTeam>
__device__ __forceinline__ double pair_loss(const Preferences& p, int64_t i, int t, int lanes,
                                            double (*part)[4]) {
  const int wave = threadIdx.x / kWave;
  const int64_t T = i < p.pairs ? p.T : 0;
  double sum[2], n[2];
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const int64_t at = (i + k * p.pairs) * p.T;
    double x = 0.0, m = 0.0;
#pragma unroll 4
    for (int64_t j = t; j < T; j += lanes) {
      const bool live = !p.mask || p.mask[at + j];
      const float rel = p.rel[at + j];  // (both loads at once)
      x += live ? (double)rel : 0.0;
      m += live ? 1.0 : 0.0;
    }
    sum[k] = lanes_sum<kWave>(x);
    n[k] = lanes_sum<kWave>(m);
    if (kTeam && (t & (kWave - 1)) == 0) {
      part[wave][k] = sum[k];
      part[wave][2 + k] = n[k];
    }
  }
  if (kTeam) {
    __syncthreads();
    const int first = wave - t / kWave;
#pragma unroll
    for (int k = 0; k < 2; ++k) {
      sum[k] = n[k] = 0.0;
      for (int w = first; w < first + lanes / kWave; ++w) {
        sum[k] += part[w][k];
        n[k] += part[w][2 + k];
      }
    }
    __syncthreads();
  }
  if (i >= p.pairs) return 0.0;
  const double w0 = p.average && n[0] > 0.0 ? 1.0 / n[0] : 1.0;
  const double w1 = p.average && n[1] > 0.0 ? 1.0 / n[1] : 1.0;
  const double r0 = p.beta * sum[0] * w0, r1 = p.beta * sum[1] * w1;
  const double m = r0 - r1 - p.margin;
  // -log sigmoid(m) = max(-m, 0) + log(1 + e^-|m|), and sigmoid(m) from the same e
  const double e = exp(-fabs(m)), soft = log1p(e);
  const double up = soft + fmax(-m, 0.0), down = soft + fmax(m, 0.0);
  const double sig = m >= 0.0 ? 1.0 / (1.0 + e) : e / (1.0 + e);
  const double not_sig = m >= 0.0 ? e / (1.0 + e) : 1.0 / (1.0 + e);
  // sigmoid(m) - (1 - smoothing), without the cancellation at m large
  const double dm = p.smoothing * sig - (1.0 - p.smoothing) * not_sig;
  if (t == 0) {
    p.rewards[i] = (float)r0;
    p.rewards[i + p.pairs] = (float)r1;
  }
  const double each = dm / (double)p.pairs * p.beta;
#pragma unroll
  for (int k = 0; k < 2; ++k) {
    const float g = (float)(each * (k ? -w1 : w0));
    const int64_t at = (i + k * p.pairs) * p.T;
#pragma unroll 4
    for (int64_t j = t; j < T; j += lanes) p.coef[at + j] = !p.mask || p.mask[at + j] ? g : 0.0f;
  }
  // (0 times an infinite part is no part; a NaN margin stays one)
  return (p.smoothing < 1.0 ? (1.0 - p.smoothing) * up : 0.0) +
         (p.smoothing > 0.0 ? p.smoothing * down : 0.0) + (m == m ? 0.0 : m);
}

// Pairs whose sequences a wave takes by itself (pairs of 31 tokens 4 us, 7 by more; 64
// pairs of 1024, past the border, take 9.2, and 7.8 by a wave each).
constexpr int64_t kWaveTokens = 512;

// Few pairs: one workgroup takes them all and their mean, one launch where two would
// take 5 us more; a wave to a pair, or up to eight pairs at once by a share of the sixteen
// waves each (a pair of 16384 tokens 140 -> 17 us).
constexpr int64_t kFewTokens = 32768, kFewPairs = 16;
__global__ void __launch_bounds__(1024) few_preferences_kernel(Preferences p, float* loss) {
  __shared__ double part[16][4], losses[16];
  const int wave = threadIdx.x / kWave, lane = threadIdx.x & (kWave - 1);
  double v = 0.0;
  if (p.pairs <= 8 && p.T > kWaveTokens) {
    const int lanes = p.pairs == 1 ? 1024 : p.pairs == 2 ? 512 : p.pairs <= 4 ? 256 : 128;
    const int t = threadIdx.x & (lanes - 1);
    v = pair_loss<true>(p, threadIdx.x / lanes, t, lanes, part);
    if (t != 0) v = 0.0;  // (a pair's loss once)
  } else if (wave < p.pairs) {
    v = pair_loss<false>(p, wave, lane, kWave, nullptr);
  }
  if (lane == 0) losses[wave] = v;
  __syncthreads();
  if (threadIdx.x != 0) return;
  double all = 0.0;
  for (int w = 0; w < 16; ++w) all += losses[w];
  *loss = (float)(all / (double)p.pairs);
}

// A wave to a pair, or a workgroup.
template <bool kTeam>
__global__ void __launch_bounds__(1024) preferences_kernel(Preferences p) {
  __shared__ double part[16][4];
  const int lanes = kTeam ? blockDim.x : kWave, teams = blockDim.x / lanes;
  const int t = threadIdx.x % lanes;
  for (int64_t i = (int64_t)blockIdx.x * teams + threadIdx.x / lanes; i < p.pairs;
       i += (int64_t)gridDim.x * teams) {
    const double v = pair_loss<kTeam>(p, i, t, lanes, part);
    if (t == 0) p.losses[i] = v;
  }
}

__global__ void __launch_bounds__(1024) mean_kernel(const double* x, int64_t n, float* out) {
  __shared__ double part[16];
  double v = 0.0;
#pragma unroll 4
  for (int64_t i = threadIdx.x; i < n; i += 1024) v += x[i];
  v = lanes_sum<kWave>(v);
  if ((threadIdx.x & (kWave - 1)) == 0) part[threadIdx.x / kWave] = v;
  __syncthreads();
  if (threadIdx.x != 0) return;
  double all = 0.0;
  for (int w = 0; w < 16; ++w) all += part[w];
  *out = (float)(all / (double)n);
}

}  // namespace
}  // namespace ppo

extern "C" size_t ppo_token_workspace_bytes(int64_t sequences, int64_t tokens, int64_t A,
                                            int dtype) {
  using namespace ppo;
  if (sequences <= 0 || tokens <= 0 || A <= 0 || !dtype_ok(dtype) ||
      !sizes_ok(sequences, tokens, A))
    return 0;
  return scratch_of(nullptr, sequences, tokens, A, dtype).bytes;
}

extern "C" int ppo_token_log_probs(const ppo_token_rows* r, const float* minus, float* log_probs,
                                   float* entropy, float* saved, void* workspace,
                                   size_t workspace_bytes, void* stream_ptr) {
  using namespace ppo;
  Rows rows;
  if (const int code = take_rows(r, true, rows)) return code;
  if (rows.n == 0) return PPO_OK;
  if (!log_probs || (saved && !aligned16(saved))) return PPO_ERR_INVALID_ARG;
  const Scratch s = scratch_of(workspace, rows.S, rows.T, rows.A, r->dtype);
  if (!workspace || !aligned16(workspace) || workspace_bytes < s.bytes) return PPO_ERR_WORKSPACE;
  return with_dtype(r->dtype, [&](auto zero) {
    using T = decltype(zero);
    hipStream_t stream = (hipStream_t)stream_ptr;
    const bool again = saved && rows.n * rows.A * (int64_t)sizeof(T) <= kReadAgain;
    auto go = [&](auto sums) {
      const LogProbs<decltype(sums)> emit = {minus, log_probs, entropy,
                                             reinterpret_cast<Saved*>(saved)};
      return entropy ? launch_statistics<T, true, true>(rows, s, emit, again, stream)
                     : launch_statistics<T, false, true>(rows, s, emit, again, stream);
    };
    return minus ? go(FineStat{}) : go(Stat{});
  });
}

extern "C" int ppo_token_log_probs_backward(const ppo_token_rows* r, const float* saved,
                                            const float* d_log_probs, const float* d_entropy,
                                            const float* scale, double held, void* dlogits,
                                            void* stream_ptr) {
  using namespace ppo;
  Rows rows;
  if (const int code = take_rows(r, true, rows)) return code;
  if (rows.n == 0) return PPO_OK;
  if (!saved || !aligned16(saved) || (!d_log_probs && !d_entropy) || !dlogits || (held != 0.0 && !scale) ||
      (uintptr_t)dlogits % dtype_size(r->dtype))
    return PPO_ERR_INVALID_ARG;
  const LogProbsGrad grad = {{}, reinterpret_cast<const Saved*>(saved), d_log_probs, d_entropy};
  return with_dtype(r->dtype, [&](auto zero) {
    using T = decltype(zero);
    hipStream_t stream = (hipStream_t)stream_ptr;
    return d_entropy
               ? launch_gradient<T, true>(rows, grad, scale, (float)held, (T*)dlogits, 0, stream)
               : launch_gradient<T, false>(rows, grad, scale, (float)held, (T*)dlogits, 0, stream);
  });
}

extern "C" size_t ppo_token_preference_workspace_bytes(int64_t sequences) {
  return sequences > 0 ? (size_t)sequences / 2 * sizeof(double) : 0;
}

extern "C" int ppo_token_preference(const float* relative, const uint8_t* mask, int64_t sequences,
                                    int64_t tokens, double beta, double margin, double smoothing,
                                    int average, float* loss, float* rewards, float* coef,
                                    void* workspace, size_t workspace_bytes, void* stream_ptr) {
  using namespace ppo;
  if (sequences <= 0 || sequences % 2 || tokens < 0 || !isfinite(beta) || !isfinite(margin) ||
      !(smoothing >= 0.0 && smoothing <= 1.0) || !loss || !rewards ||
      (tokens > 0 && (!relative || !coef)))
    return PPO_ERR_INVALID_ARG;
  if (!sizes_ok(sequences, tokens, 1)) return PPO_ERR_TOO_LARGE;
  if (!workspace || !aligned16(workspace) ||
      workspace_bytes < ppo_token_preference_workspace_bytes(sequences))
    return PPO_ERR_WORKSPACE;
  hipStream_t stream = (hipStream_t)stream_ptr;
  const Preferences p = {relative, mask, sequences / 2, tokens, beta, margin, smoothing, average,
                         static_cast<double*>(workspace), rewards, coef};
  if (sequences * tokens <= kFewTokens && p.pairs <= kFewPairs) {
    hipLaunchKernelGGL(few_preferences_kernel, dim3(1), dim3(1024), 0, stream, p, loss);
    return last_launch_status();
  }
  if (tokens <= kWaveTokens)
    hipLaunchKernelGGL(preferences_kernel<false>,
                       dim3(launch_blocks(div_up(p.pairs, 4), kMaxPartials)), dim3(256), 0, stream, p);
  else
    hipLaunchKernelGGL(preferences_kernel<true>, dim3(launch_blocks(p.pairs, kMaxPartials)),
                       dim3(tokens > 2048 ? 1024 : 256), 0, stream, p);
  hipLaunchKernelGGL(mean_kernel, dim3(1), dim3(1024), 0, stream, p.losses, p.pairs, loss);
  return last_launch_status();
}
