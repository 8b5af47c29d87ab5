/*
 * ppo_tokens.h — C ABI of `libppo_tokens.so`: token policies on MI355X (gfx950),
 * policies that pick one of A actions (up to a vocabulary) at every step of S
 * sequences of T tokens, trained from their logits.  Beside the PPO update of
 * ppo_amd.h, whose losses are made for fp32 and tens to hundreds of actions.
 *
 * Conventions are those of ppo_amd.h: device pointers owned by the caller,
 * every call only enqueues work on `stream` of the current device, dense
 * row-major layouts, PPO_OK or a PPO_ERR_* code (ppo_amd_strerror renders
 * it).  `workspace` is scratch of at least ppo_token_workspace_bytes(), 16-byte
 * aligned, whose contents on entry do not matter and mean nothing afterwards;
 * calls that share one must be ordered.  No call keeps state.
 *
 * Logits are `dtype` (fp32, bf16 or fp16), rows of any width A at any address
 * that the type allows.  With z = logits / temperature, p = softmax(z) of a row.
 * Statistics, log-probabilities and losses are held in 32 bits or more; a
 * gradient is formed in fp32 and rounded once, to nearest even.  A logit of -inf
 * is an action that cannot be taken: p = 0, no gradient, no part in the entropy (one
 * that was taken all the same has log p = -inf and, as 1 - p = 1, log p's whole gradient).
 * A row that holds +inf or NaN, or nothing but -inf, gives NaN, and so does a
 * row whose action lies outside [0, A) (it is never dereferenced).
 *
 * mask [rows], one byte each (NULL: every row counts): where it is 0 the
 * logits, the action and the row's other inputs are not read, its
 * log-probability, entropy and gradients are 0, and it has no part in a loss.
 *
 * Logits that another stream writes during a call give undefined results (top's
 * columns lie in their rows all the same).
 *
 * Rows times A up to 2^46, A up to 2^30, rows below 2^24, more where a row takes fewer than
 * 256 lanes (top: below 2^24, 2^23 and 2^22 for K up to 96, 192 and 256, and below 2^26
 * of up to 8 KB with K up to 48 or A up to 512): PPO_ERR_TOO_LARGE otherwise.
 */
#ifndef PPO_TOKENS_H
#define PPO_TOKENS_H

#include <stddef.h>
#include <stdint.h>

#include "ppo_amd.h"
#include "ppo_layers.h" /* PPO_DTYPE_* */

#ifdef __cplusplus
extern "C" {
#endif

#if defined(__GNUC__)
#pragma GCC visibility push(default)
#endif

/* The rows of a call: sequences * tokens of them, sequence by sequence. */
typedef struct ppo_token_rows {
  const void* logits;   /* [sequences, tokens, A] of dtype                     */
  const void* actions;  /* [sequences, tokens] int32 or int64                  */
  const uint8_t* mask;  /* [sequences, tokens], or NULL                        */
  int64_t sequences, tokens, A;
  int dtype;
  int actions_are_int64;
  double temperature;   /* > 0                                                 */
} ppo_token_rows;

/* Scratch of the calls below over these rows (preference and top have their own). */
size_t ppo_token_workspace_bytes(int64_t sequences, int64_t tokens, int64_t A, int dtype);

/* Floats per row of `saved`, which a forward pass writes for its backward. */
#define PPO_TOKEN_SAVED 8

/*
 * log_probs[r] = log p[action] - minus[r] (minus may be NULL: 0; the difference is
 * formed in 64 bits and rounded once), entropy[r] = -sum p log p (may be NULL).
 * saved fp32 [rows][PPO_TOKEN_SAVED], 16-byte aligned, may be NULL.
 */
int ppo_token_log_probs(const ppo_token_rows* rows, const float* minus, float* log_probs,
                        float* entropy, float* saved, void* workspace, size_t workspace_bytes,
                        void* stream);

/*
 * dlogits = up * (d_log_probs[r] dlog p[a]/dlogits + d_entropy[r] dH/dlogits) from the
 * forward's saved, either may be NULL; up = *scale (device memory, read when
 * the kernel runs), 1 without it.  held, when not 0, says that dlogits already
 * holds the gradient for up = held: the call leaves it as it is where *scale
 * equals held.
 */
int ppo_token_log_probs_backward(const ppo_token_rows* rows, const float* saved,
                                 const float* d_log_probs, const float* d_entropy,
                                 const float* scale, double held, void* dlogits, void* stream);

/* How a loss weighs its rows. */
#define PPO_TOKEN_MEAN 0     /* 1 / rows that count                             */
#define PPO_SEQUENCE_MEAN 1  /* 1 / (the sequence's rows that count * sequences
                                that have any)                                  */

/* Where a denominator and a grad_scale lie: weights are held in fp32. */
#define PPO_TOKEN_LEAST 1e-30
#define PPO_TOKEN_MOST 1e30

typedef struct ppo_token_loss {
  double clip_low, clip_high;  /* ratio within [1 - clip_low, 1 + clip_high]     */
  double kl_coef, entropy_coef; /* finite in fp32                                */
  double denominator;          /* > 0: in place of the number of rows (of
                                  sequences) that count; 0: that number          */
  double grad_scale;           /* the gradients are formed for this incoming one */
  int reduction;
  int advantages_per_sequence; /* advantages [sequences] instead of one a row    */
} ppo_token_loss;

/* Index of each scalar inside scalars[PPO_TOKEN_SCALARS]. */
#define PPO_TOKEN_SCALAR_LOSS 0
#define PPO_TOKEN_SCALAR_POLICY 1    /* clipped surrogate                          */
#define PPO_TOKEN_SCALAR_KL 2        /* to the reference policy                    */
#define PPO_TOKEN_SCALAR_ENTROPY 3
#define PPO_TOKEN_SCALAR_APPROX_KL 4 /* old_log_probs - log_probs                  */
#define PPO_TOKEN_SCALAR_CLIPFRAC 5  /* share of rows whose ratio leaves the clip  */
#define PPO_TOKEN_SCALARS 6

/*
 * The clipped policy loss with a KL term to a reference policy,
 *   ratio = exp(log p[a] - old),  d = ref - log p[a]
 *   loss  = sum_r w_r (-min(ratio adv, clip(ratio) adv)
 *                      + kl_coef (e^d - d - 1) - entropy_coef H)
 * the other scalars the same weighted sums of their terms.  The surrogate's
 * gradient is -ratio adv where the minimum takes the unclipped term (a tie
 * among them), 0 elsewhere.  ref_log_probs may be NULL when kl_coef is 0 (the KL scalar is
 * then 0).  dlogits may be NULL: no gradient.  Otherwise it receives
 * grad_scale * dloss/dlogits in the same pass over the logits, saved what
 * ppo_token_log_probs saves, and coef fp32 [2][rows] the rows' dloss/dlog p[a]
 * and dloss/dH, so that ppo_token_log_probs_backward gives the gradient for any
 * other incoming one (saved and coef may be NULL together).
 * Sums are formed in a fixed order: the same call gives the same bits.
 */
int ppo_token_policy_loss(const ppo_token_rows* rows, const float* old_log_probs,
                          const float* advantages, const float* ref_log_probs,
                          const ppo_token_loss* loss, float* scalars, float* saved, float* coef,
                          void* dlogits, void* workspace, size_t workspace_bytes, void* stream);

/*
 * The preference loss of sequence i (chosen) over sequence i + sequences / 2
 * (rejected), from relative[r] = log p[a] - ref of ppo_token_log_probs:
 *   L_s = sum_t relative (divided by the tokens that count where `average`)
 *   m_i = beta (L_chosen - L_rejected) - margin
 *   loss = mean_i of -(1 - smoothing) log sigmoid(m_i) - smoothing log sigmoid(-m_i)
 * rewards[s] = beta L_s; coef [rows] = dloss/dlog p[a], which is what
 * ppo_token_log_probs_backward takes.
 */
size_t ppo_token_preference_workspace_bytes(int64_t sequences);
int ppo_token_preference(const float* relative, const uint8_t* mask, int64_t sequences,
                         int64_t tokens, double beta, double margin, double smoothing, int average,
                         float* loss, float* rewards, float* coef, void* workspace,
                         size_t workspace_bytes, void* stream);

/*
 * Distillation from a teacher's K top logits (teacher [rows, K] of
 * teacher_dtype at the columns ids [rows, K]; K <= PPO_TOKEN_MAX_K):
 *   q = softmax(teacher / temperature) over the row's entries with ids >= 0
 *   loss = temperature^2 sum_r w_r sum_k q_k (log q_k - log p[id_k])
 * An id may come twice (its entries add up); negative ids are no entries, and a
 * row without entries, or with none but a teacher's -inf, has loss and gradient 0
 * and counts (NaN where its logits give it).  An id from A on gives NaN.
 * rows->actions is not read.  Of `loss`, reduction, denominator and grad_scale
 * count.  dlogits and saved may be NULL; backward forms the gradient for any
 * incoming one from saved, as ppo_token_log_probs_backward does.
 */
#define PPO_TOKEN_MAX_K 256
int ppo_token_distillation(const ppo_token_rows* rows, const void* teacher, int teacher_dtype,
                           const void* ids, int ids_are_int64, int64_t K,
                           const ppo_token_loss* loss, float* scalar, float* saved, void* dlogits,
                           void* workspace, size_t workspace_bytes, void* stream);
int ppo_token_distillation_backward(const ppo_token_rows* rows, const void* teacher,
                                    int teacher_dtype, const void* ids, int ids_are_int64,
                                    int64_t K, const float* saved, const float* scale,
                                    double held, void* dlogits, void* stream);

/*
 * The K largest of each row of logits [rows, A] in falling order with their
 * columns, K <= min(A, PPO_TOKEN_MAX_K).  Equal logits come in the order of
 * their columns, NaN before everything.  A up to 2^22: PPO_ERR_TOO_LARGE otherwise.
 */
size_t ppo_token_top_workspace_bytes(int64_t rows, int64_t A, int64_t K, int dtype);
int ppo_token_top(const void* logits, int dtype, int64_t rows, int64_t A, int64_t K, void* values,
                  int64_t* ids, void* workspace, size_t workspace_bytes, void* stream);

#if defined(__GNUC__)
#pragma GCC visibility pop
#endif

#ifdef __cplusplus
}
#endif

#endif /* PPO_TOKENS_H */
