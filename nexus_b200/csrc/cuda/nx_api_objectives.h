// C ABI of the operators that fine-tune a language model on rewards and preferences: log-probabilities of given tokens, clipped
// policy loss, preference loss, global gradient norm over many tensors.  Conventions as in nx_api.h.
#pragma once
#include "nx_api.h"

#ifdef __cplusplus
extern "C" {
#endif

// Logits of `rows` tokens: row r starts at logits + (r / per) * stride_outer + (r % per) * stride_inner elements (any alignment of the
// element) and has `width` elements, of which the first `vocab` are the vocabulary.  targets [rows]: int32 or int64; a row whose target is
// `ignore_index` is not read, one whose target lies outside the vocabulary gives NaN and a gradient of zeros.
typedef struct NxTokenRows {
  const void* logits;
  const void* targets;
  int64_t rows, per, stride_outer, stride_inner, ignore_index;
  int32_t dtype;         // NX_BF16, NX_F16 or NX_F32
  int32_t targets_wide;  // targets are int64
  int32_t vocab, width;
  float inv_temp;        // the logits are multiplied by it
  int32_t pad_;
} NxTokenRows;

// logp [rows] = log-probability of the target (0 where ignored); stats [rows] pairs: a logit x, and log2 of the sum of
// exp((logit - x) * inv_temp).
// status: device int, receives a non-zero nx::StatusCode when a wait timed out.
// wide [rows], may be null: logp before it is rounded to FP32.
int nx_token_logprobs(const NxTokenRows* rows, float* logp, float* stats, double* wide, int* status, nx_stream_t stream);
// A gradient has the layout and type of the logits and starts at the same place of a 16-byte line.
// grad = coef (delta_target - p) * inv_temp (zeros in ignored rows and behind the vocabulary);
// coef of row r: coef[r / coef_per] * *factor (factor: device scalar, may be null)
int nx_token_logprobs_grad(const NxTokenRows* rows, const float* stats, const float* coef, int64_t coef_per, const float* factor,
                           void* grad, nx_stream_t stream);

enum NxPolicyKl { NX_KL_K1 = 0, NX_KL_K2 = 1, NX_KL_K3 = 2 };
enum NxPolicyMean { NX_MEAN_TOKEN = 0, NX_MEAN_SEQUENCE = 1, NX_MEAN_NONE = 2 };
typedef struct NxPolicyArgs {
  const float* old_logp;    // [rows]
  const float* ref_logp;    // [rows], may be null (no KL term)
  const float* advantages;  // advantage of row r: advantages[r / adv_per]
  int64_t adv_per;
  int64_t seq_len;          // tokens of a sequence: row r belongs to sequence r / seq_len
  float clip_low, clip_high, kl_coef, entropy_coef, scale;
  int32_t kl, mean;
  int32_t write_grad;
} NxPolicyArgs;
// What a row's gradient is made of: p_j (slope (logit_j - x) + off) with p_j = 2^((logit_j - x) inv_temp log2 e - log2_s), and c more at the target.
typedef struct NxPolicySlope {
  float x, log2_s, c, slope, off;
} NxPolicySlope;
// Clipped policy loss with KL and entropy terms.  logp, kl, entropy, row_loss: [rows]; totals: three doubles, counts: [rows / seq_len],
// both scratch; loss: one float; at least one row;
// grad (write_grad; BF16, FP32): d loss / d logits in the layout and type of the logits; slopes [rows], may be null: for nx_policy_loss_grad.
int nx_policy_loss(const NxTokenRows* rows, const NxPolicyArgs* args, double* totals, int32_t* counts, float* logp, float* kl, float* entropy,
                   float* row_loss, float* loss, void* grad, NxPolicySlope* slopes, int* status, nx_stream_t stream);
// grad = *factor (device scalar) * d loss / d logits, FP16 logits only: a loss scale has to be in the gradient before it is rounded
int nx_policy_loss_grad(const NxTokenRows* rows, const NxPolicySlope* slopes, const float* factor, void* grad, nx_stream_t stream);
// x *= *factor in place, n elements (BF16, FP32); nothing is read or written where the factor is 1
int nx_scale_unless_one(void* x, const float* factor, int dtype, int64_t n, nx_stream_t stream);

enum NxPreferenceKind { NX_PREF_SIGMOID = 0, NX_PREF_HINGE = 1, NX_PREF_IPO = 2 };
typedef struct NxPreferenceArgs {
  const double* logp;      // [2 * pairs, seq_len] per token, chosen sequences first
  const void* targets;     // [2 * pairs, seq_len]
  const float* ref_logp;   // [2 * pairs], may be null
  int64_t pairs, seq_len, ignore_index;
  int32_t targets_wide, kind, average;
  float beta, smoothing, target_margin;
} NxPreferenceArgs;
// seq_logp [2 * pairs], margin [pairs], coef [2 * pairs] = d loss / d logp of each counted token, loss: one float
int nx_preference_loss(const NxPreferenceArgs* args, float* seq_logp, float* margin, float* coef, float* loss, nx_stream_t stream);

// Log-probabilities of `targets` [rows] under softmax(hidden weight^T * inv_temp), hidden [rows, width] of pitch ld_hidden, weight
// [vocab, width] of pitch ld_weight, BF16 or FP16 (16-byte bases; width and pitches multiples of 8).  `index` [rows], `count` [1] and
// `gathered` [rows rounded up to 64, width], all three or none (the gradient wants them): the rows that count are brought together before
// the products (the forward call fills index and count; `gathered` is filled by both, with `weights` by the forward call for the gradient
// too).  stats [rows] pairs, written by the forward call, read by the gradient.
typedef struct NxHeadArgs {
  const void* hidden;
  const void* weight;
  const void* targets;
  int32_t* index;
  int32_t* count;
  void* gathered;
  float* stats;
  float* part;     // [2 * (vocab / 256 rounded up), part_rows] pairs: scratch of the forward call, which takes part_rows (a multiple of 256) rows
                   // at a time; with `weights` all at once, and read by the gradient too
  void* weights;   // may be null: [rows rounded up to 256, ld_weights] of the operands' type, the logits' exponentials for the gradient
  int* status;     // receives a non-zero nx::StatusCode when a wait timed out
  int64_t part_rows, ld_weights, rows, ld_hidden, ld_weight, ignore_index;
  int32_t vocab, width, dtype, targets_wide;
  float inv_temp;
  int32_t pad_;
} NxHeadArgs;
// logp [rows] (0 where ignored, NaN where the target lies outside the vocabulary); tlogit [rows]: scratch
int nx_head_logprobs(const NxHeadArgs* args, float* logp, float* tlogit, nx_stream_t stream);
typedef struct NxHeadGrad {
  const float* coef;       // [rows] gradient of logp
  void* logit_grad;        // scratch [chunk, ld_logit_grad] of the operands' type: rows are taken `chunk` (a multiple of 256) at a time; with
                           // `weights` all at once, ld_weights apart, and it may be the same memory
  int64_t chunk, ld_logit_grad;  // ld a multiple of 64
  float* scale;            // two floats of scratch (FP16)
  void* d_hidden;          // [rows, width], may be null
  void* d_weight;          // [vocab, width], may be null
  float* slice_sums;       // slices > 1: scratch [slices, chunk, width]: the vocabulary may be cut into so many to fill the machine
  float* weight_sums;      // chunk < rows: scratch [vocab, width]
  int32_t slices, pad_;
} NxHeadGrad;
int nx_head_logprobs_grad(const NxHeadArgs* args, const NxHeadGrad* grad, nx_stream_t stream);

// Gradients of `tensors` tensors (host arrays): count elements at src, of NxDType `type & 15`; the clipped ones go to dst, of type `type >> 4`
// (dst null: in place, both types the same).
typedef struct NxGradTable {
  const void* const* src;
  void* const* dst;
  const int64_t* count;
  const uint8_t* type;
  int64_t tensors;
} NxGradTable;
// partial: 592 doubles per 256 tensors or part of them.
// out[0] = sum of squares; (float*)(out + 1) = norm = sqrt of it.  clip: the gradients times min(1, max_norm / (norm + 1e-6)); where the norm
// is not finite they stay (dst: are copied) as they are.  Sums in a fixed order.
int nx_grad_clip(const NxGradTable* table, double max_norm, int clip, double* partial, double* out, nx_stream_t stream);

#ifdef __cplusplus
}
#endif
