/*
 * envpool_amd_policy.h - C ABI of the operators a policy on the GPU needs next to the pools: the choice
 * of an action from logits under the pool's legal-action mask, the log-probability and entropy of stored
 * actions with their gradients, and a linear-attention memory per env (one step over the rows of a
 * batch; a whole rollout segment with its gradients).
 *
 * Every pointer is device memory of GPU `device_id` unless said otherwise, `stream` is a hipStream_t of
 * that GPU (NULL = the legacy default stream). Calls enqueue kernels and return: nothing is allocated,
 * copied to the host or waited for, so they can be captured into a HIP graph. Scratch memory is the
 * caller's (`workspace`, at least as many bytes as the call's *_workspace function says; its contents
 * need not be kept between calls, but two calls that may run at the same time - two streams, two
 * captured graphs - need one each). Refusals are EP_ERR_INVALID with ep_last_error() naming the argument
 * (EP_ERR_TOO_LARGE: more rows, or states, than one launch can hold, some 16 million workgroups of 256;
 * EP_ERR_NO_DEVICE: no such GPU), and nothing has been enqueued then. No counterpart in the reference: its policies live outside it and
 * see numpy arrays (envpool2/python/envpool.py:135-142).
 */
#ifndef ENVPOOL_AMD_POLICY_H_
#define ENVPOOL_AMD_POLICY_H_

#include "envpool_amd.h"

#ifdef __cplusplus
extern "C" {
#endif

/* element types beside those of envpool_amd.h */
enum {
  EP_F16 = 7,
  EP_BF16 = 8
};

/* ---- logits under a mask --------------------------------------------------------------------------
 *
 * The distribution of row b over its options j = 0 .. options-1:
 *   x = logits[b, j];  c = how often j stands in history[b, :]
 *   c > 0:  x = x > 0 ? x / repetition : x * repetition;  x -= frequency * c + presence
 *   y = (x + bias[b, j]) / temperature
 *   j is legal iff j < num_options[b] (when given) and mask[b, j] (when given)
 *   p_j = exp(y_j) / sum over the legal options;  0 for the others, whose logits, biases and history are
 *   never used (they may hold anything, NaN included).
 * A row without a legal option, or whose legal options are all -inf, is EMPTY. A row with a NaN or +inf among
 * its legal y, or a per-row temperature or (with a history) repetition that is not > 0 and finite, is BAD. */
typedef struct {
  int32_t device_id;
  int32_t dtype;          /* of the logits: EP_F32, EP_F16 or EP_BF16 */
  int64_t rows, options;  /* options >= 1, <= 2^30 */
  const void* logits;
  int64_t logits_stride;  /* elements from one row to the next (>= options for more than one row) */
  const int32_t* num_options; /* [rows] or NULL; values outside [0, options] count as the nearer end (info:num_options) */
  const void* mask;       /* NULL, bytes (nonzero = legal; aux:action_mask) or bits */
  int32_t mask_dtype;     /* EP_BOOL / EP_U8: a byte per option; EP_I32: bit j % 32 of word j / 32 */
  int64_t mask_stride;    /* elements (bytes or words) from row to row; 0 = one mask for all rows */
  const void* bias;       /* NULL or values in bias_dtype (EP_F32, or the logits' type) */
  int32_t bias_dtype;
  int64_t bias_stride;    /* elements from row to row; 0 = one row of biases for all rows */
  const int32_t* history; /* NULL or [rows][history_len]: options chosen before; entries outside [0, options) count for nothing */
  int64_t history_len, history_stride;
  /* one value per row when the pointer is given, else the value beside it for all rows
   * (temperature, repetition: > 0; all finite; ep_policy_evaluate takes them in 32 bits, which have to hold them and the
   * reciprocals of those two: a number for all rows that is used is refused otherwise, a row's own makes it BAD) */
  const float *repetition, *frequency, *presence, *temperature;
  double repetition_all, frequency_all, presence_all, temperature_all;
  void* workspace;
  int64_t workspace_bytes;
  void* stream;
} ep_policy_rows;

/* action[b] (int32), log_prob[b] and entropy[b] (float) of the choice.
 * u: one number per row in [0, 1) (u_dtype EP_F32 or EP_F64): the option at which the cumulated
 * probability first exceeds it. u NULL: the most probable option, the lowest of equals. Evaluated in
 * 64 bits throughout, so that the choice does not depend on how sums were split.
 * EMPTY rows: action -1, log_prob 0, entropy 0. BAD rows: action -1, log_prob and entropy NaN. */
int ep_policy_choose(const ep_policy_rows* rows, const void* u, int32_t u_dtype, int32_t* action, float* log_prob,
                     float* entropy);
int64_t ep_policy_choose_workspace(const ep_policy_rows* rows);

/* log_prob[b] = log p of action[b], entropy[b] = -sum p log p, in 32 bits, and in stats[b] (two floats)
 * what ep_policy_evaluate_grad needs of the row. action -1 ("none", what EMPTY rows choose): log_prob 0 without
 * gradient; an illegal action: -inf; any other value outside [0, options): NaN. EMPTY rows: entropy 0,
 * log_prob 0 (-1) or -inf; BAD rows: NaN. */
int ep_policy_evaluate(const ep_policy_rows* rows, const int32_t* action, float* log_prob, float* entropy, float* stats);
int64_t ep_policy_evaluate_workspace(const ep_policy_rows* rows);

/* The gradients of sum_b (grad_log_prob[b] * log_prob[b] + grad_entropy[b] * entropy[b]): grad_logits in the
 * logits' type (stride in elements, all options written, 0 where illegal) and, where grad_bias is not NULL, in
 * bias_dtype the bias' gradient - [options], the sum over the rows in a fixed order, when bias_stride is 0
 * (an intermediate sum is kept in 32 bits), else [rows][options] with stride grad_bias_stride. `entropy` and
 * `stats` are what ep_policy_evaluate wrote for these rows. Either gradient in may be NULL (zero), and so may one of the
 * two out (not wanted). */
int ep_policy_evaluate_grad(const ep_policy_rows* rows, const int32_t* action, const float* entropy, const float* stats,
                            const float* grad_log_prob, const float* grad_entropy, void* grad_logits,
                            int64_t grad_logits_stride, void* grad_bias, int64_t grad_bias_stride);
int64_t ep_policy_evaluate_grad_workspace(const ep_policy_rows* rows, int32_t with_bias);

/* ---- memory ----------------------------------------------------------------------------------------
 *
 * Linear attention with a decay per head. Per env (or row) and head h a state S [key_dim][value_dim] in 32
 * bits, updated once per env-step:
 *   S = exp(log_decay[h]) * S_before + k^T v   (S_before = 0 when the step is the first of an episode)
 *   out = scale * q S
 * q, out have `heads` heads; k, v `kv_heads`, a divisor of it: head h reads k, v head h / (heads / kv_heads). */
typedef struct {
  int32_t device_id;
  int32_t dtype;  /* of q, k, v, out: EP_F32, EP_F16 or EP_BF16 */
  int64_t num_envs, rows;
  int32_t heads, kv_heads, key_dim, value_dim; /* dims 1 .. 256 */
  const void *q, *k, *v;  /* [rows][heads or kv_heads][dim], the last dimension dense */
  int64_t q_stride[2], k_stride[2], v_stride[2], out_stride[2]; /* elements: row, head */
  void* out;
  const float* log_decay; /* [heads], <= 0 */
  float* state;           /* [num_envs][heads][key_dim][value_dim], dense, updated in place */
  const int32_t* env_id;  /* [rows]: row r steps env env_id[r] - env_id_offset; NULL: row r steps env r (rows <= num_envs) */
  int32_t env_id_offset;
  const void* fresh;      /* NULL (no row starts an episode), or [rows] */
  int32_t fresh_dtype;    /* EP_BOOL / EP_U8: nonzero = first step; EP_I32: zero = first step (elapsed_step) */
  float scale;
  int32_t* error;         /* NULL or a word the kernel may set to 1 (memory the GPU can write; host-mapped is fine) */
  void* workspace;
  int64_t workspace_bytes;
  void* stream;
} ep_memory_step_args;

/* One step of the rows of a batch. A row whose env id is outside [env_id_offset, env_id_offset + num_envs)
 * touches no state, gets NaN in `out` and sets *error. An env named several times is stepped several
 * times, in row order (as ep_pool_send does for host arrays). Steps of one state table must be ordered
 * by the caller (one stream, or events). */
int ep_memory_step(const ep_memory_step_args* args);
int64_t ep_memory_step_workspace(const ep_memory_step_args* args);

/* Zeroes the states of the envs that `env_id` [rows] names (NULL: envs 0 .. rows-1), as often as it names them. Of `args`
 * only device_id, num_envs, rows, heads, key_dim, value_dim, state, env_id, env_id_offset, error and stream are looked at. An
 * id outside touches nothing and sets *error, as in a step. */
int ep_memory_reset(const ep_memory_step_args* args);

/* `steps` steps of `rows` independent rows at once (a rollout segment, time first; any strides with a dense
 * last dimension). reverse != 0 runs time backwards with the recurrence of the gradients:
 *   forward:  S_t = d_t S_{t-1} + inc_scale k_t^T v_t,  d_t = fresh[t] ? 0 : exp(log_decay);  S_{-1} = state_in,
 *             out_t = out_scale q_t S_t;  state_out = S_{steps-1}
 *   reverse:  S_t = d_{t+1} S_{t+1} + inc_scale k_t^T v_t, S_{steps-1} = state_in + inc_scale k^T v;
 *             out_t = out_scale q_t S_t;  state_out = d_0 S_0
 * so that, with o = forward(q, k, v) under `scale`, grad_q = forward(do, v, k; state_in^T) with out_scale = scale,
 * grad_v = reverse(k, q, do; d state_out) and grad_k = reverse(v, do, q; (d state_out)^T), both with inc_scale = scale.
 * S and all sums are kept in 32 bits; as operands of 16-bit products S and the scores q_t k_s^T enter with 16 bits (bf16) or 22
 * (f16), before out is rounded to out_dtype once. Values that are not finite reach the steps that the recurrence takes them to
 * and no others. */
typedef struct {
  int32_t device_id;
  int32_t dtype;
  int64_t steps, rows;
  int32_t heads;                     /* states per row */
  int32_t q_group, k_group, v_group; /* state h reads head h / group of the operand (groups divide heads) */
  int32_t key_dim, value_dim;        /* 1 .. 128 each */
  const void *q, *k, *v;
  int64_t q_stride[3], k_stride[3], v_stride[3], out_stride[3]; /* elements: step, row, head */
  void* out;                         /* [steps][rows][heads][value_dim]; NULL: only state_out is wanted */
  int32_t out_dtype;                 /* dtype, or EP_F32 */
  const float* log_decay;            /* [heads], <= 0 */
  const uint8_t* fresh;              /* NULL or [steps][rows]: nonzero = first step of an episode */
  int64_t fresh_stride[2];           /* step, row */
  const float* state_in;             /* NULL (zero) or one [key_dim][value_dim] per (row, head) */
  float* state_out;                  /* NULL or the same */
  int64_t state_in_stride[4], state_out_stride[4]; /* row, head, key, value */
  float inc_scale, out_scale;
  int32_t reverse;
  void* workspace;
  int64_t workspace_bytes;
  void* stream;
} ep_memory_scan_args;
int ep_memory_scan(const ep_memory_scan_args* args);
int64_t ep_memory_scan_workspace(const ep_memory_scan_args* args);

/* Two scans as one call, both on one device and stream and naming one workspace (of what
 * ep_memory_scan_pair_workspace says, or more). The gradients of values (a) and keys (b) of one forward scan - reverse scans
 * over the same tensors: a's k is b's v and the other way round - share their reads where their sizes allow it
 * (16-bit types, dims up to 64); any other two simply follow one another. Neither's results are read by the other. */
int ep_memory_scan_pair(const ep_memory_scan_args* a, const ep_memory_scan_args* b);
int64_t ep_memory_scan_pair_workspace(const ep_memory_scan_args* a, const ep_memory_scan_args* b);

/* out[i, j] = sum of `group` neighbouring heads of src (32 bits), rounded once to `dtype`: the gradients of
 * keys and values that several heads share. src [n][heads_out * group][dim] dense, out [n][heads_out][dim] dense. */
int ep_memory_sum_heads(int32_t device_id, const float* src, int64_t n, int32_t heads_out, int32_t group, int32_t dim,
                        void* out, int32_t dtype, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* ENVPOOL_AMD_POLICY_H_ */
