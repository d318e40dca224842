/* Operators of a policy with memory, for the batched env's learners: attention with a state that decays per
 * head (a sequence at a time with its gradients, and one token at a time), and dropout whose mask is drawn
 * from the transition's own id.  The reference's policy side is SB3's PPO (gymnasium_src/scripts/regular_rl/
 * rl/train_rl.py:60-75), with a sequence feature extractor over stacked frames (:26-35).
 *
 * Attention.  For each sequence b and query head h (key / value head h / (heads / kv_heads)), with
 * a_t = 0 where starts[b][t], else exp(log_decay[h]):
 *     S_t = a_t S_{t-1} + k_t v_t^T        S_{-1} = s0 (0 when null), [dk][dv], float
 *     o_t = scale * S_t^T q_t
 * Tokens t >= lengths[b] are padding: their outputs and gradients are 0 and they leave the state alone; nothing
 * they hold is used.  Nothing in front of a start, whatever its values, reaches a token behind it.  log_decay is at
 * most 0; -inf keeps the token alone.  What a NaN or an infinity reaches by the formula is not finite, and nothing else.
 *
 * Element types: 0 float, 1 bfloat16, 2 IEEE half, the same for every token tensor of a call.  States,
 * log_decay and all sums are float.  With 16-bit tokens a float operand of a product (scores, the state where it is read out,
 * keys that enter a state without s_out or ds0) is taken to 17 bits, as two bfloat16 parts; keys that enter a state which
 * leaves to 25, as three.  With float tokens every product is float.  All pointers are device pointers on the current HIP device; strides
 * are in elements, the channels of a token are contiguous, token strides are not negative.  Outputs overlap nothing
 * else.  Work is enqueued on `stream`; nothing is kept between calls, and a call may be captured into a graph; calls that
 * may run at once need workspaces of their own.  Results do not depend on timing (no atomics).
 *
 * Limits: dk, dv in [1, 128]; b * heads below 2^22; t at most 2^30; with shared heads or less than four channels,
 * b * t * heads * ceil(channels / 4) below 2^32 - 256.
 *
 * Errors: UR3E_EINVAL / UR3E_EHIP (ur3e_batch.h) with ur3e_last_error(); nothing is launched on EINVAL.
 */
#ifndef UR3E_POLICY_H
#define UR3E_POLICY_H

#include <stddef.h>

#ifdef __cplusplus
extern "C" {
#endif

#define UR3E_F32 0
#define UR3E_BF16 1
#define UR3E_F16 2
#define UR3E_ATTN_MAX_DIM 128 /* dk, dv */

typedef struct {
  void* p;
  long long sb, st, sh; /* strides of sequence, token and head */
} ur3e_tokens_t;

typedef struct {
  int b, t, heads, kv_heads, dk, dv, dtype;
  float scale;
  ur3e_tokens_t q, k, v; /* [b][t][heads][dk], [b][t][kv_heads][dk], [b][t][kv_heads][dv] */
  const float* log_decay; /* [heads] */
  const float* s0;        /* [b][heads][dk][dv], contiguous, or null */
  const unsigned char* starts; /* nonzero where an episode starts, or null */
  long long starts_sb, starts_st;
  const int* lengths; /* [b] clamped to [0, t], or null: t */
} ur3e_attn_t;

/* out [b][t][heads][dv]; s_out [b][heads][dk][dv] the state behind the last token, or null.
   workspace: device memory of ur3e_attn_workspace(a, 0) bytes (16-byte aligned), or null when that is 0. */
int ur3e_attn_forward(const ur3e_attn_t* a, const ur3e_tokens_t* out, float* s_out, void* workspace,
                      size_t workspace_bytes, void* stream);

/* Gradients of a forward call with the same `a`: dout [b][t][heads][dv] and ds_out (null: 0) in; dq, dk, dv
   (shaped as q, k, v; dk and dv summed over the query heads that share them) and ds0 (or null) out.
   workspace: ur3e_attn_workspace(a, 1) bytes. */
int ur3e_attn_backward(const ur3e_attn_t* a, const ur3e_tokens_t* dout, const float* ds_out,
                       const ur3e_tokens_t* dq, const ur3e_tokens_t* dk, const ur3e_tokens_t* dv, float* ds0,
                       void* workspace, size_t workspace_bytes, void* stream);

/* bytes of workspace that the forward (backward = 0) or the backward call needs */
int ur3e_attn_workspace(const ur3e_attn_t* a, int backward, size_t* bytes);

/* One token (a->t must be 1): state_in -> state_out (the same buffer, two that do not overlap, or
   state_out null: the output alone), and out.  a->s0 is not used, a->lengths must be null. */
int ur3e_attn_step(const ur3e_attn_t* a, const ur3e_tokens_t* out, const float* state_in, float* state_out,
                   void* stream);

/* y[r][c] = keep ? x[r][c] * 65536 / keep_count : 0  (+ residual[r][c] when not null), keep = u16(r, c) < keep_count,
   where u16(r, 8 j + 2 w + s) is the low (s = 0) or high (s = 1) half of word w of
   Philox4x32-10(counter = (j, id low, id high, substream), key = (seed low, seed high)) and id = row_ids[r]
   (null: r).  keep_count in [0, 65536].  Rows are `*_stride` elements apart, columns contiguous. */
int ur3e_keyed_dropout(int dtype, long long rows, int cols, const void* x, long long x_stride, const void* residual,
                       long long residual_stride, void* y, long long y_stride, const long long* row_ids,
                       unsigned long long seed, unsigned int substream, int keep_count, void* stream);

#ifdef __cplusplus
}
#endif
#endif
