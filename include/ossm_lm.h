/*
 * ossm_lm.h — C ABI of libossm_scan.so's operators for serving and training language
 * models built on the Mamba mixer: the mixer over ragged prompts and over single
 * tokens with its states in a pool, the gated projection of a feed-forward block,
 * and the control of logits.
 *
 * The conventions are ossm_scan.h's: device pointers, sizes and a HIP stream (as
 * void*), asynchronous launches on that stream, status 0 or an error with
 * ossm_last_error(), outputs written and never allocated, scratch from the
 * library's workspace of the stream (grown on demand outside stream capture, which
 * waits for the stream and allocates; refused under capture with OSSM_ERR_UNSUPPORTED).
 * No other call synchronises; none reads device memory on the host or uses atomics on
 * floating-point values: results are bitwise repeatable.
 *
 * dtype: OSSM_F32 (0) or OSSM_BF16 (1), of the tensors marked E below; everything
 * else is float32.  Sums, states and statistics are held in float32, and each
 * output is rounded once.  Index tensors are int32.
 */
#ifndef OSSM_LM_H
#define OSSM_LM_H

#include "ossm_scan.h"

#ifdef __cplusplus
extern "C" {
#endif

enum { OSSM_F32 = 0, OSSM_BF16 = 1 };

/* Version of this header's entry points (ossm_abi_version() covers ossm_scan.h). */
int ossm_lm_abi_version(void);

/*
 * The Mamba mixer between its in and out projections, with states kept in a pool.
 *
 * Per channel d of Di, with x = xz[:, :Di], z = xz[:, Di:], p = R + 2N projections:
 *   u_t  = silu(conv_bias[d] + sum_k conv_w[d, k] x[t - K + 1 + k, d])
 *   p_t  = x_proj u_t            (R values for dt, N for B, N for C)
 *   dt_t = softplus(dt_proj p_t[:R] + dt_bias)
 *   h_t[n, d] = exp(-dt_t exp(A_log[d, n])) h_{t-1}[n, d] + dt_t u_t B_t[n]
 *   y_t  = (sum_n C_t[n] h_t[n, d] + skip[d] u_t) silu(z_t)
 *
 * Pools: conv_state E [slots, K - 1, Di] (a sequence's last K - 1 inputs, oldest
 * first; may be null when K = 1), ssm_state f32 [slots, N, Di].  Sequence i starts
 * from slot in_slots[i] and leaves its state in out_slots[i] (in_slots when null);
 * an index outside [0, n_slots) starts from zeros, or keeps nothing.  No out slot may
 * be the in slot of another sequence of the call, nor appear twice.
 *
 * Weights: conv_w E [Di, K], conv_bias E [Di] or null, x_proj E [R + 2N, Di],
 * dt_proj E [Di, R], dt_bias f32 [Di], a_log f32 [Di, N], skip f32 [Di] or null.
 * xz E [rows, 2 Di] with row stride ld_xz, y E [rows, Di] dense.  1 <= K <= 8; up to
 * 65535 sequences a call.
 *
 * ossm_mixer_step: one token of each of `rows` sequences; a row whose in and out
 * slot are both outside the pool is padding: its y is zero.
 *
 * ossm_mixer_prompt: `rows` packed tokens of n_seqs prompts, prompt i the rows
 * offsets[i] .. offsets[i + 1] - 1 (offsets [n_seqs + 1], not decreasing; rows before
 * offsets[0] and from offsets[n_seqs] on are padding: their y is zero).  resume
 * (uint8 [n_seqs] or null): nonzero starts prompt i from its in slot, else, or when
 * null, from zeros.  An empty prompt leaves the state it starts from.
 */
int ossm_mixer_step(int dtype, const void* xz, int64_t ld_xz, const void* conv_w, const void* conv_bias,
                    const void* x_proj, const void* dt_proj, const float* dt_bias, const float* a_log,
                    const float* skip, void* conv_state, float* ssm_state, const int32_t* in_slots,
                    const int32_t* out_slots, void* y, int64_t rows, int64_t n_slots, int64_t d_inner,
                    int64_t d_state, int64_t dt_rank, int64_t d_conv, ossm_stream_t stream);

int ossm_mixer_prompt(int dtype, const void* xz, int64_t ld_xz, const void* conv_w, const void* conv_bias,
                      const void* x_proj, const void* dt_proj, const float* dt_bias, const float* a_log,
                      const float* skip, void* conv_state, float* ssm_state, const int32_t* in_slots,
                      const int32_t* out_slots, const int32_t* offsets, const uint8_t* resume, void* y,
                      int64_t rows, int64_t n_seqs, int64_t n_slots, int64_t d_inner, int64_t d_state,
                      int64_t dt_rank, int64_t d_conv, ossm_stream_t stream);

/*
 * Penalties for repeated tokens, biases and a grammar's mask on logits, row by row:
 *   l = logits[v];  if v is in history[:length]: l = l > 0 ? l / repetition : l * repetition
 *   l -= frequency * c + presence * (c > 0),  c = how often v is in history[prompt_length:length]
 *   l += bias_values[j] for the last j with bias_ids[j] = v;  l = -inf where v is not allowed
 * logits, out E [rows, vocab] with row strides ld_* (they may be the same tensor);
 * history int32 [rows, history_len] with row stride ld_history, ids outside the
 * vocabulary count nowhere; lengths, prompt_lengths int32 [rows] or null (history_len, 0),
 * clamped to [0, history_len]; repetition, presence, frequency f32 [rows], or null
 * and the value *_all for every row; bias_ids, bias_values [rows, n_bias] with row
 * stride ld_bias (ids outside the vocabulary are padding); allowed: bit v % 32 of word
 * v / 32 of a row, int32 [rows, ceil(vocab / 32)] with row stride ld_allowed (0: one
 * row for all), or null.
 */
int ossm_control_logits(int dtype, const void* logits, int64_t ld_logits, void* out, int64_t ld_out,
                        const int32_t* history, int64_t ld_history, int64_t history_len,
                        const int32_t* lengths, const int32_t* prompt_lengths, const float* repetition,
                        float repetition_all, const float* presence, float presence_all,
                        const float* frequency, float frequency_all, const int32_t* bias_ids,
                        const float* bias_values, int64_t ld_bias, int64_t n_bias, const int32_t* allowed,
                        int64_t ld_allowed, int64_t rows, int64_t vocab, ossm_stream_t stream);

enum { OSSM_ACT_SILU = 0, OSSM_ACT_GELU = 1, OSSM_ACT_GELU_TANH = 2, OSSM_ACT_SIGMOID = 3, OSSM_ACT_RELU = 4 };

/*
 * The gated projection of a feed-forward block:
 *   a = x w_gate^T + b_gate,  b = x w_up^T + b_up,  y = act(a) b
 * x E [rows, d_in], w_* E [d_out, d_in] with row strides ld_* (up to 2^20), b_* E
 * [d_out] or null, y E [rows, d_out] dense.  a, b: f32 [rows, d_out] dense, written for the
 * backward, or both null.
 *
 * ossm_gated_backward: with grad_y E [rows, d_out] (row stride ld_grad) and the
 * forward's a and b, the gradients of x, of the weights and of the biases, all dense E;
 * a null gradient is not computed.  float32 products take three bf16 terms of
 * each operand (24 bits).  In bfloat16 the gradients of a and b enter their products
 * as two bfloat16 terms (16 bits) where rows * d_out <= 2^18, and rounded to one past
 * that: their errors then average out, and a gradient is about 1.41 times as far from the
 * exact one as that one's own rounding to bfloat16.
 */
int ossm_gated_forward(int dtype, const void* x, int64_t ld_x, const void* w_gate, int64_t ld_gate, const void* w_up,
                       int64_t ld_up, const void* b_gate, const void* b_up, int activation, void* y, float* a, float* b,
                       int64_t rows, int64_t d_in, int64_t d_out, ossm_stream_t stream);

int ossm_gated_backward(int dtype, const void* grad_y, int64_t ld_grad, const void* x, int64_t ld_x, const void* w_gate,
                        int64_t ld_gate, const void* w_up, int64_t ld_up, int activation, const float* a, const float* b,
                        void* grad_x, void* grad_w_gate, void* grad_w_up, void* grad_b_gate, void* grad_b_up,
                        int64_t rows, int64_t d_in, int64_t d_out, ossm_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* OSSM_LM_H */
