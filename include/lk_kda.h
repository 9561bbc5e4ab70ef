/*
 * C ABI of the Kimi Delta Attention (KDA) kernels: for decode the recurrent-state
 * step and its launch-fused preparation (short convolutions, gates), for
 * prompts the short convolutions and the recurrence over packed sequences.
 *
 * Same conventions as lk_w4a16.h: device pointers, element counts, a
 * hipStream_t passed as void*, LK_OK or an error code (message from
 * lk_last_error()); nothing allocates or synchronises, so every call can be
 * captured in a HIP graph. All tensors are dense row-major.
 *
 * Value dtype codes: LK_DTYPE_F32 = 0, LK_DTYPE_F16 = 1, LK_DTYPE_BF16 = 2
 * (fp16 / bf16 as uint16_t bit patterns).
 */
#ifndef LK_KDA_H
#define LK_KDA_H

#include "lk_w4a16.h"

#ifdef __cplusplus
extern "C" {
#endif

#define LK_DTYPE_F32 0
#define LK_DTYPE_F16 1
#define LK_DTYPE_BF16 2

/* ---- one decode step of the KDA recurrence, state updated in place:
 *      engine/kernels/kda_step.py:273-293 (kda_decode_step; the recurrence of
 *      kda_decode_step_reference, :173-196)
 * state fp32 [B, H, d_k, d_v]; q, k, decay fp32 [B, H, d_k]; v fp32
 * [B, H, d_v]; beta fp32 [B, H]; out fp32 [B, H, d_v]:
 *   S <- S * exp(decay) (per key row); S <- S + beta * k (v - S^T k)^T;
 *   out = S^T (q * scale).
 * d_k <= 256. */
LK_API int lk_kda_decode_step(float* state, const float* q, const float* k, const float* v,
                              const float* decay, const float* beta, float* out, int64_t batch,
                              int64_t heads, int64_t d_k, int64_t d_v, float scale,
                              void* stream);

/* ---- the three width-4 decode convolutions in one launch:
 *      engine/kernels/kda_prepare.py:479-538 (fused_short_conv_triple)
 * inputs q/k/v_in [B, 1, C] and states [B, C, 4] in value_dtype; weights
 * [C, 4] (the [C, 1, 4] conv weight) in weight_dtype; outputs [B, 1, C] in
 * value_dtype. Per channel: window = (state[1], state[2], state[3], token),
 * out = silu(sum_j window[j] * weight[j]) in fp32, rounded to value_dtype;
 * the window becomes the state. */
LK_API int lk_kda_short_conv_triple(const void* q_in, const void* k_in, const void* v_in,
                                    void* q_state, void* k_state, void* v_state,
                                    const void* q_weight, const void* k_weight,
                                    const void* v_weight, void* q_out, void* k_out, void* v_out,
                                    int64_t batch, int64_t channels, int value_dtype,
                                    int weight_dtype, void* stream);

/* ---- decay, beta and per-head q/k normalisation in one launch:
 *      engine/kernels/kda_prepare.py:630-686 (fused_kda_gates)
 * rows = batch * sequence. raw_decay [rows, H, D] (decay_dtype), dt_bias fp32
 * [H * D], a_log fp32 [H], raw_beta [rows, H] (beta_dtype), q and k
 * [rows, H * D] (qk_dtype); outputs fp32: decay [rows, H, D] =
 * -exp(a_log[h]) * softplus(raw_decay + dt_bias) (softplus(x) = x above 20),
 * beta [rows, H] = sigmoid(raw_beta), q_out / k_out [rows, H, D] = x *
 * rsqrt(sum over the head of x^2 + eps). head_dim <= 1024. */
LK_API int lk_kda_gates(const void* raw_decay, const float* dt_bias, const float* a_log,
                        const void* raw_beta, const void* q, const void* k, float* decay,
                        float* beta, float* q_out, float* k_out, int64_t rows, int64_t heads,
                        int64_t head_dim, float eps, int decay_dtype, int beta_dtype,
                        int qk_dtype, void* stream);

/* ---- a whole KDA decode layer in one launch. No reference counterpart: it
 * runs, for one token per batch row, what engine/klinear/attention.py:193-271
 * runs through fused_short_conv_triple, fused_kda_gates and kda_decode_step
 * (three launches there, plus the bf16 -> fp32 view of v), with one block
 * per (batch row, head). Inputs as lk_kda_short_conv_triple (C = heads *
 * head_dim) and lk_kda_gates (rows = batch, sequence one); state fp32
 * [B, H, D, D] and out fp32 [B, H, D] as lk_kda_decode_step with
 * d_k = d_v = D. Conv states and state are updated in place. q, k, v, decay
 * and beta are bit-identical to the three-launch chain's; the step sums its
 * row groups in another order. head_dim a multiple of 4, at most 128. */
LK_API int lk_kda_decode_layer(const void* q_in, const void* k_in, const void* v_in,
                               void* q_state, void* k_state, void* v_state,
                               const void* q_weight, const void* k_weight,
                               const void* v_weight, const void* raw_decay,
                               const float* dt_bias, const float* a_log, const void* raw_beta,
                               float* state, float* out, int64_t batch, int64_t heads,
                               int64_t head_dim, float eps, float scale, int value_dtype,
                               int weight_dtype, int decay_dtype, int beta_dtype, void* stream);

/* ---- the same layer over several blocks per head (no reference counterpart)
 * Arguments as lk_kda_decode_layer, except that the convolution states are
 * read from q/k/v_state and the shifted states written to q/k/v_state_out
 * (distinct buffers; callers alternate the two from call to call), which lets
 * a head's value columns be split over blocks of 16 without a block reading a
 * state another block already shifted. The recurrent state is updated in
 * place. q, k, v, decay and beta are bit-identical to lk_kda_decode_layer's;
 * the step sums its rows in another grouping. head_dim a multiple of 4, at
 * most 128. */
LK_API int lk_kda_decode_layer_split(const void* q_in, const void* k_in, const void* v_in,
                                     const void* q_state, const void* k_state,
                                     const void* v_state, void* q_state_out, void* k_state_out,
                                     void* v_state_out, const void* q_weight,
                                     const void* k_weight, const void* v_weight,
                                     const void* raw_decay, const float* dt_bias,
                                     const float* a_log, const void* raw_beta, float* state,
                                     float* out, int64_t batch, int64_t heads, int64_t head_dim,
                                     float eps, float scale, int value_dtype, int weight_dtype,
                                     int decay_dtype, int beta_dtype, void* stream);

/* ---- prompts: the short convolutions and the recurrence over packed sequences
 *
 * Sequences are packed one behind the other over the rows of a call: sequence
 * s has rows cu_seqlens[s] to cu_seqlens[s + 1] - 1 (int32 [sequences + 1] on
 * the device, starting with 0 and not decreasing; clamped to the rows, so that
 * others lead nowhere outside the tensors), or with a null cu_seqlens tokens /
 * sequences rows each. A sequence may be empty: its state is kept. Output
 * rows behind the last sequence are set to zero. A state may be updated in
 * place (state_out = state) or written elsewhere; nothing else that is
 * written may overlap anything. Reruns are bit-identical. */

/* the three width-4 convolutions of a prompt: what lk_kda_short_conv_triple
 * computes token by token. inputs [tokens, C] in value_dtype, row_stride
 * elements from one row to the next (the same for all three; >= C); states
 * [sequences, C, 4]; weights [C, 4] in weight_dtype; outputs [tokens, C]
 * dense, in value_dtype. 16-byte accesses where C and row_stride are
 * multiples of 16 bytes and every input and output starts on one. */
LK_API int lk_kda_short_conv_prefill(const void* q_in, const void* k_in, const void* v_in,
                                     const void* q_state, const void* k_state,
                                     const void* v_state, void* q_state_out, void* k_state_out,
                                     void* v_state_out, const void* q_weight,
                                     const void* k_weight, const void* v_weight, void* q_out,
                                     void* k_out, void* v_out, const int32_t* cu_seqlens,
                                     int64_t sequences, int64_t tokens, int64_t channels,
                                     int64_t row_stride, int value_dtype, int weight_dtype,
                                     void* stream);

/* the recurrence of a prompt: what lk_kda_decode_step computes token by token.
 * q, k, decay fp32 [tokens, H, d_k], beta fp32 [tokens, H] (lk_kda_gates
 * writes them for any number of rows), v [tokens, H, d_v] and out
 * [tokens, H, d_v] in value_dtype, state fp32 [sequences, H, d_k, d_v].
 * decay <= 0 (a log decay). d_k <= 256; tensors start on 16 bytes. All sums
 * and the state are fp32; out is rounded once. From 48 tokens a sequence on (the
 * call's mean) and up to d_k = 128, chunks of 32 steps are solved together, in which
 * the operands of the state's products are sums of two fp16 (22 bits of the largest
 * beside them), for states up to 1e36; otherwise steps follow one another in fp32.
 * The knob kda_prefill (lk_set_path) asks for one form. workspace:
 * lk_kda_prefill_workspace() bytes on 16 bytes (may be null where that is 0), by
 * the knob's setting of the call. */
LK_API int64_t lk_kda_prefill_workspace(int64_t sequences, int64_t tokens, int64_t heads,
                                        int64_t d_k, int64_t d_v);

LK_API int lk_kda_prefill(const float* state, float* state_out, const float* q, const float* k,
                          const void* v, const float* decay, const float* beta, void* out,
                          const int32_t* cu_seqlens, int64_t sequences, int64_t tokens,
                          int64_t heads, int64_t d_k, int64_t d_v, float scale, int value_dtype,
                          void* workspace, int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* LK_KDA_H */
