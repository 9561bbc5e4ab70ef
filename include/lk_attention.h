/*
 * C ABI of causal attention over whole prompts.
 *
 * Same conventions as lk_w4a16.h: device pointers, element counts, a
 * hipStream_t passed as void*, LK_OK or an error code (message from
 * lk_last_error()); nothing allocates or synchronises, so every call can be
 * captured in a HIP graph. Dtype codes are those of lk_kda.h.
 */
#ifndef LK_ATTENTION_H
#define LK_ATTENTION_H

#include "lk_kda.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- causal softmax attention of packed prompts, grouped heads. The full
 *      attention layers of engine/klinear/attention.py over a prompt, without
 *      their projections.
 * q [rows_q, heads, d_qk], k [rows_k, kv_heads, d_qk], v [rows_k, kv_heads,
 * d_v], out [rows_q, heads, d_v], all in dtype (LK_DTYPE_F16 or
 * LK_DTYPE_BF16). q, k and v are addressed as base + row * row_stride + head *
 * head_stride + i (strides in elements, multiples of 8; base on 16 bytes); out
 * is dense. heads is a multiple of kv_heads; query head h reads key head h /
 * (heads / kv_heads). d_qk is a multiple of 8 up to 192, d_v up to 128.
 *
 * cu_q [sequences + 1] (int32, device): sequence s has query rows cu_q[s] to
 * cu_q[s + 1] - 1 and key rows cu_k[s] to cu_k[s + 1] - 1; a null cu_q (cu_k)
 * means equal sequences of rows_q (rows_k) / sequences. A sequence's queries
 * are its last rows: query i of lq sees keys 0 .. i + lk - lq of lk. One that
 * sees none gets zeros, as do the rows behind the last sequence. Offsets start
 * with 0 and do not decrease; they are clamped to the rows, so that others lead
 * nowhere outside the tensors. out overlaps nothing.
 *   o_i = sum_j p_ij v_j,  p_i = softmax over the keys seen of scale * q_i . k_j
 * Scores and sums in fp32; p is rounded to dtype for its product with v. A key
 * or value row that a query does not see has no part in its result, NaN and
 * infinities included. A query whose every score is -infinity gets zeros too. fp16
 * results of finite values stay finite. Reruns are bit-identical.
 *
 * workspace: lk_attention_prefill_workspace() bytes on 16 bytes (may be null
 * where that is 0). */
LK_API int64_t lk_attention_prefill_workspace(int64_t rows_q, int64_t rows_k, int64_t sequences,
                                              int64_t heads, int64_t kv_heads, int64_t d_qk,
                                              int64_t d_v);

LK_API int lk_attention_prefill(const void* q, const void* k, const void* v, void* out,
                                const int32_t* cu_q, const int32_t* cu_k, int64_t sequences,
                                int64_t rows_q, int64_t rows_k, int64_t heads, int64_t kv_heads,
                                int64_t d_qk, int64_t d_v, int64_t q_row_stride,
                                int64_t q_head_stride, int64_t k_row_stride,
                                int64_t k_head_stride, int64_t v_row_stride,
                                int64_t v_head_stride, float scale, int dtype, void* workspace,
                                int64_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* LK_ATTENTION_H */
