/*
 * C ABI of the paged cache of full attention layers: norms and rotation of new
 * queries and keys, their write to the pages, attention on the pages, copies of
 * pages.
 *
 * Same conventions as lk_w4a16.h: device pointers (but for lk_copy_pages' lists),
 * element counts, a hipStream_t passed as void*, LK_OK or an error code (message
 * from lk_last_error()); nothing allocates device memory or synchronises, so every
 * call can be captured in a HIP graph. Dtype codes are those of lk_kda.h.
 *
 * A cache is two tensors of `pages` pages of page_rows rows of kv_heads heads:
 * row r of page p, head h is at base + p * page_stride + r * row_stride + h *
 * head_stride (strides in elements, multiples of 8, not negative; base on 16 bytes).
 * page_table [sequences, table_width] (int32, rows table_stride apart) gives each
 * sequence's pages in order: its position i is row i % page_rows of page
 * page_table[s][i / page_rows]. lengths [sequences] (int32): a sequence's positions,
 * the call's new ones included, which are its last; below 0 counts as 0. Positions beyond
 * table_width * page_rows are not written and not seen: rows keep the positions that the
 * length gives them, also where it passes that. Table entries
 * that name no page (below 0, pages and above) lead nowhere: such positions read as
 * zeros and are not written.
 * page_rows is a multiple of 16 up to 65536, table_width * page_rows at most 2^30.
 *
 * cu [sequences + 1] (int32): sequence s has new rows cu[s] to cu[s + 1] - 1; null
 * means equal sequences of rows / sequences. Offsets start with 0 and do not
 * decrease; they are clamped to the rows, so that others lead nowhere outside the
 * tensors.
 */
#ifndef LK_PAGED_H
#define LK_PAGED_H

#include "lk_kda.h"

#ifdef __cplusplus
extern "C" {
#endif

/* ---- norms of queries and keys for each head, with the position rotation
 * x is q [rows, heads, d] or k [rows, kv_heads, d] (dtype: LK_DTYPE_F32, _F16 or
 * _BF16; rows and heads at strides in elements, multiples of 8; bases on 16 bytes):
 *   y = x * rsqrt(mean(x^2) + eps) * weight        (a null weight: y = x)
 * then in the rotated slice y[offset .. offset + rotary), with c, s = cos_sin[p][i],
 * cos_sin[p][rotary / 2 + i] of the row's position p, for i < rotary / 2
 *   (y[a], y[b]) = (y[a] c - y[b] s, y[b] c + y[a] s)
 * a, b = offset + i, offset + rotary / 2 + i, or interleaved offset + 2 i, + 2 i + 1.
 * fp32 throughout, one rounding. q_out and k_out are dense and overlap nothing.
 * cos_sin [table_rows, rotary] fp32 on 16 bytes (ignored where rotary is 0);
 * positions [rows] (int32, or int64 where positions_64), clamped to the table. d
 * is a multiple of 8 up to 256, rotary and offset multiples of 8 within it. Weights
 * [d] in weight_dtype, on 16 bytes; both or neither may be null. */
LK_API int lk_qk_norm_rope(const void* q, const void* k, const void* q_weight,
                           const void* k_weight, const float* cos_sin, const void* positions,
                           void* q_out, void* k_out, int64_t rows, int64_t heads,
                           int64_t kv_heads, int64_t d, int64_t q_row_stride,
                           int64_t q_head_stride, int64_t k_row_stride, int64_t k_head_stride,
                           int64_t rotary, int64_t offset, int interleaved, int64_t table_rows,
                           int positions_64, float eps, int dtype, int weight_dtype, void* stream);

/* ---- the same for new rows of cached sequences, written to the cache
 * New row i of the n of sequence s is position p = lengths[s] - n + i: q (as above) goes
 * to q_out [rows, heads, d_qk] (dense), k (as above) and v [rows, kv_heads, d_v]
 * (as it is) to position p of k_pages and v_pages. What has no place there (p < 0,
 * beyond the table, no page) is not written; p < 0 is rotated as 0. Rows behind the last sequence
 * write nothing to the cache; their q_out is zeros. heads may be 0 (q, q_out, q_weight unused),
 * rotary 0 (no rotation). dtype is LK_DTYPE_F16 or LK_DTYPE_BF16. Two rows must
 * not go to one place: pages that take new rows belong to one sequence. The places
 * of k_pages and of v_pages do not overlap (refused where the strides show it, or the
 * two are one), nor what is read. */
LK_API int lk_paged_append(const void* q, const void* k, const void* v, const void* q_weight,
                           const void* k_weight, const float* cos_sin, const int32_t* page_table,
                           const int32_t* lengths, const int32_t* cu, void* q_out, void* k_pages,
                           void* v_pages, int64_t sequences, int64_t rows, int64_t heads,
                           int64_t kv_heads, int64_t d_qk, int64_t d_v, int64_t q_row_stride,
                           int64_t q_head_stride, int64_t k_row_stride, int64_t k_head_stride,
                           int64_t v_row_stride, int64_t v_head_stride, int64_t pages,
                           int64_t page_rows, int64_t table_width, int64_t table_stride,
                           int64_t k_page, int64_t k_page_row, int64_t k_page_head,
                           int64_t v_page, int64_t v_page_row, int64_t v_page_head,
                           int64_t rotary, int64_t offset, int interleaved, int64_t table_rows,
                           float eps, int dtype, int weight_dtype, void* stream);

/* ---- causal softmax attention of new rows on the cache, grouped heads
 * q [rows, heads, d_qk] (strided as above), out [rows, heads, d_v] (dense, overlaps
 * nothing), all in dtype (LK_DTYPE_F16 or LK_DTYPE_BF16); query head h reads key head
 * h / (heads / kv_heads). d_qk is a multiple of 8 up to 192, d_v up to 128. Query i of
 * the n of sequence s sees positions 0 .. lengths[s] - n + i, within the table. One that sees none
 * gets zeros, as do the rows behind the last sequence.
 *   o_i = sum_j p_ij v_j,  p_i = softmax over the positions seen of scale * q_i . k_j
 * Scores and sums in fp32; p is rounded to dtype for its product with v. What a query
 * does not see has no part in its result, NaN and infinities included. A query
 * whose every score is -infinity gets zeros too. fp16 results of finite values stay
 * finite. Reruns are bit-identical; how a sequence's keys are split, and so the
 * order of its sums, follows all lengths of the call.
 *
 * workspace: lk_attention_paged_workspace() bytes on 16 bytes (may be null where that
 * is 0). Calls that overlap in time take one each. */
LK_API int64_t lk_attention_paged_workspace(int64_t rows, int64_t sequences, int64_t capacity,
                                            int64_t heads, int64_t kv_heads, int64_t d_qk,
                                            int64_t d_v, int packed);

/* above: capacity is table_width * page_rows, packed whether cu is given */
LK_API int lk_attention_paged(const void* q, const void* k_pages, const void* v_pages, void* out,
                              const int32_t* page_table, const int32_t* lengths,
                              const int32_t* cu, int64_t sequences, int64_t rows, int64_t heads,
                              int64_t kv_heads, int64_t d_qk, int64_t d_v, int64_t q_row_stride,
                              int64_t q_head_stride, int64_t pages, int64_t page_rows,
                              int64_t table_width, int64_t table_stride, int64_t k_page,
                              int64_t k_page_row, int64_t k_page_head, int64_t v_page,
                              int64_t v_page_row, int64_t v_page_head, float scale, int dtype,
                              void* workspace, int64_t workspace_bytes, void* stream);

/* ---- pages copied: page src[i] to page dst[i] of every tensor
 * tensors, page_strides, page_bytes: host arrays of `count` device pointers, bytes from
 * a page to the next and bytes of a page (dense, multiples of 16, pointers on 16
 * bytes). src, dst: host arrays of `pairs` page numbers in 0 .. pages - 1; a page is
 * written once at most and is not a source too; others are refused. A pair of one page
 * with itself does nothing and counts for neither. The host's lists are read before the call
 * returns. lists: null, or device memory of 2 pairs int32 with src, then dst, which saves a launch
 * for every 192 pairs. */
LK_API int lk_copy_pages(void* const* tensors, const int64_t* page_strides,
                         const int64_t* page_bytes, int64_t count, const int32_t* src,
                         const int32_t* dst, int64_t pairs, int64_t pages,
                         const int32_t* lists, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* LK_PAGED_H */
