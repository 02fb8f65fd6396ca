/*
 * h3vae_b200_kv.h -- C ABI of the paged INT8 key/value cache: writing it, reading it back,
 * attention over it, and attention over the pages a score selects.
 *
 * The conventions of h3vae_b200.h hold (raw device pointers, int64 sizes, an explicit stream, 0 or a
 * negative H3B_E* status, h3b_last_error()).  No entry point allocates device memory or synchronises.
 *
 * The cache.  A sequence's tokens lie in pages of `page_size` tokens; token t of sequence b is in slot
 * t % page_size of page page_table[b][t / page_size].  For every (page, kv head):
 *   K and V   int8 codes [page_size, head_dim], |code| <= 127
 *   scales    one fp32 each for K and V: value = code * scale
 *   k_sum     int16 [head_dim]: the sum of the page's K codes, written when the page is complete; the
 *             summary that h3b_kv_select_i8 scores pages with
 * Device-side contents (page numbers, starts, counts, lengths) cannot be checked by the host.  A page
 * number outside [0, num_pages), or a position outside the table, is not accessed: the tokens concerned
 * are not written, read back as zero and are not attended to, and bit 3 (value 8) of the device error
 * word (h3b_device_error) is set.
 */
#ifndef H3VAE_B200_KV_H_
#define H3VAE_B200_KV_H_

#include "h3vae_b200.h"

#ifdef __cplusplus
extern "C" {
#endif

enum {
  H3B_TYPE_F16 = 0,
  H3B_TYPE_BF16 = 1,
  H3B_TYPE_F32 = 2 /* h3b_kv_write_i8 and h3b_kv_read_i8 only */
};

typedef struct h3b_kv_cache {
  int8_t* k;      /* [num_pages, kv_heads, page_size, head_dim], 16-byte aligned */
  int8_t* v;      /* likewise */
  float* k_scale; /* [num_pages, kv_heads] */
  float* v_scale; /* [num_pages, kv_heads] */
  int16_t* k_sum; /* [num_pages, kv_heads, head_dim], 16-byte aligned */
  int64_t num_pages;
  int64_t kv_heads;
  int64_t page_size; /* 16, 32, 64 or 128 */
  int64_t head_dim;  /* 64 or 128 */
} h3b_kv_cache;

/* Quantises and stores tokens start[b] .. start[b] + counts[b] - 1 of every sequence b.
 *   page_table  int32 [batch, table_width]; start int32 [batch]; counts int32 [batch] (each <= tokens)
 *               or NULL: `tokens` for every sequence
 *   k, v        type `dtype`, logical [batch, kv_heads, tokens, head_dim] at element strides
 *               {batch, head, token}, unit dim stride, any alignment
 * Per (page, head), separately for K and V, in fp32 with every operation rounded to nearest:
 *   s = max(max|x| * fp32(1/127), 1e-30) over the page's new tokens; a page that already holds earlier
 *   tokens keeps max(s, its scale), and where that grew the earlier codes become rint(code * (old / s));
 *   code = rint(x * (1 / s)).  Tokens at or after `start` that an earlier call stored are replaced.
 * A page that takes a NaN or an infinity gets the scale NaN (all its values read as NaN) until its first
 * slot is written anew.  Two sequences of one call must not write to the same page. */
int h3b_kv_write_i8(const h3b_kv_cache* cache, const int32_t* page_table, int64_t batch, int64_t table_width,
                    const int32_t* start, const int32_t* counts, const void* k, const int64_t* k_strides,
                    const void* v, const int64_t* v_strides, int64_t tokens, int dtype, h3b_stream_t stream);

/* Reads tokens start[b] .. start[b] + tokens - 1 (start NULL: from 0) back as code * scale, rounded once to
 * `dtype`; positions at or past lengths[b] are zero.  k, v: dense [batch, kv_heads, tokens, head_dim],
 * 16-byte aligned. */
int h3b_kv_read_i8(const h3b_kv_cache* cache, const int32_t* page_table, int64_t batch, int64_t table_width,
                   const int32_t* start, const int32_t* lengths, void* k, void* v, int64_t tokens, int dtype,
                   h3b_stream_t stream);

/* softmax(q k^T * scale) v over the cached tokens.
 *   q, out     fp16 or bf16, logical [batch, q_heads, tokens, head_dim] at element strides
 *              {batch, head, token}, unit dim stride, any alignment; q_heads a multiple of kv_heads: query
 *              head j reads kv head j / (q_heads / kv_heads)
 *   lengths    int32 [batch]: tokens in the cache, the queries' own included
 *   counts     int32 [batch] or NULL: query tokens of each sequence (NULL: `tokens`).  Query i of n sits at
 *              position lengths[b] - n + i; rows i >= n are padding
 *   causal     nonzero: query at position p sees keys <= p, and with window > 0 only keys > p - window;
 *              0: every query sees all lengths[b] keys (window must be 0)
 *   selected   NULL, or int32 [batch, kv_heads, tokens, n_selected] page ordinals (position / page_size) in
 *              any order without repeats, negative = none: each query sees only the keys of its pages
 *              (causal must be nonzero and window 0)
 *   lse        NULL, or fp32 [batch, q_heads, tokens]: the natural logarithm of each row's sum of exp
 * Rows that see no key (padding, an empty sequence, a position before the first key) are zero with lse
 * -infinity.  Keys a row does not see have no effect on it, whatever their page holds.  Pages of zeros, or of values
 * far below the others', count in the sum like any other beside values up to 2^77.
 * Workspace: h3b_attention_kv_i8_workspace_size(...) bytes of the same sizes, asked for with the same current
 * device (the plan goes by its number of SMs), 16-byte aligned; contents are not kept between calls.  Where that is
 * 16 the call needs none and takes NULL. */
size_t h3b_attention_kv_i8_workspace_size(int64_t batch, int64_t q_heads, int64_t kv_heads, int64_t tokens,
                                          int64_t head_dim, int64_t table_width, int64_t page_size,
                                          int64_t n_selected);
int h3b_attention_kv_i8(const void* q, const int64_t* q_strides, const h3b_kv_cache* cache,
                        const int32_t* page_table, int64_t batch, int64_t table_width, const int32_t* lengths,
                        const int32_t* counts, int64_t q_heads, int64_t tokens, float scale, int causal,
                        int64_t window, const int32_t* selected, int64_t n_selected, int dtype, void* out,
                        const int64_t* out_strides, float* lse, void* workspace, size_t workspace_bytes,
                        h3b_stream_t stream);

/* Chooses n_selected pages for each query token and kv head: the page of the query's own position, and of
 * the earlier (complete) pages those with the highest scores; ties go to the lower page.
 *   row quantisation of every query row: s = max(max|q| * fp32(1/127), 1e-30), q8 = rint(q * (1 / s))
 *   score(page) = max over the group's heads of float(q8 . k_sum[page]) * s, times k_scale[page]
 *   (whole-number products; the scores of a page whose scale is NaN rank first).  A head whose query row holds a
 *   NaN or an infinity is left out of the maximum; where no head is left, all pages count alike
 * selected: int32 [batch, kv_heads, tokens, n_selected], ascending ordinals, -1 where no page is left and for
 * rows without a position.  q, lengths and counts as in h3b_attention_kv_i8.
 * Workspace: h3b_kv_select_i8_workspace_size(...) bytes, 16-byte aligned. */
size_t h3b_kv_select_i8_workspace_size(int64_t batch, int64_t kv_heads, int64_t tokens, int64_t table_width);
int h3b_kv_select_i8(const void* q, const int64_t* q_strides, const h3b_kv_cache* cache, const int32_t* page_table,
                     int64_t batch, int64_t table_width, const int32_t* lengths, const int32_t* counts,
                     int64_t q_heads, int64_t tokens, int64_t n_selected, int dtype, int32_t* selected,
                     void* workspace, size_t workspace_bytes, h3b_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* H3VAE_B200_KV_H_ */
