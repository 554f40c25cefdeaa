/*
 * paged_hip_q4.h — the 4-bit paged KV cache of libpaged_hip.so (same library, status codes, dtypes, stream
 * and error conventions as paged_hip.h).
 *
 * K and V pools of uint8 [num_blocks, kv_heads, pa_q4_page_bytes(head_dim)], 16-byte
 * aligned, 16 tokens a page, head_dim 64 or 128; num_heads query heads share kv_heads KV heads, a multiple
 * of them: query head h reads KV head h / (num_heads / kv_heads). 64 consecutive values of a row share a
 * half-precision scale s and centre z, and 4 bits c of each stand for z + s (c - 7.5): 4.5 bits a value.
 * csrc/pa_q4.h has the bytes' places. `weights` (or NULL) is float [num_blocks, kv_heads, 16], the running
 * total of the attention weight that each slot's key has had. Page tables, lengths and
 * row visibility are those of pa_decode / pa_prefill. No reference counterpart: the reference's pools hold
 * the model's dtype.
 */
#ifndef PAGED_HIP_Q4_H_
#define PAGED_HIP_Q4_H_

#include "paged_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/* Bytes of one page of one KV head: 16 * (head_dim / 2 + 4 * head_dim / 64); 0 for other head_dims. */
size_t pa_q4_page_bytes(int32_t head_dim);

/*
 * Quantising append: rows k_new[b, h, j, :], v_new[b, h, j, :] into slot slot_mapping[b * query_len + j]
 * (as pa_kv_append; negative slots and blocks outside the pool are skipped, two rows of one slot in
 * a call leave parts of both). Per group, values clamped to +-65504: s = half((hi - lo) / 15), z = half((hi + lo) / 2), the
 * difference, the sum and their products with 1/15 and 1/2 rounded to fp32 first; c = (x - z) / s + 7.5
 * in 64 bits (difference, quotient and sum each rounded to them), then to the nearest, ties to even, in 0..15 (0
 * where s is 0). So a value stands for its own within s / 2, but for what the halves lose: a group whose spread is
 * small beside its centre (1000 +- 0.1, where z's step is 1/2) is off by up to half of z's step, all codes at one
 * end. A centre of zero is +0. A group with a NaN gets NaN for s and z. weights: the written slots' totals are
 * cleared.
 */
int pa_q4_append(const void* k_new, const void* v_new, int64_t new_stride_b, int64_t new_stride_h,
                 int64_t new_stride_t, int new_dtype,
                 void* k_pool, void* v_pool, int64_t num_blocks, float* weights,
                 const int32_t* slot_mapping,
                 int32_t batch, int32_t kv_heads, int32_t query_len, int32_t head_dim, void* stream);

/* The values that slots stand for, rounded once to out_dtype; rows whose slot is negative or whose block is
 * outside the pool are zeros. Outputs start, and their rows follow each other, at multiples of 16 bytes. */
int pa_q4_read(const void* k_pool, const void* v_pool, int64_t num_blocks, const int32_t* slot_mapping,
               void* k_out, void* v_out, int64_t out_stride_b, int64_t out_stride_h, int64_t out_stride_t,
               int out_dtype,
               int32_t batch, int32_t kv_heads, int32_t query_len, int32_t head_dim, void* stream);

/*
 * Attention over 4-bit pages: decode (query_len 1) and causal chunks, with the visibility of pa_prefill
 * (row i sees min(L, L - C + 1 + i) keys, rows without keys are zeros, keys without a page are skipped).
 * The codes enter the products exactly; with fp32 q the products keep 2^-22 and better (q and the softmax
 * weights in two fp16 parts each), with bf16 q the softmax weights are rounded to fp16. weights: for every
 * key, the sum of its softmax weights over the KV head's query heads and the real rows (i < C) is added to
 * its slot's total (a block in several rows of the page table gets the sum of all, in no fixed order).
 * scale must be positive. out must not overlap q: calls whose rows share a byte are refused, and so are those
 * whose extents meet with other strides (rows of q and out interleaved in one tensor have the same). The workspace (16-byte aligned, pa_q4_attention_workspace_size bytes for the
 * same arguments, weights != 0 where totals are asked for) needs no initial state and keeps none. Calls on one
 * stream may share one, from several threads too (a call's launches follow each other undivided); calls
 * on several streams must not.
 */
int pa_q4_attention(const void* q, int64_t q_stride_b, int64_t q_stride_h, int64_t q_stride_t,
                    void* out, int64_t out_stride_b, int64_t out_stride_h, int64_t out_stride_t, int io_dtype,
                    const void* k_pool, const void* v_pool, int64_t num_blocks,
                    const int32_t* page_table, int64_t pt_stride, int32_t max_pages,
                    const int32_t* seq_lens, const int32_t* cur_lens, float* weights,
                    int32_t batch, int32_t num_heads, int32_t kv_heads, int32_t query_len, int32_t head_dim,
                    float scale, void* workspace, size_t workspace_bytes, void* stream);

size_t pa_q4_attention_workspace_size(int io_dtype, int32_t batch, int32_t num_heads, int32_t kv_heads,
                                      int32_t query_len, int32_t head_dim, int32_t max_pages, int32_t weights);

/*
 * Eviction by accumulated weight: request b's keys, n = min(seq_lens[b], 16 * max_pages) of them, are cut
 * to min(n, keep) per KV head: the newest `window` (0 <= window <= keep) and of the others those of the
 * largest totals, the lower index where totals are equal, a NaN total above every number, a key without a
 * page below all. Their indices go, ascending, to kept[b, h, :] (int32 [batch, kv_heads, keep], -1 behind
 * the last), their rows and totals in that order into the pages of new_page_table[b, :], whose other rows
 * stay as they are, and min(n, keep) to new_seq_lens[b]. A kept key without a page moves as zeros; new
 * pages that are no blocks of the pool are skipped. The new pages must be none of the batch's old ones,
 * and hold min(keep, 16 * max_pages) keys; kept and new_seq_lens must not overlap each other, the lengths
 * or the page tables.
 */
int pa_q4_evict(void* k_pool, void* v_pool, float* weights, int64_t num_blocks,
                const int32_t* page_table, int64_t pt_stride, int32_t max_pages, const int32_t* seq_lens,
                const int32_t* new_page_table, int64_t new_pt_stride, int32_t new_max_pages,
                int32_t keep, int32_t window, int32_t* kept, int32_t* new_seq_lens,
                int32_t batch, int32_t kv_heads, int32_t head_dim, void* stream);

#ifdef __cplusplus
}
#endif

#endif /* PAGED_HIP_Q4_H_ */
