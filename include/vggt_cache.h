/*
 * vggt_cache.h — C ABI of the streaming key/value cache: rotary positions, a
 * paged cache, attention of new tokens over it, the weight that each cached
 * key has received, and eviction by that weight.
 *
 * As in vggt_sparse.h every entry point takes plain device pointers, sizes
 * and a cudaStream_t (as void*), enqueues on that stream, never synchronises
 * and never allocates.  0: enqueued; negative: argument error (message from
 * vggt_sparse_last_error()); positive: CUDA error code of the launch.
 *
 * Tensors
 *   pools        k_pages, v_pages [n_pages][kv_heads][page][dim], bf16 or
 *                fp16, both with the same strides (in elements; the last
 *                dimension contiguous, the others multiples of 8)
 *   table        [seqs][table_width] int32 page numbers; slot s of sequence b
 *                lies in page table[b][s / page] at row s % page.  Entries
 *                past a sequence's last page are never read.
 *   lengths      [seqs] int32, tokens of each sequence in the cache
 *   starts       [seqs + 1] int32: sequence b's new tokens are rows
 *                starts[b] .. starts[b + 1] of the packed tensors
 *   ids, weights [seqs][kv_heads][slots] int32 / fp32, slots =
 *                table_width * page: number and weight of the token in each
 *                slot; -1 and 0 past a sequence's length
 *
 * Device-side checks: a page number outside [0, n_pages) is never used as an
 * address (its keys and values read as zeros, nothing is written), lengths
 * and starts outside their ranges are clamped; either ORs a VGGT_STATUS_* bit
 * into *status when status is non-NULL.
 */
#ifndef VGGT_CACHE_H
#define VGGT_CACHE_H

#include <stddef.h>
#include <stdint.h>

#ifdef __cplusplus
extern "C" {
#endif

/* element type of vggt_rotary beside VGGT_DTYPE_BF16 and VGGT_DTYPE_FP16 */
#define VGGT_DTYPE_FP32 2

/* status bits beside those of vggt_sparse.h */
#define VGGT_STATUS_BAD_PAGE 16   /* a needed page number is outside [0, n_pages) */
#define VGGT_STATUS_BAD_LENGTH 32 /* a length or a start was out of range and clamped */

/* front of the workspace of vggt_paged_attention that has to be zero */
#define VGGT_PAGED_WORKSPACE_ZERO_BYTES 16384

/* which elements of a head form the pairs that are rotated */
#define VGGT_ROTARY_HALF 0        /* element i with element i + pairs */
#define VGGT_ROTARY_INTERLEAVED 1 /* element 2i with element 2i + 1 */

/*
 * Rotates the first 2 * axes * pairs elements of each head of x [tokens][heads][dim]
 * and copies the rest.  Axis a's 2 * pairs elements are turned by
 * positions[token][a] * freq[i] (radians; the angle is reduced exactly for
 * every 32-bit position), and the result is multiplied by `lengthen`.
 * `inverse` turns the other way: the gradient with respect to x.
 * out may be x.  Strides in elements; the last dimension is contiguous.
 */
int vggt_rotary(const void* x, int dtype, int64_t tokens, int heads, int dim,
                int64_t x_token_stride, int64_t x_head_stride, const int32_t* positions, int axes,
                const double* freq, int pairs, int layout, float lengthen, int inverse, void* out,
                int64_t out_token_stride, int64_t out_head_stride, void* stream);

/*
 * Writes the new tokens' keys (rotated as by vggt_rotary when positions is
 * non-NULL) and values k, v [total][kv_heads][dim] behind each sequence's
 * `before[b]` cached tokens, and before[b] + (new tokens) to after[b].  ids
 * and weights, where non-NULL, get new_ids[token] and new_weights[token] (0
 * when new_weights is NULL) in every head.  Tokens past the last slot are not
 * written (VGGT_STATUS_BAD_LENGTH).  after must not overlap before.
 */
int vggt_paged_append(const void* k, const void* v, int dtype, int64_t total,
                      int64_t k_token_stride, int64_t k_head_stride, int64_t v_token_stride,
                      int64_t v_head_stride, void* k_pages, void* v_pages, int64_t n_pages,
                      int kv_heads, int page, int dim, int64_t page_stride, int64_t head_stride,
                      int64_t row_stride, const int32_t* table, int64_t table_width, int64_t seqs,
                      const int32_t* before, const int32_t* starts, const int32_t* positions,
                      int axes, const double* freq, int pairs, int layout, float lengthen,
                      int32_t* ids, const int32_t* new_ids, float* weights,
                      const float* new_weights, int32_t* after, int32_t* status, void* stream);

/*
 * Attention of the new tokens (already in the cache: lengths[b] counts them)
 * over the cache.  q, out [total][kv_heads * group][dim] with strides that
 * are multiples of 8 elements; query head h reads key head h / group.  With
 * n = starts[b + 1] - starts[b] and causal != 0, new token i of sequence b
 * sees slots j <= lengths[b] - n + i, else all of its sequence's slots:
 *   s_ij = scale q_i . k_j,  lse_i = log sum_j exp s_ij,
 *   out_i = sum_j exp(s_ij - lse_i) v_j
 * A row that sees no key gets zeros and lse -inf.  So does a row that belongs
 * to no sequence (before starts[0], or at or past starts[seqs]), which also
 * sets VGGT_STATUS_BAD_LENGTH; with seqs == 0 nothing is written.  Slots past
 * the length are never used, whatever they hold; keys and values that only
 * later tokens see do not reach a row, finite or not.  lse
 * [total][kv_heads * group] fp32, or NULL.
 *
 * max_new and max_len are the most new tokens of a sequence and the greatest
 * length as the caller expects them; they choose the kernel and how the work
 * is cut, the result is right for any lengths.  The workspace holds at least
 * vggt_paged_attention_workspace_size bytes (same arguments), its first
 * VGGT_PAGED_WORKSPACE_ZERO_BYTES are zeroed before its first use (a call
 * leaves it ready for the next one, of any sizes), and it serves one stream at
 * a time.
 */
size_t vggt_paged_attention_workspace_size(int64_t total, int64_t seqs, int kv_heads, int group,
                                           int dim, int64_t max_new, int64_t max_len);
int vggt_paged_attention(const void* q, int dtype, int64_t total, int64_t q_token_stride,
                         int64_t q_head_stride, const void* k_pages, const void* v_pages,
                         int64_t n_pages, int kv_heads, int page, int dim, int64_t page_stride,
                         int64_t head_stride, int64_t row_stride, const int32_t* table,
                         int64_t table_width, int64_t seqs, const int32_t* lengths,
                         const int32_t* starts, int group, int causal, float scale,
                         int64_t max_new, int64_t max_len, void* out, int64_t out_token_stride,
                         int64_t out_head_stride, float* lse, int32_t* status, void* workspace,
                         size_t workspace_bytes, void* stream);

/*
 * Adds to each cached key's weight what the new tokens gave it:
 *   weights[j] = decay * weights[j] + sum_i exp(s_ij - lse_i)
 * over the rows i of its key head's group that see it (causal as above), lse
 * as vggt_paged_attention wrote it.  A weight of +inf (a token that is never
 * evicted) stays as it is, whatever the decay.  Slots past the length are left
 * alone.
 */
int vggt_paged_weights(const void* q, int dtype, int64_t total, int64_t q_token_stride,
                       int64_t q_head_stride, const float* lse, const void* k_pages,
                       int64_t n_pages, int kv_heads, int page, int dim, int64_t page_stride,
                       int64_t head_stride, int64_t row_stride, const int32_t* table,
                       int64_t table_width, int64_t seqs, const int32_t* lengths,
                       const int32_t* starts, int group, int causal, float scale, float decay,
                       int64_t max_new, int64_t max_len, float* weights, int32_t* status,
                       void* stream);

/*
 * Cuts every sequence to at most `budget` tokens, each key head by its own
 * weights.  Kept are the slots of largest weight; tokens whose id is
 * recent_from[seq] or more (recent_from non-NULL) rank as +inf, NaN below
 * everything, equal ranks by the lower slot.  Kept slots below the new length
 * min(length, budget) stay; the n-th evicted slot below it receives the n-th
 * kept slot at or past it (keys, values, weight and id).  weights, ids and
 * lengths are read, new_weights, new_ids (0 and -1 past the new length) and
 * new_lengths written; they must not overlap.  The pages of the sequences
 * must not be shared.  max_len as above.  The workspace needs no clearing.
 */
size_t vggt_paged_evict_workspace_size(int64_t seqs, int kv_heads, int64_t slots, int64_t budget);
int vggt_paged_evict(const float* weights, const int32_t* ids, int dtype, void* k_pages,
                     void* v_pages, int64_t n_pages, int kv_heads, int page, int dim,
                     int64_t page_stride, int64_t head_stride, int64_t row_stride,
                     const int32_t* table, int64_t table_width, int64_t seqs,
                     const int32_t* lengths, int64_t budget, const int32_t* recent_from,
                     int64_t max_len, float* new_weights, int32_t* new_ids, int32_t* new_lengths,
                     int32_t* status, void* workspace, size_t workspace_bytes, void* stream);

#ifdef __cplusplus
}
#endif
#endif /* VGGT_CACHE_H */
