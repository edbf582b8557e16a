/*
 * C ABI of the language model's serving operators: a paged cache of routed keys
 * and values, the attention of new tokens over it with the cached tokens'
 * accumulated weights, the choice and the move of the tokens that stay when a
 * sequence is cut, and log probabilities of tokens.  No counterpart in the
 * reference.  The conventions are those of double_attention_hip.h: device
 * pointers, element counts, the caller's stream, buffers and workspace, nothing
 * allocated, freed or synchronized, arguments checked before anything is
 * enqueued, 0 or a DA_ERR_* code returned (da_last_error has the message).
 */
#ifndef DOUBLE_ATTENTION_SERVING_H
#define DOUBLE_ATTENTION_SERVING_H

#include "double_attention_hip.h"

#ifdef __cplusplus
extern "C" {
#endif

/*
 * A paged cache of one layer.  Token t (0 <= t < page_size) of page p:
 *   key feature f    keys[p * key_page_stride + t * key_width + f]
 *   value feature d  values[p * value_page_stride + (t / 32) * 32 * value_dim + 32 * d + t % 32]
 * (elements; values lie in tiles of 32 tokens, a feature's tokens side by
 * side).  key_width is branches * routing_dim.  page_size: a multiple of 32 up
 * to 4096.  key_width: a multiple of 64 up to 1024.  value_dim: a multiple of
 * 64 up to 4096.  table_pages * page_size: up to 2^27.  Both tensors 16-byte aligned, page strides multiples of 8.
 *
 * page_table: [sequences] rows of table_pages entries, ld_table apart: the pages
 * of each sequence in order.  An entry outside [0, pages) names no page: its
 * tokens are not seen, not written and not moved.
 * lengths[b]: tokens of sequence b, the new ones of this call among them; tokens
 * behind the table's entries are not there.  New tokens are packed: those of
 * sequence b are rows offsets[b] to offsets[b + 1] of [rows] and stand at the
 * sequence's last positions (offsets: [sequences + 1], not decreasing; rows in
 * front of the first and behind the last one belong to no sequence).  A new
 * token whose position would be negative sees nothing and is not written.
 * max_chunk and max_length are what the host knows of the new tokens and the
 * tokens of a sequence (0: nothing, and all rows may be one sequence's); they
 * choose the launch, not the result.
 */
typedef struct {
  void* keys;
  int64_t key_page_stride;
  void* values;
  int64_t value_page_stride;
  int64_t pages;
  int64_t page_size;
  int64_t key_width;
  int64_t value_dim;
  const int32_t* page_table;
  int64_t ld_table;
  int64_t table_pages;
} da_paged_cache;

/* The new tokens' keys [rows, key_width] and values [rows, value_dim] (16-bit
 * elements, pitches ldk and ldv, multiples of 8) into the cache. */
int da_cache_append(const da_paged_cache* cache, const void* key, int64_t ldk, const void* value, int64_t ldv, int64_t rows,
                    const int32_t* lengths, const int32_t* offsets, int64_t sequences, int64_t max_chunk, da_stream_t stream);

/*
 * Attention of the new tokens over the cache:
 *   out[n, s] = sum_j softmax_j(scales[s] scale_mult <q_{n,s}, k_{j,s}>) v_j
 * over the tokens j of row n's sequence up to its own (causal) or all of them.
 * Map s has features [(s / map_repeat) * score_dim, + score_dim) of the rows of
 * query [rows, key_width] (pitch ldq, a multiple of 8 up to 2^22) and of the keys;
 * score_dim is a multiple of 64 up to 512, at most 64 maps.
 * out: [rows, maps, value_dim], or with mix [maps] (fp32) its sum
 * over the maps with these weights, [rows, value_dim].  Rows that see nothing,
 * and rows of no sequence, are zero.  Scores, the softmax and sums are fp32;
 * probabilities are rounded to v_dtype for the product with the values, and the
 * result once.  A value that is an infinity or a NaN makes its feature one in the
 * rows that see its token, and in no other.  A key feature that is one may make
 * the rows NaN that see its token, in the maps that read it, and the weights of
 * what those rows see.  What lies behind a sequence's last token reaches nothing.
 * Types: (qk_dtype, v_dtype) in (F16, BF16), (F16, F16), (BF16, BF16).
 *
 * weights_out (NULL: none) [sequences] rows of table_pages * page_size fp32, ld_weights apart:
 *   weights_out[b, t] = (t old ? weights_in[b, t] : 0) + sum over b's new rows and maps of their probability of t,
 * t old: in front of the call's new tokens; zero behind the last token.
 * weights_in may be NULL (zeros) or weights_out itself.
 * workspace: 16-byte aligned, as many bytes as the query returns (0: none).
 */
typedef struct {
  da_paged_cache cache;
  const void* query;
  int64_t ldq;
  int64_t rows;
  const int32_t* lengths;
  const int32_t* offsets;
  int64_t sequences;
  const void* scales;
  int scales_dtype;
  float scale_mult;
  int64_t maps;
  int64_t score_dim;
  int64_t map_repeat;
  int causal;
  const float* mix;
  int qk_dtype;
  int v_dtype;
  void* out;
  const float* weights_in;
  float* weights_out;
  int64_t ld_weights;
  int64_t max_chunk;
  int64_t max_length;
  void* workspace;
  int64_t workspace_bytes;
} da_paged_attention_args;

int64_t da_paged_attention_workspace_bytes(const da_paged_attention_args* args);
int da_paged_attention(const da_paged_attention_args* args, da_stream_t stream);

/*
 * The tokens that stay when sequences are cut to `keep` tokens: the last
 * `recent` ones and, of the others, those of the largest weights, equal ones
 * in their order (NaN is below everything).  weights: [sequences] rows of
 * capacity fp32, ld_weights apart; lengths are taken up to capacity.
 * kept: [sequences, keep], ascending, -1 behind the counts[b] that stay
 * (all, where the sequence is not longer).  0 <= recent <= keep.
 */
int da_cache_select(const float* weights, int64_t ld_weights, int64_t capacity, const int32_t* lengths, int64_t sequences,
                    int64_t keep, int64_t recent, int32_t* kept, int32_t* counts, da_stream_t stream);

/*
 * Tokens kept[b, i], i < counts[b], of `from` become tokens i of `to` (caches
 * of one key_width, value_dim and element size of 16 bits; kept: [sequences]
 * rows of keep, ld_kept apart).  Pages that `to`'s table names must not be
 * among those that `from`'s names for tokens that move.  With
 * weights_out, weights_out[b, i] = weights_in[b, kept[b, i]] for i < counts[b],
 * else 0, over all of to's table_pages * page_size entries; weights_in has
 * from's.
 */
int da_cache_compact(const da_paged_cache* from, const da_paged_cache* to, int64_t sequences, const int32_t* kept,
                     int64_t ld_kept, int64_t keep, const int32_t* counts, const float* weights_in, int64_t ld_in,
                     float* weights_out, int64_t ld_out, da_stream_t stream);

/*
 * Of logits [rows, vocab] (any dtype, pitch ldx, aligned to their elements):
 *   log_probs[r] = log softmax(logits[r])[tokens[r]]   (0 at ignore_index, NaN for other tokens outside [0, vocab))
 *   entropy[r]   = -sum_j p_j log p_j                  (NULL: not wanted)
 *   lse[r]       = (m, log sum_j exp(logits[r, j] - m)) with some m near the row's largest logit: two floats, whose
 *                  sum is the log-sum-exp                (NULL: not wanted; the backward's)
 *   top_tokens[r], top_log_probs[r]: the `top` most probable tokens in order,
 *                  equal ones the lowest first (top <= 64, top <= vocab; a NaN is never among them: -1 and NaN stand for what is missing).
 * Rows with a NaN or +infinity, and rows of -infinity throughout, have NaN log
 * probabilities, as log_softmax.  vocab <= 2^24.  workspace as above.
 */
#define DA_MAX_TOP 64
int64_t da_token_log_probs_workspace_bytes(int64_t rows, int64_t vocab, int64_t top);
int da_token_log_probs(const void* logits, int64_t rows, int64_t vocab, int64_t ldx, int dtype, const int64_t* tokens,
                       int64_t ignore_index, float* log_probs, float* entropy, float* lse, int64_t top, float* top_log_probs,
                       int64_t* top_tokens, void* workspace, int64_t workspace_bytes, da_stream_t stream);

/*
 * Its gradient at the logits, rounded once to their type, from the gradients at
 * log_probs, entropy and top_log_probs (each NULL: zero), and the lse, entropy
 * and top_tokens that the forward gave.  grad: [rows, vocab] at pitch ldg, off
 * the logits.
 */
int da_token_log_probs_backward(const void* logits, int64_t rows, int64_t vocab, int64_t ldx, int dtype, const int64_t* tokens,
                                int64_t ignore_index, const float* lse, const float* entropy, int64_t top,
                                const int64_t* top_tokens, const float* grad_log_probs, const float* grad_entropy,
                                const float* grad_top, void* grad, int64_t ldg, da_stream_t stream);

#ifdef __cplusplus
}
#endif

#endif /* DOUBLE_ATTENTION_SERVING_H */
