// Launch interfaces of the serving operators (include/double_attention_serving.h):
// the paged cache, the attention that reads it, and token log probabilities.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

namespace da {

// A cache of routed keys and values in pages, and the sequences in it.  Keys:
// token t of a page at keys + page * key_page + t * W; values: tiles of 32
// tokens, feature d of token t at values + page * value_page +
// (t / 32) * 32 * D + 32 * d + t % 32 (elements).
struct CacheView {
  void* keys;
  int64_t key_page;
  void* values;
  int64_t value_page;
  int pages;
  int tiles;            // 32-token tiles of a page
  uint32_t tiles_inv;   // ceil(2^32 / tiles), 0 for one tile
  int W;                // key features of a token (all branches)
  int D;
  const int32_t* table; // [sequences][ld_table]: the pages of each sequence, in order
  int64_t ld_table;
  int table_pages;      // entries of a row that are read
};

// Tile kt of a sequence: tile kt % tiles of the page in entry kt / tiles (exact
// for kt below 2^25: the product's error is at most kt * tiles, tiles <= 128).
__device__ __forceinline__ int entry_of(const CacheView& c, int kt) {
  return c.tiles_inv == 0 ? kt : static_cast<int>(__umulhi(static_cast<uint32_t>(kt), c.tiles_inv));
}
// A number that no kernel writes, at a uniform address: a scalar load.
template <typename T>
__device__ __forceinline__ T load_constant(const T* p) {
  return *(__attribute__((address_space(4))) const T*)(p);
}
// The page of tile kt of sequence b, or -1 where the table names none.
__device__ __forceinline__ int page_of(const CacheView& c, int b, int kt) {
  const int entry = entry_of(c, kt);
  if (entry >= c.table_pages) return -1;
  const int id = c.table[b * c.ld_table + entry];
  return static_cast<unsigned>(id) < static_cast<unsigned>(c.pages) ? id : -1;
}

// Packed new tokens: those of sequence b are rows offsets[b] .. offsets[b+1],
// and the last ones of its lengths[b] tokens.
struct NewTokens {
  int64_t N;            // rows there are
  int B;
  const int32_t* lengths;
  const int32_t* offsets;
};

struct PagedAttentionArgs {
  CacheView cache;
  NewTokens tokens;
  const void* q;        // [N] rows of W features, ldq apart
  int64_t ldq;
  const void* scales;   // [S]
  int scales_dtype;
  float scale_mult;     // every scale times this
  int S;                // score maps
  int RP;               // features of a map
  int repeat;           // maps that share one range of features
  bool causal;
  const float* mix;     // [S] weights of the maps' sum, or nullptr
  int qk_dtype, v_dtype;
  void* out;            // [N][S][D], with mix [N][D]
  float* lse2;          // [N][S] log2 of each row's sum of exponentials, or nullptr
  int max_chunk;        // new tokens of a sequence, as far as the host knows
  int max_length;       // tokens of a sequence, as far as the host knows
  // attention weights (launch_paged_weights)
  const float* weights_in;   // [B][ld_weights] or nullptr (0)
  float* weights_out;        // [B][ld_weights]
  int64_t ld_weights;
  int capacity;              // entries of a row
};
int64_t paged_attention_workspace(const PagedAttentionArgs& a);
void launch_paged_attention(const PagedAttentionArgs& a, void* workspace, hipStream_t stream);
// weights_out[b][t] = (t < old ? weights_in[b][t] : 0) + sum over the new rows
// and maps of their probabilities at t; from the row sums of the attention.
void launch_paged_weights(const PagedAttentionArgs& a, hipStream_t stream);

struct CacheAppendArgs {
  CacheView cache;
  NewTokens tokens;
  const void* key;      // [N] rows of W, ldk apart
  int64_t ldk;
  const void* value;    // [N] rows of D, ldv apart
  int64_t ldv;
  int max_chunk;
};
void launch_cache_append(const CacheAppendArgs& a, hipStream_t stream);

// kept[b]: in ascending order the last `recent` of the lengths[b] tokens and
// those of the others with the largest weights, keep in all (or all there
// are: counts[b]); -1 behind them.
struct CacheSelectArgs {
  const float* weights;
  int64_t ld_weights;
  int capacity;
  const int32_t* lengths;
  int B;
  int keep, recent;
  int32_t* kept;        // [B][keep]
  int32_t* counts;      // [B]
};
void launch_cache_select(const CacheSelectArgs& a, hipStream_t stream);

struct CacheCompactArgs {
  CacheView from, to;   // of one W, D and element size; only `to` is written
  int B;
  const int32_t* kept;  // [B][ld_kept]
  int64_t ld_kept;
  int keep;
  const int32_t* counts;
  const float* weights_in;   // [B][ld_in] or nullptr
  int64_t ld_in;
  float* weights_out;        // [B][ld_out]
  int64_t ld_out;
  int capacity_in, capacity_out;
};
void launch_cache_compact(const CacheCompactArgs& a, hipStream_t stream);

constexpr int kMaxTop = 64;
struct TokenLogProbsArgs {
  const void* logits;   // [rows] rows of V, ldx apart
  int64_t ldx;
  int64_t rows;
  int V;
  int dtype;
  const int64_t* tokens;     // [rows]
  int64_t ignore;
  float* log_probs;     // [rows]
  float* entropy;       // [rows]
  float* lse;           // [rows][2]: a reference m and log sum e^(x - m), or nullptr
  int top;
  float* top_log_probs; // [rows][top]
  int64_t* top_tokens;  // [rows][top]
  // backward: grad [rows][V] of the logits' type at
  const float* g_log_probs;       // [rows] or nullptr (0)
  const float* g_entropy;         // [rows] or nullptr
  const float* g_top;             // [rows][top] or nullptr
  void* grad;
  int64_t ldg;
};
int64_t token_log_probs_workspace(const TokenLogProbsArgs& a);
void launch_token_log_probs(const TokenLogProbsArgs& a, void* workspace, hipStream_t stream);
void launch_token_log_probs_backward(const TokenLogProbsArgs& a, hipStream_t stream);

}  // namespace da
