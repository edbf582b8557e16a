// C ABI entry points of the serving operators (declared in
// include/double_attention_serving.h): arguments are checked here, then the
// kernels are enqueued on the caller's stream.
#include <algorithm>
#include <cmath>

#include "../../include/double_attention_serving.h"
#include "da_capi.h"
#include "da_launch.h"
#include "da_serving.h"

using namespace da::capi;

namespace {

constexpr int64_t kMaxRows = 1 << 22;        // new tokens of a call
constexpr int64_t kMaxSequences = 65535;     // a grid's second dimension
constexpr int64_t kMaxTokens = 1 << 27;      // tokens of a sequence
constexpr int64_t kMaxStride = 1LL << 40;
constexpr int64_t kMaxQueryPitch = 1 << 22;  // 128 rows span less than 2^32 bytes

int validate_cache(const char* what, const da_paged_cache& c, int64_t sequences) {
  if (c.page_size < 32 || c.page_size % 32 || c.page_size > 4096)
    return fail(DA_ERR_UNSUPPORTED, "%s: page_size %lld must be a multiple of 32 in [32, 4096]", what, (long long)c.page_size);
  if (c.key_width < 64 || c.key_width % 64 || c.key_width > 1024)
    return fail(DA_ERR_UNSUPPORTED, "%s: key_width %lld must be a multiple of 64 in [64, 1024]", what, (long long)c.key_width);
  if (c.value_dim < 64 || c.value_dim % 64 || c.value_dim > 4096)
    return fail(DA_ERR_UNSUPPORTED, "%s: value_dim %lld must be a multiple of 64 in [64, 4096]", what, (long long)c.value_dim);
  if (c.pages < 1 || c.pages > 0x7fffffff) return fail(DA_ERR_INVALID_ARGUMENT, "%s: the cache has no pages", what);
  if (sequences < 0 || sequences > kMaxSequences)
    return fail(DA_ERR_UNSUPPORTED, "%s: sequences must be in [0, %lld]", what, (long long)kMaxSequences);
  if (c.table_pages < 0 || c.ld_table < c.table_pages || c.ld_table > kMaxStride || c.table_pages > kMaxTokens / c.page_size)
    return fail(DA_ERR_INVALID_ARGUMENT, "%s: a page table's row has fewer entries than are read, or more than 2^27 tokens", what);
  if (!c.keys || !c.values || (sequences > 0 && c.table_pages > 0 && !c.page_table))
    return fail(DA_ERR_INVALID_ARGUMENT, "%s: null pointer in the cache", what);
  if (!aligned(c.keys, 16) || !aligned(c.values, 16) || !aligned(c.page_table, 4) || c.key_page_stride % 8 || c.value_page_stride % 8)
    return fail(DA_ERR_ALIGNMENT, "%s: keys and values must be 16-byte aligned at page strides that are multiples of 8", what);
  if (c.key_page_stride < c.page_size * c.key_width || c.value_page_stride < c.page_size * c.value_dim ||
      c.key_page_stride > kMaxStride / 2 || c.value_page_stride > kMaxStride / 2)
    return fail(DA_ERR_INVALID_ARGUMENT, "%s: page strides are at least a page", what);
  return DA_OK;
}

da::CacheView view(const da_paged_cache& c) {
  const int64_t tiles = c.page_size / 32;
  const uint32_t inverse = tiles == 1 ? 0u : static_cast<uint32_t>((0xffffffffu + tiles) / tiles);
  return {c.keys, c.key_page_stride, c.values, c.value_page_stride, static_cast<int>(c.pages), static_cast<int>(tiles), inverse,
          static_cast<int>(c.key_width), static_cast<int>(c.value_dim), c.page_table, c.ld_table, static_cast<int>(c.table_pages)};
}
Spans pages_of(const void* p, const da_paged_cache& c, int64_t width, int64_t stride) {
  return {p, c.pages, c.page_size * width, stride, 2};
}
Spans keys_of(const da_paged_cache& c) { return pages_of(c.keys, c, c.key_width, c.key_page_stride); }
Spans values_of(const da_paged_cache& c) { return pages_of(c.values, c, c.value_dim, c.value_page_stride); }
Spans table_of(const da_paged_cache& c, int64_t sequences) { return {c.page_table, sequences, c.table_pages, c.ld_table, 4}; }

int validate_tokens(const char* what, int64_t rows, const int32_t* lengths, const int32_t* offsets) {
  if (rows < 0 || rows > kMaxRows) return fail(DA_ERR_UNSUPPORTED, "%s: rows must be in [0, %lld]", what, (long long)kMaxRows);
  if (!lengths || !offsets || !aligned(lengths, 4) || !aligned(offsets, 4))
    return fail(DA_ERR_INVALID_ARGUMENT, "%s: lengths or offsets are null or not aligned", what);
  return DA_OK;
}
int validate_rows16(const char* what, const char* name, const void* p, int64_t cols, int64_t ld) {
  if (!p) return fail(DA_ERR_INVALID_ARGUMENT, "%s: %s is null", what, name);
  if (!aligned(p, 16) || ld % 8 || ld < cols || ld > kMaxStride)
    return fail(DA_ERR_ALIGNMENT, "%s: %s must be 16-byte aligned rows at a pitch of a multiple of 8", what, name);
  return DA_OK;
}
// What the host knows of a size, as far as it can be.
int known(int64_t given, int64_t most) { return static_cast<int>(given > 0 ? std::min(given, most) : most); }

// The checks of the attention that need no pointers, and its launch arguments.
int attention_args(const da_paged_attention_args& a, da::PagedAttentionArgs& r) {
  const char* what = "paged attention";
  const bool types_ok = (a.qk_dtype == DA_F16 && half_dtype(a.v_dtype)) || (a.qk_dtype == DA_BF16 && a.v_dtype == DA_BF16);
  if (!types_ok)
    return fail(DA_ERR_UNSUPPORTED, "%s: (qk_dtype, v_dtype) must be (F16,BF16), (F16,F16) or (BF16,BF16)", what);
  if (a.maps < 1 || a.maps > 64 || a.map_repeat < 1) return fail(DA_ERR_UNSUPPORTED, "%s: 1 to 64 maps", what);
  if (a.score_dim < 64 || a.score_dim % 64 || a.score_dim > 512)
    return fail(DA_ERR_UNSUPPORTED, "%s: score_dim %lld must be a multiple of 64 in [64, 512]", what, (long long)a.score_dim);
  if (a.maps % a.map_repeat || a.maps / a.map_repeat * a.score_dim > a.cache.key_width)
    return fail(DA_ERR_INVALID_ARGUMENT, "%s: the maps' features do not fit the keys' %lld", what, (long long)a.cache.key_width);
  if (!any_dtype(a.scales_dtype) || !std::isfinite(a.scale_mult))
    return fail(DA_ERR_INVALID_ARGUMENT, "%s: bad scales", what);
  if (a.rows * a.maps > kMaxRows) return fail(DA_ERR_UNSUPPORTED, "%s: rows times maps above %lld", what, (long long)kMaxRows);
  const int64_t capacity = a.cache.table_pages * a.cache.page_size;
  r = {view(a.cache), {a.rows, static_cast<int>(a.sequences), a.lengths, a.offsets}, a.query, a.ldq, a.scales, a.scales_dtype,
       a.scale_mult, static_cast<int>(a.maps), static_cast<int>(a.score_dim), static_cast<int>(a.map_repeat), a.causal != 0, a.mix,
       a.qk_dtype, a.v_dtype, a.out, nullptr, known(a.max_chunk, a.rows), known(a.max_length, capacity), a.weights_in,
       a.weights_out, a.ld_weights, static_cast<int>(capacity)};
  return DA_OK;
}
int64_t lse_bytes(const da_paged_attention_args& a) { return a.weights_out ? align_up(a.rows * a.maps * 4) : 0; }

int validate_logits(const char* what, const void* logits, int64_t rows, int64_t vocab, int64_t ld, int dtype) {
  if (!any_dtype(dtype)) return fail(DA_ERR_INVALID_ARGUMENT, "%s: bad dtype", what);
  if (rows < 0 || rows > kMaxRows || vocab < 1 || vocab > (1 << 24))
    return fail(DA_ERR_UNSUPPORTED, "%s: rows must be in [0, %lld], vocab in [1, 2^24]", what, (long long)kMaxRows);
  if (rows == 0) return DA_OK;
  if (!logits || !aligned(logits, static_cast<int>(element_bytes(dtype))))
    return fail(DA_ERR_ALIGNMENT, "%s: the logits are null or not aligned to their elements", what);
  if (ld < vocab || ld > kMaxStride) return fail(DA_ERR_INVALID_ARGUMENT, "%s: a pitch below the vocabulary", what);
  return DA_OK;
}
int validate_top(const char* what, int64_t top, int64_t vocab) {
  if (top < 0 || top > da::kMaxTop || top > vocab)
    return fail(DA_ERR_UNSUPPORTED, "%s: top must be in [0, %d] and at most the vocabulary", what, da::kMaxTop);
  return DA_OK;
}

}  // namespace

extern "C" {

static_assert(DA_MAX_TOP == da::kMaxTop, "alternatives of a row");

int da_cache_append(const da_paged_cache* cache, const void* key, int64_t ldk, const void* value, int64_t ldv, int64_t rows,
                    const int32_t* lengths, const int32_t* offsets, int64_t sequences, int64_t max_chunk, da_stream_t stream) {
  const char* what = "cache append";
  if (!cache) return fail(DA_ERR_INVALID_ARGUMENT, "%s: no cache", what);
  int rc = validate_cache(what, *cache, sequences);
  if (rc) return rc;
  if ((rc = validate_tokens(what, rows, lengths, offsets))) return rc;
  if (rows == 0 || sequences == 0 || cache->table_pages == 0) return ok();
  if ((rc = validate_rows16(what, "key", key, cache->key_width, ldk))) return rc;
  if ((rc = validate_rows16(what, "value", value, cache->value_dim, ldv))) return rc;
  if ((rc = validate_apart(what, {keys_of(*cache), values_of(*cache)},
                           {{key, rows, cache->key_width, ldk, 2}, {value, rows, cache->value_dim, ldv, 2}, flat(lengths, sequences, 4),
                            flat(offsets, sequences + 1, 4), table_of(*cache, sequences)})))
    return rc;
  da::launch_cache_append({view(*cache), {rows, static_cast<int>(sequences), lengths, offsets}, key, ldk, value, ldv,
                           known(max_chunk, rows)},
                          reinterpret_cast<hipStream_t>(stream));
  return check_launch(what);
}

int64_t da_paged_attention_workspace_bytes(const da_paged_attention_args* args) {
  da::PagedAttentionArgs r;
  if (!args || validate_cache("paged attention", args->cache, args->sequences) || attention_args(*args, r) || args->rows < 1 ||
      args->sequences < 1)
    return 0;
  return align_up(da::paged_attention_workspace(r)) + lse_bytes(*args);
}

int da_paged_attention(const da_paged_attention_args* args, da_stream_t stream) {
  const char* what = "paged attention";
  if (!args) return fail(DA_ERR_INVALID_ARGUMENT, "%s: no arguments", what);
  const da_paged_attention_args& a = *args;
  int rc = validate_cache(what, a.cache, a.sequences);
  if (rc) return rc;
  da::PagedAttentionArgs r;
  if ((rc = attention_args(a, r))) return rc;
  if (a.sequences == 0 && a.rows > 0) return fail(DA_ERR_INVALID_ARGUMENT, "%s: rows without sequences", what);
  if (a.sequences == 0) return ok();
  if ((rc = validate_tokens(what, a.rows, a.lengths, a.offsets))) return rc;
  const int64_t capacity = a.cache.table_pages * a.cache.page_size;
  if (a.rows > 0) {
    if ((rc = validate_rows16(what, "query", a.query, a.cache.key_width, a.ldq))) return rc;
    if (a.ldq > kMaxQueryPitch) return fail(DA_ERR_UNSUPPORTED, "%s: a pitch of the queries above 2^22", what);
    if (!a.scales || !aligned(a.scales, static_cast<int>(element_bytes(a.scales_dtype))) || !aligned(a.mix, 4))
      return fail(DA_ERR_INVALID_ARGUMENT, "%s: the scales are null, or scales or mix not aligned", what);
    if (!a.out || !aligned(a.out, 16)) return fail(DA_ERR_ALIGNMENT, "%s: out must be 16-byte aligned", what);
  }
  if (a.weights_out && (a.ld_weights < capacity || a.ld_weights > kMaxStride || !aligned(a.weights_out, 4) || !aligned(a.weights_in, 4)))
    return fail(DA_ERR_INVALID_ARGUMENT, "%s: rows of weights below table_pages * page_size, or not aligned", what);
  const int64_t need = da_paged_attention_workspace_bytes(args);
  if (need > 0) {
    if (!a.workspace || a.workspace_bytes < need)
      return fail(DA_ERR_WORKSPACE, "%s: the workspace needs %lld bytes", what, (long long)need);
    if (!aligned(a.workspace, 16)) return fail(DA_ERR_ALIGNMENT, "%s: the workspace must be 16-byte aligned", what);
  }
  const int64_t out_cols = (a.mix ? 1 : a.maps) * a.cache.value_dim;
  const Spans weights_in{a.weights_in == a.weights_out ? nullptr : a.weights_in, a.sequences, capacity, a.ld_weights, 4};
  if ((rc = validate_apart(what,
                           {flat(a.rows ? a.out : nullptr, a.rows * out_cols, 2), {a.weights_out, a.sequences, capacity, a.ld_weights, 4},
                            flat(need ? a.workspace : nullptr, need, 1)},
                           {keys_of(a.cache), values_of(a.cache), table_of(a.cache, a.sequences),
                            {a.query, a.rows, a.cache.key_width, a.ldq, 2}, flat(a.lengths, a.sequences, 4),
                            flat(a.offsets, a.sequences + 1, 4), flat(a.scales, a.maps, element_bytes(a.scales_dtype)),
                            flat(a.mix, a.maps, 4), weights_in})))
    return rc;
  const hipStream_t s = reinterpret_cast<hipStream_t>(stream);
  if (a.rows > 0) {
    const int64_t lse = lse_bytes(a);
    r.lse2 = lse ? static_cast<float*>(a.workspace) : nullptr;
    da::launch_paged_attention(r, static_cast<char*>(a.workspace) + lse, s);
  }
  if (a.weights_out && capacity > 0) da::launch_paged_weights(r, s);
  return check_launch(what);
}

int da_cache_select(const float* weights, int64_t ld_weights, int64_t capacity, const int32_t* lengths, int64_t sequences,
                    int64_t keep, int64_t recent, int32_t* kept, int32_t* counts, da_stream_t stream) {
  const char* what = "cache select";
  if (sequences < 0 || sequences > kMaxSequences || capacity < 0 || capacity > kMaxTokens)
    return fail(DA_ERR_UNSUPPORTED, "%s: sequences must be in [0, %lld], rows up to 2^27 tokens", what, (long long)kMaxSequences);
  if (keep < 0 || keep > kMaxTokens || recent < 0 || recent > keep)
    return fail(DA_ERR_INVALID_ARGUMENT, "%s: needs 0 <= recent <= keep", what);
  if (sequences == 0) return ok();
  if (!lengths || !counts || (capacity > 0 && !weights) || (keep > 0 && !kept))
    return fail(DA_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (!aligned(weights, 4) || !aligned(lengths, 4) || !aligned(kept, 4) || !aligned(counts, 4))
    return fail(DA_ERR_ALIGNMENT, "%s: tensors must be aligned to their elements", what);
  if (ld_weights < capacity || ld_weights > kMaxStride) return fail(DA_ERR_INVALID_ARGUMENT, "%s: a pitch below the capacity", what);
  int rc = validate_apart(what, {flat(keep ? kept : nullptr, sequences * keep, 4), flat(counts, sequences, 4)},
                          {{weights, sequences, capacity, ld_weights, 4}, flat(lengths, sequences, 4)});
  if (rc) return rc;
  da::launch_cache_select({weights, ld_weights, static_cast<int>(capacity), lengths, static_cast<int>(sequences),
                           static_cast<int>(keep), static_cast<int>(recent), kept, counts},
                          reinterpret_cast<hipStream_t>(stream));
  return check_launch(what);
}

int da_cache_compact(const da_paged_cache* from, const da_paged_cache* to, int64_t sequences, const int32_t* kept,
                     int64_t ld_kept, int64_t keep, const int32_t* counts, const float* weights_in, int64_t ld_in,
                     float* weights_out, int64_t ld_out, da_stream_t stream) {
  const char* what = "cache compact";
  if (!from || !to) return fail(DA_ERR_INVALID_ARGUMENT, "%s: no cache", what);
  int rc = validate_cache(what, *from, sequences);
  if (rc) return rc;
  if ((rc = validate_cache(what, *to, sequences))) return rc;
  if (from->key_width != to->key_width || from->value_dim != to->value_dim)
    return fail(DA_ERR_INVALID_ARGUMENT, "%s: caches of two widths", what);
  if (keep < 0 || keep > kMaxTokens || ld_kept < keep || ld_kept > kMaxStride)
    return fail(DA_ERR_INVALID_ARGUMENT, "%s: kept has a pitch below keep", what);
  if (sequences == 0) return ok();
  if (!counts || !aligned(counts, 4) || (keep > 0 && !kept) || !aligned(kept, 4))
    return fail(DA_ERR_INVALID_ARGUMENT, "%s: kept or counts are null or not aligned", what);
  const int64_t cap_in = from->table_pages * from->page_size, cap_out = to->table_pages * to->page_size;
  if (weights_out && ((!weights_in && cap_in > 0) || ld_in < cap_in || ld_out < cap_out || ld_in > kMaxStride || ld_out > kMaxStride ||
                      !aligned(weights_in, 4) || !aligned(weights_out, 4)))
    return fail(DA_ERR_INVALID_ARGUMENT, "%s: weights are null, not aligned, or in rows below the caches' tokens", what);
  const Spans in{weights_out ? weights_in : nullptr, sequences, cap_in, ld_in, 4};
  const Spans tables[2] = {table_of(*from, sequences), table_of(*to, sequences)};
  // A cache may be compacted into other pages of its own: keys into keys, values into values.
  const bool own_keys = from->keys == to->keys && from->key_page_stride == to->key_page_stride;
  const bool own_values = from->values == to->values && from->value_page_stride == to->value_page_stride;
  if (from->page_size != to->page_size && (own_keys || own_values))
    return fail(DA_ERR_INVALID_ARGUMENT, "%s: one cache with two page sizes", what);
  const Spans from_keys = own_keys ? Spans(nullptr, 0, 0, 0, 2) : keys_of(*from);
  const Spans from_values = own_values ? Spans(nullptr, 0, 0, 0, 2) : values_of(*from);
  if ((rc = validate_apart(what, {keys_of(*to), values_of(*to), {weights_out, sequences, cap_out, ld_out, 4}},
                           {from_keys, from_values, tables[0], tables[1], {keep ? kept : nullptr, sequences, keep, ld_kept, 4},
                            flat(counts, sequences, 4), in})))
    return rc;
  da::launch_cache_compact({view(*from), view(*to), static_cast<int>(sequences), kept, ld_kept, static_cast<int>(keep), counts,
                            weights_in, ld_in, weights_out, ld_out, static_cast<int>(cap_in), static_cast<int>(cap_out)},
                           reinterpret_cast<hipStream_t>(stream));
  return check_launch(what);
}

int64_t da_token_log_probs_workspace_bytes(int64_t rows, int64_t vocab, int64_t top) {
  if (rows < 1 || rows > kMaxRows || vocab < 1 || vocab > (1 << 24) || top < 0 || top > da::kMaxTop) return 0;
  da::TokenLogProbsArgs a{};
  a.rows = rows;
  a.V = static_cast<int>(vocab);
  a.top = static_cast<int>(top);
  return align_up(da::token_log_probs_workspace(a));
}

int da_token_log_probs(const void* logits, int64_t rows, int64_t vocab, int64_t ldx, int dtype, const int64_t* tokens,
                       int64_t ignore_index, float* log_probs, float* entropy, float* lse, int64_t top, float* top_log_probs,
                       int64_t* top_tokens, void* workspace, int64_t workspace_bytes, da_stream_t stream) {
  const char* what = "token log probs";
  int rc = validate_logits(what, logits, rows, vocab, ldx, dtype);
  if (rc) return rc;
  if ((rc = validate_top(what, top, vocab))) return rc;
  if (rows == 0) return ok();
  if (!tokens || !log_probs || (top && (!top_log_probs || !top_tokens))) return fail(DA_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (!aligned(tokens, 8) || !aligned(log_probs, 4) || !aligned(entropy, 4) || !aligned(lse, 4) || !aligned(top_log_probs, 4) ||
      !aligned(top_tokens, 8))
    return fail(DA_ERR_ALIGNMENT, "%s: tensors must be aligned to their elements", what);
  const int64_t need = da_token_log_probs_workspace_bytes(rows, vocab, top);
  if (need > 0) {
    if (!workspace || workspace_bytes < need)
      return fail(DA_ERR_WORKSPACE, "%s: the workspace needs %lld bytes", what, (long long)need);
    if (!aligned(workspace, 16)) return fail(DA_ERR_ALIGNMENT, "%s: the workspace must be 16-byte aligned", what);
  }
  if ((rc = validate_apart(what,
                           {flat(log_probs, rows, 4), flat(entropy, rows, 4), flat(lse, 2 * rows, 4), flat(top ? top_log_probs : nullptr, rows * top, 4),
                            flat(top ? top_tokens : nullptr, rows * top, 8), flat(need ? workspace : nullptr, need, 1)},
                           {{logits, rows, vocab, ldx, element_bytes(dtype)}, flat(tokens, rows, 8)})))
    return rc;
  da::TokenLogProbsArgs a{};
  a.logits = logits;
  a.ldx = ldx;
  a.rows = rows;
  a.V = static_cast<int>(vocab);
  a.dtype = dtype;
  a.tokens = tokens;
  a.ignore = ignore_index;
  a.log_probs = log_probs;
  a.entropy = entropy;
  a.lse = lse;
  a.top = static_cast<int>(top);
  a.top_log_probs = top_log_probs;
  a.top_tokens = top_tokens;
  da::launch_token_log_probs(a, workspace, reinterpret_cast<hipStream_t>(stream));
  return check_launch(what);
}

int da_token_log_probs_backward(const void* logits, int64_t rows, int64_t vocab, int64_t ldx, int dtype, const int64_t* tokens,
                                int64_t ignore_index, const float* lse, const float* entropy, int64_t top,
                                const int64_t* top_tokens, const float* grad_log_probs, const float* grad_entropy,
                                const float* grad_top, void* grad, int64_t ldg, da_stream_t stream) {
  const char* what = "token log probs backward";
  int rc = validate_logits(what, logits, rows, vocab, ldx, dtype);
  if (rc) return rc;
  if ((rc = validate_top(what, top, vocab))) return rc;
  if (rows == 0) return ok();
  if ((rc = validate_logits(what, grad, rows, vocab, ldg, dtype))) return rc;
  if (!tokens || !lse || (grad_entropy && !entropy) || (grad_top && (!top_tokens || top == 0)))
    return fail(DA_ERR_INVALID_ARGUMENT, "%s: null pointer", what);
  if (!aligned(tokens, 8) || !aligned(lse, 4) || !aligned(entropy, 4) || !aligned(top_tokens, 8) || !aligned(grad_log_probs, 4) ||
      !aligned(grad_entropy, 4) || !aligned(grad_top, 4))
    return fail(DA_ERR_ALIGNMENT, "%s: tensors must be aligned to their elements", what);
  if ((rc = validate_apart(what, {{grad, rows, vocab, ldg, element_bytes(dtype)}},
                           {{logits, rows, vocab, ldx, element_bytes(dtype)}, flat(tokens, rows, 8), flat(lse, 2 * rows, 4),
                            flat(entropy, rows, 4), flat(grad_top ? top_tokens : nullptr, rows * top, 8), flat(grad_log_probs, rows, 4),
                            flat(grad_entropy, rows, 4), flat(grad_top, rows * top, 4)})))
    return rc;
  da::TokenLogProbsArgs a{};
  a.logits = logits;
  a.ldx = ldx;
  a.rows = rows;
  a.V = static_cast<int>(vocab);
  a.dtype = dtype;
  a.tokens = tokens;
  a.ignore = ignore_index;
  a.lse = const_cast<float*>(lse);
  a.entropy = const_cast<float*>(entropy);
  a.top = static_cast<int>(top);
  a.top_tokens = const_cast<int64_t*>(top_tokens);
  a.g_log_probs = grad_log_probs;
  a.g_entropy = grad_entropy;
  a.g_top = grad_top;
  a.grad = grad;
  a.ldg = ldg;
  da::launch_token_log_probs_backward(a, reinterpret_cast<hipStream_t>(stream));
  return check_launch(what);
}

}  // extern "C"
