// Attention of new tokens over a paged cache:
//   out[n, s] = sum_j softmax_j(gamma_s q_{n,s} . k_{j,s}) v_j
// over the tokens j of row n's sequence up to its own position, for each score
// map s; all maps share the values.
//
// Columns.  A sequence's (new token, map) pairs are the columns of its score
// matrix, tokens outermost, 16 to a tile.  A tile's queries are laid over all
// W key features, zero outside of their map's: one product K Q^T then serves
// every map, and keys and values are read once for all maps of few tokens.
//
// paged_token_kernel: a wave takes 32 cached tokens at a time,
//   S^T[token, column] = K Q^T     (keys straight from memory, queries in LDS)
//   O^T[feature, column] += V^T P^T (values straight from memory: their tiles
//                                    hold a feature's tokens side by side, so a
//                                    wave's load is one contiguous KiB)
// with the running maximum and sum of each column in 32 bits.  The key rows go
// to the MFMA's rows in such an order that the score accumulators are the next
// product's operand as they stand (da_common.h).  A workgroup's four waves
// take every fourth tile of its part of the tokens and add up in LDS; parts
// are joined by paged_merge_kernel.
#include <algorithm>

#include "da_common.h"
#include "da_launch.h"
#include "da_serving.h"
#include "da_tile.h"

namespace da {

namespace {

constexpr int kWaves = 4;
constexpr int kKeyChunk = 8;          // 32-feature steps whose keys a wave holds
constexpr int kMaxSplits = 1024;
constexpr float kNoScore = -3.0e38f;  // the running maximum before the first score

struct Params {
  PagedAttentionArgs a;
  int n_ct;        // column tiles a workgroup index stands for (a stride, not a bound)
  int n_slices;    // slices of the value features
  int n_split;     // parts of the cached tokens
  int units;       // B * n_split
  float* part_o;   // [n_split][N * S][D], or nullptr: rows are finished here
  float* part_m;   // [n_split][N * S]
  float* part_l;
};

// The rows and tokens of sequence b; offsets and lengths are the device's, so
// they are held against the buffers here.
struct Sequence {
  int64_t n0;      // first row
  int rows;        // new tokens
  int length;      // tokens, the new ones among them
  int cached;      // of these, those that the table has entries for
};
__device__ __forceinline__ Sequence sequence_of(const NewTokens& t, const CacheView& c, int b) {
  Sequence s;
  const int64_t first = min(max(static_cast<int64_t>(t.offsets[b]), int64_t{0}), t.N);
  const int64_t last = min(max(static_cast<int64_t>(t.offsets[b + 1]), first), t.N);
  s.n0 = first;
  s.rows = static_cast<int>(last - first);
  s.length = max(t.lengths[b], 0);
  s.cached = static_cast<int>(min(static_cast<int64_t>(s.length), static_cast<int64_t>(c.table_pages) * c.tiles * 32));
  return s;
}
// Tokens that new token i of the sequence sees.
__device__ __forceinline__ int visible_to(const Sequence& s, int i, bool causal) {
  return causal ? max(0, min(s.cached, s.length - s.rows + i + 1)) : s.cached;
}
// The page of tile kt of sequence b, or -1 where the table names none.
__device__ __forceinline__ int page_of(const CacheView& c, int b, int kt) {
  const int id = c.table[b * c.ld_table + kt / c.tiles];
  return static_cast<unsigned>(id) < static_cast<unsigned>(c.pages) ? id : -1;
}
__device__ __forceinline__ float score_scale(const PagedAttentionArgs& a, int s) {
  return load_scalar(a.scales, a.scales_dtype, s) * a.scale_mult * kLog2e;
}

// Rows of no sequence (in front of the first and behind the last one) are zero.
template <typename TV>
__device__ void clear_other_rows(const PagedAttentionArgs& a, int64_t wg, int64_t n_wg) {
  const int64_t first = min(max(static_cast<int64_t>(a.tokens.offsets[0]), int64_t{0}), a.tokens.N);
  const int64_t last = min(max(static_cast<int64_t>(a.tokens.offsets[a.tokens.B]), first), a.tokens.N);
  const int64_t width = static_cast<int64_t>(a.S) * a.cache.D;
  for (int64_t i = wg; i < a.tokens.N - (last - first); i += n_wg) {
    const int64_t n = i < first ? i : i + (last - first);
    for (int64_t d = threadIdx.x; d < width; d += blockDim.x) static_cast<TV*>(a.out)[n * width + d] = static_cast<TV>(0.f);
    if (a.lse2 && static_cast<int>(threadIdx.x) < a.S) a.lse2[n * a.S + threadIdx.x] = -INFINITY;
  }
}

}  // namespace

template <typename TQ, typename TV, int DB>
__global__ __launch_bounds__(64 * kWaves) void paged_token_kernel(Params p) {
  typedef typename Elem<TQ>::v8 q8;
  typedef typename Elem<TV>::v8 v8;
  constexpr int DS = 16 * DB, OP = DS + 4;   // pitch of the outputs in LDS
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const PagedAttentionArgs& a = p.a;
  const CacheView& cache = a.cache;
  const int lane = lane_id(), c = lane & 15, g = lane >> 4;
  const int wave = uniform_wave();
  const int S = a.S, W = cache.W, D = cache.D;
  if (p.part_o == nullptr) clear_other_rows<TV>(a, blockIdx.x, gridDim.x);

  // Workgroups are dealt to the XCDs in turn.  Those that read the same tokens
  // (a unit's column tiles and slices) go to one, for its L2.
  const int members = p.n_ct * p.n_slices;
  const int wg = static_cast<int>(blockIdx.x);
  const int unit = wg / (kXcds * members) * kXcds + wg % kXcds;
  if (unit >= p.units) return;
  const int member = wg / kXcds % members;
  const int slice = member % p.n_slices;
  const int b = unit / p.n_split, split = unit % p.n_split;
  const Sequence seq = sequence_of(a.tokens, cache, b);
  const int n_cols = seq.rows * S;

  const int d0 = slice * DS;
  const int nb = min(DB, (D - d0) / 16);       // 16-feature blocks of this slice
  const int steps = (W + 32 * kKeyChunk - 1) / (32 * kKeyChunk);
  const int qp = steps * 32 * kKeyChunk + 8;   // pitch of the queries in LDS
  TQ* qs = reinterpret_cast<TQ*>(lds);
  float* os = reinterpret_cast<float*>(lds);
  float* stats = reinterpret_cast<float*>(lds + max(16 * qp * 2, 16 * OP * 4));   // [2][kWaves][16]

  for (int ct = member / p.n_slices; ct * 16 < n_cols; ct += p.n_ct) {
    const int col0 = ct * 16;
    __syncthreads();   // the last tile's outputs have been read
    for (int i = static_cast<int>(threadIdx.x); i < 2 * (qp - 8); i += 64 * kWaves) {
      const int col = i / ((qp - 8) / 8), f = i % ((qp - 8) / 8) * 8;
      const int token = (col0 + col) / S, from = (col0 + col) % S / a.repeat * a.RP;
      u32x4 v = {0, 0, 0, 0};
      if (col0 + col < n_cols && f >= from && f < from + a.RP)
        v = load16B(static_cast<const TQ*>(a.q) + (seq.n0 + token) * a.ldq + f);
      store16B(qs + col * qp + f, v);
    }
    __syncthreads();

    // This lane's column; columns behind the last one count as seeing all.
    const int mine = min(col0 + c, n_cols - 1);
    const int vis = visible_to(seq, mine / S, a.causal);
    const float sc = score_scale(a, mine % S);
    const int limit = visible_to(seq, min(col0 + 15, n_cols - 1) / S, a.causal);
    const int all_see = visible_to(seq, col0 / S, a.causal);
    const int n_kt = (limit + 31) / 32;
    const int per = (n_kt + p.n_split - 1) / p.n_split;
    const int kt0 = min(n_kt, split * per), kt1 = min(n_kt, kt0 + per);

    f32x4 acc[DB];
#pragma unroll
    for (int i = 0; i < DB; ++i) acc[i] = zero4();
    float m_run = kNoScore, l_part = 0.f;

    q8 kf[kKeyChunk][2];
    auto load_keys = [&](const TQ* base, int step) {
#pragma unroll
      for (int k = 0; k < kKeyChunk; ++k) {
        const int f = min((step * kKeyChunk + k) * 32, W - 32);   // past the last: multiplied by zero
        kf[k][0] = load8(base + f);
        kf[k][1] = load8(base + f + 4 * W);
      }
    };
    // Block h of the scores has token 8 (c / 4) + 4 h + c % 4 in row c.
    const int key_lane = (8 * (c >> 2) + (c & 3)) * W + 8 * g;
    auto key_base = [&](int page, int kt) {
      return static_cast<const TQ*>(cache.keys) + max(page, 0) * cache.key_page +
             static_cast<int64_t>(kt % cache.tiles) * 32 * W + key_lane;
    };
    int page = -1;
    if (kt0 + wave < kt1) {
      page = page_of(cache, b, kt0 + wave);
      load_keys(key_base(page, kt0 + wave), 0);
    }
    for (int kt = kt0 + wave; kt < kt1; kt += kWaves) {
      const TV* vb = static_cast<const TV*>(cache.values) + max(page, 0) * cache.value_page +
                     static_cast<int64_t>(kt % cache.tiles) * 32 * D + 32 * (d0 + c) + 8 * g;
      v8 vf[DB];
#pragma unroll
      for (int i = 0; i < DB; ++i) vf[i] = load8(vb + 512 * min(i, nb - 1));
      __builtin_amdgcn_sched_barrier(0);
      f32x4 st[2] = {zero4(), zero4()};
      for (int step = 0; step < steps; ++step) {
        if (step > 0) load_keys(key_base(page, kt), step);
#pragma unroll
        for (int k = 0; k < kKeyChunk; ++k) {
          const q8 qv = load8(qs + c * qp + (step * kKeyChunk + k) * 32 + 8 * g);
          st[0] = Elem<TQ>::mma(kf[k][0], qv, st[0]);
          st[1] = Elem<TQ>::mma(kf[k][1], qv, st[1]);
        }
      }
      const bool whole = page >= 0 && kt * 32 + 32 <= all_see;   // nothing to mask
      const int live = page < 0 ? 0 : min(32, limit - kt * 32);
      if (kt + kWaves < kt1) {
        page = page_of(cache, b, kt + kWaves);
        load_keys(key_base(page, kt + kWaves), 0);
        __builtin_amdgcn_sched_barrier(0);
      }
      float mx = -INFINITY;
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int t = 8 * g + 4 * h + e;
          const float s = st[h][e] * sc;
          st[h][e] = whole || (t < live && kt * 32 + t < vis) ? s : -INFINITY;
          mx = fmaxf(mx, st[h][e]);
        }
      lazy_rescale<DB>(mx, 1.f, m_run, l_part, acc);
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          st[h][e] = __builtin_amdgcn_exp2f(st[h][e] - m_run);
          l_part += st[h][e];
        }
      // The probabilities are rounded to the values' type for the product, the
      // sum is of the unrounded ones.
      const v8 pv = pack_blocked<TV>(st[0], st[1]);
      if (live < 32) {   // what lies behind the last token is not multiplied
#pragma unroll
        for (int i = 0; i < DB; ++i)
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (8 * g + e >= live) vf[i][e] = static_cast<TV>(0.f);
      }
#pragma unroll
      for (int i = 0; i < DB; ++i) acc[i] = Elem<TV>::mma(vf[i], pv, acc[i]);
    }

    // The waves' sums, to the largest maximum.
    const float l_run = group_sum(l_part);
    if (g == 0) {
      stats[wave * 16 + c] = m_run;
      stats[(kWaves + wave) * 16 + c] = l_run;
    }
    __syncthreads();   // and the queries have been read
    float m_all = kNoScore, l_all = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) m_all = fmaxf(m_all, stats[w * 16 + c]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) l_all += stats[(kWaves + w) * 16 + c] * __builtin_amdgcn_exp2f(stats[w * 16 + c] - m_all);
    const float factor = __builtin_amdgcn_exp2f(m_run - m_all);
    const bool used = col0 + c < n_cols;
    for (int w = 0; w < kWaves; ++w) {
      if (wave == w && used) {
#pragma unroll
        for (int i = 0; i < DB; ++i) {
          f32x4* dst = reinterpret_cast<f32x4*>(os + c * OP + 16 * i + 4 * g);
          *dst = w == 0 ? acc[i] * factor : *dst + acc[i] * factor;
        }
      }
      __syncthreads();
    }
    const int64_t row0 = seq.n0 * S + col0;
    const int n_used = min(16, n_cols - col0);
    if (wave == 0 && g == 0 && used && slice == 0) {
      if (p.part_o) {
        p.part_m[split * a.tokens.N * S + row0 + c] = m_all;
        p.part_l[split * a.tokens.N * S + row0 + c] = l_all;
      } else if (a.lse2) {
        a.lse2[row0 + c] = l_all == 0.f ? -INFINITY : m_all + __builtin_amdgcn_logf(l_all);
      }
    }
    if (wave == 0 && g == 0) stats[c] = l_all;
    __syncthreads();
    for (int i = static_cast<int>(threadIdx.x); i < n_used * 4 * DB; i += 64 * kWaves) {
      const int col = i / (4 * DB), d = i % (4 * DB) * 4;
      if (d >= 16 * nb) continue;
      f32x4 o = *reinterpret_cast<const f32x4*>(os + col * OP + d);
      if (p.part_o) {
        *reinterpret_cast<f32x4*>(p.part_o + ((split * a.tokens.N * S + row0 + col) * D + d0 + d)) = o;
      } else {
        const float l = stats[col];
        o *= l == 0.f ? 0.f : 1.f / l;
        typename Elem<TV>::v4 r;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = static_cast<TV>(o[e]);
        *reinterpret_cast<typename Elem<TV>::v4*>(static_cast<TV*>(a.out) + (row0 + col) * D + d0 + d) = r;
      }
    }
  }
}

// The parts of a row joined: out = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i,
// summed over the maps by their weights where asked.  A workgroup takes 256
// features of a row; its waves take the parts in turn.
constexpr int kMergeWaves = 8;
template <typename TV>
__global__ __launch_bounds__(64 * kMergeWaves) void paged_merge_kernel(Params p) {
  __shared__ __attribute__((aligned(16))) float sums[kMergeWaves][256];
  const PagedAttentionArgs& a = p.a;
  const int S = a.S, D = a.cache.D;
  const int64_t rows = a.tokens.N * S;
  const int64_t n = a.mix ? blockIdx.x : blockIdx.x / S;
  const int s0 = a.mix ? 0 : static_cast<int>(blockIdx.x % S), s1 = a.mix ? S : s0 + 1;
  const int lane = lane_id(), wave = uniform_wave();
  const int d = static_cast<int>(blockIdx.y) * 256 + lane * 4;
  const bool owned = n >= a.tokens.offsets[0] && n < a.tokens.offsets[a.tokens.B];
  f32x4 total = zero4();
  for (int s = s0; s < s1; ++s) {
    const int64_t row = n * S + s;
    float m = -INFINITY;
    if (owned)
      for (int i = lane; i < p.n_split; i += 64)
        if (p.part_l[i * rows + row] != 0.f) m = fmaxf(m, p.part_m[i * rows + row]);
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
    float l = 0.f;
    f32x4 o = zero4();
    if (owned) {
      for (int i = lane; i < p.n_split; i += 64) {
        const float li = p.part_l[i * rows + row];
        if (li != 0.f) l += li * __builtin_amdgcn_exp2f(p.part_m[i * rows + row] - m);
      }
#pragma unroll 4
      for (int i = wave; i < p.n_split; i += kMergeWaves) {
        // A part that saw nothing has written nothing.
        const float li = p.part_l[i * rows + row], mi = p.part_m[i * rows + row];
        f32x4 v = zero4();
        if (li != 0.f && d < D) v = *reinterpret_cast<const f32x4*>(p.part_o + (i * rows + row) * D + d);
        o += v * (li != 0.f ? __builtin_amdgcn_exp2f(mi - m) : 0.f);
      }
    }
    l = wave_sum(l);
    if (a.lse2 && blockIdx.y == 0 && threadIdx.x == 0) a.lse2[row] = l == 0.f ? -INFINITY : m + __builtin_amdgcn_logf(l);
    total += o * (l == 0.f ? 0.f : (a.mix ? a.mix[s] : 1.f) / l);
  }
  *reinterpret_cast<f32x4*>(&sums[wave][lane * 4]) = total;
  __syncthreads();
  const int t = static_cast<int>(threadIdx.x);
  if (t < 256) {
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < kMergeWaves; ++w) v += sums[w][t];
    const int64_t at = (a.mix ? n : n * S + s0) * D + static_cast<int64_t>(blockIdx.y) * 256 + t;
    if (static_cast<int>(blockIdx.y) * 256 + t < D) static_cast<TV*>(a.out)[at] = static_cast<TV>(v);
  }
}

// Attention weights of the cached tokens: a wave takes 32 tokens of a sequence,
// holds a map's keys in registers and goes through the new tokens, 16 at a
// time; S^T = K Q^T as above, p = 2^(score - lse2), summed over the columns.
template <typename TQ, int KS>
__global__ __launch_bounds__(64 * kWaves) void paged_weights_kernel(PagedAttentionArgs a) {
  typedef typename Elem<TQ>::v8 q8;
  const CacheView& cache = a.cache;
  const int lane = lane_id(), c = lane & 15, g = lane >> 4;
  const int kt = static_cast<int>(blockIdx.x) * kWaves + uniform_wave(), b = static_cast<int>(blockIdx.y);
  if (kt * 32 >= a.capacity) return;
  const Sequence seq = sequence_of(a.tokens, cache, b);
  const int S = a.S, W = cache.W, RP = a.RP;
  f32x4 sum[2] = {zero4(), zero4()};
  const int page = kt * 32 < seq.cached ? page_of(cache, b, kt) : -1;
  if (page >= 0) {
    const TQ* kb = static_cast<const TQ*>(cache.keys) + page * cache.key_page +
                   (static_cast<int64_t>(kt % cache.tiles) * 32 + 8 * (c >> 2) + (c & 3)) * W + 8 * g;
    for (int s = 0; s < S; ++s) {
      const int from = s / a.repeat * RP;
      q8 kf[KS][2];
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        kf[k][0] = load8(kb + from + min(32 * k, RP - 32));
        kf[k][1] = load8(kb + from + min(32 * k, RP - 32) + 4 * W);
      }
      const float sc = score_scale(a, s);
      // The first new token that sees one of these tokens.
      const int first = a.causal ? max(0, kt * 32 - (seq.length - seq.rows)) / 16 : 0;
      for (int i0 = first * 16; i0 < seq.rows; i0 += 16) {
        const int i = min(i0 + c, seq.rows - 1);
        const TQ* qb = static_cast<const TQ*>(a.q) + (seq.n0 + i) * a.ldq + from + 8 * g;
        f32x4 st[2] = {zero4(), zero4()};
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          if (32 * k >= RP) break;
          const q8 qv = load8(qb + 32 * k);
          st[0] = Elem<TQ>::mma(kf[k][0], qv, st[0]);
          st[1] = Elem<TQ>::mma(kf[k][1], qv, st[1]);
        }
        const int vis = i0 + c < seq.rows ? visible_to(seq, i, a.causal) : 0;
        const float lse2 = a.lse2[(seq.n0 + i) * S + s];
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            if (kt * 32 + 8 * g + 4 * h + e < vis) sum[h][e] += __builtin_amdgcn_exp2f(st[h][e] * sc - lse2);
      }
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
#pragma unroll
      for (int x = 8; x >= 1; x >>= 1) sum[h][e] += __shfl_xor(sum[h][e], x);
      const int t = kt * 32 + 8 * g + 4 * h + e;
      if (c == 0 && t < a.capacity) {
        const float before = a.weights_in && t < seq.length - seq.rows && t < seq.cached ? a.weights_in[b * a.ld_weights + t] : 0.f;
        a.weights_out[b * a.ld_weights + t] = t < seq.cached ? before + sum[h][e] : 0.f;
      }
    }
}

namespace {

struct Plan {
  int n_ct, n_slices, db, n_split;
  bool parts;
};

Plan plan(const PagedAttentionArgs& a) {
  Plan r;
  const int64_t cols = static_cast<int64_t>(std::max(a.max_chunk, 1)) * a.S;
  r.n_slices = (a.cache.D + 511) / 512;
  r.n_ct = static_cast<int>(std::min<int64_t>((cols + 15) / 16, std::max(1, (1 << 20) / (a.tokens.B * r.n_slices))));
  r.db = static_cast<int>(round_up((a.cache.D + r.n_slices - 1) / r.n_slices, 64) / 16);
  // Workgroups for four rounds of the chip, each wave at least one tile.
  const int64_t tiles = (std::max(a.max_length, 1) + 31) / 32;
  const int64_t wgs = static_cast<int64_t>(a.tokens.B) * r.n_ct * r.n_slices;
  int64_t split = std::min<int64_t>((1024 + wgs - 1) / wgs, (tiles + kWaves - 1) / kWaves);
  r.n_split = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(split, kMaxSplits)));
  r.parts = r.n_split > 1 || a.mix != nullptr;
  return r;
}

template <typename TQ, typename TV, int DB>
void launch_token(const Params& p, hipStream_t stream) {
  const int steps = (p.a.cache.W + 32 * kKeyChunk - 1) / (32 * kKeyChunk);
  const size_t q_bytes = static_cast<size_t>(16) * (steps * 32 * kKeyChunk + 8) * 2;
  const size_t lds = std::max(q_bytes, static_cast<size_t>(16) * (16 * DB + 4) * 4) + 2 * kWaves * 16 * 4;
  const unsigned units = static_cast<unsigned>(round_up(p.units, kXcds));
  hipLaunchKernelGGL((paged_token_kernel<TQ, TV, DB>), dim3(units * p.n_ct * p.n_slices), dim3(64 * kWaves), lds, stream, p);
}

template <typename TQ, typename TV>
void launch_typed(const Params& p, int db, hipStream_t stream) {
  switch (db) {
    case 4: launch_token<TQ, TV, 4>(p, stream); break;
    case 8: launch_token<TQ, TV, 8>(p, stream); break;
    case 12: launch_token<TQ, TV, 12>(p, stream); break;
    case 16: launch_token<TQ, TV, 16>(p, stream); break;
    case 20: launch_token<TQ, TV, 20>(p, stream); break;
    case 24: launch_token<TQ, TV, 24>(p, stream); break;
    case 28: launch_token<TQ, TV, 28>(p, stream); break;
    default: launch_token<TQ, TV, 32>(p, stream); break;
  }
  if (p.part_o) {
    const dim3 grid(static_cast<unsigned>(p.a.tokens.N * (p.a.mix ? 1 : p.a.S)), static_cast<unsigned>((p.a.cache.D + 255) / 256));
    hipLaunchKernelGGL((paged_merge_kernel<TV>), grid, dim3(64 * kMergeWaves), 0, stream, p);
  }
}

}  // namespace

int64_t paged_attention_workspace(const PagedAttentionArgs& a) {
  const Plan r = plan(a);
  return r.parts ? r.n_split * a.tokens.N * a.S * (static_cast<int64_t>(a.cache.D) + 2) * 4 : 0;
}

void launch_paged_attention(const PagedAttentionArgs& a, void* workspace, hipStream_t stream) {
  const Plan r = plan(a);
  Params p{a, r.n_ct, r.n_slices, r.n_split, a.tokens.B * r.n_split, nullptr, nullptr, nullptr};
  if (r.parts) {
    const int64_t rows = r.n_split * a.tokens.N * a.S;
    p.part_o = static_cast<float*>(workspace);
    p.part_m = p.part_o + rows * a.cache.D;
    p.part_l = p.part_m + rows;
  }
  if (a.qk_dtype == kBF16) launch_typed<__bf16, __bf16>(p, r.db, stream);
  else if (a.v_dtype == kBF16) launch_typed<_Float16, __bf16>(p, r.db, stream);
  else launch_typed<_Float16, _Float16>(p, r.db, stream);
}

template <typename TQ>
static void launch_weights_typed(const PagedAttentionArgs& a, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(((a.capacity + 31) / 32 + kWaves - 1) / kWaves), static_cast<unsigned>(a.tokens.B));
  const dim3 block(64 * kWaves);
  if (a.RP <= 128) hipLaunchKernelGGL((paged_weights_kernel<TQ, 4>), grid, block, 0, stream, a);
  else if (a.RP <= 256) hipLaunchKernelGGL((paged_weights_kernel<TQ, 8>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((paged_weights_kernel<TQ, 16>), grid, block, 0, stream, a);
}

void launch_paged_weights(const PagedAttentionArgs& a, hipStream_t stream) {
  if (a.qk_dtype == kBF16) launch_weights_typed<__bf16>(a, stream);
  else launch_weights_typed<_Float16>(a, stream);
}

}  // namespace da
