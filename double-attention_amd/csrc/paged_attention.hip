// Attention of new tokens over a paged cache:
//   out[n, s] = sum_j softmax_j(gamma_s q_{n,s} . k_{j,s}) v_j
// over the tokens j of row n's sequence up to its own position, for each score
// map s; all maps share the values.
//
// Both kernels take 32 cached tokens (a tile) at a time,
//   S^T[token, column] = K Q^T     (keys straight from memory, queries in LDS)
//   O^T[feature, column] += V^T P^T (values straight from memory: their tiles
//                                    hold a feature's tokens side by side, so a
//                                    wave's load is one contiguous KiB)
// with the running maximum and sum of each column in 32 bits.  The key rows go
// to the MFMA's rows in such an order that the score accumulators are the next
// product's operand as they stand (da_common.h).  A sequence's tokens are split
// over workgroups where there are few columns; paged_merge_kernel joins the parts.
//
// Columns are 16 to a tile.  paged_token_kernel, for few new tokens: a sequence's
// (new token, map) pairs, tokens outermost.  A tile's queries are laid over all
// W key features, zero outside of their map's: one product K Q^T then serves
// every map, and keys and values are read once for all maps.  paged_chunk_kernel,
// for many: one map's tokens, with that map's features alone.
#include <algorithm>
#include <type_traits>

#include "da_common.h"
#include "da_launch.h"
#include "da_serving.h"
#include "da_tile.h"

namespace da {

namespace {

constexpr int kWaves = 4;
constexpr int kTokenGroups = 4;       // of 64 key features, at a time
constexpr int kMaxSplits = 256;
constexpr int kWantWorkgroups = 1024, kChunkWorkgroups = 256;
constexpr float kNoScore = -3.0e38f;  // the running reference before the first score

// A running reference is a whole number (log2); it moves where a score exceeds it
// by more than SLACK, to BELOW under that rounded up.  Probabilities beside it are
// rounded to the values' type, relative to their size in bf16, but by up to 2^-25 in
// fp16, below 2^-14: there the reference stays low, so that the largest ones are
// between 2^6 and 2^15.  At BELOW 0, 131072 tokens of 2^-25.1 beside one of 1 were all
// lost (0.4% of the sum); now what the rounding adds up to is below 2^-31 a token.
template <typename TV>
struct Reference {
  static constexpr bool wide = std::is_same<TV, __bf16>::value;
  static constexpr float BELOW = wide ? 0.f : 7.f, SLACK = wide ? kRescaleSlack : 15.f;
};

// Division of numbers below 2^23 by a divisor up to 2^16, by a product (the
// quotient of n and d is the whole part of n m / 2^40 with m = ceil(2^40 / d):
// the excess n (m d - 2^40) / (2^40 d) stays below 1 / d).
struct Divisor {
  uint32_t d;
  uint64_t m;
  Divisor() = default;
  explicit Divisor(int64_t n) : d(static_cast<uint32_t>(n)), m(((uint64_t{1} << 40) + d - 1) / d) {}
  __device__ __forceinline__ uint32_t divide(uint32_t n) const { return static_cast<uint32_t>(n * m >> 40); }
  __device__ __forceinline__ uint32_t remainder(uint32_t n) const { return n - divide(n) * d; }
};

struct Params {
  PagedAttentionArgs a;
  int n_ct;        // column tiles a workgroup index stands for (a stride, not a bound)
  int n_split;     // parts of a sequence's tokens
  int per;         // tiles of a part (the last one takes what is left)
  int units;       // B * n_split
  int64_t rows;    // N * S
  Divisor members; // workgroups of a unit
  Divisor sequences, slices, maps, repeats;
  float* part_o;   // [n_split][rows][D], or nullptr: rows are finished here
  float* part_m;   // [n_split][rows]
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
// b is the same in all lanes.
__device__ __forceinline__ Sequence sequence_of(const NewTokens& t, const CacheView& c, int b) {
  Sequence s;
  const int64_t first = min(max(static_cast<int64_t>(load_constant(t.offsets + b)), int64_t{0}), t.N);
  const int64_t last = min(max(static_cast<int64_t>(load_constant(t.offsets + b + 1)), first), t.N);
  s.n0 = first;
  s.rows = static_cast<int>(last - first);
  s.length = max(load_constant(t.lengths + b), 0);
  s.cached = static_cast<int>(min(static_cast<int64_t>(s.length), static_cast<int64_t>(c.table_pages) * c.tiles * 32));
  return s;
}
// Tokens that new token i of the sequence sees.
__device__ __forceinline__ int visible_to(const Sequence& s, int i, bool causal) {
  return causal ? max(0, min(s.cached, s.length - s.rows + i + 1)) : s.cached;
}
__device__ __forceinline__ int tile_of(const CacheView& c, int kt) { return kt - entry_of(c, kt) * c.tiles; }
__device__ __forceinline__ float score_scale(const PagedAttentionArgs& a, int s) {
  return load_scalar(a.scales, a.scales_dtype, s) * a.scale_mult * kLog2e;
}

// A number that the compiler takes for a new one: what is worked out from it
// stays where it is used, and out of registers elsewhere.
__device__ __forceinline__ int opaque(int x) {
  asm volatile("" : "+v"(x));
  return x;
}

// Sixteen bytes at a uniform global address and a lane's offset.
typedef __attribute__((address_space(1))) const char* global_ptr;
__device__ __forceinline__ u32x4 load_at(const char* base, uint32_t lane_offset) {
  return *reinterpret_cast<__attribute__((address_space(1))) const u32x4*>((global_ptr)(base) + lane_offset);
}

// A product multiplies every token of a tile with every column, those that do
// not see the token with zero: there an infinity or a NaN among the values is
// taken out, and the features' first such tokens are kept in LDS (`first`, this
// lane's feature).  Columns that see one are NaN in that feature at the end.
constexpr int kNoToken = 0x7fffffff;
// Bit 15 of each half where that is an infinity or a NaN.
template <typename TV>
__device__ __forceinline__ uint32_t non_finite(uint32_t halves) {
  constexpr uint32_t exponents = std::is_same<TV, __bf16>::value ? 0x7f807f80u : 0x7c007c00u;
  constexpr uint32_t step = std::is_same<TV, __bf16>::value ? 0x00800080u : 0x04000400u;
  return ((halves & exponents) + step) & 0x80008000u;
}
// v: eight tokens of a feature from `token` on.  True where any lane had one.
template <typename TV>
__device__ __forceinline__ bool take_out(u32x4& v, int* first, int token) {
  uint32_t any = 0;
#pragma unroll
  for (int e = 0; e < 4; ++e) any |= non_finite<TV>(v[e]);
  if (__ballot(any != 0) == 0) return false;
  int at = kNoToken;
#pragma unroll
  for (int e = 3; e >= 0; --e) {
    const uint32_t bits = non_finite<TV>(v[e]);
    if (bits >> 31) at = token + 2 * e + 1;
    if (bits & 0x8000u) at = token + 2 * e;
    v[e] &= ~((bits >> 15) * 0xffffu);
  }
  if (at != kNoToken) atomicMin(first, at);
  return true;
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

// NK: groups of 64 key features that a wave holds (fewer features leave the rest
// zero, more are taken in turn: eight groups at once spill with 512 value
// features, and 32 sequences of up to 4096 tokens with 512 key features take 71 us
// instead of 58); DBW: 16-feature blocks of the values of a wave.  The 16 columns
// are (token, map) pairs over all features.
//
// A step takes four tiles.  Wave w forms tile w's scores and leaves its
// probabilities in LDS; after a barrier every wave multiplies them with its own
// DBW blocks of the values of all tiles.  A wave's next keys and the next two
// tiles' values are on their way meanwhile, and the probabilities have two buffers,
// so that a step has one barrier.
//
// Bound by the cache's bytes: 64 sequences of up to 4096 tokens (keys of 256, values of
// 512 features, 254 MB) 54 us with the merge, one of 131072 tokens (201 MB) 42 us.
// Waves that held whole tiles, each with all features, had a register file too
// small for their loads in flight: 85 us for the former.
template <typename TQ, typename TV, int DBW>
__global__ __launch_bounds__(64 * kWaves, 2) void paged_token_kernel(Params p) {
  typedef typename Elem<TQ>::v8 q8;
  typedef typename Elem<TV>::v8 v8;
  constexpr int NW = kWaves, NK = kTokenGroups;
  constexpr int DS = 16 * DBW * NW;
  constexpr int FW = 64 * NK;               // features of a pass
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const PagedAttentionArgs& a = p.a;
  const CacheView& cache = a.cache;
  const int wave = uniform_wave();
  const int W = cache.W, D = cache.D;

  // Workgroups are dealt to the XCDs in turn.  Those that read the same tokens
  // (a unit's column tiles, maps and slices) go to one, for its L2.  All
  // sequences' first parts come first, so that the parts that have tiles are
  // dealt evenly.
  const uint32_t wg = blockIdx.x;
  if (p.part_o == nullptr) clear_other_rows<TV>(a, wg, gridDim.x);
  const uint32_t round = p.members.divide(wg / kXcds);
  const int unit = static_cast<int>(round * kXcds + wg % kXcds);
  if (unit >= p.units) return;
  int member = static_cast<int>(wg / kXcds - round * p.members.d);
  const int split = static_cast<int>(p.sequences.divide(unit)), b = unit - split * a.tokens.B;
  const Sequence seq = sequence_of(a.tokens, cache, b);
  if (seq.rows == 0) return;
  const int slice = static_cast<int>(p.slices.remainder(member));
  member = static_cast<int>(p.slices.divide(member));
  const int n_cols = seq.rows * a.S;
  const int passes = (W + FW - 1) / FW;
  const int QP = passes * FW + 8;           // pitch of the queries in LDS
  const int d0 = slice * DS + wave * DBW * 16;
  const int nb = max(0, min(DBW, (D - d0) / 16));   // blocks of this wave (the last slice may have fewer)

  TQ* qs = reinterpret_cast<TQ*>(lds);
  char* ps = lds + 32 * QP;                           // [2][NW][64 lanes] 16 bytes
  float* ms = reinterpret_cast<float*>(ps + 2 * NW * 1024); // [2][NW][16]
  int* moved = reinterpret_cast<int*>(ms + 2 * NW * 16);    // [2][NW]
  int* firsts = moved + 2 * NW + wave * DBW * 16;           // [NW][DBW][16], this wave's features

  for (int ct0 = member; ct0 * 16 < n_cols; ct0 += p.n_ct) {
    // Nearly always the only round: what depends on the lane is worked out in it,
    // rather than in front of it and kept in registers that there are not.
    const int tid = opaque(static_cast<int>(threadIdx.x));
    const int lane = tid & 63, c = lane & 15, g = lane >> 4;
    const int col0 = ct0 * 16, n_used = min(16, n_cols - col0);
    auto token_of = [&](int col) { return static_cast<int>(p.maps.divide(col)); };
    auto map_of = [&](int col) { return static_cast<int>(p.maps.remainder(col)); };
    const int64_t row0 = seq.n0 * a.S + col0;
    const int limit = visible_to(seq, token_of(col0 + n_used - 1), a.causal), all_see = visible_to(seq, token_of(col0), a.causal);
    const int n_kt = (limit + 31) / 32;
    const int kt0 = min(n_kt, split * p.per), kt1 = split == p.n_split - 1 ? n_kt : min(n_kt, kt0 + p.per);
    if (split > 0 && kt0 == kt1) {   // nothing left for this part
      if (slice == 0)
        for (int i = tid; i < n_used; i += 64 * NW) p.part_l[split * p.rows + row0 + i] = 0.f;
      continue;
    }

    // A tile's page is in the lane of its place in the step: the next two steps'
    // are on their way.
    auto pages_at = [&](int base) { return lane < NW && base + lane < kt1 ? page_of(cache, b, base + lane) : -1; };
    int pages = pages_at(kt0), pages_next = pages_at(kt0 + NW);

    // Queries: sixteen threads to a column.
    if (ct0 != member) lds_barrier();   // the last tiles' have been read
    for (int col = tid >> 4; col < 16; col += 4 * NW) {
      const bool used = col < n_used;
      const int from = static_cast<int>(p.repeats.divide(map_of(col0 + col))) * a.RP;
      const TQ* src = static_cast<const TQ*>(a.q) + (seq.n0 + token_of(col0 + (used ? col : 0))) * a.ldq;
      for (int f = (tid & 15) * 8; f < passes * FW; f += 128) {
        u32x4 v = {0, 0, 0, 0};
        if (used && f >= from && f < from + a.RP) v = load16B(src + f);
        store16B(qs + col * QP + f, v);
      }
    }
    // This lane's column; those behind the last one count as it.
    const int own_col = col0 + min(c, n_used - 1);
    const int vis = visible_to(seq, token_of(own_col), a.causal);
    const float sc = score_scale(a, map_of(own_col));
    float m_run = kNoScore, l_part = 0.f;
    for (int i = lane; i < DBW * 16; i += 64) firsts[i] = kNoToken;
    bool taken = false;   // some value was taken out

    // Addresses are a uniform base and a lane's 32-bit offset.  Block h of the
    // scores has token 8 (c / 4) + 4 h + c % 4 in row c.  Where there is no tile
    // or page every lane reads one place, and nothing uses it.
    const uint32_t key_lane = static_cast<uint32_t>(((8 * (c >> 2) + (c & 3)) * W + 8 * g) * 2);
    const uint32_t value_lane = static_cast<uint32_t>((32 * c + 8 * g) * 2);
    u32x4 kf[NK][4], vf[2][DBW];
    auto load_keys = [&](int kt, int page, int pass) {
      const char* base = uniform_ptr(static_cast<const char*>(cache.keys) +
                                     (max(page, 0) * cache.key_page + static_cast<int64_t>(tile_of(cache, kt)) * 32 * W) * 2);
      const uint32_t at = page < 0 ? 0 : key_lane;
#pragma unroll
      for (int j = 0; j < NK; ++j) {   // a group past the last feature is multiplied by zero
        const char* from = base + 128 * min(pass * NK + j, W / 64 - 1);
#pragma unroll
        for (int i = 0; i < 4; ++i) kf[j][i] = load_at(from + (i & 1) * 8 * W, at + 64 * (i >> 1));
      }
    };
    auto load_values = [&](u32x4 (&v)[DBW], int kt, int page) {
      const char* base = uniform_ptr(static_cast<const char*>(cache.values) +
                                     (max(page, 0) * cache.value_page + (static_cast<int64_t>(tile_of(cache, kt)) * D + (nb > 0 ? d0 : 0)) * 32) * 2);
      const uint32_t at = page < 0 ? 0 : value_lane;
#pragma unroll
      for (int i = 0; i < DBW; ++i) v[i] = load_at(base + 1024 * max(0, min(i, nb - 1)), at);
    };
    load_keys(kt0 + wave, __builtin_amdgcn_readlane(pages, wave), 0);
    load_values(vf[0], kt0, __builtin_amdgcn_readlane(pages, 0));
    load_values(vf[1], kt0 + 1, __builtin_amdgcn_readlane(pages, 1));
    f32x4 acc[DBW];
#pragma unroll
    for (int j = 0; j < DBW; ++j) acc[j] = zero4();
    __builtin_amdgcn_sched_barrier(0);
    lds_barrier();   // the queries are there

    int buf = 0;
    for (int base = kt0; base < kt1; base += NW) {
      const int pages_after = pages_at(base + 2 * NW);
      const int kt = base + wave, page = __builtin_amdgcn_readlane(pages, wave);
      const int live = page < 0 ? 0 : min(32, limit - kt * 32);
      char* mine = ps + (buf * NW + wave) * 1024 + lane * 16;
      bool any = false;
      // Scores of this wave's tile, and its probabilities.
      f32x4 st[2] = {zero4(), zero4()};
      auto scores = [&](int pass) {
#pragma unroll
        for (int j = 0; j < 2 * NK; ++j) {
          const q8 qf = load8(qs + c * QP + pass * FW + 32 * j + 8 * g);
          st[0] = Elem<TQ>::mma(__builtin_bit_cast(q8, kf[j >> 1][2 * (j & 1)]), qf, st[0]);
          st[1] = Elem<TQ>::mma(__builtin_bit_cast(q8, kf[j >> 1][2 * (j & 1) + 1]), qf, st[1]);
        }
      };
      scores(0);
      for (int pass = 1; pass < passes; ++pass) {
        load_keys(kt, page, pass);
        scores(pass);
      }
      const int seen = min(live, vis - kt * 32) - 8 * g;   // of this lane's eight tokens
      float mx, sum;
      auto scaled = [&] {
        mx = -INFINITY;
        sum = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const float s = e < seen ? st[e >> 2][e & 3] * sc : -INFINITY;
          st[e >> 2][e & 3] = s;
          mx = fmaxf(mx, s);
          sum += s;
        }
      };
      scaled();
      if (__ballot(sum != sum)) {
        // An infinity or a NaN among another map's features makes a score NaN, times
        // this map's zeros there: each map's features alone, and each lane's own sum.
        const char* base = uniform_ptr(static_cast<const char*>(cache.keys) +
                                       (max(page, 0) * cache.key_page + static_cast<int64_t>(tile_of(cache, kt)) * 32 * W) * 2);
        const int c = opaque(tid) & 15, g = (opaque(tid) & 63) >> 4;
        const int own = static_cast<int>(p.repeats.divide(map_of(col0 + min(c, n_used - 1))));
        f32x4 mine[2] = {zero4(), zero4()};
#pragma nounroll
        for (int r = 0; r < a.S / a.repeat; ++r) {
          f32x4 part[2] = {zero4(), zero4()};
#pragma nounroll
          for (int f = r * a.RP; f < (r + 1) * a.RP; f += 32) {
            const q8 qf = load8(qs + c * QP + f + 8 * g);
#pragma unroll
            for (int h = 0; h < 2; ++h) part[h] = Elem<TQ>::mma(__builtin_bit_cast(q8, load_at(base + 2 * f + h * 8 * W, key_lane)), qf, part[h]);
          }
          if (r == own) {
            mine[0] = part[0];
            mine[1] = part[1];
          }
        }
        st[0] = mine[0];
        st[1] = mine[1];
        scaled();
      }
      // What a moving reference scales stays exact (but for fp16 probabilities that
      // fall below 2^-14).
      float m = m_run;
      if (__ballot(mx > m + Reference<TV>::SLACK)) {
        const float tile_max = group_max(mx);
        if (tile_max > m + Reference<TV>::SLACK) m = __builtin_ceilf(tile_max) - Reference<TV>::BELOW;
        any = true;
      }
      float l = 0.f;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const float s = __builtin_amdgcn_exp2f(st[e >> 2][e & 3] - m);
        st[e >> 2][e & 3] = s;
        l += s;
      }
      if (any) l_part *= __builtin_amdgcn_exp2f(m_run - m);
      l_part += l;
      // The probabilities are rounded to the values' type for the product, the
      // sum is of the unrounded ones.
      *reinterpret_cast<v8*>(mine) = pack_blocked<TV>(st[0], st[1]);
      ms[(buf * NW + wave) * 16 + c] = m;
      if (lane == 0) moved[buf * NW + wave] = any;
      __builtin_amdgcn_sched_barrier(0);
      load_keys(kt + NW, __builtin_amdgcn_readlane(pages_next, wave), 0);
      __builtin_amdgcn_sched_barrier(0);
      lds_barrier();
      int moves = 0;
#pragma unroll
      for (int w = 0; w < NW; ++w) moves |= moved[buf * NW + w];
      if (__builtin_amdgcn_readfirstlane(moves)) {
        // To the largest of the waves' references: this wave's probabilities and
        // sums, and what has been added up.
        const float own = ms[(buf * NW + wave) * 16 + c];
        float m = own;
#pragma unroll
        for (int w = 0; w < NW; ++w) m = fmaxf(m, ms[(buf * NW + w) * 16 + c]);
        const float f = __builtin_amdgcn_exp2f(own - m), fa = __builtin_amdgcn_exp2f(m_run - m);
        m_run = m;
        l_part *= f;
#pragma unroll
        for (int j = 0; j < DBW; ++j) acc[j] *= fa;
        v8 pv = *reinterpret_cast<const v8*>(mine);
#pragma unroll
        for (int e = 0; e < 8; ++e) pv[e] = static_cast<TV>(static_cast<float>(pv[e]) * f);
        *reinterpret_cast<v8*>(mine) = pv;
        lds_barrier();
      }
      const char* probs = ps + buf * NW * 1024 + lane * 16;
#pragma unroll
      for (int t = 0; t < NW; ++t) {
        const int page_t = __builtin_amdgcn_readlane(pages, t), at = (base + t) * 32;
        v8 vv[DBW];
        if (page_t >= 0 && at + 32 <= all_see) {
#pragma unroll
          for (int j = 0; j < DBW; ++j) vv[j] = __builtin_bit_cast(v8, vf[t & 1][j]);
        } else {   // what lies behind the last token is not multiplied: it may hold anything
          const int live_t = page_t < 0 ? 0 : min(32, limit - at);
          const int c = opaque(tid) & 15, g = (opaque(tid) & 63) >> 4;
          u32x4 keep;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            keep[e] = (8 * g + 2 * e < live_t ? 0xffffu : 0u) | (8 * g + 2 * e + 1 < live_t ? 0xffff0000u : 0u);
#pragma unroll
          for (int j = 0; j < DBW; ++j) {
            u32x4 v = vf[t & 1][j] & keep;
            if (at + live_t > all_see) taken |= take_out<TV>(v, firsts + 16 * j + c, at + 8 * g);
            vv[j] = __builtin_bit_cast(v8, v);
          }
        }
        const v8 pv = *reinterpret_cast<const v8*>(probs + t * 1024);
#pragma unroll
        for (int j = 0; j < DBW; ++j) acc[j] = Elem<TV>::mma(vv[j], pv, acc[j]);
        const int next = t + 2 < NW ? __builtin_amdgcn_readlane(pages, t + 2 < NW ? t + 2 : 0)
                                    : __builtin_amdgcn_readlane(pages_next, t + 2 < NW ? 0 : t + 2 - NW);
        load_values(vf[t & 1], base + t + 2, next);
        __builtin_amdgcn_sched_barrier(0);
      }
      pages = pages_next;
      pages_next = pages_after;
      buf ^= 1;
    }

    // The waves' sums of exponentials; the rest of a column is in one wave.
    float* ls = reinterpret_cast<float*>(ps);
    lds_barrier();   // the probabilities have been read
    l_part = group_sum(l_part);
    if (g == 0) ls[wave * 16 + c] = l_part;
    lds_barrier();
    if (c >= n_used) continue;
    float l = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) l += ls[w * 16 + c];
    const int64_t row = row0 + c;
    if (taken) {
#pragma unroll
      for (int j = 0; j < DBW; ++j)
#pragma unroll
        for (int e = 0; e < 4; ++e)
          if (vis > firsts[16 * j + 4 * g + e]) acc[j][e] = __builtin_nanf("");
    }
    if (wave == 0 && g == 0 && slice == 0) {
      if (p.part_o) {
        p.part_m[split * p.rows + row] = m_run;
        p.part_l[split * p.rows + row] = l;
      } else if (a.lse2) {
        a.lse2[row] = l == 0.f ? -INFINITY : m_run + __builtin_amdgcn_logf(l);
      }
    }
    if (p.part_o) {
      float* to = p.part_o + (split * p.rows + row) * D + d0 + 4 * g;
#pragma unroll
      for (int j = 0; j < DBW; ++j)
        if (j < nb) *reinterpret_cast<f32x4*>(to + 16 * j) = acc[j];
    } else {
      const float f = l == 0.f ? 0.f : 1.f / l;
      TV* to = static_cast<TV*>(a.out) + row * D + d0 + 4 * g;
#pragma unroll
      for (int j = 0; j < DBW; ++j) {
        typename Elem<TV>::v4 r;
#pragma unroll
        for (int e = 0; e < 4; ++e) r[e] = static_cast<TV>(acc[j][e] * f);
        if (j < nb) *reinterpret_cast<typename Elem<TV>::v4*>(to + 16 * j) = r;
      }
    }
  }
}

// Many new tokens.  A workgroup of eight waves takes 16 CT tokens of one map;
// a step takes four tiles.  Wave w forms the scores of half a tile (16 tokens)
// for all columns, with its keys in registers and the queries in LDS, and
// leaves its probabilities in LDS; after a barrier every wave multiplies them
// with its own DBW blocks of the values, straight from memory.
// Where a score exceeds the reference that all waves share by too much a wave
// raises its own, and the waves agree on the largest behind the barrier.
constexpr int kChunkWaves = 8, kChunkTiles = 4;
template <int NK, int CT>
struct ChunkLds {   // bytes
  static constexpr int REFS = 0;                                    // [16 CT] floats: the shared references
  static constexpr int SEES = 64 * CT;                              // [16 CT] ints: tokens that a column sees
  static constexpr int OWN = 2 * 64 * CT;                           // [waves][16 CT] floats: the waves' references
  static constexpr int MOVED = OWN + kChunkWaves * 64 * CT;         // [2][waves] ints
  static constexpr int QUERIES = MOVED + 2 * kChunkWaves * 4;       // [CT][2 NK][64 lanes] 16 bytes
  static constexpr int PROBS = QUERIES + 2 * NK * CT * 1024;        // [2][tiles][CT][64 lanes] 16 bytes
  static constexpr int FIRSTS = PROBS + 2 * kChunkTiles * CT * 1024; // [waves][4 blocks][16] ints: see take_out
  static constexpr int BYTES = FIRSTS + kChunkWaves * 4 * 64;
};

template <typename TQ, typename TV, int NK, int DBW, int CT>
__global__ __launch_bounds__(64 * kChunkWaves, 2) void paged_chunk_kernel(Params p) {
  typedef typename Elem<TQ>::v8 q8;
  typedef typename Elem<TV>::v8 v8;
  typedef typename Elem<TV>::v4 v4;
  typedef ChunkLds<NK, CT> Lds;
  constexpr int NW = kChunkWaves, TS = kChunkTiles;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const PagedAttentionArgs& a = p.a;
  const CacheView& cache = a.cache;
  const int wave = uniform_wave();
  const int W = cache.W, D = cache.D;

  // As above; members are slices, then maps, then column tiles.
  const uint32_t wg = blockIdx.x;
  if (p.part_o == nullptr) clear_other_rows<TV>(a, wg, gridDim.x);
  const uint32_t round = p.members.divide(wg / kXcds);
  const int unit = static_cast<int>(round * kXcds + wg % kXcds);
  if (unit >= p.units) return;
  int member = static_cast<int>(wg / kXcds - round * p.members.d);
  const int split = static_cast<int>(p.sequences.divide(unit)), b = unit - split * a.tokens.B;
  const Sequence seq = sequence_of(a.tokens, cache, b);
  const int slice = static_cast<int>(p.slices.remainder(member));
  member = static_cast<int>(p.slices.divide(member));
  const int map = static_cast<int>(p.maps.remainder(member)), f0 = static_cast<int>(p.repeats.divide(map)) * a.RP;
  member = static_cast<int>(p.maps.divide(member));
  const int d0 = (slice * NW + wave) * DBW * 16;
  const int nb = max(0, min(DBW, (D - d0) / 16));   // blocks of this wave (the last slice may have fewer)
  const int wt = wave >> 1, wh = wave & 1;          // this wave's tile of a step, and half of it
  const float sc = score_scale(a, map);

  float* refs = reinterpret_cast<float*>(lds + Lds::REFS);
  float* own = reinterpret_cast<float*>(lds + Lds::OWN) + wave * 16 * CT;
  int* sees = reinterpret_cast<int*>(lds + Lds::SEES);
  int* moved = reinterpret_cast<int*>(lds + Lds::MOVED);
  int* firsts = reinterpret_cast<int*>(lds + Lds::FIRSTS) + wave * DBW * 16;

  for (int ct0 = member; ct0 * 16 * CT < seq.rows; ct0 += p.n_ct) {
    const int tid = opaque(static_cast<int>(threadIdx.x));   // as above
    const int lane = tid & 63, c = lane & 15, g = lane >> 4;
    const q8* qs = reinterpret_cast<const q8*>(lds + Lds::QUERIES) + lane;
    const int col0 = ct0 * 16 * CT, n_used = min(16 * CT, seq.rows - col0);
    auto row_of = [&](int col) { return (seq.n0 + col0 + col) * a.S + map; };
    const int limit = visible_to(seq, col0 + n_used - 1, a.causal), all_see = visible_to(seq, col0, a.causal);
    const int n_kt = (limit + 31) / 32;
    const int kt0 = min(n_kt, split * p.per), kt1 = split == p.n_split - 1 ? n_kt : min(n_kt, kt0 + p.per);
    if (split > 0 && kt0 == kt1) {   // nothing left for this part
      if (slice == 0)
        for (int i = tid; i < n_used; i += 64 * NW) p.part_l[split * p.rows + row_of(i)] = 0.f;
      continue;
    }

    // A tile's page is in the lane of its place in the step.
    auto pages_at = [&](int base) { return lane < TS && base + lane < kt1 ? page_of(cache, b, base + lane) : -1; };
    int pages = pages_at(kt0), pages_next = pages_at(kt0 + TS);

    // Queries, as the fragments that the products read; zero behind the last
    // column and feature.  Thread t has the chunks t, t + 512, ... of the columns.
    if (ct0 != member) lds_barrier();   // the last tiles' have been read
    constexpr int CHUNKS = 8 * NK, COLS = 64 * NW / CHUNKS, LOADS = 16 * CT / COLS;
    const int q_col = tid / CHUNKS, q_f = tid % CHUNKS * 8;
    const uint32_t q_lane = static_cast<uint32_t>((q_col * static_cast<int>(a.ldq) + q_f) * 2);
    u32x4 qv[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const char* rows = uniform_ptr(static_cast<const char*>(a.q) + ((seq.n0 + col0 + min(i * COLS, n_used - 1)) * a.ldq + f0) * 2);
      const bool there = i * COLS + q_col < n_used && q_f < a.RP;
      qv[i] = load_at(rows, there ? q_lane : 0);
    }
    for (int i = tid; i < 16 * CT; i += 64 * NW) {
      sees[i] = visible_to(seq, col0 + min(i, n_used - 1), a.causal);
      refs[i] = kNoScore;
    }
    for (int i = lane; i < 16 * CT; i += 64) own[i] = kNoScore;
    for (int i = lane; i < 16 * DBW; i += 64) firsts[i] = kNoToken;
    bool taken = false;   // some value was taken out

    // Addresses as above.
    const uint32_t key_lane = static_cast<uint32_t>(((8 * (c >> 2) + 4 * wh + (c & 3)) * W + 8 * g) * 2);
    const uint32_t value_lane = static_cast<uint32_t>((32 * c + 8 * g) * 2);
    u32x4 kf[2 * NK], vf[2][DBW];
    auto load_keys = [&](int kt, int page) {
      const char* base = uniform_ptr(static_cast<const char*>(cache.keys) +
                                     (max(page, 0) * cache.key_page + static_cast<int64_t>(tile_of(cache, kt)) * 32 * W + f0) * 2);
      const uint32_t at = page < 0 ? 0 : key_lane;
#pragma unroll
      for (int j = 0; j < NK; ++j) {   // a group past the last feature is multiplied by zero
        const char* from = base + 128 * min(j, a.RP / 64 - 1);
        kf[2 * j] = load_at(from, at);
        kf[2 * j + 1] = load_at(from, at + 64);
      }
    };
    auto load_values = [&](u32x4 (&v)[DBW], int kt, int page) {
      const char* base = uniform_ptr(static_cast<const char*>(cache.values) +
                                     (max(page, 0) * cache.value_page + (static_cast<int64_t>(tile_of(cache, kt)) * D + (nb > 0 ? d0 : 0)) * 32) * 2);
      const uint32_t at = page < 0 ? 0 : value_lane;
#pragma unroll
      for (int i = 0; i < DBW; ++i) v[i] = load_at(base + 1024 * max(0, min(i, nb - 1)), at);
    };
    load_keys(kt0 + wt, __builtin_amdgcn_readlane(pages, wt));
    load_values(vf[0], kt0, __builtin_amdgcn_readlane(pages, 0));
    load_values(vf[1], kt0 + 1, __builtin_amdgcn_readlane(pages, 1));
#pragma unroll
    for (int i = 0; i < LOADS; ++i) {
      const int col = i * COLS + q_col;
      if (col >= n_used || q_f >= a.RP) qv[i] = u32x4{0, 0, 0, 0};
      store16B(lds + Lds::QUERIES + ((col / 16 * 2 * NK + q_f / 32) * 64 + q_f % 32 * 2 + col % 16) * 16, qv[i]);
    }
    f32x4 acc[CT][DBW];
    float l_part[CT];   // sums of this lane's probabilities
#pragma unroll
    for (int i = 0; i < CT; ++i)
#pragma unroll
      for (int j = 0; j < DBW; ++j) acc[i][j] = zero4();
#pragma unroll
    for (int i = 0; i < CT; ++i) l_part[i] = 0.f;
    __builtin_amdgcn_sched_barrier(0);
    lds_barrier();   // the queries are there

    int buf = 0;
    for (int base = kt0; base < kt1; base += TS) {
      const int pages_after = pages_at(base + 2 * TS);
      const int kt = base + wt, page = __builtin_amdgcn_readlane(pages, wt);
      const int live = page < 0 ? 0 : min(32, limit - kt * 32);
      char* mine = lds + Lds::PROBS + (buf * TS + wt) * CT * 1024 + lane * 16 + 8 * wh;
      bool raises = false;
      // Probabilities of column tiles i and i + 1 for this wave's tokens.
      auto probabilities = [&](int i, auto masked) {
        constexpr int PAIR = 2, READS = PAIR * 2 * NK, AHEAD = 4;
        f32x4 st[PAIR];
#pragma unroll
        for (int u = 0; u < PAIR; ++u) st[u] = zero4();
#pragma unroll
        for (int j = 0; j < 2 * NK; ++j)
#pragma unroll
          for (int u = 0; u < PAIR; ++u)
            st[u] = Elem<TQ>::mma(__builtin_bit_cast(q8, kf[j]), qs[((i + u) * 2 * NK + j) * 64], st[u]);
        // Four fragments stay in flight ahead of their MFMAs (left to itself the
        // compiler reads one, waits, and multiplies).
        __builtin_amdgcn_sched_group_barrier(0x100, AHEAD, 0);
#pragma unroll
        for (int n = 0; n < READS - AHEAD; ++n) {
          __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, AHEAD, 0);
#pragma unroll
        for (int u = 0; u < PAIR; ++u) {
          const int col = 16 * (i + u) + c;
          float m = refs[col];
          const int seen = masked ? min(live, sees[col] - kt * 32) - (opaque(tid) & 48) / 2 - 4 * wh : 4;   // of this lane's four tokens
          f32x4 x;
#pragma unroll
          for (int e = 0; e < 4; ++e) x[e] = masked && e >= seen ? -INFINITY : st[u][e] * sc;
          const float mx = fmaxf(fmaxf(x[0], x[1]), fmaxf(x[2], x[3]));
          if (__ballot(mx > m + Reference<TV>::SLACK)) {   // as above
            const float before = m, most = group_max(mx);
            if (most > m + Reference<TV>::SLACK) m = __builtin_ceilf(most) - Reference<TV>::BELOW;
            own[col] = m;
            l_part[i + u] *= __builtin_amdgcn_exp2f(before - m);
            raises = true;
          }
          v4 pv;
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float v = __builtin_amdgcn_exp2f(x[e] - m);
            l_part[i + u] += v;
            pv[e] = static_cast<TV>(v);
          }
          *reinterpret_cast<v4*>(mine + (i + u) * 1024) = pv;
        }
        __builtin_amdgcn_sched_barrier(0);
      };
      constexpr std::true_type yes{};
      constexpr std::false_type no{};
      if (live == 32 && kt * 32 + 32 <= all_see) {
#pragma unroll
        for (int i = 0; i < CT; i += 2) probabilities(i, no);
      } else {
#pragma unroll
        for (int i = 0; i < CT; i += 2) probabilities(i, yes);
      }
      if (lane == 0) moved[buf * NW + wave] = raises;
      __builtin_amdgcn_sched_barrier(0);
      load_keys(kt + TS, __builtin_amdgcn_readlane(pages_next, wt));
      __builtin_amdgcn_sched_barrier(0);
      lds_barrier();
      int moves = 0;
#pragma unroll
      for (int w = 0; w < NW; ++w) moves |= moved[buf * NW + w];
      if (__builtin_amdgcn_readfirstlane(moves)) {
        // To the largest of the waves' references: this wave's probabilities, and
        // what has been added up.
        const int c = opaque(tid) & 15;
#pragma unroll
        for (int i = 0; i < CT; ++i) {
          const float* all = reinterpret_cast<const float*>(lds + Lds::OWN) + 16 * i + c;
          float m = all[0];
#pragma unroll
          for (int w = 1; w < NW; ++w) m = fmaxf(m, all[w * 16 * CT]);
          const float f = __builtin_amdgcn_exp2f(own[16 * i + c] - m), fa = __builtin_amdgcn_exp2f(refs[16 * i + c] - m);
          l_part[i] *= f;
#pragma unroll
          for (int j = 0; j < DBW; ++j) acc[i][j] *= fa;
          v4 pv = *reinterpret_cast<const v4*>(mine + i * 1024);
#pragma unroll
          for (int e = 0; e < 4; ++e) pv[e] = static_cast<TV>(static_cast<float>(pv[e]) * f);
          *reinterpret_cast<v4*>(mine + i * 1024) = pv;
          __builtin_amdgcn_sched_barrier(0);
        }
        lds_barrier();
        for (int i = tid; i < 16 * CT; i += 64 * NW) {
          float* all = reinterpret_cast<float*>(lds + Lds::OWN) + i;
          float m = all[0];
          for (int w = 1; w < NW; ++w) m = fmaxf(m, all[w * 16 * CT]);
          refs[i] = m;
          for (int w = 0; w < NW; ++w) all[w * 16 * CT] = m;
        }
        lds_barrier();
      }
      const char* probs = lds + Lds::PROBS + buf * TS * CT * 1024 + lane * 16;
#pragma unroll
      for (int t = 0; t < TS; ++t) {
        const int page_t = __builtin_amdgcn_readlane(pages, t);
        const int at = (base + t) * 32, live_t = page_t < 0 ? 0 : min(32, limit - at);
        u32x4(&v)[DBW] = vf[t & 1];
        if (live_t < 32) {   // what lies behind the last token is not multiplied: it may hold anything
          const int g = (opaque(tid) & 63) >> 4;
          u32x4 keep;
#pragma unroll
          for (int e = 0; e < 4; ++e)
            keep[e] = (8 * g + 2 * e < live_t ? 0xffffu : 0u) | (8 * g + 2 * e + 1 < live_t ? 0xffff0000u : 0u);
#pragma unroll
          for (int j = 0; j < DBW; ++j) v[j] &= keep;
        }
        if (live_t > 0 && at + live_t > all_see) {
          const int c = opaque(tid) & 15, g = (opaque(tid) & 63) >> 4;
#pragma unroll
          for (int j = 0; j < DBW; ++j) taken |= take_out<TV>(v[j], firsts + 16 * j + c, at + 8 * g);
        }
#pragma unroll
        for (int i = 0; i < CT; ++i) {
          const v8 pv = *reinterpret_cast<const v8*>(probs + (t * CT + i) * 1024);
#pragma unroll
          for (int j = 0; j < DBW; ++j) acc[i][j] = Elem<TV>::mma(__builtin_bit_cast(v8, v[j]), pv, acc[i][j]);
        }
        __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
#pragma unroll
        for (int i = 0; i < CT - 2; ++i) {
          __builtin_amdgcn_sched_group_barrier(0x008, DBW, 0);
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x008, 2 * DBW, 0);
        const int next = t + 2 < TS ? __builtin_amdgcn_readlane(pages, t + 2) : __builtin_amdgcn_readlane(pages_next, t + 2 - TS);
        load_values(v, base + t + 2, next);
        __builtin_amdgcn_sched_barrier(0);
      }
      pages = pages_next;
      pages_next = pages_after;
      buf ^= 1;
    }

    // The waves' sums of exponentials; the rest of a column is in one wave.
    float* ls = reinterpret_cast<float*>(lds + Lds::OWN);
    lds_barrier();
#pragma unroll
    for (int i = 0; i < CT; ++i) {
      const float l = group_sum(l_part[i]);
      if (g == 0) ls[wave * 16 * CT + 16 * i + c] = l;
    }
    lds_barrier();
#pragma unroll
    for (int i = 0; i < CT; ++i) {
      const int col = 16 * i + c;
      float l = 0.f;
#pragma unroll
      for (int w = 0; w < NW; ++w) l += ls[w * 16 * CT + col];
      const float m = refs[col];
      const int64_t row = row_of(min(col, n_used - 1));
      if (taken) {
#pragma unroll
        for (int j = 0; j < DBW; ++j)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            acc[i][j][e] = sees[col] > firsts[16 * j + 4 * g + e] ? __builtin_nanf("") : acc[i][j][e];
      }
      if (wave == 0 && g == 0 && slice == 0 && col < n_used) {
        if (p.part_o) {
          p.part_m[split * p.rows + row] = m;
          p.part_l[split * p.rows + row] = l;
        } else if (a.lse2) {
          a.lse2[row] = l == 0.f ? -INFINITY : m + __builtin_amdgcn_logf(l);
        }
      }
      if (p.part_o) {
        float* to = p.part_o + (split * p.rows + row) * D + d0 + 4 * g;
#pragma unroll
        for (int j = 0; j < DBW; ++j)
          if (j < nb && col < n_used) *reinterpret_cast<f32x4*>(to + 16 * j) = acc[i][j];
      } else {
        const float f = l == 0.f ? 0.f : 1.f / l;
        TV* to = static_cast<TV*>(a.out) + row * D + d0 + 4 * g;
#pragma unroll
        for (int j = 0; j < DBW; ++j) {
          v4 r;
#pragma unroll
          for (int e = 0; e < 4; ++e) r[e] = static_cast<TV>(acc[i][j][e] * f);
          if (j < nb && col < n_used) *reinterpret_cast<v4*>(to + 16 * j) = r;
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
}

// The parts of a row joined: out = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i,
// summed over the maps by their weights where asked.  A workgroup takes 64
// features of a row; a wave reads them of four parts at once.
constexpr int kMergeWaves = 16;
template <typename TV>
__global__ __launch_bounds__(64 * kMergeWaves) void paged_merge_kernel(Params p) {
  __shared__ __attribute__((aligned(16))) float sums[kMergeWaves][64];
  const PagedAttentionArgs& a = p.a;
  const int S = a.S, D = a.cache.D;
  const uint32_t block = blockIdx.x;
  const int64_t n = a.mix ? block : p.maps.divide(block);
  const int s0 = a.mix ? 0 : static_cast<int>(p.maps.remainder(block)), s1 = a.mix ? S : s0 + 1;
  const int lane = lane_id(), wave = uniform_wave(), waves = static_cast<int>(blockDim.x) / 64;
  const int d = static_cast<int>(blockIdx.y) * 64 + (lane & 15) * 4;
  const bool owned = n >= load_constant(a.tokens.offsets) && n < load_constant(a.tokens.offsets + a.tokens.B);
  f32x4 total = zero4();
  for (int s = s0; s < s1 && owned; ++s) {
    const int64_t row = n * S + s;
    // A part that saw nothing (l = 0) has written nothing else.
    float m = -INFINITY, l = 0.f;
    for (int i = lane; i < p.n_split; i += 64) {
      const float li = p.part_l[i * p.rows + row], mi = p.part_m[i * p.rows + row];
      if (li != 0.f) m = fmaxf(m, mi);
    }
#pragma unroll
    for (int x = 32; x >= 1; x >>= 1) m = fmaxf(m, __shfl_xor(m, x));
    f32x4 o = zero4();
#pragma unroll 4
    for (int i = wave * 4 + (lane >> 4); i < p.n_split; i += waves * 4) {
      const float li = p.part_l[i * p.rows + row], mi = p.part_m[i * p.rows + row];
      if (li != 0.f && d < D) o += *reinterpret_cast<const f32x4*>(p.part_o + (i * p.rows + row) * D + d) * __builtin_amdgcn_exp2f(mi - m);
    }
    for (int i = lane; i < p.n_split; i += 64) {
      const float li = p.part_l[i * p.rows + row], mi = p.part_m[i * p.rows + row];
      if (li != 0.f) l += li * __builtin_amdgcn_exp2f(mi - m);
    }
    l = wave_sum(l);
    if (a.lse2 && blockIdx.y == 0 && threadIdx.x == 0) a.lse2[row] = l == 0.f ? -INFINITY : m + __builtin_amdgcn_logf(l);
    total += o * (l == 0.f ? 0.f : (a.mix ? a.mix[s] : 1.f) / l);
  }
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    total[e] += __shfl_xor(total[e], 16);
    total[e] += __shfl_xor(total[e], 32);
  }
  if (lane < 16) *reinterpret_cast<f32x4*>(&sums[wave][lane * 4]) = total;
  __syncthreads();
  const int t = static_cast<int>(threadIdx.x), at = static_cast<int>(blockIdx.y) * 64 + t;
  if (t < 64 && at < D) {
    float v = 0.f;
    for (int w = 0; w < waves; ++w) v += sums[w][t];
    static_cast<TV*>(a.out)[(a.mix ? n : n * S + s0) * D + at] = static_cast<TV>(v);
  }
}

// Attention weights of the cached tokens: p = 2^(score - lse2), summed over the
// columns.  A wave takes 32 tokens of a sequence, holds a map's keys in registers
// and goes through the new tokens, 16 at a time, the next ones' queries on their
// way; S^T = K Q^T as above.  With many new tokens `share` waves of a workgroup
// take the same tokens and a part of the maps and new tokens each.
template <typename TQ, int KS>
__global__ __launch_bounds__(64 * kWaves) void paged_weights_kernel(PagedAttentionArgs a, int share) {
  typedef typename Elem<TQ>::v8 q8;
  __shared__ float sums[kWaves][32];
  const CacheView& cache = a.cache;
  const int lane = lane_id(), c = lane & 15, g = lane >> 4;
  const int wave = uniform_wave(), part = wave % share;
  const int kt = (static_cast<int>(blockIdx.x) * kWaves + wave) / share, b = static_cast<int>(blockIdx.y);
  const Sequence seq = sequence_of(a.tokens, cache, b);
  const int S = a.S, W = cache.W, RP = a.RP;
  f32x4 sum[2] = {zero4(), zero4()};
  const int page = kt * 32 < seq.cached ? page_of(cache, b, kt) : -1;
  // The first sixteen new tokens that see one of these tokens, and how many
  // sixteens follow, over all maps.
  const int first = a.causal ? max(0, kt * 32 - (seq.length - seq.rows)) / 16 : 0;
  const int blocks = max(0, (seq.rows + 15) / 16 - first);
  if (page >= 0 && blocks > 0) {
    const TQ* kb = static_cast<const TQ*>(cache.keys) + page * cache.key_page +
                   (static_cast<int64_t>(tile_of(cache, kt)) * 32 + 8 * (c >> 2) + (c & 3)) * W + 8 * g;
    const int64_t total = static_cast<int64_t>(S) * blocks;
    int64_t at = total * part / share;
    const int64_t end = total * (part + 1) / share;
    q8 qf[KS];
    float lse2 = 0.f;
    int vis = 0;
    auto load_queries = [&](int s, int i0) {
      const int i = min(i0 + c, seq.rows - 1);
      const TQ* qb = static_cast<const TQ*>(a.q) + (seq.n0 + i) * a.ldq + s / a.repeat * RP + 8 * g;
#pragma unroll
      for (int k = 0; k < KS; ++k) qf[k] = load8(qb + min(32 * k, RP - 32));
      lse2 = a.lse2[(seq.n0 + i) * S + s];
      vis = i0 + c < seq.rows ? visible_to(seq, i, a.causal) : 0;
    };
    while (at < end) {
      const int s = static_cast<int>(at / blocks), from = s / a.repeat * RP;
      const int r0 = static_cast<int>(at - static_cast<int64_t>(s) * blocks);
      const int r1 = static_cast<int>(min(static_cast<int64_t>(blocks), r0 + (end - at)));
      at += r1 - r0;
      q8 kf[KS][2];
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        kf[k][0] = load8(kb + from + min(32 * k, RP - 32));
        kf[k][1] = load8(kb + from + min(32 * k, RP - 32) + 4 * W);
      }
      const float sc = score_scale(a, s);
      load_queries(s, (first + r0) * 16);
      for (int r = r0; r < r1; ++r) {
        f32x4 st[2] = {zero4(), zero4()};
#pragma unroll
        for (int k = 0; k < KS; ++k) {
          if (32 * k < RP) {
            st[0] = Elem<TQ>::mma(kf[k][0], qf[k], st[0]);
            st[1] = Elem<TQ>::mma(kf[k][1], qf[k], st[1]);
          }
        }
        const float l = lse2;
        const int seen = vis - kt * 32 - 8 * g;
        if (r + 1 < r1) load_queries(s, (first + r + 1) * 16);
#pragma unroll
        for (int h = 0; h < 2; ++h)
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            const float x = __builtin_amdgcn_exp2f(__builtin_fmaf(st[h][e], sc, -l));
            sum[h][e] += 4 * h + e < seen ? x : 0.f;
          }
      }
    }
  }
#pragma unroll
  for (int h = 0; h < 2; ++h)
#pragma unroll
    for (int e = 0; e < 4; ++e) {
#pragma unroll
      for (int x = 8; x >= 1; x >>= 1) sum[h][e] += __shfl_xor(sum[h][e], x);
      if (c == 0) sums[wave][8 * g + 4 * h + e] = sum[h][e];
    }
  __syncthreads();
  const int t = kt * 32 + lane;
  if (part == 0 && lane < 32 && t < a.capacity) {
    float v = a.weights_in && t < seq.length - seq.rows && t < seq.cached ? a.weights_in[b * a.ld_weights + t] : 0.f;
    for (int w = 0; w < share; ++w) v += sums[wave + w][lane];
    a.weights_out[b * a.ld_weights + t] = t < seq.cached ? v : 0.f;
  }
}

namespace {

// How a call is cut: one of the kernel's forms, and parts of the tokens.
struct Plan {
  bool one;        // columns of one map: paged_chunk_kernel
  int ct, nw;      // column tiles and waves of a workgroup
  int n_slices, dbw, members, n_ct, n_split, per;
  bool parts;
};

Plan plan(const PagedAttentionArgs& a) {
  Plan r;
  // Measured (us, columns of one map / all maps): 32 sequences over 2000 cached
  // tokens, 32 new ones 50 / 49, 64 58 / 63, 128 69 / 97; on two maps 32 72 / 79, on
  // four 96 / 125; one sequence, 256 new ones 39 / 25 over 2000 cached and 170 / 146
  // over 65536, 512 43 / 33 and 188 / 258.  A launch has fewer than 2^32 threads.
  const int most = 512;   // features of a workgroup
  r.n_slices = (a.cache.D + most - 1) / most;
  r.one = a.max_chunk >= 32 && a.max_chunk * a.S >= 64 && a.tokens.N * a.S >= 512 &&
          static_cast<int64_t>(a.tokens.B) * r.n_slices * a.S < (1 << 22);
  r.ct = r.one ? a.RP <= 256 ? 8 : 4 : 1;
  r.nw = r.one ? 8 : 4;
  const int64_t cols = static_cast<int64_t>(std::max(a.max_chunk, 1)) * (r.one ? 1 : a.S);
  r.dbw = (a.cache.D + r.n_slices * 16 * r.nw - 1) / (r.n_slices * 16 * r.nw);
  const int per_ct = r.n_slices * (r.one ? a.S : 1);
  r.n_ct = static_cast<int>(std::max<int64_t>(1, std::min<int64_t>((cols + 16 * r.ct - 1) / (16 * r.ct), 16384 / (a.tokens.B * per_ct) + 1)));
  r.members = r.n_ct * per_ct;
  // Parts of whole steps.  Few columns: as many as make kWantWorkgroups where all
  // sequences are as long as the longest.  Many: as many as fill the chip once
  // (one workgroup for each CU), going by the tiles that the rows fill and the
  // triangle that a causal chunk leaves out.
  const int64_t tiles = (std::max(a.max_length, 1) + 31) / 32;
  int64_t items = static_cast<int64_t>(a.tokens.B) * r.members, want = kWantWorkgroups;
  if (r.one) {
    const double filled = std::min<double>(a.tokens.B * r.n_ct, static_cast<double>(a.tokens.N) / (16 * r.ct) + 0.5 * a.tokens.B);
    const double seen = a.causal ? 1 - 0.5 * std::min(1.0, static_cast<double>(a.max_chunk) / std::max(a.max_length, 1)) : 1;
    items = std::max<int64_t>(1, static_cast<int64_t>(filled * seen * per_ct));
    want = kChunkWorkgroups;
  }
  const int64_t split = std::min<int64_t>({std::max<int64_t>(1, want / items), kMaxSplits, tiles});
  r.per = static_cast<int>(round_up((tiles + split - 1) / split, 4));
  r.n_split = static_cast<int>((tiles + r.per - 1) / r.per);
  r.parts = r.n_split > 1 || a.mix != nullptr;
  return r;
}

template <typename TQ, typename TV, int DBW>
void launch_token(const Params& p, hipStream_t stream) {
  const int QP = static_cast<int>(round_up(p.a.cache.W, 64 * kTokenGroups)) + 8;
  const size_t lds = static_cast<size_t>(32) * QP + 2 * kWaves * (1024 + 64 + 4) + kWaves * DBW * 64;
  const unsigned units = static_cast<unsigned>(round_up(p.units, kXcds));
  hipLaunchKernelGGL((paged_token_kernel<TQ, TV, DBW>), dim3(units * p.members.d), dim3(64 * kWaves), lds, stream, p);
}

template <typename TQ, typename TV, int NK, int DBW, int CT>
void launch_chunk_kernel(const Params& p, hipStream_t stream) {
  const unsigned units = static_cast<unsigned>(round_up(p.units, kXcds));
  hipLaunchKernelGGL((paged_chunk_kernel<TQ, TV, NK, DBW, CT>), dim3(units * p.members.d), dim3(64 * kChunkWaves), (ChunkLds<NK, CT>::BYTES),
                     stream, p);
}
template <typename TQ, typename TV, int DBW>
void launch_chunk(const Params& p, hipStream_t stream) {
  if (p.a.RP <= 128) launch_chunk_kernel<TQ, TV, 2, DBW, 8>(p, stream);
  else if (p.a.RP <= 256) launch_chunk_kernel<TQ, TV, 4, DBW, 8>(p, stream);
  else launch_chunk_kernel<TQ, TV, 8, DBW, 4>(p, stream);
}

template <typename TQ, typename TV>
void launch_typed(const Params& p, const Plan& r, hipStream_t stream) {
  if (r.one) {
    switch (r.dbw) {
      case 1: launch_chunk<TQ, TV, 1>(p, stream); break;
      case 2: launch_chunk<TQ, TV, 2>(p, stream); break;
      case 3: launch_chunk<TQ, TV, 3>(p, stream); break;
      default: launch_chunk<TQ, TV, 4>(p, stream); break;
    }
  } else switch (r.dbw) {
    case 1: launch_token<TQ, TV, 1>(p, stream); break;
    case 2: launch_token<TQ, TV, 2>(p, stream); break;
    case 3: launch_token<TQ, TV, 3>(p, stream); break;
    case 4: launch_token<TQ, TV, 4>(p, stream); break;
    case 5: launch_token<TQ, TV, 5>(p, stream); break;
    case 6: launch_token<TQ, TV, 6>(p, stream); break;
    case 7: launch_token<TQ, TV, 7>(p, stream); break;
    default: launch_token<TQ, TV, 8>(p, stream); break;
  }
  if (p.part_o) {
    const dim3 grid(static_cast<unsigned>(p.a.tokens.N * (p.a.mix ? 1 : p.a.S)), static_cast<unsigned>((p.a.cache.D + 63) / 64));
    const int waves = std::max(1, std::min(kMergeWaves, (p.n_split + 15) / 16));
    hipLaunchKernelGGL((paged_merge_kernel<TV>), grid, dim3(64 * waves), 0, stream, p);
  }
}

}  // namespace

int64_t paged_attention_workspace(const PagedAttentionArgs& a) {
  const Plan r = plan(a);
  return r.parts ? r.n_split * a.tokens.N * a.S * (static_cast<int64_t>(a.cache.D) + 2) * 4 : 0;
}

void launch_paged_attention(const PagedAttentionArgs& a, void* workspace, hipStream_t stream) {
  const Plan r = plan(a);
  Params p{};
  p.a = a;
  p.n_ct = r.n_ct;
  p.n_split = r.n_split;
  p.per = r.per;
  p.units = a.tokens.B * r.n_split;
  p.rows = a.tokens.N * a.S;
  p.members = Divisor(r.members);
  p.sequences = Divisor(a.tokens.B);
  p.slices = Divisor(r.n_slices);
  p.maps = Divisor(a.S);
  p.repeats = Divisor(a.repeat);
  if (r.parts) {
    p.part_o = static_cast<float*>(workspace);
    p.part_m = p.part_o + r.n_split * p.rows * a.cache.D;
    p.part_l = p.part_m + r.n_split * p.rows;
  }
  if (a.qk_dtype == kBF16) launch_typed<__bf16, __bf16>(p, r, stream);
  else if (a.v_dtype == kBF16) launch_typed<_Float16, __bf16>(p, r, stream);
  else launch_typed<_Float16, _Float16>(p, r, stream);
}

template <typename TQ>
static void launch_weights_typed(const PagedAttentionArgs& a, hipStream_t stream) {
  const int64_t blocks = static_cast<int64_t>(a.S) * ((std::max(a.max_chunk, 1) + 15) / 16);
  const int share = blocks >= 4 ? 4 : blocks >= 2 ? 2 : 1;
  const dim3 grid(static_cast<unsigned>((static_cast<int64_t>((a.capacity + 31) / 32) * share + kWaves - 1) / kWaves),
                  static_cast<unsigned>(a.tokens.B));
  const dim3 block(64 * kWaves);
  if (a.RP <= 128) hipLaunchKernelGGL((paged_weights_kernel<TQ, 4>), grid, block, 0, stream, a, share);
  else if (a.RP <= 256) hipLaunchKernelGGL((paged_weights_kernel<TQ, 8>), grid, block, 0, stream, a, share);
  else hipLaunchKernelGGL((paged_weights_kernel<TQ, 16>), grid, block, 0, stream, a, share);
}

void launch_paged_weights(const PagedAttentionArgs& a, hipStream_t stream) {
  if (a.qk_dtype == kBF16) launch_weights_typed<__bf16>(a, stream);
  else launch_weights_typed<_Float16>(a, stream);
}

}  // namespace da
