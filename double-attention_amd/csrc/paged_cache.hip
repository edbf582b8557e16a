// The paged cache's own moves: new tokens into their pages, the choice of the
// tokens that stay when a sequence is cut, and their move into other pages.
// All are bound by their bytes.
#include <algorithm>

#include "da_common.h"
#include "da_launch.h"
#include "da_serving.h"

namespace da {

namespace {

constexpr int kMoveThreads = 256;

__device__ __forceinline__ uint16_t* key_row(const CacheView& c, int page, int t) {
  return static_cast<uint16_t*>(c.keys) + page * c.key_page + static_cast<int64_t>(t) * c.W;
}
__device__ __forceinline__ uint16_t* value_tile(const CacheView& c, int page, int tile) {
  return static_cast<uint16_t*>(c.values) + page * c.value_page + static_cast<int64_t>(tile) * 32 * c.D;
}

typedef uint16_t u16x8 __attribute__((ext_vector_type(8)));

// Eight features of each of eight tokens, turned to eight tokens of each
// feature, and written for the tokens of `mask`.
__device__ __forceinline__ void store_turned(uint16_t* dst, const u16x8 (&rows)[8], unsigned mask) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    u16x8 v;
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = rows[i][e];
    uint16_t* at = dst + 32 * e;
    if (mask == 0xffu) {
      *reinterpret_cast<u16x8*>(at) = v;
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i)
        if (mask >> i & 1) at[i] = v[i];
    }
  }
}

}  // namespace

// A workgroup takes a 32-token tile of a sequence that new tokens reach.  Keys
// are copied row by row; of the values a thread takes eight features of eight
// tokens, which it turns in registers (a wave's loads are 256 contiguous bytes
// of a token, its stores 64 of a feature).
__global__ __launch_bounds__(kMoveThreads) void cache_append_kernel(CacheAppendArgs a, int n_tiles) {
  const CacheView& cache = a.cache;
  const int b = static_cast<int>(blockIdx.y);
  const int64_t first = min(max(static_cast<int64_t>(a.tokens.offsets[b]), int64_t{0}), a.tokens.N);
  const int64_t last = min(max(static_cast<int64_t>(a.tokens.offsets[b + 1]), first), a.tokens.N);
  const int64_t rows = last - first;
  const int64_t length = max(a.tokens.lengths[b], 0);
  // Positions in front of the sequence or behind its pages take nothing.
  const int64_t begin = max(length - rows, int64_t{0});
  const int64_t end = min(length, static_cast<int64_t>(cache.table_pages) * cache.tiles * 32);
  const int64_t row0 = first - (length - rows);   // row of position 0
  for (int64_t kt = begin / 32 + blockIdx.x; kt * 32 < end; kt += n_tiles) {
    const int page = page_of(cache, b, static_cast<int>(kt));
    if (page < 0) continue;
    const int tile = static_cast<int>(kt % cache.tiles);
    const int t0 = static_cast<int>(max(begin - kt * 32, int64_t{0})), t1 = static_cast<int>(min(end - kt * 32, int64_t{32}));
    const uint16_t* key = static_cast<const uint16_t*>(a.key) + (row0 + kt * 32) * a.ldk;
    const int chunks = cache.W / 8;
    for (int i = static_cast<int>(threadIdx.x); i < (t1 - t0) * chunks; i += kMoveThreads) {
      const int t = t0 + i / chunks, f = i % chunks * 8;
      store16B(key_row(cache, page, tile * 32 + t) + f, load16B(key + t * a.ldk + f));
    }
    const uint16_t* value = static_cast<const uint16_t*>(a.value) + (row0 + kt * 32) * a.ldv;
    uint16_t* out = value_tile(cache, page, tile);
    for (int i = static_cast<int>(threadIdx.x); i < cache.D / 2; i += kMoveThreads) {
      const int tg = (i & 3) * 8, d = (i >> 2) * 8;
      u16x8 v[8];
      unsigned mask = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v[e] = u16x8{0, 0, 0, 0, 0, 0, 0, 0};
        if (tg + e >= t0 && tg + e < t1) {
          v[e] = *reinterpret_cast<const u16x8*>(value + (tg + e) * a.ldv + d);
          mask |= 1u << e;
        }
      }
      if (mask) store_turned(out + 32 * d + tg, v, mask);
    }
  }
}

void launch_cache_append(const CacheAppendArgs& a, hipStream_t stream) {
  const int n_tiles = std::min((std::max(a.max_chunk, 1) + 31) / 32 + (a.max_chunk > 1 ? 1 : 0), std::max(1, (1 << 20) / a.tokens.B));
  hipLaunchKernelGGL(cache_append_kernel, dim3(static_cast<unsigned>(n_tiles), static_cast<unsigned>(a.tokens.B)), dim3(kMoveThreads),
                     0, stream, a, n_tiles);
}

namespace {

// Weights in an order of whole numbers: larger ones are larger, both zeros
// equal, NaN below everything.
__device__ __forceinline__ uint32_t weight_key(float w) {
  if (w != w) return 0;
  const uint32_t u = __float_as_uint(w + 0.f);   // -0 becomes +0
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}

constexpr int kSelectThreads = 1024;
constexpr int kSelectWaves = kSelectThreads / 64;
constexpr int kDigit = 256;
constexpr int kCopies = 4;   // of the bins

}  // namespace

// The `need` largest of a sequence's older tokens by the digits of their keys
// from the highest: four counts of 256 bins find the key of the last one that
// stays and how many of its equals do (the first ones).  Each wave has a
// contiguous part of the tokens, read once where they fit its registers (32768
// in all), and writes its kept ones in order.  The first digits of most weights
// are alike, so the lanes of a wave share four copies of the bins: atomics of
// one address wait for each other.  Bound by its passes on one CU: 1001 tokens of
// each sequence 7 us, 32768 of them 22 us (46 us with one copy and the weights read
// again at each pass).
template <int KEYS>
__device__ void select_older(const float* w, int32_t* kept, int older, int need, int rounds) {
  __shared__ int copies[kCopies * (kDigit + 1)];
  __shared__ int picked[2];
  __shared__ int counts[2][kSelectWaves];
  const int tid = static_cast<int>(threadIdx.x), lane = lane_id(), wave = wave_id();
  const int i0 = wave * rounds * 64, i1 = min(older, i0 + rounds * 64);
  uint32_t keys[KEYS > 0 ? KEYS : 1];
  if constexpr (KEYS > 0) {
#pragma unroll
    for (int j = 0; j < KEYS; ++j)   // all in flight
      if (j < rounds) keys[j] = __float_as_uint(w[min(i0 + j * 64 + lane, older - 1)]);
#pragma unroll
    for (int j = 0; j < KEYS; ++j)
      if (j < rounds) keys[j] = weight_key(__uint_as_float(keys[j]));
  }
  // f(first token of the round, this lane's key, whether it has one)
  auto each = [&](auto f) {
    if constexpr (KEYS > 0) {
#pragma unroll
      for (int j = 0; j < KEYS; ++j)
        if (j < rounds) f(i0 + j * 64, keys[j], i0 + j * 64 + lane < i1);
    } else {
      for (int i = i0; i < i1; i += 64) f(i, i + lane < i1 ? weight_key(w[i + lane]) : 0, i + lane < i1);
    }
  };
  uint32_t prefix = 0, mask = 0;
  int equals = need;   // of the tokens with the key's digits so far, those that stay
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = tid; i < kCopies * (kDigit + 1); i += kSelectThreads) copies[i] = 0;
    __syncthreads();
    int* mine = copies + (lane & (kCopies - 1)) * (kDigit + 1);
    each([&](int, uint32_t key, bool there) {
      if (there && (key & mask) == prefix) atomicAdd(&mine[key >> shift & 255], 1);
    });
    __syncthreads();
    if (wave == 0) {
      // Lane l has bins 255 - 4 l down to 252 - 4 l; the sum in front of them
      // tells which lane's bins reach the number that stays.
      int n[4], own = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        n[e] = 0;
#pragma unroll
        for (int c = 0; c < kCopies; ++c) n[e] += copies[c * (kDigit + 1) + 255 - 4 * lane - e];
        own += n[e];
      }
      int before = own;
#pragma unroll
      for (int x = 1; x < 64; x <<= 1) {
        const int v = __shfl_up(before, x);
        if (lane >= x) before += v;
      }
      before -= own;
      if (before < equals && before + own >= equals) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          if (before < equals && before + n[e] >= equals) {
            picked[0] = 255 - 4 * lane - e;
            picked[1] = equals - before;
          }
          before += n[e];
        }
      }
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(picked[0]) << shift;
    mask |= 255u << shift;
    equals = picked[1];
  }
  // Above the key: all stay; at the key: the first `equals`.
  int above = 0, at = 0;
  each([&](int, uint32_t key, bool there) {
    above += there && key > prefix;
    at += there && key == prefix;
  });
#pragma unroll
  for (int x = 32; x >= 1; x >>= 1) {
    above += __shfl_xor(above, x);
    at += __shfl_xor(at, x);
  }
  if (lane == 0) {
    counts[0][wave] = above;
    counts[1][wave] = at;
  }
  __syncthreads();
  int put = 0, seen = 0;   // kept tokens, and tokens at the key, in front
  for (int v = 0; v < wave; ++v) {
    put += counts[0][v];
    seen += counts[1][v];
  }
  put += min(seen, equals);
  const uint64_t below = (uint64_t{1} << lane) - 1;
  each([&](int i, uint32_t key, bool there) {
    const bool equal = there && key == prefix;
    const uint64_t ties = __ballot(equal);
    const bool stays = there && (key > prefix || (equal && seen + __popcll(ties & below) < equals));
    const uint64_t all = __ballot(stays);
    if (stays) kept[put + __popcll(all & below)] = i + lane;
    put += __popcll(all);
    seen += __popcll(ties);
  });
}

__global__ __launch_bounds__(kSelectThreads) void cache_select_kernel(CacheSelectArgs a) {
  const int b = static_cast<int>(blockIdx.x), tid = static_cast<int>(threadIdx.x);
  const int length = min(max(a.lengths[b], 0), a.capacity);
  const int count = min(length, a.keep);
  const int recent = min(a.recent, count);
  const int older = length - recent;            // tokens to choose from
  const int need = count - recent;
  const float* w = a.weights + b * a.ld_weights;
  int32_t* kept = a.kept + static_cast<int64_t>(b) * a.keep;
  if (tid == 0) a.counts[b] = count;
  for (int i = tid; i < recent; i += kSelectThreads) kept[need + i] = older + i;
  for (int i = count + tid; i < a.keep; i += kSelectThreads) kept[i] = -1;
  if (need == older) {   // all stay
    for (int i = tid; i < need; i += kSelectThreads) kept[i] = i;
    return;
  }
  if (need == 0) return;
  // Up to 4096 and 32768 tokens in registers, longer rows read again at each pass.
  const int rounds = (older + kSelectThreads - 1) / kSelectThreads;   // of 64 tokens of a wave
  if (rounds <= 4) select_older<4>(w, kept, older, need, rounds);
  else if (rounds <= 32) select_older<32>(w, kept, older, need, rounds);
  else select_older<0>(w, kept, older, need, rounds);
}

void launch_cache_select(const CacheSelectArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL(cache_select_kernel, dim3(static_cast<unsigned>(a.B)), dim3(kSelectThreads), 0, stream, a);
}

// A workgroup takes 32 kept tokens of a sequence, a tile of the new pages, and a
// part (blockIdx.z) of their features.  The tokens' values lie 64 bytes apart in
// their tiles, a feature's 32 side by side, so that most of the old tiles' lines
// are read: bound by bytes (8192 of 32768 tokens of four sequences, keys of 256
// and values of 512 features: 200 MB in 40 us).
__global__ __launch_bounds__(kMoveThreads) void cache_compact_kernel(CacheCompactArgs a) {
  __shared__ int64_t key_at[32], value_at[32];   // where the tokens come from, or -1
  const int b = static_cast<int>(blockIdx.y), kt = static_cast<int>(blockIdx.x), tid = static_cast<int>(threadIdx.x);
  const int count = min(max(a.counts[b], 0), a.keep);
  const int D = a.to.D, W = a.to.W;
  const int nz = static_cast<int>(gridDim.z), z = static_cast<int>(blockIdx.z);
  if (a.weights_out && tid < 32 && z == 0) {
    const int i = kt * 32 + tid;
    const int t = i < count ? a.kept[b * a.ld_kept + i] : -1;
    if (i < a.capacity_out) a.weights_out[b * a.ld_out + i] = t >= 0 && t < a.capacity_in ? a.weights_in[b * a.ld_in + t] : 0.f;
  }
  if (kt * 32 >= count) return;
  const int page = page_of(a.to, b, kt);
  if (page < 0) return;
  if (tid < 32) {
    const int i = kt * 32 + tid;
    const int t = i < count ? a.kept[b * a.ld_kept + i] : -1;
    const int from = t >= 0 ? page_of(a.from, b, t / 32) : -1;
    const int at = t % (a.from.tiles * 32);
    key_at[tid] = from < 0 ? -1 : from * a.from.key_page + static_cast<int64_t>(at) * W;
    value_at[tid] = from < 0 ? -1 : from * a.from.value_page + static_cast<int64_t>(at / 32) * 32 * D + at % 32;
  }
  __syncthreads();
  const int tile = kt % a.to.tiles;
  const uint16_t* keys = static_cast<const uint16_t*>(a.from.keys);
  const uint16_t* values = static_cast<const uint16_t*>(a.from.values);
  const int chunks = W / 8;
  for (int i = z * kMoveThreads + tid; i < 32 * chunks; i += nz * kMoveThreads) {
    const int t = i / chunks, f = i % chunks * 8;
    if (key_at[t] >= 0) store16B(key_row(a.to, page, tile * 32 + t) + f, load16B(keys + key_at[t] + f));
  }
  uint16_t* out = value_tile(a.to, page, tile);
  for (int i = z * kMoveThreads + tid; i < 4 * D; i += nz * kMoveThreads) {
    const int tg = (i & 3) * 8, d = i >> 2;
    u16x8 v;
    unsigned mask = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      v[e] = 0;
      if (value_at[tg + e] >= 0) {
        v[e] = values[value_at[tg + e] + 32 * d];
        mask |= 1u << e;
      }
    }
    uint16_t* at = out + 32 * d + tg;
    if (mask == 0xffu) {
      *reinterpret_cast<u16x8*>(at) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (mask >> e & 1) at[e] = v[e];
    }
  }
}

void launch_cache_compact(const CacheCompactArgs& a, hipStream_t stream) {
  // The new weights are written to the end of their rows.
  const int tokens = std::max(a.keep, a.weights_out ? a.capacity_out : 0);
  if (tokens == 0) return;
  // A tile's features in parts while its workgroups do not fill the chip (128
  // tiles of 512 features: 14 us whole, 7 us in four; 1024 tiles of them: 40 and
  // 45 us), 128 features and two rounds of a thread's loads in each.
  const int64_t tiles = (tokens + 31) / 32;
  const int64_t fill = 1024 / std::max<int64_t>(1, tiles * a.B);
  const unsigned parts = static_cast<unsigned>(std::min<int64_t>(std::max<int64_t>(1, fill), std::max(1, a.to.D / 128)));
  hipLaunchKernelGGL(cache_compact_kernel, dim3(static_cast<unsigned>(tiles), static_cast<unsigned>(a.B), parts),
                     dim3(kMoveThreads), 0, stream, a);
}

}  // namespace da
