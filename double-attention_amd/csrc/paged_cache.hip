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

}  // namespace

// The `need` largest of a sequence's older tokens by the digits of their keys
// from the highest: four counts of 256 bins find the key of the last one that
// stays and how many of its equals do (the first ones).  Each wave then takes
// a contiguous part of the tokens and writes the kept ones in order.
__global__ __launch_bounds__(kSelectThreads) void cache_select_kernel(CacheSelectArgs a) {
  __shared__ int bins[kDigit];
  __shared__ int picked[2];
  __shared__ int counts[2][kSelectWaves];
  const int b = static_cast<int>(blockIdx.x), tid = static_cast<int>(threadIdx.x);
  const int lane = lane_id(), wave = wave_id();
  const int length = min(max(a.lengths[b], 0), a.capacity);
  const int count = min(length, a.keep);
  const int recent = min(a.recent, count);
  const int older = length - recent;            // tokens to choose from
  int need = count - recent;
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
  uint32_t prefix = 0, mask = 0;
  int equals = need;   // of the tokens with the key's digits so far, those that stay
  for (int shift = 24; shift >= 0; shift -= 8) {
    if (tid < kDigit) bins[tid] = 0;
    __syncthreads();
    for (int i = tid; i < older; i += kSelectThreads) {
      const uint32_t key = weight_key(w[i]);
      if ((key & mask) == prefix) atomicAdd(&bins[key >> shift & 255], 1);
    }
    __syncthreads();
    if (wave == 0) {
      // Lane l has bins 255 - 4 l down to 252 - 4 l; the sum in front of them
      // tells which lane's bins reach the number that stays.
      int n[4], own = 0;
#pragma unroll
      for (int e = 0; e < 4; ++e) own += n[e] = bins[255 - 4 * lane - e];
      int before = own;
#pragma unroll
      for (int x = 1; x < 64; x <<= 1) {
        const int v = __shfl_up(before, x);
        if (lane >= x) before += v;
      }
      before -= own;
      if (before < equals && before + own >= equals) {
        int e = 0;
        while (before + n[e] < equals) before += n[e++];
        picked[0] = 255 - 4 * lane - e;
        picked[1] = equals - before;
      }
    }
    __syncthreads();
    prefix |= static_cast<uint32_t>(picked[0]) << shift;
    mask |= 255u << shift;
    equals = picked[1];
  }
  // Above the key: all stay; at the key: the first `equals`.
  const int part = (older + kSelectThreads - 1) / kSelectThreads * 64;   // tokens of a wave
  const int i0 = min(older, wave * part), i1 = min(older, i0 + part);
  int above = 0, at = 0;
  for (int i = i0 + lane; i < i1; i += 64) {
    const uint32_t key = weight_key(w[i]);
    above += key > prefix;
    at += key == prefix;
  }
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
  for (int i = i0; i < i1; i += 64) {
    const uint32_t key = i + lane < i1 ? weight_key(w[i + lane]) : 0;
    const bool equal = i + lane < i1 && key == prefix;
    const uint64_t ties = __ballot(equal);
    const uint64_t below = (uint64_t{1} << lane) - 1;
    const bool stays = i + lane < i1 && (key > prefix || (equal && seen + __popcll(ties & below) < equals));
    const uint64_t all = __ballot(stays);
    if (stays) kept[put + __popcll(all & below)] = i + lane;
    put += __popcll(all);
    seen += __popcll(ties);
  }
}

void launch_cache_select(const CacheSelectArgs& a, hipStream_t stream) {
  hipLaunchKernelGGL(cache_select_kernel, dim3(static_cast<unsigned>(a.B)), dim3(kSelectThreads), 0, stream, a);
}

// A workgroup takes 32 kept tokens of a sequence: a tile of the new pages.
__global__ __launch_bounds__(kMoveThreads) void cache_compact_kernel(CacheCompactArgs a) {
  __shared__ int64_t key_at[32], value_at[32];   // where the tokens come from, or -1
  const int b = static_cast<int>(blockIdx.y), kt = static_cast<int>(blockIdx.x), tid = static_cast<int>(threadIdx.x);
  const int count = min(max(a.counts[b], 0), a.keep);
  const int D = a.to.D, W = a.to.W;
  if (a.weights_out && tid < 32) {
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
  for (int i = tid; i < 32 * chunks; i += kMoveThreads) {
    const int t = i / chunks, f = i % chunks * 8;
    if (key_at[t] >= 0) store16B(key_row(a.to, page, tile * 32 + t) + f, load16B(keys + key_at[t] + f));
  }
  uint16_t* out = value_tile(a.to, page, tile);
  for (int i = tid; i < 4 * D; i += kMoveThreads) {
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
  hipLaunchKernelGGL(cache_compact_kernel, dim3(static_cast<unsigned>((tokens + 31) / 32), static_cast<unsigned>(a.B)),
                     dim3(kMoveThreads), 0, stream, a);
}

}  // namespace da
