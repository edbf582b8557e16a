// Log probabilities of given tokens, the entropy of each row's distribution and
// its most probable tokens, in one pass over the logits; and the gradient.
//
// With m a reference near a row's maximum, s = sum e^(x - m) and
// t = sum e^(x - m) (x - m):
//   log p(j) = (x_j - m) - log s,   H = log s - t / s.
// Every lane keeps its own (m, s, t) over its 16-byte chunks in 32 bits and
// moves m only where a chunk exceeds it by more than kSlack.  The largest
// values are compared as whole numbers, the value's order in the high half and
// the token's in the low half, so that equal values come in the order of their
// tokens whatever the order they are met in.  Rows are cut into parts where there
// are few of them.  Bound by the bytes: 4096 x 32000 bf16 logits in 52 us (5.0
// TB/s) where the last level of cache still has most of them, 77 us after the
// gradient of others; their gradient in 86 us (6.1 TB/s).
// Backward: dx_j = -p_j (G + g_H (log p_j + H)) + what is given for j itself,
// with G the sum of the gradients at log probabilities of the row.  It gets m and
// log s apart: their rounded sum would shift every log p_j of a row whose logits
// are far from zero (by up to 2^-8 at 10^5), and be m where that is the lowest value.
#include <algorithm>
#include <type_traits>

#include "da_common.h"
#include "da_launch.h"
#include "da_serving.h"

namespace da {

namespace {

constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr float kSlack = 8.f;
constexpr float kLowest = -3.402823466e38f;
// Differences below this have no weight in 32 bits (e^-200 = 0).
constexpr float kNoWeight = -200.f, kNoWeight2 = -300.f;   // (base 2)
constexpr float kLn2 = 0.6931471805599453f;
typedef unsigned long long Key;

struct Sums {
  float m, s, t;
};

__device__ __forceinline__ float fast_exp(float x) { return __builtin_amdgcn_exp2f(x * kLog2e); }

// b's sums joined to a's.
__device__ __forceinline__ Sums join(Sums a, Sums b) {
  Sums r;
  r.m = fmaxf(a.m, b.m);
  const float da = fmaxf(a.m - r.m, kNoWeight), db = fmaxf(b.m - r.m, kNoWeight);
  const float fa = fast_exp(da), fb = fast_exp(db);
  r.s = a.s * fa + b.s * fb;
  r.t = (a.t + a.s * da) * fa + (b.t + b.s * db) * fb;
  return r;
}
__device__ __forceinline__ Sums join_wave(Sums v) {
#pragma unroll
  for (int x = 32; x >= 1; x >>= 1) v = join(v, Sums{__shfl_xor(v.m, x), __shfl_xor(v.s, x), __shfl_xor(v.t, x)});
  return v;
}

// Larger for larger values, then for earlier tokens; 0 for NaN.
__device__ __forceinline__ Key key_of(float x, int token) {
  if (x != x) return 0;
  const uint32_t u = __float_as_uint(x + 0.f);
  return static_cast<Key>(u & 0x80000000u ? ~u : u | 0x80000000u) << 32 | static_cast<uint32_t>(~token);
}
__device__ __forceinline__ float key_value(Key k) {
  const uint32_t u = static_cast<uint32_t>(k >> 32);
  return k == 0 ? __builtin_nanf("") : __uint_as_float(u & 0x80000000u ? u & 0x7fffffffu : ~u);
}
__device__ __forceinline__ int key_token(Key k) { return k == 0 ? -1 : static_cast<int>(~static_cast<uint32_t>(k)); }

__device__ __forceinline__ Key read_lane(Key k, int lane) {
  const uint32_t lo = __builtin_amdgcn_readlane(static_cast<uint32_t>(k), lane);
  const uint32_t hi = __builtin_amdgcn_readlane(static_cast<uint32_t>(k >> 32), lane);
  return static_cast<Key>(hi) << 32 | lo;
}

// The `top` largest keys, lane i with the i-th; those behind are not used.
struct TopList {
  Key mine, last;   // this lane's; the top-th one's (0: not that many yet)
  int top;
  __device__ __forceinline__ void insert(Key k) {   // k: the same in all lanes, larger than last
    const int at = __popcll(__ballot(mine > k));
    // The lane in front's key (wave_shr:1 of both halves).
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, static_cast<uint32_t>(mine), 0x138, 0xf, 0xf, false);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, static_cast<uint32_t>(mine >> 32), 0x138, 0xf, 0xf, false);
    const Key up = static_cast<Key>(hi) << 32 | lo;
    const int lane = lane_id();
    mine = lane < at ? mine : lane == at ? k : up;
    last = read_lane(mine, top - 1);
  }
  __device__ __forceinline__ void offer(Key k) {   // one key a lane (0: none)
    for (uint64_t more = __ballot(k > last); more;) {
      const int from = __builtin_ctzll(more);
      insert(read_lane(k, from));
      more = __ballot(k > last) & ~((uint64_t{2} << from) - 1);
    }
  }
  __device__ __forceinline__ float floor() const { return last == 0 ? -INFINITY : key_value(last); }
};

// A row's aligned 16-byte chunks, and the elements in front of and behind them.
template <typename T>
struct RowShape {
  int head, chunks, tail;
  __device__ RowShape(const T* x, int V) {
    const int off = static_cast<int>(reinterpret_cast<uintptr_t>(x) & 15) / static_cast<int>(sizeof(T));
    head = min(V, off ? 16 / static_cast<int>(sizeof(T)) - off : 0);
    chunks = (V - head) / 8;
    tail = V - head - 8 * chunks;
  }
};
template <typename T>
struct Chunk {
  typename Elem<T>::v8 v;
  __device__ __forceinline__ void load(const T* p) { v = load8(p); }
  __device__ __forceinline__ float operator[](int e) const { return static_cast<float>(v[e]); }
};
template <>
struct Chunk<float> {
  f32x4 v[2];
  __device__ __forceinline__ void load(const float* p) {
    v[0] = *reinterpret_cast<const f32x4*>(p);
    v[1] = *reinterpret_cast<const f32x4*>(p + 4);
  }
  __device__ __forceinline__ float operator[](int e) const { return v[e >> 2][e & 3]; }
};

struct Params {
  TokenLogProbsArgs a;
  int parts;
  Sums* sums;    // [rows][parts]
  Key* keys;     // [rows][parts][top]
};

__device__ void finish_row(const TokenLogProbsArgs& a, int64_t row, Sums v, float logit) {
  const float log_s = logf(v.s);
  const int64_t token = a.tokens[row];
  float lp = (logit - v.m) - log_s;
  if (token < 0 || token >= a.V) lp = __builtin_nanf("");
  if (token == a.ignore) lp = 0.f;
  a.log_probs[row] = lp;
  if (a.entropy) a.entropy[row] = log_s - v.t / v.s;
  if (a.lse) {
    a.lse[2 * row] = v.m;
    a.lse[2 * row + 1] = log_s;
  }
}
template <typename T>
__device__ __forceinline__ float token_logit(const TokenLogProbsArgs& a, int64_t row) {
  const int64_t token = a.tokens[row];
  return token < 0 || token >= a.V ? 0.f : static_cast<float>(static_cast<const T*>(a.logits)[row * a.ldx + token]);
}

}  // namespace

namespace {

// Where the alternatives of a row (or a part of it) are found.  Each lane keeps
// the largest values of three of its chunks and the places of two; the top-th
// largest of the lanes' first ones is a bound that `top` values reach.  Chunks
// that reach it are read again and their values that do are gathered.  Where a
// lane may have more such chunks, or the values do not fit (equal logits, masked
// vocabularies), the waves go through the row again with sorted lists.
constexpr int kMaxCandidates = 256;
struct LaneTop {
  float m1, m2, m3;
  int c1, c2;
  __device__ __forceinline__ void add(float largest, int c) {
    const bool first = largest > m1, second = largest > m2;
    m3 = fmaxf(m3, second ? m2 : largest);
    m2 = first ? m1 : second ? largest : m2;
    c2 = first ? c1 : second ? c : c2;
    m1 = first ? largest : m1;
    c1 = first ? c : c1;
  }
};
struct TopShared {
  Key candidates[kMaxCandidates];
  float maxima[kThreads];
  volatile float bounds[kWaves];
  float bound;
  int count, survivors, again;
};

}  // namespace

template <typename T, bool TOP>
__global__ __launch_bounds__(kThreads) void token_log_probs_kernel(Params p) {
  __shared__ Sums wave_sums[kWaves];
  __shared__ typename std::conditional<TOP, TopShared, int>::type top_shared;
  const TokenLogProbsArgs& a = p.a;
  const int lane = lane_id(), wave = wave_id(), tid = static_cast<int>(threadIdx.x);
  const int64_t row = blockIdx.x / p.parts;
  const int part = static_cast<int>(blockIdx.x % p.parts);
  const T* x = static_cast<const T*>(a.logits) + row * a.ldx;
  const RowShape<T> shape(x, a.V);
  const int per = (shape.chunks + p.parts - 1) / p.parts;
  const int c0 = min(shape.chunks, part * per), c1 = min(shape.chunks, c0 + per);
  const T* body = x + shape.head;

  // In this loop t is in units of log 2.  The difference to m is taken first: a
  // rounded m log2(e) would shift all terms where the logits are far from zero.
  Sums v{kLowest, 0.f, 0.f};
  auto add = [&](float value) {
    const float d = (value - v.m) * kLog2e;
    const float e = __builtin_amdgcn_exp2f(d);
    v.s += e;
    v.t += e * fmaxf(d, kNoWeight2);
  };
  auto raise = [&](float largest) {   // the reference to this chunk's largest value
    if (largest > v.m + kSlack || (v.s == 0.f && largest > v.m)) {
      const float d = fmaxf(v.m - largest, kNoWeight), f = fast_exp(d);
      v.t = (v.t + v.s * d * kLog2e) * f;
      v.s *= f;
      v.m = largest;
    }
  };
  // The first lanes of wave 0 have the elements in front of the chunks, the
  // lanes from 8 on those behind them (-1: none).
  const int extra = wave != 0 ? -1
                    : part == 0 && lane < shape.head ? lane
                    : part == p.parts - 1 && lane >= 8 && lane < 8 + shape.tail ? a.V - shape.tail + lane - 8 : -1;
  if (extra >= 0) {
    const float value = static_cast<float>(x[extra]);
    raise(value);
    add(value);
  }
  LaneTop best{-INFINITY, -INFINITY, -INFINITY, 0, 0};
  constexpr int U = 4;
  Chunk<T> ch[U];
  auto fetch = [&](int base) {
#pragma unroll
    for (int u = 0; u < U; ++u) ch[u].load(body + static_cast<int64_t>(min(base + u * kThreads + lane, c1 - 1)) * 8);
  };
  const int first = c0 + wave * 64;
  if (first < c1) fetch(first);
  for (int base = first; base < c1; base += kThreads * U) {
    Chunk<T> now[U];
#pragma unroll
    for (int u = 0; u < U; ++u) now[u] = ch[u];
    if (base + kThreads * U < c1) fetch(base + kThreads * U);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int c = base + u * kThreads + lane;
      if (c < c1) {
        float largest = now[u][0];
#pragma unroll
        for (int e = 1; e < 8; ++e) largest = fmaxf(largest, now[u][e]);
        raise(largest);
#pragma unroll
        for (int e = 0; e < 8; ++e) add(now[u][e]);
        if constexpr (TOP) best.add(largest, c);
      }
    }
  }
  v.t *= kLn2;

  v = join_wave(v);
  if (lane == 0) wave_sums[wave] = v;
  if constexpr (TOP) {
    if (tid == 0) top_shared.count = top_shared.survivors = top_shared.again = 0;
    // The top-th largest of each wave's maxima.
    int rank = 0;
    for (int i = 0; i < 64; ++i) {
      const float other = __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(best.m1), i));
      rank += other > best.m1 || (other == best.m1 && i < lane);
    }
    if (rank == a.top - 1) top_shared.bounds[wave] = best.m1;
  }
  __syncthreads();
  v = wave_sums[0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) v = join(v, wave_sums[w]);
  const bool last = p.parts == 1;
  if (tid == 0) {
    if (last) finish_row(a, row, v, token_logit<T>(a, row));
    else p.sums[row * p.parts + part] = v;
  }
  if constexpr (TOP) {
    float bound = top_shared.bounds[0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) bound = fmaxf(bound, top_shared.bounds[w]);
    // The top-th largest of all waves' maxima that reach the largest of these.
    // (In which order they come does not matter: the bound is a value.)
    if (best.m1 >= bound) top_shared.maxima[atomicAdd(&top_shared.survivors, 1)] = best.m1;
    __syncthreads();
    const int survivors = top_shared.survivors;
    if (tid < survivors) {
      const float mine = top_shared.maxima[tid];
      int rank = 0;
      for (int i = 0; i < survivors; ++i) rank += top_shared.maxima[i] > mine || (top_shared.maxima[i] == mine && i < tid);
      if (rank == a.top - 1) top_shared.bound = mine;
    }
    __syncthreads();
    bound = top_shared.bound;
    auto gather = [&](float value, int j) {
      if (value >= bound) {
        const int at = atomicAdd(&top_shared.count, 1);
        if (at < kMaxCandidates) top_shared.candidates[at] = key_of(value, j);
      }
    };
    if (best.m3 >= bound) top_shared.again = 1;
    if (bound > -INFINITY) {
      if (extra >= 0) gather(static_cast<float>(x[extra]), extra);
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        if ((i == 0 ? best.m1 : best.m2) >= bound) {
          const int c = i == 0 ? best.c1 : best.c2;
          Chunk<T> again;
          again.load(body + static_cast<int64_t>(c) * 8);
#pragma unroll
          for (int e = 0; e < 8; ++e) gather(again[e], shape.head + 8 * c + e);
        }
      }
    }
    __syncthreads();
    int total = top_shared.count;
    if (top_shared.again || total > kMaxCandidates) {
      TopList list{0, 0, a.top};
      float floor = -INFINITY;
      if (tid < kWaves) top_shared.bounds[tid] = -INFINITY;   // now the waves' lists' last values, as far as they are known
      __syncthreads();
      auto offer = [&](float value, int j, bool valid) {
        // (An equal value may be of an earlier token than the list's last one.)
        const bool wanted = valid && value >= bound && value >= floor;
        if (__ballot(wanted)) {
          list.offer(wanted ? key_of(value, j) : 0);
          floor = list.floor();
        }
      };
      const float mine = extra >= 0 ? static_cast<float>(x[extra]) : 0.f;
      if (wave == 0) offer(mine, extra, extra >= 0 && lane < 8);
      // Chunks come in the order of their tokens: what only equals the floor
      // stays behind it.
      for (int base = first; base < c1; base += kThreads) {
        const int c = base + lane;
        const bool valid = c < c1;
        Chunk<T> now;
        now.load(body + static_cast<int64_t>(min(c, c1 - 1)) * 8);
        float largest = now[0];
#pragma unroll
        for (int e = 1; e < 8; ++e) largest = fmaxf(largest, now[e]);
        if (__ballot(valid && largest >= bound && (largest > floor || list.last == 0))) {
          // No less than what the other waves' lists end with (equal values may
          // come in front of theirs).
#pragma unroll
          for (int w = 0; w < kWaves; ++w) bound = fmaxf(bound, top_shared.bounds[w]);
#pragma unroll
          for (int e = 0; e < 8; ++e) offer(now[e], shape.head + 8 * c + e, valid);
          if (lane == 0) top_shared.bounds[wave] = floor;
        }
      }
      if (wave == 0) offer(mine, extra, extra >= 0 && lane >= 8);
      if (lane < a.top) top_shared.candidates[wave * a.top + lane] = list.mine;
      total = kWaves * a.top;
      __syncthreads();
    }
    // A key's place is the number of larger ones; missing keys (0) stand at the end.
    if (tid < total) {
      const Key k = top_shared.candidates[tid];
      int at = 0;
      for (int i = 0; i < total; ++i) at += top_shared.candidates[i] > k || (top_shared.candidates[i] == k && i < tid);
      if (at < a.top) {
        if (last) {
          a.top_log_probs[row * a.top + at] = (key_value(k) - v.m) - logf(v.s);
          a.top_tokens[row * a.top + at] = key_token(k);
        } else {
          p.keys[(row * p.parts + part) * a.top + at] = k;
        }
      }
    }
  }
}

// A row's parts joined, by a wave.
template <typename T>
__global__ __launch_bounds__(64) void token_log_probs_join_kernel(Params p) {
  const TokenLogProbsArgs& a = p.a;
  const int lane = lane_id();
  const int64_t row = blockIdx.x;
  Sums v{kLowest, 0.f, 0.f};
  for (int i = lane; i < p.parts; i += 64) v = join(v, p.sums[row * p.parts + i]);
  v = join_wave(v);
  if (lane == 0) finish_row(a, row, v, token_logit<T>(a, row));
  if (a.top) {
    TopList list{0, 0, a.top};
    const int total = p.parts * a.top;
    for (int i = 0; i < total; i += 64) list.offer(i + lane < total ? p.keys[row * total + i + lane] : 0);
    if (lane < a.top) {
      a.top_log_probs[row * a.top + lane] = (key_value(list.mine) - v.m) - logf(v.s);
      a.top_tokens[row * a.top + lane] = key_token(list.mine);
    }
  }
}

template <typename T>
__global__ __launch_bounds__(kThreads) void token_log_probs_backward_kernel(TokenLogProbsArgs a, int parts) {
  const int tid = static_cast<int>(threadIdx.x);
  const int64_t row = blockIdx.x / parts;
  const int part = static_cast<int>(blockIdx.x % parts);
  const T* x = static_cast<const T*>(a.logits) + row * a.ldx;
  T* out = static_cast<T*>(a.grad) + row * a.ldg;
  const int64_t token = a.tokens[row];
  const float m = a.lse[2 * row], log_s = a.lse[2 * row + 1];
  const float g_h = a.g_entropy ? a.g_entropy[row] : 0.f, h = a.entropy ? a.entropy[row] : 0.f;
  float g_token = a.g_log_probs && token != a.ignore ? a.g_log_probs[row] : 0.f;
  if (token != a.ignore && (token < 0 || token >= a.V)) g_token = __builtin_nanf("");
  float g_all = g_token;
  if (a.g_top)
    for (int i = 0; i < a.top; ++i) g_all += a.g_top[row * a.top + i];
  // g_H H + G, once.
  const float base = g_all + g_h * h;
  auto at = [&](float value) {
    const float lp = (value - m) - log_s;
    return -fast_exp(lp) * (base + g_h * fmaxf(lp, kNoWeight));
  };
  const RowShape<T> shape(x, a.V);
  const int per = (shape.chunks + parts - 1) / parts;
  const int c0 = min(shape.chunks, part * per), c1 = min(shape.chunks, c0 + per);
  const T* body = x + shape.head;
  T* to = out + shape.head;
  const bool whole = (reinterpret_cast<uintptr_t>(to) & 15) == 0;
  for (int c = c0 + tid; c < c1; c += kThreads) {
    Chunk<T> ch;
    ch.load(body + static_cast<int64_t>(c) * 8);
    T o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = static_cast<T>(at(ch[e]));
    T* dst = to + static_cast<int64_t>(c) * 8;
    if (whole) {
#pragma unroll
      for (int q = 0; q < static_cast<int>(sizeof(T)) / 2; ++q)
        store16B(reinterpret_cast<char*>(dst) + 16 * q, reinterpret_cast<const u32x4*>(o)[q]);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) dst[e] = o[e];
    }
  }
  if (part == 0 && tid < shape.head) out[tid] = static_cast<T>(at(static_cast<float>(x[tid])));
  if (part == parts - 1 && tid < shape.tail) {
    const int j = a.V - shape.tail + tid;
    out[j] = static_cast<T>(at(static_cast<float>(x[j])));
  }
  __syncthreads();   // the entries below have been written
  // Entries with gradients of their own; an entry that is named twice gets the
  // sum both times.
  const int named = 1 + (a.g_top ? a.top : 0);
  if (tid < named) {
    const int64_t j = tid == 0 ? token : a.top_tokens[row * a.top + tid - 1];
    if (j < 0 || j >= a.V || (tid == 0 && token == a.ignore)) return;
    const int c = j < shape.head ? -1 : static_cast<int>((j - shape.head) / 8);
    const bool mine = c < 0 ? part == 0 : c >= shape.chunks ? part == parts - 1 : c >= c0 && c < c1;
    if (!mine) return;
    float own = j == token && token != a.ignore ? g_token : 0.f;
    if (a.g_top)
      for (int i = 0; i < a.top; ++i)
        if (a.top_tokens[row * a.top + i] == j) own += a.g_top[row * a.top + i];
    out[j] = static_cast<T>(at(static_cast<float>(x[j])) + own);
  }
}

namespace {

// Parts of a row: workgroups for four rounds of the chip, each with two steps
// of its waves at least.
int row_parts(int64_t rows, int V) {
  const int64_t want = (1024 + rows - 1) / std::max<int64_t>(rows, 1);
  return static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(want, V / (2 * kThreads * 8))));
}

template <typename T>
void launch_typed(const Params& p, hipStream_t stream) {
  const dim3 grid(static_cast<unsigned>(p.a.rows * p.parts));
  if (p.a.top) hipLaunchKernelGGL((token_log_probs_kernel<T, true>), grid, dim3(kThreads), 0, stream, p);
  else hipLaunchKernelGGL((token_log_probs_kernel<T, false>), grid, dim3(kThreads), 0, stream, p);
  if (p.parts > 1)
    hipLaunchKernelGGL((token_log_probs_join_kernel<T>), dim3(static_cast<unsigned>(p.a.rows)), dim3(64), 0, stream, p);
}

}  // namespace

int64_t token_log_probs_workspace(const TokenLogProbsArgs& a) {
  const int64_t parts = row_parts(a.rows, a.V);
  return parts == 1 ? 0 : a.rows * parts * (static_cast<int64_t>(sizeof(Key)) * a.top + static_cast<int64_t>(sizeof(Sums)));
}

void launch_token_log_probs(const TokenLogProbsArgs& a, void* workspace, hipStream_t stream) {
  Params p{a, row_parts(a.rows, a.V), nullptr, nullptr};
  p.keys = static_cast<Key*>(workspace);
  p.sums = reinterpret_cast<Sums*>(p.keys + a.rows * p.parts * a.top);
  if (a.dtype == kF32) launch_typed<float>(p, stream);
  else if (a.dtype == kF16) launch_typed<_Float16>(p, stream);
  else launch_typed<__bf16>(p, stream);
}

void launch_token_log_probs_backward(const TokenLogProbsArgs& a, hipStream_t stream) {
  const int parts = row_parts(a.rows, a.V);
  const dim3 grid(static_cast<unsigned>(a.rows * parts));
  if (a.dtype == kF32) hipLaunchKernelGGL((token_log_probs_backward_kernel<float>), grid, dim3(kThreads), 0, stream, a, parts);
  else if (a.dtype == kF16) hipLaunchKernelGGL((token_log_probs_backward_kernel<_Float16>), grid, dim3(kThreads), 0, stream, a, parts);
  else hipLaunchKernelGGL((token_log_probs_backward_kernel<__bf16>), grid, dim3(kThreads), 0, stream, a, parts);
}

}  // namespace da
