// Rows kept in 8 bits with a scale for every 128 columns (int8_rows.h): kept,
// restored, and GELU with its backward from the kept rows.
//
//   save      q, scale = int8(x)
//   restore   out = q scale                        (also rows with one scale each)
//   GELU      u = z Phi(z), and q, scale = int8(z)
//   backward  with zt = q scale:  dz = du (Phi(zt) + zt phi(zt)),  u = zt Phi(zt)
//
// Phi and phi are the normal distribution's function and density (the exact
// GELU, nn.GELU()).  The backward forms u again, which the weight gradient of
// the layer behind needs, so the forward keeps one byte an element where the
// 16-bit path keeps z and u, four.
//
// One pass over memory: 16 lanes hold a group, eight columns each, so a
// group's largest magnitude is a reduction within a lane row (four DPP
// rotations) and every access is a 16-byte one (8 bytes for the integers).
#include "da_erf.h"
#include "da_launch.h"
#include "int8_rows.h"

namespace da {

enum : int { kOpSave = 0, kOpRestore = 1, kOpGelu = 2, kOpGeluBackward = 3 };

// The group's largest magnitude, over its 16 lanes.  16-bit floats are
// compared as they were loaded, two at a time (unsigned integers order alike);
// a row's partial chunk is compared from its floats.
template <typename T>
__device__ __forceinline__ uint32_t group_amax(const RawChunk<T>& raw, int n, const float (&v)[8]) {
  uint32_t m = 0;
  if (sizeof(T) == 2 && n >= 8) {
    const uint32_t pair = max_pairs(raw.lo, 0);
    m = magnitude_bits(half_value<T>(max(pair & 0xffffu, pair >> 16)));
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) m = max(m, magnitude_bits(v[e]));
  }
  return row16_max(m);
}

// One chunk a thread: two or four of them in flight a thread take the same
// time or longer (GELU over 4096 x 1536 8.6 us; 9.5 with two, 10.4 with four).
constexpr int kGroupThreads = 256;

template <typename T, int OP>
__global__ __launch_bounds__(kGroupThreads) void int8_group_kernel(Int8GroupArgs a, FastDiv groups, uint32_t total) {
  const int lane16 = static_cast<int>(threadIdx.x) & 15;
  const uint32_t id = blockIdx.x * (kGroupThreads / 16) + (threadIdx.x >> 4);
  const int64_t row = fast_div(id, groups);
  const uint32_t g = id - static_cast<uint32_t>(row) * groups.d;
  const int col = static_cast<int>(g) * kInt8Group + lane16 * 8;
  const int n = id < total ? min(a.cols - col, 8) : 0;   // columns of this chunk
  const bool wide = a.cols >= 8;
  const T* x = static_cast<const T*>(a.x) + row * a.ldx + col;
  T* out = static_cast<T*>(a.out) + row * a.ldo + col;
  int8_t* values = a.values + row * a.ldv + col;
  float* scale = a.scales + (a.row_scale ? row : row * groups.d + g);
  float v[8], o[8];
  if constexpr (OP == kOpSave || OP == kOpGelu) {
    const RawChunk<T> raw = fetch_chunk(x, n, wide);
    chunk_floats(raw, x, n, wide, v);
    const Int8Scale s = int8_scale<T>(group_amax(raw, n, v));
    if (n > 0) {
      store_bytes(values, pack_int8<T>(v, s));
      if (lane16 == 0) *scale = s.scale;
    }
    if constexpr (OP == kOpGelu) {
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = gelu(v[e]);
      store_chunk(out, n, o);
    }
  } else {
    if (n <= 0) return;
    const u32x2 bytes = load_bytes(values);
    const float step = *scale;
    if constexpr (OP == kOpRestore) {
      unpack_int8(bytes, step, o);
      store_chunk(out, n, o);
    } else {
      float d[8];
      chunk_floats(fetch_chunk(x, n, wide), x, n, wide, d);
      unpack_int8(bytes, step, v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float density;
        const float below = normal_cdf(v[e], density);
        o[e] = v[e] * below;
        d[e] *= __builtin_fmaf(v[e] * kInvSqrt2Pi, density, below);
      }
      store_chunk(out, n, d);
      if (a.again) store_chunk(static_cast<T*>(a.again) + row * a.ldo + col, n, o);
    }
  }
}

template <typename T, int OP>
static void launch_group(const Int8GroupArgs& a, hipStream_t stream) {
  const uint32_t groups = static_cast<uint32_t>((a.cols + kInt8Group - 1) / kInt8Group);
  const uint32_t total = static_cast<uint32_t>(a.rows * groups);   // < 2^28 (checked by the caller)
  constexpr uint32_t per = kGroupThreads / 16;
  hipLaunchKernelGGL((int8_group_kernel<T, OP>), dim3((total + per - 1) / per), dim3(kGroupThreads), 0, stream, a,
                     make_fast_div(groups), total);
}

template <int OP>
static void launch_group_t(const Int8GroupArgs& a, hipStream_t stream) {
  if (a.dtype == kF16) launch_group<_Float16, OP>(a, stream);
  else if (a.dtype == kBF16) launch_group<__bf16, OP>(a, stream);
  else if constexpr (OP == kOpSave || OP == kOpRestore) launch_group<float, OP>(a, stream);
}

void launch_int8_save(const Int8GroupArgs& a, hipStream_t stream) { launch_group_t<kOpSave>(a, stream); }
void launch_int8_restore(const Int8GroupArgs& a, hipStream_t stream) { launch_group_t<kOpRestore>(a, stream); }
void launch_gelu_int8(const Int8GroupArgs& a, hipStream_t stream) { launch_group_t<kOpGelu>(a, stream); }
void launch_gelu_int8_backward(const Int8GroupArgs& a, hipStream_t stream) { launch_group_t<kOpGeluBackward>(a, stream); }

}  // namespace da
