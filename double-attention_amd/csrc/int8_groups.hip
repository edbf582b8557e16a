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

__device__ __forceinline__ uint32_t group_amax(const float (&v)[8]) {
  uint32_t m = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) m = max(m, magnitude_bits(v[e]));
  return row16_max(m);
}

constexpr int kGroupThreads = 256;

template <typename T, int OP, int U>
__global__ __launch_bounds__(kGroupThreads) void int8_group_kernel(Int8GroupArgs a, FastDiv groups, uint32_t total) {
  const int lane16 = static_cast<int>(threadIdx.x) & 15;
  const uint32_t first = blockIdx.x * (kGroupThreads / 16 * U) + (threadIdx.x >> 4);
  const T* x = static_cast<const T*>(a.x);
  T* out = static_cast<T*>(a.out);
  int64_t row[U];
  int col[U], n[U];
  RawChunk<T> raw[U];
  u32x2 bytes[U];
  float scale[U];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    const uint32_t id = first + u * (kGroupThreads / 16);
    const uint32_t r = fast_div(id, groups);
    const uint32_t g = id - r * groups.d;
    row[u] = r;
    col[u] = static_cast<int>(g) * kInt8Group + lane16 * 8;
    n[u] = id < total ? min(a.cols - col[u], 8) : 0;
    if constexpr (OP != kOpRestore) raw[u] = fetch_chunk(x + row[u] * a.ldx + col[u], n[u]);
    if constexpr (OP == kOpRestore || OP == kOpGeluBackward) {
      bytes[u] = u32x2{0, 0};
      scale[u] = 0.f;
      if (n[u] > 0) {
        bytes[u] = load_bytes(a.values + row[u] * a.ldv + col[u]);
        scale[u] = a.scales[a.row_scale ? row[u] : row[u] * groups.d + g];
      }
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    float v[8], o[8];
    if constexpr (OP == kOpSave || OP == kOpGelu) {
      chunk_floats(raw[u], x + row[u] * a.ldx + col[u], n[u], v);
      const Int8Scale s = int8_scale(group_amax(v));
      if (n[u] > 0) {
        store_bytes(a.values + row[u] * a.ldv + col[u], pack_int8(v, s.inverse, s.keep));
        if (lane16 == 0) a.scales[row[u] * groups.d + col[u] / kInt8Group] = s.scale;
      }
      if constexpr (OP == kOpGelu) {
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = 0.5f * v[e] * (1.f + erf_fast(v[e] * kSqrtHalf));
        store_chunk(out + row[u] * a.ldo + col[u], n[u], o);
      }
    } else if constexpr (OP == kOpRestore) {
      unpack_int8(bytes[u], scale[u], o);
      store_chunk(out + row[u] * a.ldo + col[u], n[u], o);
    } else {
      float d[8];
      chunk_floats(raw[u], x + row[u] * a.ldx + col[u], n[u], d);
      unpack_int8(bytes[u], scale[u], v);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        float density;
        const float below = 0.5f + 0.5f * erf_density(v[e] * kSqrtHalf, density);   // density = exp(-v^2 / 2)
        o[e] = v[e] * below;
        d[e] *= __builtin_fmaf(v[e] * kInvSqrt2Pi, density, below);
      }
      store_chunk(out + row[u] * a.ldo + col[u], n[u], d);
      if (a.again) store_chunk(static_cast<T*>(a.again) + row[u] * a.ldo + col[u], n[u], o);
    }
  }
}

template <typename T, int OP, int U>
static void launch_group(const Int8GroupArgs& a, hipStream_t stream) {
  const uint32_t groups = static_cast<uint32_t>((a.cols + kInt8Group - 1) / kInt8Group);
  const uint32_t total = static_cast<uint32_t>(a.rows * groups);   // < 2^31 (checked by the caller)
  constexpr uint32_t per = kGroupThreads / 16 * U;
  hipLaunchKernelGGL((int8_group_kernel<T, OP, U>), dim3((total + per - 1) / per), dim3(kGroupThreads), 0, stream, a,
                     make_fast_div(groups), total);
}

template <int OP>
static void launch_group_t(const Int8GroupArgs& a, hipStream_t stream) {
  constexpr int U = 2;
  if (a.dtype == kF16) launch_group<_Float16, OP, U>(a, stream);
  else if (a.dtype == kBF16) launch_group<__bf16, OP, U>(a, stream);
  else if constexpr (OP == kOpSave || OP == kOpRestore) launch_group<float, OP, U>(a, stream);
}

void launch_int8_save(const Int8GroupArgs& a, hipStream_t stream) { launch_group_t<kOpSave>(a, stream); }
void launch_int8_restore(const Int8GroupArgs& a, hipStream_t stream) { launch_group_t<kOpRestore>(a, stream); }
void launch_gelu_int8(const Int8GroupArgs& a, hipStream_t stream) { launch_group_t<kOpGelu>(a, stream); }
void launch_gelu_int8_backward(const Int8GroupArgs& a, hipStream_t stream) { launch_group_t<kOpGeluBackward>(a, stream); }

}  // namespace da
