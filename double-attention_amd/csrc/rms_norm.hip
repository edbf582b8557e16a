// Rows in 8 bits with one scale each, and the root-mean-square norm with the
// residual's addition in front of it.
//
//   s = x + r (rounded to the activations' type: the model carries it on)
//   n = s rstd w,  rstd = 1 / sqrt(mean(s^2) + eps)          fp32 statistics
//   out = n (one rounding), and / or  q, scale = int8(n)     (int8_rows.h)
//
// One pass over memory: NT threads hold a row in registers (CH chunks of
// eight columns each).  The scale of the integers needs no second reduction:
// max |n| = rstd max |s w|, so the sum of squares and the largest |s w| are
// reduced together, and q = rint(s w (rstd / scale)): one multiplication by a
// rounded factor, so where n / scale is within its roundings (some 2^-15 of a
// step) of a half of a step, either neighbour may come out.  Products s w of 16-bit
// numbers do have exact halves of steps: max |s w| / 2 without weights.
//
// Backward at dy = dL/dn and ds = dL/ds (the gradient that reaches s past the
// norm), with xh = s rstd and g = dy w:
//   dx = dr = rstd (g - xh mean(g xh)) + ds          (one rounding)
//   dw = sum over rows of dy xh                      (fp32)
// The weight's gradient is added up in an order fixed by the sizes alone: a
// thread over its workgroup's rows, the workgroups' sums by a second, small
// launch.
#include "da_launch.h"
#include "int8_rows.h"

namespace da {

// Eight parameters of type pdt from column c on, of which n exist (1 without
// parameters, 0 behind the row), fetched and used as a chunk of a row is.
__device__ __forceinline__ RawChunk<float> fetch_weight(const void* p, int pdt, int64_t c, int n, bool wide) {
  if (p == nullptr) return RawChunk<float>{u32x4{0, 0, 0, 0}, u32x4{0, 0, 0, 0}};
  if (pdt == kF32) return fetch_chunk(static_cast<const float*>(p) + c, n, wide);
  return RawChunk<float>{fetch_chunk(static_cast<const _Float16*>(p) + c, n, wide).lo, u32x4{0, 0, 0, 0}};
}
__device__ __forceinline__ void weight_floats(const RawChunk<float>& r, const void* p, int pdt, int64_t c, int n, bool wide,
                                              float (&w)[8]) {
  if (p == nullptr) {
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = 1.f;
  } else if (pdt == kF32) {
    chunk_floats(r, static_cast<const float*>(p) + c, n, wide, w);
  } else if (pdt == kF16) {
    chunk_floats(RawChunk<_Float16>{r.lo, r.hi}, static_cast<const _Float16*>(p) + c, n, wide, w);
  } else {
    chunk_floats(RawChunk<__bf16>{r.lo, r.hi}, static_cast<const __bf16*>(p) + c, n, wide, w);
  }
}

// Elements of a row from column c on, of which a chunk takes at most 8.  Rows of
// whole chunks (TAIL false) have kernels without the code for partial ones (4096 x
// 8192: forward 43 us against 52, backward 49 against 58).
template <bool TAIL>
__device__ __forceinline__ int row_left(int dim, int c) {
  return TAIL ? dim - c : c < dim ? 8 : 0;
}

// The row's sum and largest magnitude over its NT threads.
template <int NT>
__device__ __forceinline__ void row_reduce(float& sum, uint32_t& amax, float* lds) {
  sum = wave_sum_dpp(sum);
  amax = wave_max_bits(amax);
  if constexpr (NT > 64) {
    constexpr int W = NT / 64;
    if (lane_id() == 0) {
      lds[wave_id()] = sum;
      lds[W + wave_id()] = __uint_as_float(amax);
    }
    __syncthreads();
    sum = 0.f;
    amax = 0;
#pragma unroll
    for (int w = 0; w < W; ++w) {
      sum += lds[w];
      amax = max(amax, __float_as_uint(lds[W + w]));
    }
  }
}

template <int NT>
constexpr int row_block() { return NT < 256 ? 256 : NT; }

template <typename T, int NT, int CH, bool NORM, bool TAIL>
__global__ __launch_bounds__(row_block<NT>()) void row_int8_kernel(RowInt8Args a) {
  __shared__ float lds[2 * (NT / 64)];
  constexpr int ROWS = row_block<NT>() / NT;
  const int t = static_cast<int>(threadIdx.x) % NT;
  const int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / NT;
  if (row >= a.rows) return;   // whole waves of a workgroup without barriers (NT == 64)
  const T* x = static_cast<const T*>(a.x) + row * a.ldx;
  const T* r = static_cast<const T*>(a.residual) + row * a.ldr;
  const bool wide = !TAIL || a.dim >= 8;
  auto left = [&](int c) { return row_left<TAIL>(a.dim, c); };
  RawChunk<T> rx[CH], rr[CH];
  RawChunk<float> rw[CH];
#pragma unroll
  for (int k = 0; k < CH; ++k) rx[k] = fetch_chunk(x + (k * NT + t) * 8, left((k * NT + t) * 8), wide);
  if constexpr (NORM) {
    if (a.residual != nullptr) {
#pragma unroll
      for (int k = 0; k < CH; ++k) rr[k] = fetch_chunk(r + (k * NT + t) * 8, left((k * NT + t) * 8), wide);
    }
#pragma unroll
    for (int k = 0; k < CH; ++k) rw[k] = fetch_weight(a.weight, a.param_dtype, (k * NT + t) * 8, left((k * NT + t) * 8), wide);
  }
  float v[CH][8], w[CH][8];
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    const int c = (k * NT + t) * 8;
    chunk_floats(rx[k], x + c, left(c), wide, v[k]);
  }
  float sum = 0.f;
  uint32_t amax = 0;
  if constexpr (NORM) {
    if (a.residual != nullptr) {
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        const int c = (k * NT + t) * 8;
        chunk_floats(rr[k], r + c, left(c), wide, w[k]);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[k][e] = static_cast<float>(static_cast<T>(v[k][e] + w[k][e]));
        store_chunk(static_cast<T*>(a.sum) + row * a.dim + c, left(c), v[k]);
      }
    }
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const int c = (k * NT + t) * 8;
      weight_floats(rw[k], a.weight, a.param_dtype, c, left(c), wide, w[k]);
    }
#pragma unroll
    for (int k = 0; k < CH; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        sum = __builtin_fmaf(v[k][e], v[k][e], sum);
        v[k][e] *= w[k][e];
      }
  }
#pragma unroll
  for (int k = 0; k < CH; ++k)
#pragma unroll
    for (int e = 0; e < 8; ++e) amax = max(amax, magnitude_bits(v[k][e]));
  row_reduce<NT>(sum, amax, lds);
  float rstd = 1.f;
  if constexpr (NORM) rstd = 1.f / sqrtf(sum / static_cast<float>(a.dim) + a.eps);
  if constexpr (NORM) {
    if (a.out != nullptr) {
      T* out = static_cast<T*>(a.out) + row * a.dim;
#pragma unroll
      for (int k = 0; k < CH; ++k) {
        const int c = (k * NT + t) * 8;
        float o[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = v[k][e] * rstd;
        store_chunk(out + c, left(c), o);
      }
    }
    if (a.values == nullptr) return;
  }
  // The norm's values are no 16-bit floats: one rounding of s w * inverse.
  const Int8Scale s = NORM ? int8_scale<float>(amax, rstd) : int8_scale<T>(amax);
  // A row whose scale is the floor may have an inverse beyond fp32.
  const float inverse = fminf(rstd * s.inverse, 3.4028234e38f);
  int8_t* q = a.values + row * a.ldv;
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    const int c = (k * NT + t) * 8;
    if (c < a.dim) store_bytes(q + c, NORM ? pack_int8(v[k], inverse, s.keep) : pack_int8<T>(v[k], s));
  }
  if (t == 0) a.scales[row] = s.scale;
}

// Rows blockIdx.x, blockIdx.x + gridDim.x, ... of ROWS each.  `partials`
// [gridDim.x][dim]: the workgroup's share of the weight's gradient.
template <int NT>
constexpr int backward_block() { return NT == 64 ? 512 : NT; }

template <typename T, int NT, int CH, bool TAIL>
__global__ __launch_bounds__(backward_block<NT>()) void rms_norm_backward_kernel(RmsNormBackwardArgs a) {
  constexpr int ROWS = backward_block<NT>() / NT;
  // Row reductions (two sets of slots), or the sums of waves that hold a row each.
  extern __shared__ __attribute__((aligned(16))) float lds[];
  const int t = static_cast<int>(threadIdx.x) % NT;
  // A row's loads are issued while the row before it is reduced (the widest
  // rows take the registers for that, and for moving a partial chunk, themselves).
  constexpr bool EARLY = NT * CH <= 1024;
  const bool wide = EARLY && (!TAIL || a.dim >= 8);
  auto left = [&](int c) { return row_left<TAIL>(a.dim, c); };
  RawChunk<float> rw[CH];
  float w[CH][8], gw[CH][8];
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    const int c = (k * NT + t) * 8;
    rw[k] = fetch_weight(a.weight, a.param_dtype, c, left(c), wide);
#pragma unroll
    for (int e = 0; e < 8; ++e) gw[k][e] = 0.f;
  }
  const float inv_dim = 1.f / static_cast<float>(a.dim);
  const int64_t step = static_cast<int64_t>(gridDim.x) * ROWS;
  int64_t row = static_cast<int64_t>(blockIdx.x) * ROWS + threadIdx.x / NT;
  const T* const sum = static_cast<const T*>(a.sum);
  const T* const grad = static_cast<const T*>(a.grad);
  const T* const grad_sum = static_cast<const T*>(a.grad_sum);
  RawChunk<T> rv[CH], rg[CH], rs[CH];
  auto fetch_row = [&](int64_t r) {
    if (r >= a.rows) return;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const int c = (k * NT + t) * 8;
      rv[k] = fetch_chunk(sum + r * a.ldsum + c, left(c), wide);
      rg[k] = fetch_chunk(grad + r * a.ldg + c, left(c), wide);
      if (grad_sum != nullptr) rs[k] = fetch_chunk(grad_sum + r * a.ldgs + c, left(c), wide);
    }
  };
  if constexpr (EARLY) fetch_row(row);
#pragma unroll
  for (int k = 0; k < CH; ++k) {
    const int c = (k * NT + t) * 8;
    weight_floats(rw[k], a.weight, a.param_dtype, c, left(c), wide, w[k]);
  }
  int turn = 0;
  for (; row < a.rows; row += step, turn ^= 1) {
    if constexpr (!EARLY) fetch_row(row);
    // The masks of a wide row's last, partial chunk are formed again for each row:
    // kept over the loop they take more registers than there are.
    int dim = a.dim;
    if constexpr (TAIL && EARLY && NT >= 512) asm volatile("" : "+s"(dim));
    auto left_here = [&](int c) { return row_left<TAIL>(dim, c); };
    float v[CH][8], g[CH][8], d[CH][8];
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const int c = (k * NT + t) * 8;
      chunk_floats(rv[k], sum + row * a.ldsum + c, left_here(c), wide, v[k]);
      chunk_floats(rg[k], grad + row * a.ldg + c, left_here(c), wide, g[k]);
      if (grad_sum != nullptr) {
        chunk_floats(rs[k], grad_sum + row * a.ldgs + c, left_here(c), wide, d[k]);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) d[k][e] = 0.f;
      }
    }
    if constexpr (EARLY) fetch_row(row + step);
    __builtin_amdgcn_sched_barrier(0);
    float ss = 0.f, sg = 0.f;
#pragma unroll
    for (int k = 0; k < CH; ++k)
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        ss = __builtin_fmaf(v[k][e], v[k][e], ss);
        sg = __builtin_fmaf(g[k][e] * w[k][e], v[k][e], sg);
      }
    ss = wave_sum_dpp(ss);
    sg = wave_sum_dpp(sg);
    if constexpr (NT > 64) {
      // Two sets of slots, taken in turn: a wave that runs ahead writes the
      // set that no wave is reading any more.
      constexpr int W = NT / 64;
      float* slot = lds + turn * 2 * W;
      if (lane_id() == 0) {
        slot[wave_id()] = ss;
        slot[W + wave_id()] = sg;
      }
      __syncthreads();
      ss = sg = 0.f;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        ss += slot[i];
        sg += slot[W + i];
      }
    }
    const float rstd = 1.f / sqrtf(ss * inv_dim + a.eps);
    const float mean = sg * inv_dim * rstd * rstd;   // mean(g xh) rstd
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const int c = (k * NT + t) * 8;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        gw[k][e] = __builtin_fmaf(g[k][e], v[k][e] * rstd, gw[k][e]);
        d[k][e] += rstd * (g[k][e] * w[k][e] - v[k][e] * mean);
      }
      store_chunk(static_cast<T*>(a.grad_x) + row * a.dim + c, left_here(c), d[k]);
    }
  }
  if (a.partials == nullptr) return;
  float* part = a.partials + static_cast<int64_t>(blockIdx.x) * a.dim;
  if constexpr (NT > 64) {
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      const int c = (k * NT + t) * 8;
      store_chunk(part + c, left(c), gw[k]);
    }
  } else {
    // The waves' sums side by side in LDS, then added in the waves' order.
#pragma unroll
    for (int k = 0; k < CH; ++k) {
      float* at = lds + (wave_id() * CH + k) * 512 + t * 8;
      *reinterpret_cast<f32x4*>(at) = f32x4{gw[k][0], gw[k][1], gw[k][2], gw[k][3]};
      *reinterpret_cast<f32x4*>(at + 4) = f32x4{gw[k][4], gw[k][5], gw[k][6], gw[k][7]};
    }
    __syncthreads();
    for (int c = static_cast<int>(threadIdx.x); c < a.dim; c += backward_block<NT>()) {
      float sum = lds[c];
#pragma unroll
      for (int q = 1; q < ROWS; ++q) sum += lds[q * CH * 512 + c];
      part[c] = sum;
    }
  }
}

// out[c] = sum over the workgroups b of partials[b][c].  A workgroup takes 16
// columns, 64 threads each: thread r adds workgroups r, r + 64, ... in order,
// the sums meet four to a wave and then wave by wave.
constexpr int kSumCols = 16, kSumRuns = 64;
template <typename T>
__global__ __launch_bounds__(kSumCols * kSumRuns) void rms_norm_weight_kernel(const float* partials, int blocks, int dim, T* out) {
  __shared__ float lds[kSumRuns / 4][kSumCols];
  const int c = static_cast<int>(threadIdx.x) % kSumCols, r = static_cast<int>(threadIdx.x) / kSumCols;
  const int col = static_cast<int>(blockIdx.x) * kSumCols + c;
  const float* p = partials + min(col, dim - 1);
  float sum = 0.f;
  for (int b0 = r; b0 < blocks; b0 += 8 * kSumRuns) {
    float v[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) v[u] = p[static_cast<int64_t>(min(b0 + u * kSumRuns, blocks - 1)) * dim];
#pragma unroll
    for (int u = 0; u < 8; ++u) sum += b0 + u * kSumRuns < blocks ? v[u] : 0.f;
  }
  sum = group_sum(sum);   // the wave's four threads of this column
  if (lane_id() < kSumCols) lds[wave_id()][c] = sum;
  __syncthreads();
  if (r == 0 && col < dim) {
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < kSumRuns / 4; ++i) sum += lds[i][c];
    out[col] = static_cast<T>(sum);
  }
}

template <typename T, int NT, int CH, bool NORM>
static void launch_row_k(const RowInt8Args& a, hipStream_t stream) {
  constexpr int ROWS = row_block<NT>() / NT;
  const dim3 grid(static_cast<unsigned>((a.rows + ROWS - 1) / ROWS)), block(row_block<NT>());
  if (a.dim % 8) hipLaunchKernelGGL((row_int8_kernel<T, NT, CH, NORM, true>), grid, block, 0, stream, a);
  else hipLaunchKernelGGL((row_int8_kernel<T, NT, CH, NORM, false>), grid, block, 0, stream, a);
}

template <typename T, bool NORM>
static void launch_row_t(const RowInt8Args& a, hipStream_t stream) {
  if (a.dim <= 512) launch_row_k<T, 64, 1, NORM>(a, stream);
  else if (a.dim <= 1024) launch_row_k<T, 64, 2, NORM>(a, stream);
  else if (a.dim <= 2048) launch_row_k<T, 256, 1, NORM>(a, stream);
  else if (a.dim <= 4096) launch_row_k<T, 256, 2, NORM>(a, stream);
  else if (a.dim <= 8192) launch_row_k<T, 256, 4, NORM>(a, stream);
  else if (a.dim <= 16384) launch_row_k<T, 1024, 2, NORM>(a, stream);
  else if constexpr (!NORM) {
    if (a.dim <= 32768) launch_row_k<T, 1024, 4, NORM>(a, stream);
    else launch_row_k<T, 1024, 8, NORM>(a, stream);
  }
}

void launch_row_int8(const RowInt8Args& a, bool norm, hipStream_t stream) {
  if (norm) {
    if (a.dtype == kF16) launch_row_t<_Float16, true>(a, stream);
    else launch_row_t<__bf16, true>(a, stream);
  } else if (a.dtype == kF16) {
    launch_row_t<_Float16, false>(a, stream);
  } else if (a.dtype == kBF16) {
    launch_row_t<__bf16, false>(a, stream);
  } else {
    launch_row_t<float, false>(a, stream);
  }
}

// Eight waves a CU, in one workgroup where a wave holds a row (half the partial
// sums of two workgroups: 3885 x 1001 11.2 us and 2.8 for the sums against 11.7
// and 3.9), else in two of four (or of eight, over 4096 columns).  16384 x 2048 with
// two took 49 us, with one 65 (the rows' loads do not fill the memory's queues),
// with four 55 (the partial sums).
int rms_norm_backward_blocks(int64_t rows, int dim) {
  const int64_t per = dim <= 1024 ? 8 : 1, most = dim <= 1024 ? 256 : 512;
  const int64_t blocks = (rows + per - 1) / per;
  return static_cast<int>(blocks < most ? blocks : most);
}

template <typename T, int NT, int CH>
static void launch_backward_k(const RmsNormBackwardArgs& a, hipStream_t stream) {
  const size_t lds = NT > 64 ? 4 * (NT / 64) * sizeof(float) : backward_block<NT>() / NT * CH * 512 * sizeof(float);
  const dim3 grid(rms_norm_backward_blocks(a.rows, a.dim)), block(backward_block<NT>());
  if (a.dim % 8) hipLaunchKernelGGL((rms_norm_backward_kernel<T, NT, CH, true>), grid, block, lds, stream, a);
  else hipLaunchKernelGGL((rms_norm_backward_kernel<T, NT, CH, false>), grid, block, lds, stream, a);
}

template <typename T>
static void launch_backward_t(const RmsNormBackwardArgs& a, hipStream_t stream) {
  if (a.dim <= 512) launch_backward_k<T, 64, 1>(a, stream);
  else if (a.dim <= 1024) launch_backward_k<T, 64, 2>(a, stream);
  else if (a.dim <= 2048) launch_backward_k<T, 256, 1>(a, stream);
  else if (a.dim <= 4096) launch_backward_k<T, 256, 2>(a, stream);
  else if (a.dim <= 8192) launch_backward_k<T, 512, 2>(a, stream);
  else launch_backward_k<T, 512, 4>(a, stream);
}

void launch_rms_norm_backward(const RmsNormBackwardArgs& a, hipStream_t stream) {
  if (a.rows == 0) {
    // No rows: the weight's gradient is a sum over no workgroups.
  } else if (a.dtype == kF16) launch_backward_t<_Float16>(a, stream);
  else launch_backward_t<__bf16>(a, stream);
  if (a.partials == nullptr) return;
  const int blocks = rms_norm_backward_blocks(a.rows, a.dim);
  const dim3 grid((a.dim + kSumCols - 1) / kSumCols);
  if (a.param_dtype == kF32)
    hipLaunchKernelGGL((rms_norm_weight_kernel<float>), grid, dim3(kSumCols * kSumRuns), 0, stream, a.partials, blocks, a.dim, static_cast<float*>(a.grad_weight));
  else if (a.param_dtype == kF16)
    hipLaunchKernelGGL((rms_norm_weight_kernel<_Float16>), grid, dim3(kSumCols * kSumRuns), 0, stream, a.partials, blocks, a.dim, static_cast<_Float16*>(a.grad_weight));
  else
    hipLaunchKernelGGL((rms_norm_weight_kernel<__bf16>), grid, dim3(kSumCols * kSumRuns), 0, stream, a.partials, blocks, a.dim, static_cast<__bf16*>(a.grad_weight));
}

}  // namespace da
