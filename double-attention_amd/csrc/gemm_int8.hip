// Linear layer on 8-bit integers:
//
//   out[j][i] = act(xs[j] ws[i] sum_k X[j][k] W[i][k] + bias[i])  (+ residual[j][i])
//
// X [rows, K] are tokens and W [N, K] output channels, both 8-bit rows with
// one fp32 scale each (int8_rows.h).  The sums are 32-bit integers, so they
// are exact for any order of k (K <= 65536: |sum| <= 2^14 K <= 2^30); the
// scales, bias, GELU and the residual are fp32, the result is rounded once
// and, with a residual, added and rounded again (the order of an unfused
// x + linear(...)).
//
// Tiles: 128 channels x 128 tokens per workgroup, four waves of 64 x 64 in
// 16x16x64 MFMA blocks (v_mfma_i32_16x16x64_i8), K in stages of 128 bytes
// through a ring of two XOR-swizzled LDS buffers filled by global->LDS DMA:
// the layout of the 16-bit GEMM at twice the k per byte.  A stage's chunks
// behind K (the pitch is a multiple of 16, the bytes between K and the pitch
// are anything) are cut off in W's fragments: zero times anything is zero.
#include "da_erf.h"
#include "da_launch.h"
#include "da_tile.h"
#include "int8_rows.h"

namespace da {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kI8Tile = 128;
constexpr int kI8Stage = 128;   // bytes of k
typedef XorTile<kI8Tile, kI8Stage / 16, false> TileI8;

// The first n of a fragment's 16 bytes, zeros behind.
__device__ __forceinline__ i32x4 first_bytes(i32x4 v, int n) {
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const int have = n - 4 * d;
    v[d] = have >= 4 ? v[d] : have <= 0 ? 0 : static_cast<int>(static_cast<uint32_t>(v[d]) & (0xffffffffu >> (32 - 8 * have)));
  }
  return v;
}

template <typename T, int EPI>
__global__ __launch_bounds__(256) void linear_int8_kernel(LinearInt8Args a, int tiles_i, int tiles_j) {
  constexpr int STAGE = 2 * TileI8::BYTES;
  constexpr int PER_WAVE = 2 * TileI8::LOADS / 4;
  __shared__ __attribute__((aligned(1024))) char lds[2 * STAGE];
  const int tiles = tiles_i * tiles_j;
  const int w = static_cast<int>(blockIdx.x);
  // Workgroups go to the XCDs round-robin: one XCD takes a contiguous range
  // of tiles, whose blocks of the larger operand its L2 then fetches once.
  const int xcd = w % kXcds;
  const int per = tiles / kXcds, rem = tiles % kXcds;
  const int tile = xcd * per + min(xcd, rem) + w / kXcds;
  const bool i_fast = tiles_i <= tiles_j;
  const int64_t i0 = static_cast<int64_t>(i_fast ? tile % tiles_i : tile / tiles_j) * kI8Tile;
  const int64_t j0 = static_cast<int64_t>(i_fast ? tile / tiles_i : tile % tiles_j) * kI8Tile;
  const int lane = lane_id();
  const int c = lane & 15;
  const int g = lane >> 4;
  const int wave = uniform_wave();
  const int wi = wave & 1, wj = wave >> 1;
  const int K = a.K;
  const int n_stages = (K + kI8Stage - 1) / kI8Stage;
  const int last_chunk = (K - 1) / 16 * 16;

  const int8_t* src[PER_WAVE];
  int kchunk[PER_WAVE], slot[PER_WAVE];
#pragma unroll
  for (int n = 0; n < PER_WAVE; ++n) {
    const int j = n * 4 + wave;
    slot[n] = j * 1024;
    int r, ck;
    if (j < TileI8::LOADS) {
      TileI8::slot_chunk(j * 64 + lane, r, ck);
      src[n] = a.w + min(i0 + r, a.N - 1) * a.ldw;
    } else {
      TileI8::slot_chunk((j - TileI8::LOADS) * 64 + lane, r, ck);
      src[n] = a.x + min(j0 + r, a.rows - 1) * a.ldx;
    }
    kchunk[n] = ck * 16;
  }
  auto issue = [&](char* buf, int k0) {
#pragma unroll
    for (int n = 0; n < PER_WAVE; ++n) dma16(src[n] + min(k0 + kchunk[n], last_chunk), buf + slot[n]);
  };

  i32x4 acc[4][4];
#pragma unroll
  for (int p = 0; p < 4; ++p)
#pragma unroll
    for (int q = 0; q < 4; ++q) acc[p][q] = i32x4{0, 0, 0, 0};
  const int afrag[2] = {TileI8::base(wi * 64 + c, g, 0), TileI8::base(wi * 64 + c, g, 1)};
  const int bfrag[2] = {TileI8::BYTES + TileI8::base(wj * 64 + c, g, 0), TileI8::BYTES + TileI8::base(wj * 64 + c, g, 1)};

  auto step = [&](int st, char* cur, char* nxt) {
    wait_vmem();
    lds_barrier();
    i32x4 af[2][4], bf[2][4];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
#pragma unroll
      for (int p = 0; p < 4; ++p) af[kk][p] = *reinterpret_cast<const i32x4*>(cur + afrag[kk] + p * TileI8::ROW_BLOCK);
#pragma unroll
      for (int q = 0; q < 4; ++q) bf[kk][q] = *reinterpret_cast<const i32x4*>(cur + bfrag[kk] + q * TileI8::ROW_BLOCK);
    }
    if (st + 1 < n_stages) issue(nxt, (st + 1) * kI8Stage);
    const int left = K - st * kI8Stage;
    if (left < kI8Stage) {
#pragma unroll
      for (int kk = 0; kk < 2; ++kk)
#pragma unroll
        for (int p = 0; p < 4; ++p) af[kk][p] = first_bytes(af[kk][p], left - kk * 64 - g * 16);
    }
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int p = 0; p < 4; ++p)
#pragma unroll
        for (int q = 0; q < 4; ++q) acc[p][q] = __builtin_amdgcn_mfma_i32_16x16x64_i8(af[kk][p], bf[kk][q], acc[p][q], 0, 0, 0);
  };
  issue(lds, 0);
  int st = 0;
  for (; st + 1 < n_stages; st += 2) {
    step(st, lds, lds + STAGE);
    step(st + 1, lds + STAGE, lds);
  }
  if (st < n_stages) step(st, lds, lds + STAGE);

  // Lane (c, g) holds rows i = 16p + 4g + r of column j = 16q + c.  Each wave
  // stages its 64 x 64 block in LDS as [j][i] rows and writes them back in
  // 16-byte chunks along i.
  constexpr int ROWB = 64 * 2 + 16;
  static_assert(64 * ROWB <= STAGE / 2, "a wave's staging block fits its quarter of the stage buffers");
  __syncthreads();
  char* stage_w = lds + wave * (STAGE / 2);
  float ws[4][4], bias[4][4];
#pragma unroll
  for (int p = 0; p < 4; ++p)
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int64_t i = min(i0 + wi * 64 + p * 16 + 4 * g + r, a.N - 1);
      ws[p][r] = a.w_scales[i];
      bias[p][r] = a.bias ? load_scalar(a.bias, a.bias_dtype, i) : 0.f;
    }
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const float xs = a.x_scales[min(j0 + wj * 64 + q * 16 + c, a.rows - 1)];
#pragma unroll
    for (int p = 0; p < 4; ++p) {
      typename Elem<T>::v4 o;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        float v = __builtin_fmaf(static_cast<float>(acc[p][q][r]) * xs, ws[p][r], bias[p][r]);
        if constexpr ((EPI & kGemmActGelu) != 0) v = 0.5f * v * (1.f + erf_fast(v * kSqrtHalf));
        o[r] = static_cast<T>(v);
      }
      *reinterpret_cast<typename Elem<T>::v4*>(stage_w + (q * 16 + c) * ROWB + (p * 16 + 4 * g) * 2) = o;
    }
  }
  T* out = static_cast<T*>(a.out);
#pragma unroll
  for (int pass = 0; pass < 8; ++pass) {
    const int jr = pass * 8 + lane / 8;
    const int ic = (lane % 8) * 8;
    const int64_t j = j0 + wj * 64 + jr;
    const int64_t i = i0 + wi * 64 + ic;
    const u32x4 v = *reinterpret_cast<const u32x4*>(stage_w + jr * ROWB + ic * 2);
    if (j >= a.rows || i >= a.N) continue;
    const int n = static_cast<int>(min(a.N - i, static_cast<int64_t>(8)));
    T* dst = out + j * a.N + i;
    const typename Elem<T>::v8 e8 = __builtin_bit_cast(typename Elem<T>::v8, v);
    if constexpr ((EPI & 2) != 0) {
      float res[8];
      load_chunk(static_cast<const T*>(a.residual) + j * a.ldr + i, n, res);
#pragma unroll
      for (int e = 0; e < 8; ++e) res[e] += static_cast<float>(e8[e]);
      store_chunk(dst, n, res);
    } else if (n == 8) {
      store16B_any(dst, v);
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e)
        if (e < n) dst[e] = e8[e];
    }
  }
}

template <typename T, int EPI>
static void launch_linear_int8_k(const LinearInt8Args& a, hipStream_t stream) {
  const int ti = static_cast<int>((a.N + kI8Tile - 1) / kI8Tile), tj = static_cast<int>((a.rows + kI8Tile - 1) / kI8Tile);
  hipLaunchKernelGGL((linear_int8_kernel<T, EPI>), dim3(ti * tj), dim3(256), 0, stream, a, ti, tj);
}

template <typename T>
static void launch_linear_int8_t(const LinearInt8Args& a, hipStream_t stream) {
  switch ((a.act == kGemmActGelu ? kGemmActGelu : 0) | (a.residual ? 2 : 0)) {
    case 0: launch_linear_int8_k<T, 0>(a, stream); break;
    case kGemmActGelu: launch_linear_int8_k<T, kGemmActGelu>(a, stream); break;
    case 2: launch_linear_int8_k<T, 2>(a, stream); break;
    default: launch_linear_int8_k<T, kGemmActGelu | 2>(a, stream); break;
  }
}

void launch_linear_int8(const LinearInt8Args& a, hipStream_t stream) {
  if (a.dtype == kF16) launch_linear_int8_t<_Float16>(a, stream);
  else launch_linear_int8_t<__bf16>(a, stream);
}

}  // namespace da
