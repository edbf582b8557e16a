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
// The tile kernel takes BI channels x BJ tokens a workgroup in 16x16x64 MFMA
// blocks (v_mfma_i32_16x16x64_i8), K in stages of 128 bytes through a ring of
// NST XOR-swizzled LDS buffers filled by global->LDS DMA: the layout of the
// 16-bit GEMM at twice the k per byte.  A stage is two halves of 64 bytes, and
// the fragments of a half are read from LDS while the half before it is
// multiplied; the workgroup's one barrier a stage falls between the halves, so
// the matrix cores have operands on both sides of it, and the buffer that it
// frees is loaded again at once.  A stage's chunks behind K (the pitch is a
// multiple of 16, the bytes between K and the pitch are anything) are cut off
// in W's fragments: zero times anything is zero.
#include "da_erf.h"
#include "da_launch.h"
#include "da_tile.h"
#include "int8_rows.h"

namespace da {

typedef int i32x4 __attribute__((ext_vector_type(4)));

constexpr int kI8Stage = 128;   // bytes of k

// The layer's result in fp32, the same bits in every kernel: two roundings
// (the scaled sum, the sum with the bias), then GELU's.  The empty statement
// keeps the compiler from folding the last of them into a conversion to 16
// bits (v_fma_mixlo_f16 rounds once where v_fma_f32 and v_cvt_f16_f32 round
// twice), which it would do in one kernel and not in another.
template <int EPI>
__device__ __forceinline__ float linear_result(int sum, float x_scale, float w_scale, float bias) {
  float y = __builtin_fmaf(static_cast<float>(sum) * x_scale, w_scale, bias);
  if constexpr ((EPI & kGemmActGelu) != 0) y = gelu(y);
  asm("" : "+v"(y));
  return y;
}

// The first n of a fragment's 16 bytes, zeros behind.
__device__ __forceinline__ i32x4 first_bytes(i32x4 v, int n) {
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    const int have = n - 4 * d;
    v[d] = have >= 4 ? v[d] : have <= 0 ? 0 : static_cast<int>(static_cast<uint32_t>(v[d]) & (0xffffffffu >> (32 - 8 * have)));
  }
  return v;
}

// lds_barrier() with waits that the compiler takes into its own accounts: it
// then knows that the fragments read before the barrier have arrived, and
// does not wait for the ones read behind it before using them.
__device__ __forceinline__ void counted_barrier() {
  __builtin_amdgcn_s_waitcnt(0xC07F);   // lgkmcnt(0)
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
}

// A workgroup's tile: BI channels x BJ tokens over NWI x NWJ waves, NST stages
// in LDS.  AHEAD > 0: stages that the L2 is asked for AHEAD stages before they
// are multiplied (see below).  XS > 0: the tokens are 16-bit rows of up to XS
// stages, quantized into LDS by the workgroup, and only W goes through the ring.
template <int BI, int BJ, int NWI, int NWJ, int NST, int AHEAD = 0, int XS = 0>
struct I8Cfg {
  static constexpr int kAhead = AHEAD, kXS = XS;
  static constexpr int kBI = BI, kBJ = BJ, kNWI = NWI, kNWJ = NWJ, kNST = NST;
  static constexpr int WAVES = NWI * NWJ;
  static constexpr int WI = BI / NWI, WJ = BJ / NWJ;    // a wave's block
  static constexpr int NA = WI / 16, NB = WJ / 16;      // its MFMA blocks
  typedef XorTile<BI, kI8Stage / 16, false> TileW;
  typedef XorTile<BJ, kI8Stage / 16, false> TileX;
  static constexpr int STAGE = TileW::BYTES + (XS ? 0 : TileX::BYTES);
  static constexpr int STAGE_LOADS = TileW::LOADS + (XS ? 0 : TileX::LOADS);
  static constexpr int LOADS = STAGE_LOADS / WAVES;     // a wave's, each stage
  static_assert(STAGE_LOADS % WAVES == 0, "every wave loads as much");
  // Behind the ring: the corner that the L2's asking writes, the quantized
  // tokens and their scales.
  static constexpr int X_AT = NST * STAGE + (AHEAD ? 256 : 0);
  static constexpr int LDS = X_AT + XS * TileX::BYTES + (XS ? 4 * BJ : 0);
  static constexpr int ROWB = WI * 2 + 16;              // bytes of a staged output row
  static_assert(TileW::LOADS % WAVES == 0 && WAVES % 2 == 0, "a load of all waves is of one operand, and 16 rows or a multiple");
  static constexpr int PARAMS = 2 * BI + BJ;            // floats that the epilogue reads
  static_assert(16 * ROWB * WAVES + 4 * PARAMS <= NST * STAGE, "the epilogue's rows and parameters fit the stage buffers");
  static_assert(BI <= 64 * WAVES && BJ <= 64 * WAVES, "a thread fetches one channel's and one token's parameters");
};

// Tile `t` of the launch's tiles: bands of eight channel tiles, token tiles
// outside of channel tiles in each, so that the tiles in flight on an XCD (a
// contiguous range of t) share both operands in its L2.
__device__ __forceinline__ void i8_tile(int t, int tiles_i, int tiles_j, int& ti, int& tj) {
  const int band = t / (8 * tiles_j);
  const int wide = min(8, tiles_i - band * 8);
  const int r = t - band * 8 * tiles_j;
  ti = band * 8 + r % wide;
  tj = r / wide;
}

// The scales of a wave's rows, lane r's of row r: a chain of some 25
// instructions, formed once instead of for each row.  `largest`: 16-bit
// magnitudes.
template <typename T>
struct LaneScales {
  Int8Scale own;
  uint64_t divide;
  __device__ __forceinline__ explicit LaneScales(uint32_t largest)
      : own(int8_scale<T>(magnitude_bits(half_value<T>(largest)))), divide(__builtin_amdgcn_ballot_w64(own.divide)) {}
  __device__ __forceinline__ Int8Scale of(int r) const {
    const auto lane_r = [&](uint32_t v) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(v, r)); };
    return Int8Scale{__uint_as_float(lane_r(__float_as_uint(own.scale))), __uint_as_float(lane_r(__float_as_uint(own.inverse))),
                     lane_r(own.keep), (divide >> r & 1) != 0};
  }
};

// Eight 16-bit floats as they were loaded, in their row's scale.
template <typename T>
__device__ __forceinline__ u32x2 pack_bits(u32x4 bits, const Int8Scale& s) {
  const typename Elem<T>::v8 h = __builtin_bit_cast(typename Elem<T>::v8, bits);
  float v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = static_cast<float>(h[e]);
  return pack_int8<T>(v, s);
}

// The tokens' 8-bit rows in LDS, in the layout of their stages (XS > 0; zeros
// behind K), and their scales.  A wave takes every WAVES-th row, its lanes eight
// columns each of 512 at a time; W's first stages (`first_loads`) are asked for
// behind the tokens' and arrive while these are quantized.
template <typename T, typename Cfg, typename F>
__device__ __forceinline__ void quantize_tokens(const LinearInt8Args& a, int64_t j0, int n_stages, char* lds, F first_loads) {
  if constexpr (Cfg::kXS == 0) {
    first_loads();
  } else {
    typedef typename Cfg::TileX TileX;
    constexpr int ROWS = Cfg::kBJ / Cfg::WAVES, PASSES = (Cfg::kXS * kI8Stage + 511) / 512;
    char* const values = lds + Cfg::X_AT;
    float* const scales = reinterpret_cast<float*>(values + Cfg::kXS * TileX::BYTES);
    const int lane = lane_id(), wave = uniform_wave();
    u32x4 raw[ROWS][PASSES];
    const bool wide = a.K >= 8;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const T* x = static_cast<const T*>(a.x) + min(j0 + wave + r * Cfg::WAVES, a.rows - 1) * a.ldx;
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const int k = p * 512 + lane * 8;
        raw[r][p] = fetch_bits(x + k, a.K - k, wide);
      }
    }
    first_loads();
    if (a.K % 8) {
#pragma unroll
      for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int p = 0; p < PASSES; ++p) raw[r][p] = chunk_bits(raw[r][p], a.K - p * 512 - lane * 8, wide);
    }
    uint32_t mine = 0;
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      uint32_t pair = 0;
#pragma unroll
      for (int p = 0; p < PASSES; ++p) pair = max_pairs(raw[r][p], pair);
      const uint32_t largest = wave_max_bits(max(pair & 0xffffu, pair >> 16));
      mine = lane == r ? largest : mine;
    }
    const LaneScales<T> rows(mine);
#pragma unroll
    for (int r = 0; r < ROWS; ++r) {
      const Int8Scale s = rows.of(r);
      const int row = wave + r * Cfg::WAVES;
#pragma unroll
      for (int p = 0; p < PASSES; ++p) {
        const int k = p * 512 + lane * 8, st = k / kI8Stage;
        const u32x2 q = pack_bits<T>(raw[r][p], s);
        if (st < n_stages)
          *reinterpret_cast<u32x2*>(values + st * TileX::BYTES + TileX::offset(row, k % kI8Stage / 16) + k % 16) = q;
      }
    }
    if (lane < ROWS) scales[wave + lane * Cfg::WAVES] = rows.own.scale;
  }
}

template <typename T, int EPI, typename Cfg>
__global__ __launch_bounds__(64 * Cfg::WAVES) void linear_int8_kernel(LinearInt8Args a, int tiles_i, int tiles_j) {
  typedef typename Cfg::TileW TileW;
  typedef typename Cfg::TileX TileX;
  constexpr int NA = Cfg::NA, NB = Cfg::NB, NST = Cfg::kNST, STAGE = Cfg::STAGE, LOADS = Cfg::LOADS;
  constexpr int AHEAD = Cfg::kAhead, EXTRA = AHEAD ? 1 : 0, XS = Cfg::kXS;
  __shared__ __attribute__((aligned(1024))) char lds[Cfg::LDS];
  const int tiles = tiles_i * tiles_j;
  const int w = static_cast<int>(blockIdx.x);
  // Workgroups go to the XCDs round-robin: one XCD takes a contiguous range.
  const int xcd = w % kXcds;
  const int per = tiles / kXcds, rem = tiles % kXcds;
  int ti, tj;
  i8_tile(xcd * per + min(xcd, rem) + w / kXcds, tiles_i, tiles_j, ti, tj);
  const int64_t i0 = static_cast<int64_t>(ti) * Cfg::kBI;
  const int64_t j0 = static_cast<int64_t>(tj) * Cfg::kBJ;
  const int lane = lane_id();
  const int c = lane & 15;
  const int g = lane >> 4;
  const int wave = uniform_wave();
  const int wi = wave % Cfg::kNWI, wj = wave / Cfg::kNWI;
  const int K = a.K;
  const int n_stages = (K + kI8Stage - 1) / kI8Stage;
  const int last_chunk = (K - 1) / 16 * 16;

  // The epilogue's scales and biases, one channel and one token a thread,
  // fetched ahead of the stages and without branches: they land with the first.
  const int tid = static_cast<int>(threadIdx.x);
  const int64_t chan = min(i0 + min(tid, Cfg::kBI - 1), a.N - 1);
  const float chan_scale = a.w_scales[chan];
  const float tok_scale = XS ? 0.f : a.x_scales[min(j0 + min(tid, Cfg::kBJ - 1), a.rows - 1)];
  const bool has_bias = a.bias != nullptr;
  const ScalarHalves bias_raw = fetch_scalar(has_bias ? a.bias : a.w_scales, has_bias ? a.bias_dtype : kF32, chan);

  // A wave's loads of a stage: lane offsets from the tile's first row
  // (its rows span less than 2^32 bytes: the host checks the pitches).
  uint32_t off[LOADS];
  int kchunk = 0;
#pragma unroll
  for (int n = 0; n < LOADS; ++n) {
    const int j = n * Cfg::WAVES + wave;
    int r, ck;
    if (j < TileW::LOADS) {
      TileW::slot_chunk(j * 64 + lane, r, ck);
      off[n] = static_cast<uint32_t>(min(static_cast<int64_t>(r), a.N - 1 - i0) * a.ldw);
    } else {
      TileX::slot_chunk((j - TileW::LOADS) * 64 + lane, r, ck);
      off[n] = static_cast<uint32_t>(min(static_cast<int64_t>(r), a.rows - 1 - j0) * a.ldx);
    }
    kchunk = ck * 16;   // the same for all n: their rows are 8 WAVES apart, and the swizzle repeats every 16
  }
  const int8_t* const w0 = a.w + i0 * a.ldw;
  const int8_t* const x0 = static_cast<const int8_t*>(a.x) + j0 * a.ldx;
  // A stage's loads from..to: scalar bases (made anew, or the compiler keeps a
  // 64-bit address a load) plus the lane's offset.
  struct StageLoads {
    const int8_t* w;
    const int8_t* x;
    uint32_t kc;
    char* buf;
  };
  auto stage_loads = [&](int st) {
    const int k0 = st * kI8Stage;
    return StageLoads{uniform_ptr(w0 + k0), uniform_ptr(x0 + k0), static_cast<uint32_t>(min(kchunk, last_chunk - k0)),
                      lds + (st % NST) * STAGE + wave * 1024};
  };
  auto issue = [&](const StageLoads& l, int from, int to) {
#pragma unroll
    for (int n = 0; n < LOADS; ++n)
      if (n >= from && n < to) dma16((n * Cfg::WAVES < TileW::LOADS ? l.w : l.x) + (off[n] + l.kc), l.buf + n * Cfg::WAVES * 1024);
  };

  // The DMA's loads of a stage wait for the L2's misses, and a CU has only so
  // many in flight.  The tiles in flight on an XCD (8 of channels x 4 of
  // tokens, i8_tile) share their operands 4-fold and 8-fold, so each asks the
  // L2 for its part of a later stage's lines, a dword each, into a corner of
  // LDS that nobody reads (8192 x 4096 x 4096: 124 -> 117 us).
  uint32_t aoff = 0;
  bool asks = false, asks_w = false;
  if constexpr (AHEAD > 0) {
    constexpr int WL = Cfg::kBI / 4 / Cfg::WAVES, XL = Cfg::kBJ / 8 / Cfg::WAVES;
    asks_w = lane < WL;
    asks = lane < WL + XL;
    const int r = asks_w ? (tj % 4) * (Cfg::kBI / 4) + wave * WL + lane : (ti % 8) * (Cfg::kBJ / 8) + wave * XL + min(lane - WL, XL - 1);
    aoff = asks_w ? static_cast<uint32_t>(min(static_cast<int64_t>(r), a.N - 1 - i0) * a.ldw)
                  : static_cast<uint32_t>(min(static_cast<int64_t>(r), a.rows - 1 - j0) * a.ldx);
  }
  auto ask = [&](int st) {
    if constexpr (AHEAD > 0) {
      const int k0 = min(st * kI8Stage, last_chunk);
      if (asks) __builtin_amdgcn_global_load_lds((asks_w ? w0 : x0) + k0 + aoff, (lds_void_t*)(lds + NST * STAGE), 4, 0, 0);
    }
  };

  i32x4 acc[NA][NB];
#pragma unroll
  for (int p = 0; p < NA; ++p)
#pragma unroll
    for (int q = 0; q < NB; ++q) acc[p][q] = i32x4{0, 0, 0, 0};
  const int afrag[2] = {TileW::base(wi * Cfg::WI + c, g, 0), TileW::base(wi * Cfg::WI + c, g, 1)};
  const int bfrag[2] = {TileX::base(wj * Cfg::WJ + c, g, 0), TileX::base(wj * Cfg::WJ + c, g, 1)};
  i32x4 af[2][NA], bf[2][NB];
  // Fragments from..to of half kk of stage st: NB of the tokens', then NA of
  // the channels'.
  auto read = [&](int st, int kk, int from, int to) {
    const char* buf = lds + (st % NST) * STAGE;
    const char* xbuf = XS ? lds + Cfg::X_AT + st * TileX::BYTES : buf + TileW::BYTES;
#pragma unroll
    for (int f = 0; f < NA + NB; ++f) {
      if (f < from || f >= to) continue;
      if (f < NB) bf[kk][f] = *reinterpret_cast<const i32x4*>(xbuf + bfrag[kk] + f * TileX::ROW_BLOCK);
      else af[kk][f - NB] = *reinterpret_cast<const i32x4*>(buf + afrag[kk] + (f - NB) * TileW::ROW_BLOCK);
    }
  };
  auto multiply = [&](int kk, int p) {
#pragma unroll
    for (int q = 0; q < NB; ++q) acc[p][q] = __builtin_amdgcn_mfma_i32_16x16x64_i8(af[kk][p], bf[kk][q], acc[p][q], 0, 0, 0);
  };
  // The products of a half go in NA groups with the other half's fragment
  // reads between the first of them, and a stage's loads between the last:
  // a wave issues in order, so a run of reads or loads would keep its matrix
  // core waiting behind them.
  constexpr int READ_GROUPS = NA / 2, READS = (NA + NB + READ_GROUPS - 1) / READ_GROUPS;
  constexpr int LOAD_GROUPS = NA - READ_GROUPS, LOADS_EACH = (LOADS + LOAD_GROUPS - 1) / LOAD_GROUPS;

  // Stages 0 .. NST - 1 are in flight before the loop.  In the middle of
  // stage st, the wave waits for its loads of stage st + 1 (the NST - 2 later
  // ones may stay in flight) and its reads of stage st; behind the barrier
  // every wave's are done, so stage st + 1 is readable and stage st + NST may
  // be loaded into stage st's buffer.
  quantize_tokens<T, Cfg>(a, j0, n_stages, lds, [&] {
#pragma unroll
    for (int st = 0; st < NST; ++st)
      if (st < n_stages) issue(stage_loads(st), 0, LOADS);
  });
  if constexpr (AHEAD > 0) {
#pragma unroll
    for (int st = NST; st < AHEAD; ++st) ask(st);
    if (n_stages >= NST) wait_vmem_at_most<(NST - 1) * LOADS + AHEAD - NST>();
    else wait_vmem();
  } else if (n_stages >= NST) {
    wait_vmem_at_most<(NST - 1) * LOADS>();
  } else {
    wait_vmem();
  }
  counted_barrier();
  read(0, 0, 0, NA + NB);
  for (int st = 0; st + 1 < n_stages; ++st) {
#pragma unroll
    for (int p = 0; p < NA; ++p) {
      multiply(0, p);
      __builtin_amdgcn_sched_barrier(0);
      if (p < READ_GROUPS) read(st, 1, p * READS, (p + 1) * READS);
      __builtin_amdgcn_sched_barrier(0);
    }
    if (st + NST - 1 < n_stages) wait_vmem_at_most<(NST - 2) * (LOADS + EXTRA) + EXTRA>();
    else wait_vmem();
    counted_barrier();
    const StageLoads next = stage_loads(st + NST);
    const bool load = st + NST < n_stages;
#pragma unroll
    for (int p = 0; p < NA; ++p) {
      multiply(1, p);
      __builtin_amdgcn_sched_barrier(0);
      if (p < READ_GROUPS) read(st + 1, 0, p * READS, (p + 1) * READS);
      else if (load) issue(next, (p - READ_GROUPS) * LOADS_EACH, (p - READ_GROUPS + 1) * LOADS_EACH);
      if (load && p == NA - 1) ask(st + AHEAD);
      __builtin_amdgcn_sched_barrier(0);
    }
  }
  read(n_stages - 1, 1, 0, NA + NB);
  const int left = K - (n_stages - 1) * kI8Stage;
  if (left < kI8Stage) {
#pragma unroll
    for (int kk = 0; kk < 2; ++kk)
#pragma unroll
      for (int p = 0; p < NA; ++p) af[kk][p] = first_bytes(af[kk][p], left - kk * 64 - g * 16);
  }
#pragma unroll
  for (int kk = 0; kk < 2; ++kk)
#pragma unroll
    for (int p = 0; p < NA; ++p) multiply(kk, p);

  // Lane (c, g) holds rows i = 16p + 4g + r of column j = 16q + c.  A wave
  // stages 16 columns at a time in LDS as [j][i] rows and writes them back in
  // 16-byte chunks along i.
  __syncthreads();   // every wave is done reading the stage buffers
  char* stage_w = lds + wave * (16 * Cfg::ROWB);
  float* const chan_scales = reinterpret_cast<float*>(lds + NST * STAGE) - Cfg::PARAMS;
  float* const chan_biases = chan_scales + Cfg::kBI;
  float* const token_scales = chan_biases + Cfg::kBI;
  if (tid < Cfg::kBI) {
    chan_scales[tid] = chan_scale;
    chan_biases[tid] = has_bias ? scalar_value(bias_raw, a.bias_dtype) : 0.f;
  }
  if (tid < Cfg::kBJ)
    token_scales[tid] = XS ? reinterpret_cast<const float*>(lds + Cfg::X_AT + XS * TileX::BYTES)[tid] : tok_scale;
  __syncthreads();
  T* out = static_cast<T*>(a.out);
  constexpr int CHUNKS = Cfg::WI / 8;             // 16-byte chunks of a staged row
  constexpr int ROWS = 64 / CHUNKS;               // rows written at a time
  constexpr int PASSES = 16 / ROWS;
  const int ic = (lane % CHUNKS) * 8;
  const int64_t i = i0 + wi * Cfg::WI + ic;
  const int n = static_cast<int>(min(a.N - i, static_cast<int64_t>(8)));   // channels of this lane's chunks
  // All of a wave's residual chunks, before the stores that could be theirs.
  RawChunk<T> res[(EPI & 2) ? NB : 1][(EPI & 2) ? PASSES : 1];
  if constexpr ((EPI & 2) != 0) {
#pragma unroll
    for (int q = 0; q < NB; ++q)
#pragma unroll
      for (int pass = 0; pass < PASSES; ++pass) {
        const int64_t j = j0 + wj * Cfg::WJ + q * 16 + pass * ROWS + lane / CHUNKS;
        if (j < a.rows) res[q][pass] = fetch_chunk(static_cast<const T*>(a.residual) + j * a.ldr + i, n, a.N >= 8);
      }
  }
#pragma unroll
  for (int q = 0; q < NB; ++q) {
    const int64_t jq = j0 + wj * Cfg::WJ + q * 16;
    const float xs = token_scales[wj * Cfg::WJ + q * 16 + c];
#pragma unroll
    for (int p = 0; p < NA; ++p) {
      const int at = wi * Cfg::WI + p * 16 + 4 * g;
      const f32x4 ws = *reinterpret_cast<const f32x4*>(chan_scales + at);
      const f32x4 bias = *reinterpret_cast<const f32x4*>(chan_biases + at);
      typename Elem<T>::v4 o;
#pragma unroll
      for (int r = 0; r < 4; ++r) o[r] = static_cast<T>(linear_result<EPI>(acc[p][q][r], xs, ws[r], bias[r]));
      *reinterpret_cast<typename Elem<T>::v4*>(stage_w + c * Cfg::ROWB + (p * 16 + 4 * g) * 2) = o;
    }
#pragma unroll
    for (int pass = 0; pass < PASSES; ++pass) {
      const int jr = pass * ROWS + lane / CHUNKS;
      const int64_t j = jq + jr;
      const u32x4 v = *reinterpret_cast<const u32x4*>(stage_w + jr * Cfg::ROWB + ic * 2);
      if (j >= a.rows || n <= 0) continue;
      T* dst = out + j * a.N + i;
      const typename Elem<T>::v8 e8 = __builtin_bit_cast(typename Elem<T>::v8, v);
      if constexpr ((EPI & 2) != 0) {
        float r[8];
        chunk_floats(res[q][pass], static_cast<const T*>(a.residual) + j * a.ldr + i, n, a.N >= 8, r);
#pragma unroll
        for (int e = 0; e < 8; ++e) r[e] += static_cast<float>(e8[e]);
        store_chunk(dst, n, r);
      } else if (n == 8) {
        store16B_any(dst, v);
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
          if (e < n) dst[e] = e8[e];
      }
    }
  }
}

// Few tokens (MT tiles of 16): the weights' bytes bound the call, so the work
// is split over K inside the workgroup.  A workgroup takes 16 channels; its
// eight waves take K's steps of 64 bytes in turn, two neighbours at a time (a
// row's whole 128-byte line), straight from memory into MFMA fragments, eight
// steps in flight.  Their integer sums meet in LDS (in any order: they are
// exact).  With 16-bit tokens (XT = T, MT = 1) each workgroup quantizes them
// itself instead of waiting for another launch: a wave takes two tokens whole,
// in loads of 1 KiB, and leaves their integers in LDS (16 x 4096 -> 4096 9.2 us, 1
// x 4096 -> 16384 16.3; 10.6 and 26.6 where each wave read the tokens' fragments
// and quantized all 16 rows of its steps; 6.9 and 15 for 8-bit tokens).
constexpr int kFewWaves = 8;
constexpr int kFewBatch = 8;    // steps of a wave in flight
// Calls whose tokens are quantized in the kernel: one tile of tokens, 64 KiB of LDS.
constexpr int kFewRows = 16, kFewCols = 64 * kFewWaves * kFewBatch;

template <typename T, typename XT, int MT, int EPI>
__global__ __launch_bounds__(64 * kFewWaves) void linear_int8_few_kernel(LinearInt8Args a) {
  constexpr bool QUANT = sizeof(XT) == 2;
  static_assert(!QUANT || MT == 1, "one tile of tokens is quantized here");
  __shared__ __attribute__((aligned(16))) int part[kFewWaves][MT * 256];
  // The tokens' integers, at a pitch that puts a step's 16 rows into 16 different
  // groups of banks.
  constexpr int PITCH = kFewCols + 16, TOKENS = kFewRows / kFewWaves, PASSES = kFewCols / 512;
  __shared__ __attribute__((aligned(16))) char integers[QUANT ? kFewRows * PITCH : 16];
  __shared__ float token_scale[kFewRows];
  const int lane = lane_id();
  const int c = lane & 15;
  const int g = lane >> 4;
  const int wave = uniform_wave();
  const int K = a.K;
  const int steps = (K + 63) / 64;
  const int last_chunk = (K - 1) / 16 * 16;
  const int64_t i0 = static_cast<int64_t>(blockIdx.x) * 16;
  const int8_t* w = a.w + min(i0 + c, a.N - 1) * a.ldw;
  const XT* x[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m)
    x[m] = static_cast<const XT*>(a.x) + min(static_cast<int64_t>(m * 16 + c), a.rows - 1) * a.ldx;
  // This wave's 16-bit tokens.
  u32x4 raw[TOKENS][PASSES];
  auto token_of = [&](int r) { return wave + r * kFewWaves; };
  // The u-th step of this wave's batch that starts at step s0.
  auto step_of = [&](int s0, int u) { return s0 + (u >> 1) * (2 * kFewWaves) + 2 * wave + (u & 1); };
  constexpr int BATCH = kFewWaves * kFewBatch;   // steps of a batch, over the waves

  // A batch's weights and 8-bit tokens.
  i32x4 wf[kFewBatch];
  i32x4 xf[QUANT ? 1 : kFewBatch][MT];
  auto fetch_w = [&](int s0) {
#pragma unroll
    for (int u = 0; u < kFewBatch; ++u) {
      const int s = step_of(s0, u);
      if (s < steps) wf[u] = *reinterpret_cast<const i32x4*>(w + min(s * 64 + g * 16, last_chunk));
    }
  };
  auto fetch_x = [&](int s0) {
    if constexpr (QUANT) {
#pragma unroll
      for (int r = 0; r < TOKENS; ++r) {
        if (token_of(r) >= a.rows) continue;
        const T* token = static_cast<const T*>(a.x) + token_of(r) * a.ldx;
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
          const int k = p * 512 + lane * 8;
          if (p * 512 < K) raw[r][p] = fetch_bits(token + k, K - k, K >= 8);
        }
      }
    } else {
#pragma unroll
      for (int u = 0; u < kFewBatch; ++u) {
        const int s = step_of(s0, u);
        if (s >= steps) continue;
#pragma unroll
        for (int m = 0; m < MT; ++m) xf[u][m] = *reinterpret_cast<const i32x4*>(x[m] + min(s * 64 + g * 16, last_chunk));
      }
    }
  };

  fetch_x(0);
  fetch_w(0);   // on their way while the tokens are quantized

  // This thread's outputs, token e / 16 and channel e % 16 of the workgroup's,
  // and what their epilogue reads.
  constexpr int OUTS = (MT * 256 + 64 * kFewWaves - 1) / (64 * kFewWaves);
  float w_scale[OUTS], x_scale[OUTS], res[OUTS];
  ScalarHalves bias_raw[OUTS];
  const bool has_bias = a.bias != nullptr;
#pragma unroll
  for (int o = 0; o < OUTS; ++o) {
    const int e = static_cast<int>(threadIdx.x) + o * 64 * kFewWaves;
    const int64_t j = min(static_cast<int64_t>(e / 16), a.rows - 1), i = min(i0 + e % 16, a.N - 1);
    w_scale[o] = a.w_scales[i];
    bias_raw[o] = fetch_scalar(has_bias ? a.bias : a.w_scales, has_bias ? a.bias_dtype : kF32, i);
    x_scale[o] = QUANT ? 0.f : a.x_scales[j];
    if constexpr ((EPI & 2) != 0) res[o] = static_cast<float>(static_cast<const T*>(a.residual)[j * a.ldr + i]);
  }
  if constexpr (QUANT) {
    const int tokens = wave >= a.rows ? 0 : wave + kFewWaves < a.rows ? 2 : 1;
    static_assert(TOKENS == 2, "two tokens a wave");
    uint32_t mine = 0;
#pragma unroll
    for (int r = 0; r < TOKENS; ++r) {
      if (r >= tokens) continue;
      if (K % 8) {
#pragma unroll
        for (int p = 0; p < PASSES; ++p) raw[r][p] = chunk_bits(raw[r][p], K - p * 512 - lane * 8, K >= 8);
      }
      uint32_t pair = 0;
#pragma unroll
      for (int p = 0; p < PASSES; ++p)
        if (p * 512 < K) pair = max_pairs(raw[r][p], pair);
      const uint32_t largest = wave_max_bits(max(pair & 0xffffu, pair >> 16));
      mine = lane == r ? largest : mine;
    }
    if (tokens > 0) {
      const LaneScales<T> scales(mine);
#pragma unroll
      for (int r = 0; r < TOKENS; ++r) {
        if (r >= tokens) continue;
        const Int8Scale s = scales.of(r);
        char* const row = integers + token_of(r) * PITCH;
#pragma unroll
        for (int p = 0; p < PASSES; ++p) {
          const int k = p * 512 + lane * 8;
          if (p * 512 >= K) continue;   // the whole wave: a shorter loop
          if (k < K) *reinterpret_cast<u32x2*>(row + k) = pack_bits<T>(raw[r][p], s);
        }
      }
      if (lane < tokens) token_scale[token_of(lane)] = scales.own.scale;
    }
    __syncthreads();
  }

  i32x4 acc[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[m] = i32x4{0, 0, 0, 0};
  for (int s0 = 0; s0 < steps; s0 += BATCH) {
    if (s0) {
      fetch_x(s0);
      fetch_w(s0);
    }
#pragma unroll
    for (int u = 0; u < kFewBatch; ++u) {
      const int s = step_of(s0, u);
      if (s >= steps) continue;
      const int k = s * 64 + g * 16;
      if (s * 64 + 64 > K) wf[u] = first_bytes(wf[u], K - k);
      if constexpr (QUANT) {
        const i32x4 q = *reinterpret_cast<const i32x4*>(integers + c * PITCH + k);
        acc[0] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[u], q, acc[0], 0, 0, 0);
      } else {
#pragma unroll
        for (int m = 0; m < MT; ++m) acc[m] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[u], xf[u][m], acc[m], 0, 0, 0);
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m) *reinterpret_cast<i32x4*>(&part[wave][m * 256 + c * 16 + 4 * g]) = acc[m];
  __syncthreads();
  T* out = static_cast<T*>(a.out);
#pragma unroll
  for (int o = 0; o < OUTS; ++o) {
    const int e = static_cast<int>(threadIdx.x) + o * 64 * kFewWaves;
    const int64_t j = e / 16, i = i0 + e % 16;
    if (e >= MT * 256 || j >= a.rows || i >= a.N) continue;
    int sum = 0;
#pragma unroll
    for (int v = 0; v < kFewWaves; ++v) sum += part[v][e];
    const float bias = has_bias ? scalar_value(bias_raw[o], a.bias_dtype) : 0.f;
    T t = static_cast<T>(linear_result<EPI>(sum, QUANT ? token_scale[j] : x_scale[o], w_scale[o], bias));
    if constexpr ((EPI & 2) != 0) t = static_cast<T>(static_cast<float>(t) + res[o]);
    out[j * a.N + i] = t;
  }
}

typedef I8Cfg<256, 256, 2, 4, 2, 3> Tile256;   // one workgroup a CU (128 KiB of LDS)
typedef I8Cfg<128, 128, 2, 4, 2> Tile128;      // two a CU
typedef I8Cfg<128, 128, 2, 4, 3> Tile128Deep;  // one a CU, two stages ahead
typedef I8Cfg<128, 64, 2, 2, 2> Tile128x64;    // three a CU
typedef I8Cfg<64, 64, 2, 2, 4> Tile64;         // two a CU, three stages ahead

template <typename T, int EPI, typename Cfg>
static void launch_tiles(const LinearInt8Args& a, hipStream_t stream) {
  const int ti = static_cast<int>((a.N + Cfg::kBI - 1) / Cfg::kBI), tj = static_cast<int>((a.rows + Cfg::kBJ - 1) / Cfg::kBJ);
  hipLaunchKernelGGL((linear_int8_kernel<T, EPI, Cfg>), dim3(ti * tj), dim3(64 * Cfg::WAVES), 0, stream, a, ti, tj);
}

template <typename T, typename XT, int MT, int EPI>
static void launch_few(const LinearInt8Args& a, hipStream_t stream) {
  hipLaunchKernelGGL((linear_int8_few_kernel<T, XT, MT, EPI>), dim3(static_cast<unsigned>((a.N + 15) / 16)),
                     dim3(64 * kFewWaves), 0, stream, a);
}

typedef I8Cfg<128, 64, 4, 2, 2, 0, 4> Token128;      // 64 KiB of LDS: two a CU
typedef I8Cfg<64, 64, 2, 4, 4, 0, 4> Token64;        // 64 KiB
typedef I8Cfg<64, 64, 2, 4, 4, 0, 8> Token64x1024;   // 96 KiB: one a CU

// How a call runs.  Measured in us, bf16 without GELU unless said; rows x K -> N.
enum class I8Plan { kFew, kFew32, kToken64, kToken64x1024, kToken128, k256, k128, k128x64, k128Deep, k64 };
static int64_t tiles_of(int64_t rows, int64_t N, int bi, int bj) { return ((N + bi - 1) / bi) * ((rows + bj - 1) / bj); }
static I8Plan plan_linear_int8(int64_t rows, int64_t K, int64_t N, bool quantize) {
  // (32 x 4096 -> 4096: 8.5 of the split K against 11.0 of the 64-tiles; 64 rows: 12.9 against 11.0.)
  if (rows <= kFewRows && (!quantize || K <= kFewCols)) return I8Plan::kFew;
  if (rows <= 32 && !quantize) return I8Plan::kFew32;
  // 16-bit tokens are quantized again by every workgroup that multiplies them,
  // instead of once in a launch of its own.  While the workgroups are one round
  // and K is at most 512, that is faster (both from a captured graph: 4096 x 512
  // -> 512 6.8 against 8.2, 1024 x 512 -> 1536 6.7 against 7.3, 64 x 512 -> 1536 5.8
  // against 6.0, 16384 x 512 -> 256 9.6 against 13.7).  With K up to 1024 it is
  // as fast or up to a fifth slower on the GPU (777 x 1000 -> 1111 8.7 against 8.8,
  // 300 x 1000 -> 300 8.3 against 7.7, 64 x 1024 -> 1024 7.8 against 7.2, 200 x 700
  // -> 2000 8.6 against 7.1): taken for the host's 3 us of a launch, which bound
  // such a call; a captured graph, which has no host to wait for, is the slower
  // for it.  Over 1024 it loses (2500 x 1300 -> 3000 64 against 26).
  // Beyond one round whole calls go either way: the tiles take 16384 x 512 -> 640 in
  // 20.1 against 23.1, 16384 x 512 -> 512 with GELU 19.8 against 22.6, 32768 x 256
  // -> 256 15.3 against 18.0 and 32768 x 384 -> 256 16.3 against 19.1, are alike at
  // 4096 x 512 -> 1536 (16.0 and 15.8) and 16384 x 512 -> 768 (23.2 and 23.3), and
  // lose at 32768 x 512 -> 512 (29.9 against 26.5), 65536 x 512 -> 512 (57.6 against
  // 49.5), 16384 x 300 -> 512 (17.8 against 16.6) and, with K over 512, 4096 x 1024
  // -> 1024 (19 against 14): the launch is taken there.
  // Between the two tiles: 64 x 512 -> 1536, 24 64-tiles, 6.3 against 6.8; 1024 x
  // 512 -> 1536, 384 of them, 9.2 against 7.4.
  if (quantize && K <= 1024 && tiles_of(rows, N, 64, 64) <= 256) return K <= 512 ? I8Plan::kToken64 : I8Plan::kToken64x1024;
  if (quantize && K <= 512 && tiles_of(rows, N, 128, 64) <= 512) return I8Plan::kToken128;
  // Tiles by how the output fills the 256 CUs:
  //   256-tiles cost 1.22 times less for the same products than 128-tiles, but
  //     come in rounds of 256 (8192 x 4096 -> 4096: 117 against 147; 2048 x
  //     4096 -> 6144, 192 tiles: 48 against 55; 16384 x 512 -> 512: 14 against 10);
  //   up to 384 128-tiles leave a third of the slots of their one round empty,
  //     halves of them fill three a CU (4096 x 512 -> 1536: 8.9 against 9.1, with
  //     GELU 11.3 against 12.6; 16384 x 512 -> 512, 512 tiles: 12.0 against 9.9);
  //   with at most one a CU a third stage buffer is free (2048^3: 12.4 against
  //     14.3);
  //   few of them leave CUs idle that 64-tiles use (512 x 4096 -> 4096, 128
  //     tiles: 15.6 against 18.2; 4096 x 1536 -> 512: 8.6 against 9.6; at 256
  //     tiles 17.3 against 12.4).
  const int64_t t256 = tiles_of(rows, N, 256, 256), t128 = tiles_of(rows, N, 128, 128);
  if ((t256 + 255) / 256 * 100 <= (t128 + 511) / 512 * 61) return I8Plan::k256;
  if (t128 > 384) return I8Plan::k128;
  if (t128 > 256) return I8Plan::k128x64;
  return t128 > 144 ? I8Plan::k128Deep : I8Plan::k64;
}

template <typename T, int EPI>
static void launch_linear_int8_k(const LinearInt8Args& a, hipStream_t stream) {
  const bool quantize = a.x_dtype != kI8;
  switch (plan_linear_int8(a.rows, a.K, a.N, quantize)) {
    case I8Plan::kFew:
      if (quantize) launch_few<T, T, 1, EPI>(a, stream);
      else launch_few<T, int8_t, 1, EPI>(a, stream);
      break;
    case I8Plan::kFew32: launch_few<T, int8_t, 2, EPI>(a, stream); break;
    case I8Plan::kToken64: launch_tiles<T, EPI, Token64>(a, stream); break;
    case I8Plan::kToken64x1024: launch_tiles<T, EPI, Token64x1024>(a, stream); break;
    case I8Plan::kToken128: launch_tiles<T, EPI, Token128>(a, stream); break;
    case I8Plan::k256: launch_tiles<T, EPI, Tile256>(a, stream); break;
    case I8Plan::k128: launch_tiles<T, EPI, Tile128>(a, stream); break;
    case I8Plan::k128x64: launch_tiles<T, EPI, Tile128x64>(a, stream); break;
    case I8Plan::k128Deep: launch_tiles<T, EPI, Tile128Deep>(a, stream); break;
    case I8Plan::k64: launch_tiles<T, EPI, Tile64>(a, stream); break;
  }
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

bool linear_int8_quantizes(int64_t rows, int64_t K, int64_t N) {
  const I8Plan plan = plan_linear_int8(rows, K, N, true);
  return plan == I8Plan::kFew || plan == I8Plan::kToken64 || plan == I8Plan::kToken64x1024 || plan == I8Plan::kToken128;
}

void launch_linear_int8(const LinearInt8Args& a, hipStream_t stream) {
  if (a.dtype == kF16) launch_linear_int8_t<_Float16>(a, stream);
  else launch_linear_int8_t<__bf16>(a, stream);
}

}  // namespace da
