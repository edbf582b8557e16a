// Device helpers of the 8-bit rows: signed integers from -127 to 127 with an
// fp32 scale for each row, or for each 128 columns of a row.
//
//   scale = max(amax, 127 * 2^-126) / 127,   q = rint(x / scale)
//
// The floor on the scale keeps 1 / scale finite (an all-zero row has the
// least scale and zeros).  A row (group) that holds an infinity or a NaN has
// no such integers: its scale is NaN and its integers are 0, so that all of it
// stands for NaN instead of for some finite numbers.
#pragma once

#include "da_common.h"

namespace da {

constexpr int kI8 = 3;                      // dtype code of 8-bit rows
constexpr int kInt8Group = 128;             // columns that share a scale in grouped rows
constexpr float kInt8Least = 0x1p-126f;     // the least scale
// A multiple of 2^23 added to a float in its last place's range: x + kRoundMagic
// rounds x to an integer (ties to even) and leaves it in the sum's low bits, in
// two's complement.  |x| < 2^22.
constexpr float kRoundMagic = 12582912.f;   // 1.5 * 2^23

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
// 16-byte accesses at any 2-byte (4-byte for fp32 rows) address: rows of odd
// widths start there, and the hardware takes such accesses whole.
typedef u32x4 u32x4_any __attribute__((aligned(2)));

__device__ __forceinline__ u32x4 load16B_any(const void* p) { return *static_cast<const u32x4_any*>(p); }
__device__ __forceinline__ void store16B_any(void* p, u32x4 v) { *static_cast<u32x4_any*>(p) = v; }

// Eight elements of a row from column c on, of which n (<= 8) exist; the
// others are 0.
template <typename T>
__device__ __forceinline__ void load_chunk(const T* p, int n, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    if (n >= 8) {
      const u32x4 a = load16B_any(p), b = load16B_any(p + 4);
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        v[e] = __uint_as_float(a[e]);
        v[e + 4] = __uint_as_float(b[e]);
      }
      return;
    }
  } else {
    if (n >= 8) {
      const typename Elem<T>::v8 a = __builtin_bit_cast(typename Elem<T>::v8, load16B_any(p));
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] = static_cast<float>(a[e]);
      return;
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e) v[e] = e < n ? static_cast<float>(p[e]) : 0.f;
}

// Raw loads of a chunk, kept apart from their use so that all of a thread's are
// in flight before the first is waited for.  A row's last, partial chunk is read
// as the row's last eight elements (`wide`: rows of eight columns or more) and
// moved into place when it is used: no load waits for another, or for a branch.
template <typename T>
struct RawChunk {
  u32x4 lo, hi;
};

template <typename T>
__device__ __forceinline__ RawChunk<T> fetch_chunk(const T* p, int n, bool wide) {
  RawChunk<T> r{u32x4{0, 0, 0, 0}, u32x4{0, 0, 0, 0}};
  if (n > (wide ? 0 : 7)) {
    p += min(n - 8, 0);
    r.lo = load16B_any(p);
    if constexpr (sizeof(T) == 4) r.hi = load16B_any(p + 4);
  }
  return r;
}

// A row's last eight 16-bit elements as its last n (1 to 7), and zeros: a shift of
// 128 bits.
__device__ __forceinline__ u32x4 moved_down(u32x4 d, int n) {
  const uint64_t lo = static_cast<uint64_t>(d[1]) << 32 | d[0], hi = static_cast<uint64_t>(d[3]) << 32 | d[2];
  const int shift = 16 * (8 - n);   // 16 to 112
  const uint64_t top = hi >> (shift & 63);
  const uint64_t low = shift >= 64 ? top : lo >> (shift & 63) | hi << (-shift & 63);
  const uint64_t high = shift >= 64 ? 0 : top;
  return u32x4{static_cast<uint32_t>(low), static_cast<uint32_t>(low >> 32), static_cast<uint32_t>(high), static_cast<uint32_t>(high >> 32)};
}

// The chunk's floats.
template <typename T>
__device__ __forceinline__ void chunk_floats(const RawChunk<T>& r, const T* p, int n, bool wide, float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int e = 0; e < 4; ++e) {
      v[e] = __uint_as_float(r.lo[e]);
      v[e + 4] = __uint_as_float(r.hi[e]);
    }
    if (wide && n > 0 && n < 8) {
#pragma unroll
      for (int step = 4; step; step /= 2)
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = (8 - n) & step ? (e + step < 8 ? v[e + step] : 0.f) : v[e];
    }
  } else {
    u32x4 d = r.lo;
    if (wide && n > 0 && n < 8) d = moved_down(d, n);
    const typename Elem<T>::v8 a = __builtin_bit_cast(typename Elem<T>::v8, d);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = static_cast<float>(a[e]);
  }
  if (!wide && n > 0 && n < 8) load_chunk(p, n, v);
}

template <typename T>
__device__ __forceinline__ void store_chunk(T* p, int n, const float (&v)[8]) {
  if constexpr (sizeof(T) == 4) {
    if (n >= 8) {
      store16B_any(p, u32x4{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])});
      store16B_any(p + 4, u32x4{__float_as_uint(v[4]), __float_as_uint(v[5]), __float_as_uint(v[6]), __float_as_uint(v[7])});
      return;
    }
  } else {
    if (n >= 8) {
      typename Elem<T>::v8 o;
#pragma unroll
      for (int e = 0; e < 8; ++e) o[e] = static_cast<T>(v[e]);
      store16B_any(p, __builtin_bit_cast(u32x4, o));
      return;
    }
  }
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (e < n) p[e] = static_cast<T>(v[e]);
}

// Largest magnitude as the bits of a non-negative float: unsigned integers
// order like the floats, and infinities and NaN come out on top, so the
// maximum does not lose them.
__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// A chunk of eight 16-bit elements as they lie in memory; n of them exist (the
// others are 0).  Fetched like a RawChunk, and put in place by chunk_bits.
template <typename T>
__device__ __forceinline__ u32x4 fetch_bits(const T* p, int n, bool wide) {
  u32x4 d = fetch_chunk(p, n, wide).lo;
  if (!wide && n > 0) {
    const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
    for (int e = 0; e < 7; ++e)
      if (e < n) d[e / 2] |= static_cast<uint32_t>(h[e]) << (16 * (e % 2));
  }
  return d;
}
__device__ __forceinline__ u32x4 chunk_bits(u32x4 d, int n, bool wide) { return wide && n > 0 && n < 8 ? moved_down(d, n) : d; }

// Largest magnitudes of the 16-bit floats in d, as pairs of 16-bit integers.
__device__ __forceinline__ uint32_t max_pairs(u32x4 d, uint32_t pair) {
  u16x2 m = __builtin_bit_cast(u16x2, pair);
#pragma unroll
  for (int i = 0; i < 4; ++i) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, d[i] & 0x7fff7fffu));
  return __builtin_bit_cast(uint32_t, m);
}

// The float of a 16-bit float's bits.
template <typename T>
__device__ __forceinline__ float half_value(uint32_t bits) {
  if constexpr (sizeof(T) == 2) return static_cast<float>(__builtin_bit_cast(T, static_cast<uint16_t>(bits)));
  else return 0.f;
}

// All-lane reductions over the 16 lanes of a row (DPP rotations), then over
// the wave's four rows.
template <int R>
__device__ __forceinline__ uint32_t row_rotate(uint32_t v) {
  return __builtin_amdgcn_update_dpp(0, v, 0x120 + R, 0xf, 0xf, false);
}
__device__ __forceinline__ uint32_t row16_max(uint32_t v) {
  v = max(v, row_rotate<8>(v));
  v = max(v, row_rotate<4>(v));
  v = max(v, row_rotate<2>(v));
  return max(v, row_rotate<1>(v));
}
__device__ __forceinline__ float row16_sum(float v) {
  v += __uint_as_float(row_rotate<8>(__float_as_uint(v)));
  v += __uint_as_float(row_rotate<4>(__float_as_uint(v)));
  v += __uint_as_float(row_rotate<2>(__float_as_uint(v)));
  return v + __uint_as_float(row_rotate<1>(__float_as_uint(v)));
}
__device__ __forceinline__ uint32_t wave_max_bits(uint32_t v) {
  v = row16_max(v);
  const auto a = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  v = max(a[0], a[1]);
  const auto b = __builtin_amdgcn_permlane16_swap(v, v, false, false);
  return max(b[0], b[1]);
}
__device__ __forceinline__ float wave_sum_dpp(float v) { return group_sum(row16_sum(v)); }

// The integers are those of a plain fp32 division, rint(x / scale) with ties to
// even, at the price of a multiplication.  x * inverse would do but for the
// halves of a step, which roundings of the scale and of its inverse push either
// way.  In a row of 16-bit floats (p = 8 or 11 bits) a quotient 127 x / amax is
// such a half or at least 2^-19 of itself from one (|254 x - (2 k + 1) amax| is
// a unit of x's place or more), so any inverse within some 2^-21 of 1 / scale
// gives the others.  The halves are
//   * amax / 2, 63.5 steps, in all rows: the inverse is set two units, more
//     than both roundings together, to the side on which the division falls;
//   * odd multiples of amax / 254 where 127 divides amax's p bits, so that
//     the scale is exact, amax = 127 scale: 254 for bf16, a power of two as a
//     scale, where x * inverse is exact too; 127 j, j <= 16, for fp16, where
//     eight rows of 1024 take the division's steps (fp32 rows take them all).
// The tests hold every pair of significands up to 2^-11 of each other against
// fp32 division.  (The norm's rows are not such floats: rms_norm.hip.)
template <typename T> inline constexpr bool kInt8Divides = true;        // all of fp32's rows
template <> inline constexpr bool kInt8Divides<__bf16> = false;
struct Int8Scale {
  float scale;     // what a step of the integers stands for; NaN: the row has no integers
  float inverse;   // 1 / scale, or two units beside it
  uint32_t keep;   // all ones, 0 where the scale is NaN
  bool divide;     // the integers need the rounded quotient
};

// v / scale as fp32 rounds it: one step of Newton's iteration on the product with
// the rounded inverse (Markstein, "Computation of elementary functions on the
// IBM RISC System/6000 processor", 1990).  The residual is exact in an FMA.
__device__ __forceinline__ float quotient(float v, float scale, float inverse) {
#pragma clang fp contract(off)
  const float t = v * inverse;
  return __builtin_fmaf(__builtin_fmaf(-t, scale, v), inverse, t);
}

template <typename T>
__device__ __forceinline__ Int8Scale int8_scale(uint32_t amax_bits, float factor = 1.f) {
  const bool finite = amax_bits < 0x7f800000u;
  const float amax = __uint_as_float(amax_bits) * factor;
  const float s = fmaxf(amax * (1.f / 127.f), kInt8Least);
  float inverse;
  bool divide = true;
  if constexpr (sizeof(T) == 4) {
    inverse = 1.f / s;
  } else {
    // The hardware's reciprocal (one unit off at most) and a step of Newton's
    // iteration: a hair over half a unit, and rounded like a division for the
    // scales j 2^k of the rows that divide.
    inverse = __builtin_amdgcn_rcpf(s);
    inverse = __builtin_fmaf(__builtin_fmaf(-s, inverse, 1.f), inverse, inverse);
    // amax / 2 over the scale rounds to 63.5 or more from 63.5 - 2^-19 on; the
    // difference is exact.
    const float beyond = __builtin_fmaf(-127.f, s, amax);
    const float beside = __uint_as_float(__float_as_uint(inverse) + (__builtin_fmaf(0x1p-18f, s, beyond) >= 0.f ? 2u : -2u));
    divide = kInt8Divides<T> && beyond == 0.f;
    if (kInt8Divides<T> ? !divide : (__float_as_uint(s) & 0x7fffffu) != 0) inverse = beside;
  }
  return Int8Scale{finite ? s : __uint_as_float(0x7fc00000u), inverse, finite ? 0xffffffffu : 0u, divide};
}

// Eight bytes of sums with kRoundMagic.
__device__ __forceinline__ u32x2 pack_rounded(const uint32_t (&t)[8], uint32_t keep) {
  u32x2 r;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const uint32_t lo = __builtin_amdgcn_perm(t[4 * h + 1], t[4 * h], 0x0c0c0400u);
    const uint32_t hi = __builtin_amdgcn_perm(t[4 * h + 3], t[4 * h + 2], 0x04000c0cu);
    r[h] = (lo | hi) & keep;
  }
  return r;
}

// Eight integers rint(v * inverse) as bytes.  |v * inverse| <= 127 (1 + 2^-21)
// by the choice of the scale, so rounding keeps them in [-127, 127].
__device__ __forceinline__ u32x2 pack_int8(const float (&v)[8], float inverse, uint32_t keep) {
  uint32_t t[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) t[e] = __float_as_uint(__builtin_fmaf(v[e], inverse, kRoundMagic));
  return pack_rounded(t, keep);
}

// Eight elements of a row of T's in their row's scale.
template <typename T>
__device__ __forceinline__ u32x2 pack_int8(const float (&v)[8], const Int8Scale& s) {
  if (kInt8Divides<T> && s.divide) {
    uint32_t t[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) t[e] = __float_as_uint(quotient(v[e], s.scale, s.inverse) + kRoundMagic);
    return pack_rounded(t, s.keep);
  }
  return pack_int8(v, s.inverse, s.keep);
}

// The eight floats that stored bytes stand for.
__device__ __forceinline__ void unpack_int8(u32x2 q, float scale, float (&v)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    const int b = static_cast<int>(q[e / 4] << (24 - 8 * (e % 4))) >> 24;
    v[e] = static_cast<float>(b) * scale;
  }
}

// A chunk's bytes, whole also where the row ends inside it: the pitch is a
// multiple of 16, and the columns behind the row are the storage's own.
__device__ __forceinline__ void store_bytes(int8_t* p, u32x2 q) { *reinterpret_cast<u32x2*>(p) = q; }
__device__ __forceinline__ u32x2 load_bytes(const int8_t* p) { return *reinterpret_cast<const u32x2*>(p); }

// n / d for 0 <= n < 2^31 by a multiplication (d >= 1; Granlund and
// Montgomery, "Division by invariant integers using multiplication", 1994).
struct FastDiv {
  uint32_t d, mul, shift;
};
inline FastDiv make_fast_div(uint32_t d) {
  uint32_t s = 0;
  while ((1ull << s) < d) ++s;
  const uint64_t m = ((1ull << 32) * ((1ull << s) - d)) / d + 1;
  return FastDiv{d, static_cast<uint32_t>(m), s};
}
__device__ __forceinline__ uint32_t fast_div(uint32_t n, FastDiv f) { return (__umulhi(n, f.mul) + n) >> f.shift; }

}  // namespace da
