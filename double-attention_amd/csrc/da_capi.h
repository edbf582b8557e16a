// Host-side helpers of the C entry points: the error text, checks of types and
// alignment, and of tensors that share memory.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <cstdarg>
#include <cstdio>
#include <initializer_list>
#include <string>

#include "../../include/double_attention_hip.h"

namespace da {
namespace capi {

inline thread_local std::string g_error;

inline int fail(int code, const char* fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof(buf), fmt, ap);
  va_end(ap);
  g_error = buf;
  return code;
}

inline bool aligned(const void* p, int bytes) { return (reinterpret_cast<uintptr_t>(p) % bytes) == 0; }
inline bool half_dtype(int d) { return d == DA_F16 || d == DA_BF16; }
inline bool any_dtype(int d) { return d == DA_F32 || d == DA_F16 || d == DA_BF16; }

inline int ok() {
  g_error.clear();
  return DA_OK;
}

inline int check_launch(const char* what) {
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(DA_ERR_LAUNCH, "%s: launch failed: %s", what, hipGetErrorString(e));
  g_error.clear();
  return DA_OK;
}

constexpr int64_t kAlign = 256;
inline int64_t align_up(int64_t v) { return (v + kAlign - 1) / kAlign * kAlign; }

inline int64_t element_bytes(int dtype) { return dtype == DA_F32 ? 4 : 2; }

// The bytes of a tensor: `count` spans of `length`, `pitch` apart, up to `last`.
struct Spans {
  typedef __int128 wide;
  wide first, last, count, length, pitch;
  // `rows` rows of `cols` elements of `bytes`, `ld` elements apart; nothing for a null pointer.
  Spans(const void* p, int64_t rows, int64_t cols, int64_t ld, int64_t bytes)
      : first(reinterpret_cast<uintptr_t>(p)), last(first), count(p ? rows : 0), length(static_cast<wide>(cols) * bytes),
        pitch(static_cast<wide>(ld) * bytes) {
    if (count > 0) last = first + (count - 1) * pitch + length;
    if (count > 1 && pitch == length) {
      length *= count;
      count = 1;
    }
  }
};
inline Spans flat(const void* p, int64_t count, int64_t bytes) { return {p, 1, count, count, bytes}; }
// 8-bit rows that a call writes: with the rest of the last chunk of 16.
inline Spans written_int8(const void* p, int64_t rows, int64_t cols, int64_t ldv) { return {p, rows, (cols + 15) / 16 * 16, ldv, 1}; }
// Whether spans whose ranges meet share a byte.  Rows of x between rows of y
// (columns of one wider matrix) do not; where both have gaps and their pitches
// differ, their ranges decide.
inline bool share_a_byte(Spans x, Spans y) {
  typedef Spans::wide wide;
  // A single span has whichever pitch suits.
  if (x.count == 1) x.pitch = y.pitch;
  if (y.count == 1) y.pitch = x.pitch;
  if ((x.count == 1 && y.count == 1) || x.pitch != y.pitch) return true;
  // Spans i of x and j of y meet where -y.length < apart + k pitch < x.length with k = j - i.
  const auto floor_div = [](wide n, wide d) { return n / d - (n % d != 0 && n < 0 ? 1 : 0); };
  const wide apart = y.first - x.first, pitch = x.pitch;
  const wide least = floor_div(-y.length - apart, pitch) + 1, most = -floor_div(apart - x.length, pitch) - 1;
  return (least > -(x.count - 1) ? least : -(x.count - 1)) <= (most < y.count - 1 ? most : y.count - 1);
}
inline bool overlap(const Spans& x, const Spans& y) {
  return x.count > 0 && y.count > 0 && x.first < y.last && y.first < x.last && share_a_byte(x, y);
}

// Workgroups read rows that others write without an order between them, and a
// row's last columns in loads that begin before them: what a call writes stays
// off what it reads, and off what else it writes.
inline int validate_apart(const char* what, std::initializer_list<Spans> outputs, std::initializer_list<Spans> inputs) {
  for (const Spans* out = outputs.begin(); out != outputs.end(); ++out) {
    for (const Spans& in : inputs)
      if (overlap(*out, in)) return fail(DA_ERR_INVALID_ARGUMENT, "%s: an output overlaps an input", what);
    for (const Spans* other = out + 1; other != outputs.end(); ++other)
      if (overlap(*out, *other)) return fail(DA_ERR_INVALID_ARGUMENT, "%s: an output overlaps another output", what);
  }
  return DA_OK;
}

}  // namespace capi
}  // namespace da
