// ytm_decode.h -- what the answering operators (ytm_readout.hip, ytm_scores.hip) share: their
// element types and bounds.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ytm.h"

namespace ytm {

typedef _Float16 f16;
struct bf16 {
  uint16_t bits;
};

__device__ __forceinline__ float to_float(float v) { return v; }
__device__ __forceinline__ float to_float(f16 v) { return (float)v; }
__device__ __forceinline__ float to_float(bf16 v) { return __uint_as_float((uint32_t)v.bits << 16); }

// Rounds to nearest, ties to even; a NaN stays one.
template <typename T>
__device__ __forceinline__ T from_float(float v);
template <>
__device__ __forceinline__ float from_float<float>(float v) {
  return v;
}
template <>
__device__ __forceinline__ f16 from_float<f16>(float v) {
  return (f16)v;
}
template <>
__device__ __forceinline__ bf16 from_float<bf16>(float v) {
  const uint32_t u = __float_as_uint(v);
  if (v != v) return bf16{(uint16_t)(u >> 16 | 0x40u)};
  return bf16{(uint16_t)((u + 0x7FFFu + (u >> 16 & 1u)) >> 16)};
}

// Rows go along a grid's second axis.
constexpr int64_t kDecodeRows = 65535;
// Scores of a row: their masses, at most 2^40 each, add up below 2^63.
constexpr int64_t kMaxScores = 1 << 23;

// Clauses of a readout: fewer than 65536 steps of 32.
constexpr int64_t kMaxClauses = 65535 * 32;

// Bytes from a row to the next of a readout's operands: a block's rows or outputs lie within 2^31.
constexpr int64_t kMaxApart = 8 << 20;
constexpr int kMaxTogether = 256;
static_assert(kMaxApart * kMaxTogether <= (int64_t)1 << 31, "");

// An operand's `n` rows of `width` bytes, each `stride` after the one before (0: one row for all).
struct Rows {
  const void* p;
  int64_t n, stride, width;
};
inline Rows rows_of(const void* p, int64_t n, int64_t width, int64_t stride, int64_t size) {
  if (n <= 1 || stride == 0) return Rows{p, 1, 0, width * size};
  const int64_t most = INT64_MAX / size / n;  // a larger distance is no memory's
  return Rows{p, n, (stride < most ? stride : most) * size, width * size};
}
inline Rows block_of(const void* p, int64_t bytes) { return Rows{p, 1, 0, bytes}; }

// Whether two operands share a byte; none of a null one.  Rows of the same distance may lie between
// each other.
inline bool share_bytes(const Rows& a, const Rows& b) {
  if (!a.p || !b.p || a.width < 1 || b.width < 1) return false;
  const uintptr_t p = (uintptr_t)a.p, q = (uintptr_t)b.p;
  const auto end = [](const Rows& r) {
    return (uintptr_t)r.p + (uintptr_t)((r.n - 1) * r.stride) + (uintptr_t)r.width;
  };
  if (end(a) <= q || end(b) <= p) return false;
  if (a.n > 1 && b.n > 1 && a.stride == b.stride) {
    // row j of b begins d + (j - i) stride after row i of a; the least j - i at which it ends past a's beginning
    const int64_t d = (int64_t)(q - p), over = -b.width - d;
    int64_t k = over >= 0 ? over / a.stride + 1 : -((-over - 1) / a.stride);
    if (k < 1 - a.n) k = 1 - a.n;
    return k < b.n && d + k * a.stride < a.width;
  }
  for (int64_t i = 0, j = 0; i < a.n && j < b.n;) {
    const uintptr_t x = p + (uintptr_t)(i * a.stride), y = q + (uintptr_t)(j * b.stride);
    if (x + (uintptr_t)a.width <= y)
      ++i;
    else if (y + (uintptr_t)b.width <= x)
      ++j;
    else
      return true;
  }
  return false;
}

inline bool decode_float(int dtype) {
  return dtype == YTM_DTYPE_F32 || dtype == YTM_DTYPE_F16 || dtype == YTM_DTYPE_BF16;
}

}  // namespace ytm
