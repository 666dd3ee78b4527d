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

// Bytes from a row to the next of a readout's operands: a block's rows, 192 at most, lie within 2^31.
constexpr int64_t kMaxApart = 8 << 20;

inline bool decode_float(int dtype) {
  return dtype == YTM_DTYPE_F32 || dtype == YTM_DTYPE_F16 || dtype == YTM_DTYPE_BF16;
}

}  // namespace ytm
