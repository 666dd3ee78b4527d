// ytm_readout.hip -- class sums from clause outputs through weights held in 4 bits: the entry
// points ytm_readout and ytm_readout_workspace of include/ytm.h and their gfx950 kernels.
//
//   out[n][o] = sum over groups q of scale[o][q] * sum over clauses c of q of x[n][c] value(code[o][c])
//
// A code is an E2M1 float (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), exact in float16 and
// bfloat16, into which gfx950 converts two codes an instruction; so the inner sums run on the
// matrix cores in f32 with operands that are no less exact than x: bits, float16 and bfloat16 as
// they are, float32 as the sum of three bfloat16 (8 + 8 + 8 bits of its fraction), a product each.
// The scale multiplies each group's f32 sum.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <algorithm>

#include "ytm_decode.h"
#include "ytm_internal.h"

namespace ytm {

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef short v8s __attribute__((ext_vector_type(8)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

constexpr int kWave = 64;
constexpr int kTile = 16;   // rows and outputs of a product
constexpr int kStep = 32;   // clauses of a product
constexpr int kChunk = 128; // clauses of a 16-byte load of codes by each lane

struct ReadoutArgs {
  const void* x;
  int x_dtype;
  int64_t x_stride, N, C;
  const uint8_t* codes;
  int64_t code_stride;
  const void* scales;
  int64_t scale_stride, group, K;
  void* out;
  int out_dtype;
  int64_t out_stride;
  v4u* frag;
  int64_t steps, row_tiles;
};

// ------------------------------------------------------------------------------- row operands
// The value of clause c in row n as float32 bits, whatever x's type.
__device__ __forceinline__ float x_at(const ReadoutArgs& a, int64_t n, int64_t c) {
  const int64_t i = n * a.x_stride;
  switch (a.x_dtype) {
    case YTM_DTYPE_BITS: return (float)(((const uint32_t*)a.x)[i + c / 32] >> (c % 32) & 1u);
    case YTM_DTYPE_F16: return to_float(((const f16*)a.x)[i + c]);
    case YTM_DTYPE_BF16: return to_float(((const bf16*)a.x)[i + c]);
    default: return ((const float*)a.x)[i + c];
  }
}

// Row operands frag[plane][step][row tile][lane], lane l holding 8 values (clauses 32 step +
// 8 (l / 16) ...) of row l % 16, zero past the last clause or row.  Planes: one, or for float32
// three whose sum it is, each cut (not rounded) to a bfloat16, so that nothing overflows; where
// the first is infinite or NaN the others are zero.
__global__ __launch_bounds__(256) void rows_kernel(ReadoutArgs a) {
  const int64_t each = a.steps * a.row_tiles * kWave;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < each; i += (int64_t)gridDim.x * blockDim.x) {
    const int l = (int)(i % kWave);
    const int64_t n = i / kWave % a.row_tiles * kTile + l % 16;
    const int64_t c0 = i / kWave / a.row_tiles * kStep + 8 * (l / 16);
    v4u plane[3];
    for (int p = 0; p < 3; ++p) plane[p] = v4u{0u, 0u, 0u, 0u};
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      float v = n < a.N && c0 + j < a.C ? x_at(a, n, c0 + j) : 0.0f;
      const int sh = 16 * (j & 1);
      if (a.x_dtype == YTM_DTYPE_F16) {
        plane[0][j / 2] |= (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)v) << sh;
        continue;
      }
      const uint32_t hi = __float_as_uint(v) >> 16;
      plane[0][j / 2] |= hi << sh;
      if (a.x_dtype == YTM_DTYPE_F32 && (hi & 0x7F80u) != 0x7F80u) {
        v -= __uint_as_float(hi << 16);
        const uint32_t mid = __float_as_uint(v) >> 16;
        plane[1][j / 2] |= mid << sh;
        v -= __uint_as_float(mid << 16);
        plane[2][j / 2] |= __float_as_uint(v) >> 16 << sh;
      }
    }
    a.frag[i] = plane[0];
    if (a.x_dtype == YTM_DTYPE_F32) {
      a.frag[each + i] = plane[1];
      a.frag[2 * each + i] = plane[2];
    }
  }
}

// ------------------------------------------------------------------------------------ products
template <bool HALF>
__device__ __forceinline__ v4u codes_to_16(uint32_t w) {
  v4u r;
  if (HALF) {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 0));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 1));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 2));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w, 1.0f, 3));
  } else {
    r[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 0));
    r[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 1));
    r[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 2));
    r[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 3));
  }
  return r;
}

template <bool HALF>
__device__ __forceinline__ v4f product(v4u x, v4u w, v4f d) {
  if (HALF)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, x), __builtin_bit_cast(v8h, w), d, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, x), __builtin_bit_cast(v8bf, w), d, 0, 0, 0);
}

// A lane of group g = l / 16 holds codes of clauses 32 g .. 32 g + 31 in four words; after this
// word s holds those of clauses 32 s + 8 g ..., so that a product's clauses are 32 in a row and
// belong to one scale.  A 4 x 4 transposition in two exchanges of bits of (group, word).
__device__ __forceinline__ v4u turn(v4u w) {
  auto a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
  auto b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
  auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
  auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  return v4u{c[0], c[1], d[0], d[1]};
}

__device__ __forceinline__ void store_out(const ReadoutArgs& a, int64_t n, int64_t o, float v) {
  const int64_t i = n * a.out_stride + o;
  switch (a.out_dtype) {
    case YTM_DTYPE_F16: ((f16*)a.out)[i] = from_float<f16>(v); break;
    case YTM_DTYPE_BF16: ((bf16*)a.out)[i] = from_float<bf16>(v); break;
    default: ((float*)a.out)[i] = v; break;
  }
}

// A block of four waves per tile of 16 outputs and 16 rows, the clauses split among the waves
// chunk by chunk and their sums joined in LDS in the waves' order.  Lane l takes the codes of
// output l % 16 as the second operand and gets sums of rows 4 (l / 16) .. + 3 of that output.
// GRAIN: clauses after which sums are scaled, 32, 64 or 128, a divisor of the group.
constexpr int kWaves = 4;
template <int PLANES, bool HALF, int GRAIN, typename Scale>
__global__ __launch_bounds__(kWaves* kWave) void readout_kernel(ReadoutArgs a) {
  __shared__ v4f sums[kWaves][kWave];
  const int l = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const int64_t o = blockIdx.x * (int64_t)kTile + l % 16;
  const int64_t tile = blockIdx.y;
  const bool real = o < a.K;
  const uint8_t* codes = a.codes + (real ? o : 0) * a.code_stride;
  const Scale* scales = (const Scale*)a.scales + (real ? o : 0) * a.scale_stride;
  const int64_t bytes = (a.C + 31) / 32 * 16, chunks = (a.C + kChunk - 1) / kChunk;
  const int64_t each = a.steps * a.row_tiles * kWave;
  v4f total = {0.0f, 0.0f, 0.0f, 0.0f};
  for (int64_t t = wave; t < chunks; t += kWaves) {
    const int64_t at = t * 64 + l / 16 * 16;
    v4u w = {0u, 0u, 0u, 0u};
    if (at < bytes) w = *(const v4u*)(codes + at);
    w = turn(w);
    v4f sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const int64_t c = t * kChunk + s * kStep;
      if (c < a.C) {
        const v4u b = codes_to_16<HALF>(w[s]);
        const v4u* frag = a.frag + ((t * 4 + s) * a.row_tiles + tile) * kWave + l;
#pragma unroll
        for (int p = PLANES - 1; p >= 0; --p) sum = product<HALF>(frag[p * each], b, sum);
        if ((s + 1) * kStep % GRAIN == 0 || c + kStep >= a.C) {
          const float scale = to_float(scales[c / a.group]);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            total[r] += scale * sum[r];
            sum[r] = 0.0f;
          }
        }
      }
    }
  }
  sums[wave][l] = total;
  __syncthreads();
  if (wave == 0) {
    for (int w = 1; w < kWaves; ++w) total += sums[w][l];
    for (int r = 0; r < 4; ++r) {
      const int64_t n = tile * kTile + l / 16 * 4 + r;
      if (real && n < a.N) store_out(a, n, o, total[r]);
    }
  }
}

int planes_of(int x_dtype) { return x_dtype == YTM_DTYPE_F32 ? 3 : 1; }
int64_t steps_of(int64_t C) { return (C + kStep - 1) / kStep; }
int64_t tiles_of(int64_t n) { return (n + kTile - 1) / kTile; }

template <int PLANES, bool HALF, int GRAIN>
void launch_scale(const ReadoutArgs& a, int scale_dtype, hipStream_t s) {
  const dim3 grid((unsigned)tiles_of(a.K), (unsigned)a.row_tiles);
  switch (scale_dtype) {
    case YTM_DTYPE_F16: readout_kernel<PLANES, HALF, GRAIN, f16><<<grid, kWaves * kWave, 0, s>>>(a); break;
    case YTM_DTYPE_BF16: readout_kernel<PLANES, HALF, GRAIN, bf16><<<grid, kWaves * kWave, 0, s>>>(a); break;
    default: readout_kernel<PLANES, HALF, GRAIN, float><<<grid, kWaves * kWave, 0, s>>>(a); break;
  }
}

template <int PLANES, bool HALF>
hipError_t launch_readout(const ReadoutArgs& a, int scale_dtype, hipStream_t s) {
  const int64_t items = a.steps * a.row_tiles * kWave;
  if (items) rows_kernel<<<(unsigned)std::min<int64_t>((items + 255) / 256, 4096), 256, 0, s>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  if (a.group % 128 == 0)
    launch_scale<PLANES, HALF, 128>(a, scale_dtype, s);
  else if (a.group % 64 == 0)
    launch_scale<PLANES, HALF, 64>(a, scale_dtype, s);
  else
    launch_scale<PLANES, HALF, 32>(a, scale_dtype, s);
  return hipGetLastError();
}

}  // namespace

}  // namespace ytm

using ytm::fail;

extern "C" {

int ytm_readout_workspace(int x_dtype, int64_t N, int64_t C, int64_t K, int64_t* bytes) {
  if (!bytes || (x_dtype != YTM_DTYPE_BITS && !ytm::decode_float(x_dtype)) || N < 0 || C < 0 || K < 0 ||
      N > ytm::kDecodeRows || C > INT32_MAX || K > INT32_MAX)
    return fail(YTM_EINVAL, "bad readout_workspace arguments");
  *bytes = ytm::planes_of(x_dtype) * ytm::steps_of(C) * ytm::tiles_of(N) * ytm::kWave * 16;
  return YTM_OK;
}

int ytm_readout(const void* x, int x_dtype, int64_t x_stride, int64_t N, int64_t C, const uint8_t* codes,
                int64_t code_stride, const void* scales, int scale_dtype, int64_t scale_stride, int64_t group,
                int64_t K, void* out, int out_dtype, int64_t out_stride, void* workspace, int64_t workspace_bytes,
                void* stream) {
  if (x_dtype != YTM_DTYPE_BITS && !ytm::decode_float(x_dtype))
    return fail(YTM_EINVAL, "readout takes bits, float32, float16 or bfloat16");
  if (!ytm::decode_float(scale_dtype) || !ytm::decode_float(out_dtype))
    return fail(YTM_EINVAL, "readout scales and sums are float32, float16 or bfloat16");
  if (N < 0 || C < 0 || K < 0 || N > ytm::kDecodeRows || C > INT32_MAX || K > INT32_MAX)
    return fail(YTM_EINVAL, "readout takes at most 65535 rows");
  if (group < 32 || group % 32) return fail(YTM_EINVAL, "readout groups are multiples of 32 clauses");
  if (N == 0 || K == 0) return YTM_OK;
  if (!out || (C > 0 && (!x || !codes || !scales))) return fail(YTM_EINVAL, "bad readout arguments");
  if (C > 0 && ((uintptr_t)codes | (K > 1 ? (uint64_t)code_stride : 0u)) % 16)
    return fail(YTM_EINVAL, "readout codes start at multiples of 16 bytes, every output's");
  const int64_t width = x_dtype == YTM_DTYPE_BITS ? (C + 31) / 32 : C;
  if ((K > 1 && (code_stride < (C + 31) / 32 * 16 || scale_stride < (C + group - 1) / group)) ||
      (N > 1 && (x_stride < width || out_stride < K)))
    return fail(YTM_EINVAL, "readout: rows overlap");
  int64_t need = 0;
  if (int rc = ytm_readout_workspace(x_dtype, N, C, K, &need)) return rc;
  if (need > 0 && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
    return fail(YTM_EINVAL, "readout: the workspace is too small or not at a multiple of 16 bytes");
  ytm::ReadoutArgs a{x, x_dtype, x_stride, N, C, codes, code_stride, scales, scale_stride, group, K, out, out_dtype,
                     out_stride, (ytm::v4u*)workspace, ytm::steps_of(C), ytm::tiles_of(N)};
  hipStream_t s = (hipStream_t)stream;
  const hipError_t e = x_dtype == YTM_DTYPE_F16   ? ytm::launch_readout<1, true>(a, scale_dtype, s)
                       : x_dtype == YTM_DTYPE_F32 ? ytm::launch_readout<3, false>(a, scale_dtype, s)
                                                  : ytm::launch_readout<1, false>(a, scale_dtype, s);
  if (e != hipSuccess) return fail(YTM_EHIP, std::string("readout failed: ") + hipGetErrorString(e));
  return YTM_OK;
}

}  // extern "C"
