// ytm_readout.hip -- class sums from clause outputs through weights held in 4 bits: the entry
// point ytm_readout of include/ytm.h and its gfx950 kernels.
//
//   out[n][o] = sum over groups q of scale[o][q] * sum over clauses c of q of x[n][c] value(code[o][c])
//
// A code is an E2M1 float (0, 0.5, 1, 1.5, 2, 3, 4, 6 and their negatives), exact in float16 and
// bfloat16, into which gfx950 converts two codes an instruction; so the inner sums run on the
// matrix cores in f32 with operands that are no less exact than x: float16 and bfloat16 as they
// are, float32 as the sum of three bfloat16 (8 + 8 + 8 bits of its fraction), a product each.  Bits
// are E2M1 floats themselves, 0 and 1, which the matrix cores multiply with the codes as they are.
// The scale multiplies each group's f32 sum.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "ytm_decode.h"
#include "ytm_internal.h"

namespace ytm {

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef int v8i __attribute__((ext_vector_type(8)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

constexpr int kWave = 64;
constexpr int kTile = 16;    // rows and outputs of a product
constexpr int kStep = 32;    // clauses of a product
constexpr int kChunk = 128;  // clauses of a 16-byte load of codes by each lane, four products
constexpr int kPieces = 16;  // of 8 clauses, in a chunk: a lane's part of a product's row operand
constexpr int kWords = 4;    // of 32 bits, in a chunk: the same of a product with bits, which takes a whole chunk

struct ReadoutArgs {
  const void* x;
  int64_t x_stride;
  int N, C;
  const uint8_t* codes;
  int64_t code_stride;
  const void* scales;
  int scale_dtype;
  int64_t scale_stride;
  uint32_t inverse;  // (step + 1) * inverse >> 32 is the group of clauses 32 step ..
  int K;
  void* out;
  int out_dtype;
  int64_t out_stride;
  int chunks, part_chunks, out_tiles, row_tiles;
  float* parts;  // the workspace, of few rows' sums or many rows' operands
  v4u* frag;
};

// What x is: its element, the number of 16-bit operands it is the sum of, whether these are float16.
template <int X>
constexpr int kSize = X == YTM_DTYPE_BITS || X == YTM_DTYPE_F32 ? 4 : 2;  // bytes of what x_stride counts
template <int X>
struct Kind;
template <>
struct Kind<YTM_DTYPE_BITS> {
  static constexpr int kPlanes = 1;
  static constexpr bool kHalf = false;
};
template <int X>
constexpr bool kBits = X == YTM_DTYPE_BITS;
template <>
struct Kind<YTM_DTYPE_F16> {
  static constexpr int kPlanes = 1;
  static constexpr bool kHalf = true;
};
template <>
struct Kind<YTM_DTYPE_BF16> {
  static constexpr int kPlanes = 1;
  static constexpr bool kHalf = false;
};
template <>
struct Kind<YTM_DTYPE_F32> {
  static constexpr int kPlanes = 3;
  static constexpr bool kHalf = false;
};

// Operands that 16 rows' clauses of a chunk make, 1 KB each.
constexpr int operands_of(int x_dtype) {
  return x_dtype == YTM_DTYPE_BITS ? 1 : x_dtype == YTM_DTYPE_F32 ? 12 : 4;
}
template <int X>
constexpr int kOperands = operands_of(X);

// ------------------------------------------------------------------------------- row operands
// Eight clauses of a row as they are in memory, and as 16-bit operands: float32
// as the sum of three bfloat16, each cut (not rounded) to one, so that nothing overflows; where
// the first is infinite or NaN the others are zero.  What a float has below 2^-133, the least bfloat16,
// is left out.
//
// The load has no branch (rows have eight clauses or more), so that others can follow it before
// it is there: a piece that would pass the row's end is taken from its last eight clauses, and moved
// to its place, with zeros after it, when it becomes operands.
template <int X>
struct Piece {
  static constexpr int kWords = X == YTM_DTYPE_F32 ? 8 : 4;
  uint32_t raw[kWords];

  // of the row `off` bytes from x's uniform address `x`, clauses c .. c + 7
  __device__ __forceinline__ void load(const ReadoutArgs& a, const char* x, uint32_t off, int c) {
    const int at = c < a.C - 8 ? c : a.C - 8;
    __builtin_memcpy(raw, x + (off + at * (X == YTM_DTYPE_F32 ? 4 : 2)), sizeof raw);
  }

  // the operands of clauses c .. c + 7, which load() was asked for
  __device__ __forceinline__ void operands(const ReadoutArgs& a, int c, v4u (&plane)[Kind<X>::kPlanes]) const {
    const int over = c + 8 - a.C;  // of the eight, past the last clause
    uint32_t r[kWords];
#pragma unroll
    for (int q = 0; q < kWords; ++q) r[q] = raw[q];
    if (over > 0) {  // what is in place `over` moves to place 0
      if (X == YTM_DTYPE_F32) {
#pragma unroll
        for (int d = 1; d < 8; d <<= 1)
#pragma unroll
          for (int q = 0; q < kWords; ++q) r[q] = over & d ? (q + d < kWords ? r[(q + d) % kWords] : 0u) : r[q];
      } else {
#pragma unroll
        for (int q = 0; q < kWords; ++q) {
          const uint32_t next = q + 1 < kWords ? r[(q + 1) % kWords] : 0u;
          r[q] = over & 1 ? r[q] >> 16 | next << 16 : r[q];
        }
#pragma unroll
        for (int d = 1; d < 4; d <<= 1)
#pragma unroll
          for (int q = 0; q < kWords; ++q) r[q] = over & 2 * d ? (q + d < kWords ? r[(q + d) % kWords] : 0u) : r[q];
      }
      if (over >= 8) {
#pragma unroll
        for (int q = 0; q < kWords; ++q) r[q] = 0u;
      }
    }
    if (X != YTM_DTYPE_F32) {
#pragma unroll
      for (int q = 0; q < 4; ++q) plane[0][q] = r[q % kWords];
      return;
    }
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      uint32_t part[3][2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const uint32_t u = r[(2 * q + h) % kWords];
        const bool finite = (u & 0x7F800000u) != 0x7F800000u;
        const float rest = finite ? __uint_as_float(u) - __uint_as_float(u & 0xFFFF0000u) : 0.0f;
        part[0][h] = (u & 0x7FFFFFFFu) > 0x7F800000u ? u | 0x00400000u : u;  // a NaN stays one
        part[1][h] = __float_as_uint(rest);
        part[2][h] = __float_as_uint(rest - __uint_as_float(part[1][h] & 0xFFFF0000u));
      }
#pragma unroll
      for (int p = 0; p < Kind<X>::kPlanes; ++p)
        plane[p][q] = __builtin_amdgcn_perm(part[p][1], part[p][0], 0x07060302u);
    }
  }
};

// Word i of a row's bits, and as E2M1 floats: a bit's 1 is 0010.
__device__ __forceinline__ uint32_t load_bits(const ReadoutArgs& a, const char* x, uint32_t off, int i) {
  const int last = (a.C - 1) / 32;
  return *(const uint32_t*)(x + (off + 4 * (i < last ? i : last)));
}
__device__ __forceinline__ v4u bit_operand(const ReadoutArgs& a, uint32_t bits, int i) {
  const int left = a.C - 32 * i;
  bits = left >= 32 ? bits : left > 0 ? bits & ((1u << left) - 1u) : 0u;
  v4u r;
#pragma unroll
  for (int q = 0; q < 4; ++q) {  // eight bits four places apart
    uint32_t u = bits >> 8 * q & 0xFFu;
    u = (u | u << 12) & 0x000F000Fu;
    u = (u | u << 6) & 0x03030303u;
    u = (u | u << 3) & 0x11111111u;
    r[q] = u << 1;
  }
  return r;
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

// A whole chunk's product of bits and codes, each lane's 32 clauses of a row and of an output.
__device__ __forceinline__ v4f bit_product(v4u x, v4u w) {
  const v8i p = {(int)x[0], (int)x[1], (int)x[2], (int)x[3], 0, 0, 0, 0};
  const v8i q = {(int)w[0], (int)w[1], (int)w[2], (int)w[3], 0, 0, 0, 0};
  return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(p, q, v4f{0.0f, 0.0f, 0.0f, 0.0f}, 4, 4, 0, 0, 0, 0);
}

// A lane of group g = l / 16 holds a chunk's clauses 32 g .. 32 g + 31 in four words of codes, and
// a product takes one word of each lane.  Where a scale holds for the whole chunk (GRAIN 128),
// product s takes word s as it is: clauses 32 g + 8 s .., the row operands' alike.  Where it does
// not (GRAIN 32), the words are exchanged first so that product s has clauses 32 s + 8 g ..:
// a 4 x 4 transposition in two exchanges of bits of (group, word).  A product with bits takes all
// four words, and where a scale does not hold for the chunk, one for each group of lanes, with zeros for
// the other groups' bits: as many cycles as the four of 16-bit operands, without their conversion.
__device__ __forceinline__ v4u only(v4u w, int group) {
  const bool mine = threadIdx.x % kWave / 16 == group;
  return v4u{mine ? w[0] : 0u, mine ? w[1] : 0u, mine ? w[2] : 0u, mine ? w[3] : 0u};
}
template <int GRAIN>
__device__ __forceinline__ v4u turn(v4u w) {
  if (GRAIN == kChunk) return w;
  auto a = __builtin_amdgcn_permlane32_swap(w[0], w[2], false, false);
  auto b = __builtin_amdgcn_permlane32_swap(w[1], w[3], false, false);
  auto c = __builtin_amdgcn_permlane16_swap(a[0], b[0], false, false);
  auto d = __builtin_amdgcn_permlane16_swap(a[1], b[1], false, false);
  return v4u{c[0], c[1], d[0], d[1]};
}
// (step, lane group) of piece i (clauses 8 i ..) of a chunk, as 4 step + group.
template <int GRAIN>
__device__ __forceinline__ int place_of(int i) {
  return GRAIN == kChunk ? 4 * (i % 4) + i / 4 : i;
}

// A scale from its two halves, or the same 16 bits twice.
__device__ __forceinline__ float scale_value(const ReadoutArgs& a, uint16_t low, uint16_t high) {
  const float half = (float)__builtin_bit_cast(_Float16, high);
  const float full = __uint_as_float((uint32_t)high << 16 | (a.scale_dtype == YTM_DTYPE_F32 ? low : 0u));
  return a.scale_dtype == YTM_DTYPE_F16 ? half : full;
}

// A chunk's codes of one output a lane, and a scale: that of the whole chunk (GRAIN 128), or of the
// 32 clauses whose codes the lane holds, which turn() then hands to all.  WIDE: scales are float32.
template <int GRAIN, bool WIDE>
struct Codes {
  v4u w;
  typename std::conditional<WIDE, float, uint16_t>::type scale;

  // of the output whose codes are `code` bytes from the uniform address `codes` and whose scales are
  // `at` bytes from `scales`.  Past the last clause the last codes are taken: the rows are zero there.
  __device__ __forceinline__ void load(const ReadoutArgs& a, const uint8_t* codes, uint32_t code, const char* scales,
                                       uint32_t at, int chunk) {
    const uint32_t steps = (a.C + kStep - 1) / kStep;
    const uint32_t mine = chunk * 4 + threadIdx.x % kWave / 16;
    w = *(const v4u*)(codes + (code + 16 * (mine < steps ? mine : steps - 1)));
    const uint32_t step = GRAIN == kChunk ? chunk * 4 : mine;
    const uint32_t q = __umulhi(step < steps ? step + 1 : steps, a.inverse);
    scale = *(const decltype(scale)*)(scales + (at + q * (uint32_t)sizeof scale));
  }
  // scales of the four products, zero past the last clause: infinity by the zeros there would be NaN
  __device__ __forceinline__ void scaled(const ReadoutArgs& a, int chunk, float (&f)[4]) const {
    uint32_t u;
    if constexpr (WIDE)
      u = __float_as_uint(scale);
    else
      u = __float_as_uint(scale_value(a, scale, scale));
    const v4u t = turn<GRAIN>(v4u{u, u, u, u});
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const uint32_t there = GRAIN == kChunk ? ~0u : (uint32_t)((chunk * 4 + s - (a.C + kStep - 1) / kStep) >> 31);
      f[s] = __uint_as_float(t[s] & there);
    }
  }
};

__device__ __forceinline__ void store_out(const ReadoutArgs& a, int n, int o, float v) {
  const int64_t i = n * a.out_stride + o;
  switch (a.out_dtype) {
    case YTM_DTYPE_F16: ((f16*)a.out)[i] = from_float<f16>(v); break;
    case YTM_DTYPE_BF16: ((bf16*)a.out)[i] = from_float<bf16>(v); break;
    default: ((float*)a.out)[i] = v; break;
  }
}

// A chunk's products of a row tile, whose operands lie at from[plane * .. + step * ..], and OB output
// tiles, added to the sums so far.  One output tile after the other, so that the scaling of one can go
// beside the products of the next; code(b, w, scale) gives tile b's codes and the scales of its four
// products.
template <int X, int GRAIN, int OB, typename Code>
__device__ __forceinline__ void add_chunk(const v4u* from, int plane, int step, v4f (&total)[OB], Code code) {
  constexpr int kPlanes = Kind<X>::kPlanes;
  constexpr bool kHalf = Kind<X>::kHalf;
  v4u x[4][kPlanes];
#pragma unroll
  for (int s = 0; s < 4; ++s)
#pragma unroll
    for (int p = 0; p < kPlanes; ++p) x[s][p] = from[p * plane + s * step];
#pragma unroll
  for (int b = 0; b < OB; ++b) {
    v4u w;
    float scale[4];
    code(b, w, scale);
    w = turn<GRAIN>(w);
    v4f sum;
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const v4u y = codes_to_16<kHalf>(w[s]);
      if (s * kStep % GRAIN == 0) sum = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int p = kPlanes - 1; p >= 0; --p) sum = product<kHalf>(x[s][p], y, sum);
      if ((s + 1) * kStep % GRAIN == 0) {
#pragma unroll
        for (int r = 0; r < 4; ++r) total[b][r] = __builtin_fmaf(scale[s], sum[r], total[b][r]);
      }
    }
  }
}

// Many rows: their operands in the order in which products take them, frag[chunk][plane][step][row
// tile][lane], zero past the last clause, the last row's past the last row.  A block makes a chunk
// (the grid's first axis) of a row tile, a thread a piece; 16 of them read 256 or 512 bytes in a row.
template <int X, int GRAIN>
__global__ __launch_bounds__(kPieces* kTile) void rows_kernel(ReadoutArgs a) {
  if constexpr (kBits<X>) {  // frag[chunk][row tile][lane]: a block makes four chunks of a row tile
    const int row = threadIdx.x / kPieces, i = threadIdx.x % kPieces, chunk = blockIdx.x * 4 + i / kWords;
    const int tile = blockIdx.y, n = tile * kTile + row < a.N ? tile * kTile + row : a.N - 1;
    const uint32_t bits = load_bits(a, (const char*)a.x + n * a.x_stride * 4, 0, blockIdx.x * kPieces + i);
    a.frag[((int64_t)chunk * a.row_tiles + tile) * kWave + i % kWords * 16 + row] =
        bit_operand(a, bits, blockIdx.x * kPieces + i);
    return;
  }
  constexpr int kPlanes = Kind<X>::kPlanes;
  const int chunk = blockIdx.x, tile = blockIdx.y, row = threadIdx.x / kPieces, i = threadIdx.x % kPieces;
  const int place = place_of<GRAIN>(i), c = chunk * kChunk + i * 8;
  const int n = tile * kTile + row < a.N ? tile * kTile + row : a.N - 1;
  Piece<X> piece;
  v4u plane[kPlanes];
  piece.load(a, (const char*)a.x + n * a.x_stride * kSize<X>, 0, c);
  piece.operands(a, c, plane);
#pragma unroll
  for (int p = 0; p < kPlanes; ++p)
    a.frag[(((int64_t)(chunk * kPlanes + p) * 4 + place / 4) * a.row_tiles + tile) * kWave + place % 4 * 16 + row] =
        plane[p];
}

// ---------------------------------------------------------------------- copies into LDS, and waits
// A wave's copy from memory into LDS that passes no register: lane l's 16 bytes (4 or 2, which take
// a word each) from `off` bytes after the uniform address `from`, to `at` (uniform) and on, lane after
// lane.  The compiler knows nothing of them: await() waits for all but the wave's youngest LEFT copies
// and for its reads of LDS, and then for the block's other waves.  What it loads itself meanwhile only
// makes that wait longer.
__device__ __forceinline__ uint32_t lds_address(const void* p) {
  return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}
template <int BYTES>
__device__ __forceinline__ void copy_to_lds(const void* from, uint32_t off, uint32_t at) {
  if (BYTES == 16)
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(from), "s"(at)
                 : "memory", "m0");
  else if (BYTES == 4)
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1" ::"v"(off), "s"(from), "s"(at)
                 : "memory", "m0");
  else
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_ushort %0, %1" ::"v"(off), "s"(from), "s"(at)
                 : "memory", "m0");
}
template <int LEFT>
__device__ __forceinline__ void await() {
  static_assert(LEFT < 64, "what the counter of loads holds");
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"n"(LEFT) : "memory");
}

// A block takes 16 NT RW rows and 16 OB WO outputs; its waves are WK groups, each with pairs of chunks of
// clauses of its own, of WO x RW waves, each with NT tiles of rows and OB of outputs.  Lane l takes
// the codes of output l % 16 as a product's second operand and gets sums of rows 4 (l / 16) .. + 3
// of that output.
//
// A group's chunks pass through LDS: the rows' operands in a ring of three chunks (two where three do
// not fit), the outputs' codes and scales in one of two pairs, of which each output's codes are 128
// bytes in a row.  A wave has a chunk's operands in registers before the chunk begins, so that there
// is one wait a chunk, at its start: for the next chunk to be in LDS, and for all waves to have read this
// one, whose place then takes the chunk after the ring's last.  Copies are thus under way for
// two chunks, which eight waves a CU, in step, have nothing else to hide.  A group's sums are scaled
// beside the products of the next.
//
// 512 rows x 20000 clauses x 10000 outputs of bfloat16 (groups of 128): 200 us, 1.0 PFLOP/s; with loads
// through registers a chunk ahead and LDS read where it was needed, 256.  Of the 200 about 40 go without
// the copies; the rest is the matrix unit at the clock that it leaves, and vector work that shares
// its issue: per product of 16 cycles two conversions, and one multiply-add and one other instruction.
// Bits, with a quarter of the products and no conversion: 10000 x 10000, 512 rows 62 us (109 through 16 bits).
template <int X, int GRAIN, int NT, int RW, int OB, int WO, int WK>
__global__ __launch_bounds__(kWave* RW* WO* WK) void tile_kernel(ReadoutArgs a) {
  constexpr int kPlanes = Kind<X>::kPlanes;
  constexpr bool kHalf = Kind<X>::kHalf;
  constexpr int kGroupWaves = RW * WO;
  constexpr int kTiles = NT * RW;               // of rows
  constexpr int kFrags = kOperands<X> * kTiles;  // operands of a chunk, 1 KB each
  constexpr int kOuts = kTile * OB * WO;
  static_assert(kOuts <= kMaxTogether, "32-bit distances of codes and scales");
  constexpr int kGrains = kChunk / GRAIN;  // scales of a chunk
  // copies a wave makes, the last of them twice where they do not come out even
  constexpr int kRowCopies = (kFrags + kGroupWaves - 1) / kGroupWaves;
  constexpr int kCodeCopies = (kOuts / 8 + kGroupWaves - 1) / kGroupWaves;
  constexpr int kScaleAll = 2 * kGrains * kOuts / kWave;
  constexpr int kScaleCopies = (kScaleAll + kGroupWaves - 1) / kGroupWaves;
  static_assert(2 * kGrains * kOuts % kWave == 0, "");
  constexpr int kPairSpace = 2 * WK * (kOuts * 8 * 16 + 2 * kGrains * kOuts * 4);
  constexpr int kSlots = 3 * WK * kFrags * 1024 + kPairSpace <= 160 * 1024 ? 3 : 2;
  constexpr int kJoin = (WK - 1) * kGroupWaves * NT * OB;
  static_assert(kJoin <= kSlots * WK * kFrags + 2 * WK * kOuts * 8 / kWave, "");
  constexpr int kRowSpace = kSlots * WK * kFrags * kWave;
  __shared__ v4u held[kRowSpace + 2 * WK * kOuts * 8];  // rows, then codes
  v4u(*held_rows)[WK][kFrags * kWave] = (v4u(*)[WK][kFrags * kWave])held;
  v4u(*held_codes)[WK][kOuts * 8] = (v4u(*)[WK][kOuts * 8])(held + kRowSpace);
  __shared__ __attribute__((aligned(16))) uint32_t held_scales[2][WK][kOuts * 2 * kGrains];

  // blocks of the same outputs one after the other on the same XCD, whose L2 then has the codes
  const int row_blocks = (a.row_tiles + kTiles - 1) / kTiles;
  const int slot = blockIdx.x / 8;
  const int out_tile = slot / row_blocks * 8 + blockIdx.x % 8, row_block = slot % row_blocks;
  if (out_tile >= a.out_tiles) return;
  const int l = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int group = wave / kGroupWaves, mine = wave % kGroupWaves, wo = mine / RW, rw = mine % RW;
  const int block_out = out_tile * kOuts;

  // uniform addresses and 32-bit distances from them take fewer registers than addresses
  const bool wide = a.scale_dtype == YTM_DTYPE_F32;
  const uint32_t size = wide ? 4 : 2;
  const uint8_t* codes = a.codes + block_out * a.code_stride;
  const char* scales = (const char*)a.scales + block_out * a.scale_stride * size;
  // outputs past the last take its codes and are not stored
  const auto output = [&](int o) { return (uint32_t)((block_out + o < a.K ? block_out + o : a.K - 1) - block_out); };
  const auto code_copy = [&](int e) {  // which 8 outputs' codes
    const int f = e * kGroupWaves + mine;
    return f < kOuts / 8 ? f : kOuts / 8 - 1;
  };
  const auto row_copy = [&](int e) {
    const int f = e * kGroupWaves + mine;
    return f < kFrags ? f : kFrags - 1;
  };
  const auto scale_copy = [&](int e) {
    const int f = e * kGroupWaves + mine;
    return f < kScaleAll ? f : kScaleAll - 1;
  };
  // Piece p of output o's eight in a pair lies at place p ^ o % 8 of its 128 bytes, so that 16 outputs'
  // same piece is in different banks.
  uint32_t code_off[kCodeCopies], scale_off[kScaleCopies];
#pragma unroll
  for (int e = 0; e < kCodeCopies; ++e) code_off[e] = output(code_copy(e) * 8 + l / 8) * (uint32_t)a.code_stride;
#pragma unroll
  for (int e = 0; e < kScaleCopies; ++e)
    scale_off[e] = output((scale_copy(e) * kWave + l) / (2 * kGrains)) * (uint32_t)a.scale_stride * size;
  const int all_pairs = (a.chunks + 2 * WK - 1) / (2 * WK);
  const int first_pair = blockIdx.y * a.part_chunks;  // of this part; part_chunks counts pairs here
  const int pairs = all_pairs - first_pair < a.part_chunks ? all_pairs - first_pair : a.part_chunks;
  const uint32_t steps = (a.C + kStep - 1) / kStep;
  const int padded = all_pairs * 2 * WK;
  // What is copied past the part's end is not used: copies are made all the same, so that their
  // number is known where they are waited for.  Rows are zero from the last clause to the last pair's end.
  const auto chunk_of = [&](int i) { return ((first_pair + i / 2) * WK + group) * 2 + i % 2; };
  const auto copy_rows = [&](int i, int to) {  // of the group's chunk i
    const int own = chunk_of(i), chunk = own < padded ? own : padded - 1;
    const uint32_t at = lds_address(held_rows) + (to * WK + group) * kFrags * 1024;
#pragma unroll
    for (int e = 0; e < kRowCopies; ++e) {  // row tiles past the last take its rows and are not stored
      const int f = row_copy(e), tile = row_block * kTiles + f % kTiles;
      const v4u* from = a.frag + (((int64_t)chunk * kOperands<X> + f / kTiles) * a.row_tiles +
                                  (tile < a.row_tiles ? tile : a.row_tiles - 1)) * kWave;
      copy_to_lds<16>(from, l * 16, at + f * 1024);
    }
  };
  const auto copy_codes = [&](int pair) {
    const uint32_t first = chunk_of(2 * pair) * 4;  // step
    const int place = pair % 2 * WK + group;
    const uint32_t step = first + (l % 8 ^ l / 8);
#pragma unroll
    for (int e = 0; e < kCodeCopies; ++e)
      copy_to_lds<16>(codes, code_off[e] + 16 * (step < steps ? step : steps - 1),
                      lds_address(held_codes) + place * kOuts * 128 + code_copy(e) * 1024);
    const uint32_t at = lds_address(held_scales) + place * kOuts * 2 * kGrains * 4;
#pragma unroll
    for (int e = 0; e < kScaleCopies; ++e) {
      const uint32_t of = first + l % (2 * kGrains) * (4 / kGrains);
      const uint32_t off = scale_off[e] + __umulhi(of < steps ? of + 1 : steps, a.inverse) * size;
      if (wide)
        copy_to_lds<4>(scales, off, at + scale_copy(e) * 256);
      else
        copy_to_lds<2>(scales, off, at + scale_copy(e) * 256);
    }
  };

  v4f total[NT][OB];
#pragma unroll
  for (int b = 0; b < OB; ++b)
#pragma unroll
    for (int n = 0; n < NT; ++n) total[n][b] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  struct Operands {  // a wave's of a chunk
    v4u x[kOperands<X>][NT], w[OB];
    uint32_t scale[OB][kGrains];
  };
  const auto read = [&](int i, int from, Operands& to) {
#pragma unroll
    for (int b = 0; b < OB; ++b) {
      const int place = i / 2 % 2, half = i % 2, o = (wo * OB + b) * kTile + l % 16;
      to.w[b] = held_codes[place][group][o * 8 + ((half * 4 + l / 16) ^ l % 8)];
#pragma unroll
      for (int g = 0; g < kGrains; ++g) to.scale[b][g] = held_scales[place][group][(o * 2 + half) * kGrains + g];
    }
#pragma unroll
    for (int q = 0; q < kOperands<X>; ++q)
#pragma unroll
      for (int n = 0; n < NT; ++n) to.x[q][n] = held_rows[from][group][(q * kTiles + rw * NT + n) * kWave + l];
  };
  const int shift = wide ? 0 : 16;
  const uint32_t halves = a.scale_dtype == YTM_DTYPE_F16 ? ~0u : 0u;
  v4f last[NT];  // the sums before these, and their scale
  float due = 0.0f;
#pragma unroll
  for (int n = 0; n < NT; ++n) last[n] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  const auto scaled = [&](int b) {
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
      for (int r = 0; r < 4; ++r) total[n][b][r] = __builtin_fmaf(due, last[n][r], total[n][b][r]);
  };

  Operands now[2];
  copy_codes(0);
  copy_rows(0, 0);
#pragma unroll
  for (int i = 1; i < kSlots; ++i) copy_rows(i, i);
  copy_codes(1);
  await<(kSlots - 1) * kRowCopies + kCodeCopies + kScaleCopies>();
  read(0, 0, now[0]);
  int at = 0;  // the chunk's place in the ring
  for (int pair = 0; pair < pairs; ++pair) {
#pragma unroll
    for (int half = 0; half < 2; ++half) {
      const int i = 2 * pair + half, next = at + 1 < kSlots ? at + 1 : 0;
      // Of what is younger than the next chunk's: a chunk's rows in a ring of three, and where
      // this chunk is the first of its pair, the codes that its predecessor asked for.
      if (half == 0)
        await<(kSlots - 2) * kRowCopies + kCodeCopies + kScaleCopies>();
      else
        await<(kSlots - 2) * kRowCopies>();
      copy_rows(i + kSlots, at);
      if (half == 1) copy_codes(pair + 2);
      read(i + 1, next, now[1 - half]);
      const Operands& o = now[half];
      const uint32_t first = chunk_of(i) * 4;
#pragma unroll
      for (int b = 0; b < OB; ++b) {
        const v4u w = kBits<X> ? o.w[b] : turn<GRAIN>(o.w[b]);
#pragma unroll
        for (int g = 0; g < kGrains; ++g) {
          v4f sum[NT];
          if constexpr (kBits<X>) {
            const v4u y = kGrains == 1 ? w : only(w, g);
#pragma unroll
            for (int n = 0; n < NT; ++n) sum[n] = bit_product(o.x[0][n], y);
          } else {
#pragma unroll
            for (int n = 0; n < NT; ++n) sum[n] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int s = 4 / kGrains * g; s < 4 / kGrains * (g + 1); ++s) {
              const v4u y = codes_to_16<kHalf>(w[s]);
#pragma unroll
              for (int p = kPlanes - 1; p >= 0; --p)
#pragma unroll
                for (int n = 0; n < NT; ++n) sum[n] = product<kHalf>(o.x[p * 4 + s][n], y, sum[n]);
            }
          }
          scaled(g > 0 ? b : b > 0 ? b - 1 : OB - 1);
          // Zero past the last clause, as in few rows.  By masks, since uniform choices become branches,
          // which keep products and scaling apart.
          const uint32_t u = o.scale[b][g];
          const uint32_t half_bits = __float_as_uint((float)__builtin_bit_cast(_Float16, (uint16_t)u));
          const uint32_t there = (uint32_t)((int32_t)(first + g * (4 / kGrains) - steps) >> 31);
          due = __uint_as_float(((half_bits & halves) | (u << shift & ~halves)) & there);
#pragma unroll
          for (int n = 0; n < NT; ++n) last[n] = sum[n];
          // or the compiler puts the products of all groups first, whose sums take more registers than there are
          if (kGrains > 1) __builtin_amdgcn_sched_barrier(0);
        }
      }
      at = next;
    }
  }
  scaled(OB - 1);
  await<0>();  // no copy comes after the block's end, or into the sums to be joined
  v4f* join = (v4f*)held;
  if (WK > 1) {
    if (group > 0) {
#pragma unroll
      for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int b = 0; b < OB; ++b)
          join[(((group - 1) * kGroupWaves + mine) * NT * OB + n * OB + b) * kWave + l] = total[n][b];
    }
    __syncthreads();
    if (group > 0) return;
  }
#pragma unroll
  for (int n = 0; n < NT; ++n)
#pragma unroll
    for (int b = 0; b < OB; ++b) {
      v4f v = total[n][b];
      for (int g = 0; g < WK - 1; ++g) v += join[((g * kGroupWaves + mine) * NT * OB + n * OB + b) * kWave + l];
      const int o = block_out + (wo * OB + b) * kTile + l % 16;
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int row = (row_block * kTiles + rw * NT + n) * kTile + l / 16 * 4 + r;
        if (o >= a.K || row >= a.N) continue;
        if (gridDim.y > 1)
          a.parts[((int64_t)blockIdx.y * a.N + row) * a.K + o] = v[r];
        else
          store_out(a, row, o, v[r]);
      }
    }
}

// The parts' sums added in their order.
__global__ __launch_bounds__(256) void parts_kernel(ReadoutArgs a, int parts) {
  const int64_t each = (int64_t)a.N * a.K;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < each; i += (int64_t)gridDim.x * blockDim.x) {
    float v = a.parts[i];
    for (int p = 1; p < parts; ++p) v += a.parts[p * each + i];
    store_out(a, (int)(i / a.K), (int)(i % a.K), v);
  }
}
hipError_t launch_parts(const ReadoutArgs& a, int parts, hipStream_t s) {
  const int64_t blocks = ((int64_t)a.N * a.K + 255) / 256;
  parts_kernel<<<(unsigned)(blocks < 4096 ? blocks : 4096), 256, 0, s>>>(a, parts);
  return hipGetLastError();
}

// What a block of tile_kernel takes: 32 or 64 rows where there are no more; float32, whose operands
// take three times the LDS, up to 64; else 64, 96 or 128 rows by the rounds in which the 256 CUs take the
// blocks, at 4, 5 and 7 units of time each (fewer blocks than half the CUs are cut into parts, and
// count as what they are).  10000 clauses x 10000 outputs in groups of 32, blocks of 64 and of 96 rows:
// 192 rows 86 and 106 us (one round each), 320 rows 129 and 160 (two), 500 rows 243 and 207 (three, two).
// With four scales a chunk (grain 32) 128 rows' sums and operands do not fit the registers and take
// three times as long.
struct Tile {
  int rows, outs, groups;
};
Tile tile_of(int operands, int grain, int N, int K) {
  const bool whole = grain == kChunk;
  if (operands > 4) return N <= 32 ? Tile{32, 128, 1} : Tile{64, whole ? 128 : 96, 1};
  if (N <= 32) return Tile{32, 128, 2};
  const Tile tiles[3] = {{64, 128, whole ? 2 : 1}, {96, 128, 1}, {128, 160, 1}};
  constexpr int kTime[3] = {4, 5, 7};
  int best = 0;
  int64_t least = 0;
  for (int i = 0; i < (N <= 64 ? 1 : whole ? 3 : 2); ++i) {
    const int64_t blocks =
        (int64_t)((N + tiles[i].rows - 1) / tiles[i].rows) * ((K + tiles[i].outs - 1) / tiles[i].outs);
    const int64_t time = (blocks > 128 ? (blocks + 255) / 256 * 256 : blocks) * kTime[i];
    if (i == 0 || time < least) least = time, best = i;
  }
  return tiles[best];
}
// Pairs of chunks in a part of the clauses: all, or where that leaves half of the 256 CUs without
// a block, as many as give each CU one (103 rows x 10012 clauses x 22 outputs, one block: 909 us;
// two pairs a part: 21).
int part_pairs_of(int operands, int grain, int N, int chunks, int K) {
  const Tile t = tile_of(operands, grain, N, K);
  const int64_t blocks = (int64_t)((N + t.rows - 1) / t.rows) * ((K + t.outs - 1) / t.outs);
  const int pairs = (chunks + 2 * t.groups - 1) / (2 * t.groups);
  if (blocks > 128 || pairs < 4) return pairs;
  const int parts = (int)(256 / blocks) < pairs / 2 ? (int)(256 / blocks) : pairs / 2;
  return (pairs + parts - 1) / parts;
}
int tile_parts_of(int operands, int grain, int N, int chunks, int K) {
  const Tile t = tile_of(operands, grain, N, K);
  const int each = part_pairs_of(operands, grain, N, chunks, K);
  return ((chunks + 2 * t.groups - 1) / (2 * t.groups) + each - 1) / each;
}
// Chunks of the rows' operands: whole pairs for each group of waves, of which a block has up to two.
int padded_of(int chunks) { return (chunks + 3) / 4 * 4; }
int64_t frag_bytes(int operands, int N, int chunks) {
  return (int64_t)(N + kTile - 1) / kTile * padded_of(chunks) * operands * kWave * 16;
}

template <int X, int GRAIN, int NT, int RW, int OB, int WO, int WK>
hipError_t launch_tile(ReadoutArgs a, hipStream_t s) {
  a.row_tiles = (a.N + kTile - 1) / kTile;
  a.part_chunks = part_pairs_of(kOperands<X>, GRAIN, a.N, a.chunks, a.K);
  a.parts = (float*)((char*)a.frag + frag_bytes(kOperands<X>, a.N, a.chunks));
  const int parts = tile_parts_of(kOperands<X>, GRAIN, a.N, a.chunks, a.K);
  rows_kernel<X, GRAIN><<<dim3(padded_of(a.chunks) / (kBits<X> ? 4 : 1), a.row_tiles), kPieces * kTile, 0, s>>>(a);
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  // A launch counts its threads in 32 bits, and one of more leaves blocks out without an error, so more
  // outputs than that take several (never in parts, which few blocks are cut into).
  constexpr int kThreads = kWave * RW * WO * WK, kOuts = kTile * OB * WO;
  const int64_t row_blocks = (a.row_tiles + NT * RW - 1) / (NT * RW), K = a.K;
  const int64_t most = (int64_t)UINT32_MAX / kThreads / row_blocks / 8 * 8 * kOuts;
  const int out_size = a.out_dtype == YTM_DTYPE_F32 ? 4 : 2, scale_size = a.scale_dtype == YTM_DTYPE_F32 ? 4 : 2;
  for (int64_t done = 0; done < K; done += most) {
    a.K = (int)(K - done < most ? K - done : most);
    a.out_tiles = (a.K + kOuts - 1) / kOuts;
    const unsigned grid = (unsigned)((a.out_tiles + 7) / 8 * 8 * row_blocks);
    tile_kernel<X, GRAIN, NT, RW, OB, WO, WK><<<dim3(grid, parts), kThreads, 0, s>>>(a);
    e = hipGetLastError();
    if (e != hipSuccess) return e;
    if (done + most >= K) break;  // and the addresses stay within their tensors
    a.codes += most * a.code_stride;
    a.scales = (const char*)a.scales + most * a.scale_stride * scale_size;
    a.out = (char*)a.out + most * out_size;
  }
  return parts == 1 ? e : launch_parts(a, parts, s);
}
template <int X, int GRAIN>
hipError_t launch_tiles(const ReadoutArgs& a, hipStream_t s) {
  const int rows = tile_of(kOperands<X>, GRAIN, a.N, a.K).rows;
  if constexpr (Kind<X>::kPlanes > 1) {
    if (rows == 32) return launch_tile<X, GRAIN, 2, 1, 2, 4, 1>(a, s);
    if constexpr (GRAIN == kChunk) return launch_tile<X, GRAIN, 2, 2, 2, 4, 1>(a, s);
    else return launch_tile<X, GRAIN, 1, 4, 3, 2, 1>(a, s);
  } else {
    if (rows == 32) return launch_tile<X, GRAIN, 2, 1, 2, 4, 2>(a, s);
    if (rows == 96) return launch_tile<X, GRAIN, 3, 2, 2, 4, 1>(a, s);
    if constexpr (GRAIN == kChunk)
      return rows == 64 ? launch_tile<X, GRAIN, 4, 1, 2, 4, 2>(a, s) : launch_tile<X, GRAIN, 2, 4, 5, 2, 1>(a, s);
    else
      return launch_tile<X, GRAIN, 2, 2, 2, 4, 1>(a, s);
  }
}

// Few rows (up to 16), bound by the codes' bytes: one row of 9973 bits x 10000 outputs takes 14.5 us,
// 3.6 TB/s (through products of 16-bit operands 18.5: two thirds of the vector work was their
// conversion).  A block has 16 OB WO outputs and the clauses of one of the parts that the
// grid's second axis counts, whose row operands lie in LDS from the start (without those of rows
// that are not there), so that nothing waits between its first and last chunk.  WK waves share
// an output tile's chunks, two at a time (128 bytes of codes); each loads kAhead of them before the
// first is looked at.  With more
// than one part the sums go to the workspace, [part][row][output].
template <int OB>
constexpr int kAhead = OB == 1 ? 4 : 2;
template <int X, int GRAIN, int OB, int WO, int WK, bool WIDE>
__global__ __launch_bounds__(kWave* WO* WK) void held_kernel(ReadoutArgs a) {
  constexpr int kPlanes = Kind<X>::kPlanes;
  constexpr int kDeep = kAhead<OB>;
  extern __shared__ v4u held[];
  __shared__ v4f join[WO * WK][OB][kWave];
  const int l = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wo = wave / WK, wk = wave % WK;
  const int begin = blockIdx.y * a.part_chunks;
  const int end = begin + a.part_chunks < a.chunks ? begin + a.part_chunks : a.chunks;
  const int first_out = (blockIdx.x * WO + wo) * OB * kTile + l % 16;
  const int block_out = blockIdx.x * WO * OB * kTile;
  static_assert(WO * OB * kTile <= kMaxTogether, "32-bit distances of codes and scales");
  constexpr int size = WIDE ? 4 : 2;
  const uint8_t* codes = a.codes + block_out * a.code_stride;
  const char* scales = (const char*)a.scales + block_out * a.scale_stride * size;
  uint32_t code_off[OB], scale_off[OB];
#pragma unroll
  for (int b = 0; b < OB; ++b) {
    const uint32_t o = (first_out + b * kTile < a.K ? first_out + b * kTile : a.K - 1) - block_out;
    code_off[b] = o * (uint32_t)a.code_stride;
    scale_off[b] = o * (uint32_t)a.scale_stride * size;
  }
  Codes<GRAIN, WIDE> code[kDeep][OB];
  // this wave's u-th chunk from `first` on
  const auto chunk_at = [&](int first, int u) { return first + u / 2 * (2 * WK) + u % 2; };
  const auto load = [&](int first) {
#pragma unroll
    for (int u = 0; u < kDeep; ++u)
#pragma unroll
      for (int b = 0; b < OB; ++b)
        code[u][b].load(a, codes, code_off[b], scales, scale_off[b], chunk_at(first, u));
  };
  load(begin + 2 * wk);
  const int count = (end - begin) * (kBits<X> ? kWords : kPieces);
  constexpr int kAtOnce = kPlanes == 1 ? 4 : 2;
  if constexpr (kBits<X>) {
    for (int j = threadIdx.x; j < a.N * count; j += kWave * WO * WK) {
      const int n = j / count, i = j - n * count;
      const uint32_t bits = load_bits(a, (const char*)a.x, n * (uint32_t)a.x_stride * 4, begin * kWords + i);
      held[i * a.N + n] = bit_operand(a, bits, begin * kWords + i);
    }
  } else {
    for (int first = threadIdx.x; first < a.N * count; first += kAtOnce * kWave * WO * WK) {
      Piece<X> piece[kAtOnce];
#pragma unroll
      for (int e = 0; e < kAtOnce; ++e) {
        const int j = first + e * kWave * WO * WK;
        const int n = j < a.N * count ? j / count : 0;
        piece[e].load(a, (const char*)a.x, n * (uint32_t)a.x_stride * kSize<X>,
                      begin * kChunk + 8 * (j < a.N * count ? j - n * count : 0));
      }
#pragma unroll
      for (int e = 0; e < kAtOnce; ++e) {
        const int j = first + e * kWave * WO * WK;
        if (j >= a.N * count) break;
        const int n = j / count, i = j - n * count;
        v4u plane[kPlanes];
        piece[e].operands(a, begin * kChunk + 8 * i, plane);
        const int place = i / kPieces * kPieces + place_of<GRAIN>(i % kPieces);
#pragma unroll
        for (int p = 0; p < kPlanes; ++p) held[(p * count + place) * a.N + n] = plane[p];
      }
    }
  }
  __syncthreads();
  const v4u* from = held + l / 16 * a.N + (l % 16 < a.N ? l % 16 : 0);
  v4f total[OB];
#pragma unroll
  for (int b = 0; b < OB; ++b) total[b] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  for (int first = begin + 2 * wk; first < end; first += kDeep * WK) {
    Codes<GRAIN, WIDE> now[kDeep][OB];
#pragma unroll
    for (int u = 0; u < kDeep; ++u)
#pragma unroll
      for (int b = 0; b < OB; ++b) now[u][b] = code[u][b];
    if (first + kDeep * WK < end) load(first + kDeep * WK);
#pragma unroll
    for (int u = 0; u < kDeep; ++u) {
      const int chunk = chunk_at(first, u);
      if (chunk >= end) break;
      if constexpr (kBits<X>) {
        const v4u x = from[(chunk - begin) * kWords * a.N];
#pragma unroll
        for (int b = 0; b < OB; ++b) {
          float scale[4];
          now[u][b].scaled(a, chunk, scale);
#pragma unroll
          for (int g = 0; g < kChunk / GRAIN; ++g) {
            const v4f sum = bit_product(GRAIN == kChunk ? x : only(x, g), now[u][b].w);
#pragma unroll
            for (int r = 0; r < 4; ++r) total[b][r] = __builtin_fmaf(scale[g], sum[r], total[b][r]);
          }
        }
        continue;
      }
      add_chunk<X, GRAIN, OB>(from + (chunk - begin) * kPieces * a.N, count * a.N, 4 * a.N, total,
                              [&](int b, v4u& w, float(&scale)[4]) {
                                w = now[u][b].w;
                                now[u][b].scaled(a, chunk, scale);
                              });
    }
  }
#pragma unroll
  for (int b = 0; b < OB; ++b) join[wave][b][l] = total[b];
  __syncthreads();
  if (wk > 0) return;
#pragma unroll
  for (int b = 0; b < OB; ++b) {
    v4f v = total[b];
    for (int w = 1; w < WK; ++w) v += join[wave + w][b][l];
    const int o = first_out + b * kTile;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const int n = l / 16 * 4 + r;
      if (o >= a.K || n >= a.N) continue;
      if (gridDim.y > 1)
        a.parts[((int64_t)blockIdx.y * a.N + n) * a.K + o] = v[r];
      else
        store_out(a, n, o, v[r]);
    }
  }
}

// A chunk's row operands take 64 bytes of LDS a row for each operand of 16 rows; a part has as many
// chunks as kHeldLimit takes, which leaves room for two blocks on a CU; bits, whose products leave
// the codes' loads to wait for, half of that (16 rows x 20000 clauses x 10000 outputs: 64 KB 48 us, 32 KB
// 38, 150 KB 64).
constexpr int64_t kHeldLimit = 64 * 1024;
int part_chunks_of(int operands, int N, int chunks) {
  const int64_t most = kHeldLimit / (operands == 1 ? 2 : 1) / ((int64_t)operands * N * 64);
  if (most >= chunks) return chunks;
  const int64_t parts = (chunks + most - 1) / most;
  return (int)((chunks + parts - 1) / parts);
}
int parts_of(int operands, int N, int chunks) {
  const int each = part_chunks_of(operands, N, chunks);
  return (chunks + each - 1) / each;
}

template <int X, int GRAIN, int OB, int WO, int WK>
hipError_t launch_held(ReadoutArgs a, hipStream_t s) {
  const int parts = parts_of(kOperands<X>, a.N, a.chunks);
  a.part_chunks = part_chunks_of(kOperands<X>, a.N, a.chunks);
  const size_t lds = (size_t)a.N * kOperands<X> * a.part_chunks * 64;
  const dim3 grid((unsigned)((a.K + kTile * OB * WO - 1) / (kTile * OB * WO)), (unsigned)parts);
  if (a.scale_dtype == YTM_DTYPE_F32)
    held_kernel<X, GRAIN, OB, WO, WK, true><<<grid, kWave * WO * WK, lds, s>>>(a);
  else
    held_kernel<X, GRAIN, OB, WO, WK, false><<<grid, kWave * WO * WK, lds, s>>>(a);
  const hipError_t e = hipGetLastError();
  return e != hipSuccess || parts == 1 ? e : launch_parts(a, parts, s);
}

constexpr int kFewRows = 16;

// Fewer than eight clauses, which no load of a piece fits: a thread an output.
template <int X>
__global__ __launch_bounds__(256) void short_kernel(ReadoutArgs a) {
  const int64_t each = (int64_t)a.N * a.K;
  for (int64_t i = blockIdx.x * (int64_t)blockDim.x + threadIdx.x; i < each; i += (int64_t)gridDim.x * blockDim.x) {
    const int n = (int)(i / a.K), o = (int)(i % a.K);
    float sum = 0.0f;
    for (int c = 0; c < a.C; ++c) {
      const int64_t at = n * a.x_stride + c;
      const float x = X == YTM_DTYPE_BITS   ? (float)(((const uint32_t*)a.x)[n * a.x_stride] >> c & 1u)
                      : X == YTM_DTYPE_F16  ? to_float(((const f16*)a.x)[at])
                      : X == YTM_DTYPE_BF16 ? to_float(((const bf16*)a.x)[at])
                                            : ((const float*)a.x)[at];
      const uint32_t code = a.codes[o * a.code_stride + c / 2] >> (c % 2 * 4) & 15u;
      const uint32_t m = code & 7u;  // 0 and 0.5, then two to each power of two
      const float v = m < 2 ? 0.5f * m : __uint_as_float((126u + (m >> 1)) << 23 | (m & 1u) << 22);
      sum = __builtin_fmaf(x, code & 8u ? -v : v, sum);
    }
    if (a.C > 0) {
      const int64_t at = o * a.scale_stride;
      sum *= a.scale_dtype == YTM_DTYPE_F32   ? ((const float*)a.scales)[at]
             : a.scale_dtype == YTM_DTYPE_F16 ? to_float(((const f16*)a.scales)[at])
                                              : to_float(((const bf16*)a.scales)[at]);
    }
    store_out(a, n, o, sum);
  }
}

template <int X, int GRAIN>
hipError_t launch_rows(const ReadoutArgs& a, hipStream_t s) {
  if (a.N > kFewRows) return launch_tiles<X, GRAIN>(a, s);
  // Parts of 16-bit operands in blocks of 256 outputs, so that fewer blocks lay out the same rows (8 rows x
  // 20000 clauses x 5000 outputs, float32: 32 us, in blocks of 16 outputs 73), unless that makes few blocks
  // (2 rows x 10027 clauses x 1792 outputs, float32: 14 blocks 40 us, blocks of 16 outputs 15).  Bits are
  // laid out quickly (12 rows x 14000 clauses x 2000 outputs: 40 us, 15).
  if constexpr (!kBits<X>) {
    const int parts = parts_of(kOperands<X>, a.N, a.chunks);
    if (parts > 1 && (int64_t)(a.K + 255) / 256 * parts >= 40) return launch_held<X, GRAIN, 2, 8, 1>(a, s);
  }
  // A block's waves share its 16 outputs' clauses: 16 where there are few outputs, or 4.  With float32 and
  // groups of 32, 16 waves leave too few registers and 48 to 52 are spilled.
  return a.K <= 4096 ? launch_held<X, GRAIN, 1, 1, 16>(a, s) : launch_held<X, GRAIN, 1, 1, 4>(a, s);
}

template <int X>
hipError_t launch_readout(const ReadoutArgs& a, int64_t group, hipStream_t s) {
  if (a.C < 8) {
    const int64_t blocks = ((int64_t)a.N * a.K + 255) / 256;
    short_kernel<X><<<(unsigned)(blocks < 4096 ? blocks : 4096), 256, 0, s>>>(a);
    return hipGetLastError();
  }
  return group % kChunk == 0 ? launch_rows<X, kChunk>(a, s) : launch_rows<X, kStep>(a, s);
}

}  // namespace

}  // namespace ytm

using ytm::fail;

extern "C" {

int ytm_readout_workspace(int x_dtype, int64_t N, int64_t C, int64_t K, int64_t* bytes) {
  if (!bytes || (x_dtype != YTM_DTYPE_BITS && !ytm::decode_float(x_dtype)) || N < 0 || C < 0 || K < 0 ||
      N > ytm::kDecodeRows || C > ytm::kMaxClauses || K > ytm::kMaxScores)
    return fail(YTM_EINVAL, "bad readout_workspace arguments");
  *bytes = 0;
  if (N == 0 || K == 0 || C < 8) return YTM_OK;
  const int operands = ytm::operands_of(x_dtype), chunks = (int)((C + 127) / 128);
  if (N > ytm::kFewRows) {
    *bytes = ytm::frag_bytes(operands, (int)N, chunks);
    const int whole = ytm::tile_parts_of(operands, ytm::kChunk, (int)N, chunks, (int)K);
    const int four = ytm::tile_parts_of(operands, ytm::kStep, (int)N, chunks, (int)K);
    if (whole > 1 || four > 1) *bytes += (whole > four ? whole : four) * N * K * 4;
  } else {
    const int parts = ytm::parts_of(operands, (int)N, chunks);
    if (parts > 1) *bytes = parts * N * K * 4;
  }
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
  if (N < 0 || C < 0 || K < 0 || N > ytm::kDecodeRows || C > ytm::kMaxClauses || K > ytm::kMaxScores)
    return fail(YTM_EINVAL, "readout takes at most 65535 rows, 2097120 clauses and 8388608 outputs");
  if (group < 32 || group % 32) return fail(YTM_EINVAL, "readout groups are multiples of 32 clauses");
  if (N == 0 || K == 0) return YTM_OK;
  if (!out || (C > 0 && (!x || !codes || !scales))) return fail(YTM_EINVAL, "bad readout arguments");
  if (C > 0 && ((uintptr_t)codes | (K > 1 ? (uint64_t)code_stride : 0u)) % 16)
    return fail(YTM_EINVAL, "readout codes start at multiples of 16 bytes, every output's");
  const int64_t width = x_dtype == YTM_DTYPE_BITS ? (C + 31) / 32 : C;
  if ((K > 1 && ((code_stride != 0 && code_stride < (C + 31) / 32 * 16) ||
                 (scale_stride != 0 && scale_stride < (C + group - 1) / group))) ||
      (N > 1 && ((x_stride != 0 && x_stride < width) || out_stride < K)))
    return fail(YTM_EINVAL, "readout: rows overlap");
  const int64_t x_size = x_dtype == YTM_DTYPE_BITS || x_dtype == YTM_DTYPE_F32 ? 4 : 2;
  const int64_t scale_size = scale_dtype == YTM_DTYPE_F32 ? 4 : 2;
  if (N == 1) x_stride = 0;
  if (K == 1) code_stride = scale_stride = 0;
  if (x_stride > ytm::kMaxApart / x_size || code_stride > ytm::kMaxApart || scale_stride > ytm::kMaxApart / scale_size)
    return fail(YTM_EINVAL, "readout rows, codes and scales are at most 8 MiB apart");
  int64_t need = 0;
  if (int rc = ytm_readout_workspace(x_dtype, N, C, K, &need)) return rc;
  if (need > 0 && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
    return fail(YTM_EINVAL, "readout: the workspace is too small or not at a multiple of 16 bytes");
  const ytm::Rows written[] = {ytm::rows_of(out, N, K, out_stride, out_dtype == YTM_DTYPE_F32 ? 4 : 2),
                               ytm::block_of(workspace, need)};
  const ytm::Rows read[] = {ytm::rows_of(x, N, width, x_stride, x_size),
                            ytm::rows_of(codes, K, (C + 31) / 32 * 16, code_stride, 1),
                            ytm::rows_of(scales, K, (C + group - 1) / group, scale_stride, scale_size)};
  bool overlap = ytm::share_bytes(written[0], written[1]);
  for (const ytm::Rows& w : written)
    for (const ytm::Rows& r : read) overlap |= ytm::share_bytes(w, r);
  if (overlap) return fail(YTM_EINVAL, "readout: what is written overlaps what is read");
  const int64_t steps = (C + 31) / 32, units = group / 32;
  // (step + 1) * floor((2^32 - 1) / units) >> 32 is step / units while (step + 1) * units < 2^32
  const uint32_t inverse = units >= steps ? 0u : (uint32_t)(0xFFFFFFFFu / units);
  const ytm::ReadoutArgs a{x, x_stride, (int)N, (int)C, codes, code_stride, scales, scale_dtype, scale_stride, inverse,
                           (int)K, out, out_dtype, out_stride, (int)((C + 127) / 128), 0, 0, 0, (float*)workspace,
                           (ytm::v4u*)workspace};
  hipStream_t s = (hipStream_t)stream;
  hipError_t e;
  switch (x_dtype) {
    case YTM_DTYPE_BITS: e = ytm::launch_readout<YTM_DTYPE_BITS>(a, group, s); break;
    case YTM_DTYPE_F16: e = ytm::launch_readout<YTM_DTYPE_F16>(a, group, s); break;
    case YTM_DTYPE_BF16: e = ytm::launch_readout<YTM_DTYPE_BF16>(a, group, s); break;
    default: e = ytm::launch_readout<YTM_DTYPE_F32>(a, group, s); break;
  }
  if (e != hipSuccess) return fail(YTM_EHIP, std::string("readout failed: ") + hipGetErrorString(e));
  return YTM_OK;
}

}  // extern "C"
