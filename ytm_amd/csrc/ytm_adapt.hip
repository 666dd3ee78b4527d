// ytm_adapt.hip -- low-rank adapters of many requests beside the readout, and their gradients: the
// entry points ytm_adapt and ytm_adapt_gradient of include/ytm.h and their gfx950 kernels.
//
//   hidden[n] = down[a] x[n], out[n] = scores[n] + scale * up[a] hidden[n], a = which[n]
//   d_up[a] = scale * sum over n of a of grad[n] hidden[n]^T, back[n] = scale * up[a]^T grad[n],
//   d_down[a] = sum over n of a of back[n] x[n]^T
//
// Rows are taken in the order of their adapters (ties in the order of rows), sixteen of that order,
// a window, at a time: a window's rows of one adapter are a segment, whose weights are read once.
// Sums run on the matrix cores in f32 with exact operands: of one 16-bit type as they are, a f32 beside
// values that bfloat16 holds as the sum of three of these, all else as f32, one value a lane.  Sums that
// several blocks share are joined in a fixed order by a kernel that comes after.
//
// What bounds them is latency: a block's chain of waits (the order, the rows that it names, their values, the
// parts' sums) takes 3 us at least, and memory is read and written at 1.6 to 3 TB/s.  Hence few launches, loads
// asked for before what they wait beside, and as many blocks a CU as the registers hold.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "ytm_decode.h"
#include "ytm_internal.h"

namespace ytm {

namespace {

typedef float v4f __attribute__((ext_vector_type(4)));

constexpr int kWave = 64;
constexpr int kTile = 16;  // rows, outputs, ranks or clauses of a product
constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kInline = kThreads;  // rows that every block sorts by itself
constexpr int kMaxRank = 256;
constexpr int64_t kMaxAdapters = 65535;

// A gradient's sums over many rows: windows of `rows` rows of the order, whose adapters `slots` blocks share;
// what a window has of an adapter that others have rows of goes to `partial`.
struct RowWindows {
  int count, rows, slots;
  float* partial;
};

struct AdaptArgs {
  const void* scores;  // or their gradient
  int dtype;
  int64_t stride;
  int N, K;
  const void* x;
  int64_t x_stride;
  int C;
  const void* down;
  int64_t down_adapter, down_rank;
  const void* up;
  int64_t up_adapter, up_output;
  int M, r;
  const int32_t* which;
  float scale;
  float* hidden;  // NULL where nobody asks
  int64_t hidden_stride;
  void* out;  // or the gradient of up
  int out_dtype;
  int64_t out_stride;
  void* d_down;
  int64_t d_down_adapter, d_down_rank;
  int64_t d_up_adapter, d_up_output;
  int windows, slots;     // slots: blocks that share a window's segments
  int tiles;              // blocks that share a window's outputs
  int tile_blocks;        // blocks of 64 outputs of each
  bool tiles_first;       // whether these have numbers in a row
  int parts, part_steps;  // of a sum over clauses or outputs
  int padded;             // r, to whole tiles
  float* part;            // [parts][N in order][padded]
  float* back;            // [back_parts][N in order][padded]
  int back_parts;
  uint32_t* order;  // [N], of more than kInline rows; then [begins] where adapters begin
  int begins;       // M + 1 where they are asked for
  int w_dtype;
  int d_dtype;  // of the gradients: w_dtype, or float32 where that one's range is too small for them
  int odd;  // 16-bit rows that do not all begin at multiples of 4
  int first;  // adapter of a launch of gradients
  RowWindows up_windows, down_windows;
};

// ----------------------------------------------------------------------------------- elements
template <int X>
struct Element;
template <>
struct Element<YTM_DTYPE_F32> {
  typedef float type;
};
template <>
struct Element<YTM_DTYPE_F16> {
  typedef f16 type;
};
template <>
struct Element<YTM_DTYPE_BF16> {
  typedef bf16 type;
};

// E values in a row at p, of which `left` are there, as float; the others are 0.
// WHOLE: all are, which leaves no branch, so that other loads can follow before these are there.
template <int E, bool WHOLE = false, typename T>
__device__ __forceinline__ void load_floats(const T* p, int left, float (&v)[E]) {
  T raw[E];
  if (WHOLE || left >= E) {
    __builtin_memcpy(raw, p, sizeof raw);
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = to_float(raw[e]);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = e < left ? to_float(p[e]) : 0.0f;
  }
}
template <int E, typename T>
__device__ __forceinline__ void store_floats(T* p, int left, const float (&v)[E]) {
  T raw[E];
#pragma unroll
  for (int e = 0; e < E; ++e) raw[e] = from_float<T>(v[e]);
  if (left >= E) {
    __builtin_memcpy(p, raw, sizeof raw);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e)
      if (e < left) p[e] = raw[e];
  }
}
template <int E>
__device__ __forceinline__ void store_floats(void* p, int64_t at, int dtype, int left, const float (&v)[E]) {
  switch (dtype) {
    case YTM_DTYPE_F16: store_floats<E>((f16*)p + at, left, v); break;
    case YTM_DTYPE_BF16: store_floats<E>((bf16*)p + at, left, v); break;
    default: store_floats<E>((float*)p + at, left, v); break;
  }
}

// Clauses c .. c + E - 1 of row n (E divides 32, c a multiple of E), 0 past the last clause.
template <int X, int E, bool WHOLE = false>
__device__ __forceinline__ void load_clauses(const AdaptArgs& a, int64_t n, int c, float (&v)[E]) {
  const int left = a.C - c;
  if constexpr (X == YTM_DTYPE_BITS) {
    const uint32_t word = WHOLE || left > 0 ? ((const uint32_t*)a.x)[n * a.x_stride + c / 32] >> c % 32 : 0u;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = WHOLE || e < left ? (float)(word >> e & 1u) : 0.0f;
  } else {
    load_floats<E, WHOLE>((const typename Element<X>::type*)a.x + n * a.x_stride + c, left, v);
  }
}

// What is loaded before stays before the products after it.
__device__ __forceinline__ void loads_first() { __builtin_amdgcn_sched_barrier(0); }

__device__ __forceinline__ v4f product(float a, float b, v4f d) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, d, 0, 0, 0);
}

// ---------------------------------------------------------------------------------- the order
// A row's place among the rows is the number of smaller codes, a code being the row's adapter (M where it
// has none) above its number; both have 16 bits.
__device__ __forceinline__ uint32_t code_of(const AdaptArgs& a, int n) {
  const uint32_t w = (uint32_t)a.which[n];
  return (w < (uint32_t)a.M ? w : (uint32_t)a.M) << 16 | (uint32_t)n;
}
__device__ __forceinline__ int key_of(uint32_t code) { return (int)(code >> 16); }
__device__ __forceinline__ int row_of(uint32_t code) { return (int)(code & 0xFFFFu); }

// How many of four codes are smaller.
__device__ __forceinline__ int smaller(uint4 v, uint32_t mine) {
  return (v.x < mine) + (v.y < mine) + (v.z < mine) + (v.w < mine);
}

// More than kInline rows: a block places 64 of them, its waves share the codes that they are compared with.  After
// the rows come the adapters, as codes before all of theirs, whose places are where their rows begin.
constexpr int kOrderThreads = 1024;
__global__ __launch_bounds__(kOrderThreads) void order_kernel(AdaptArgs a) {
  __shared__ uint4 codes[kOrderThreads];
  __shared__ int places[kOrderThreads / kWave][kWave];
  const int l = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int n = blockIdx.x * kWave + l;
  const uint32_t mine = n < a.N ? code_of(a, n) : (uint32_t)(n - a.N) << 16;
  int place = 0;
  for (int first = 0; first < a.N; first += 4 * kOrderThreads) {
    uint32_t v[4];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int m = first + 4 * threadIdx.x + q;
      v[q] = m < a.N ? code_of(a, m) : UINT32_MAX;
    }
    __syncthreads();
    codes[threadIdx.x] = uint4{v[0], v[1], v[2], v[3]};
    __syncthreads();
    const int left = (a.N - first + 3) / 4, last = left < kOrderThreads ? left : kOrderThreads;
#pragma unroll 4
    for (int m = wave; m < last; m += kOrderThreads / kWave) place += smaller(codes[m], mine);
  }
  places[wave][l] = place;
  __syncthreads();
  if (wave > 0 || n >= a.N + a.begins) return;
  place = 0;
#pragma unroll
  for (int w = 0; w < kOrderThreads / kWave; ++w) place += places[w][l];
  if (n < a.N)
    a.order[place] = mine;
  else
    a.order[n] = (uint32_t)place;
}

// What a block knows of the order: with at most kInline rows all of it, made by itself.
struct Order {
  uint32_t code[kInline];
  __attribute__((aligned(16))) uint32_t all[kInline];

  __device__ __forceinline__ void make(const AdaptArgs& a) {
    const int n = threadIdx.x;
    const uint32_t mine = n < a.N ? code_of(a, n) : UINT32_MAX;
    if (n < kInline) {
      all[n] = mine;
      code[n] = UINT32_MAX;
    }
    __syncthreads();
    int place = 0;
#pragma unroll 4
    for (int m = 0; m < (a.N + 3) / 4; ++m) place += smaller(((const uint4*)all)[m], mine);
    if (n < a.N) code[place] = mine;
    __syncthreads();
  }
  // the codes of a window, at code[0 ..]; past the last row none
  __device__ __forceinline__ const uint32_t* window(const AdaptArgs& a, int w) {
    if (a.N <= kInline) {
      make(a);
      return code + w * kTile;
    }
    if (threadIdx.x < kTile) {
      const int i = w * kTile + threadIdx.x;
      code[threadIdx.x] = i < a.N ? a.order[i] : UINT32_MAX;
    }
    __syncthreads();
    return code;
  }
  // where adapter `key` begins: the number of codes of smaller keys; after make() where the block makes it
  __device__ __forceinline__ int begin(const AdaptArgs& a, int key) const {
    if (a.N > kInline) return __builtin_amdgcn_readfirstlane((int)a.order[a.N + key]);
    const uint32_t least = (uint32_t)key << 16;
    int before = 0;
    for (int first = 0; first < a.N; first += kWave) {
      const int i = first + (int)threadIdx.x % kWave;
      before += __popcll(__ballot(i < a.N && code[i % kInline] < least));
    }
    return before;
  }
};

// The segments of a window that block `slot` of `slots` takes: body(key, first place, end).  A place begins one
// where its key is not that of the place before.  Blocks of the same slot have numbers in a row: those of later
// slots often find nothing, and by turns they would leave every other XCD without work (adapt of 512 rows of
// one adapter, 20000 clauses, 10000 outputs, rank 32: 39.9 us, 33.1 in a row).
template <typename Body>
__device__ __forceinline__ void segments(const uint32_t* code, int slot, int slots, Body body) {
  const int i = threadIdx.x % kTile;
  const uint32_t mine = code[i], before = code[i ? i - 1 : 0];
  const uint64_t there = __ballot(mine != UINT32_MAX) & 0xFFFFu;
  const int rows = __popcll(there);
  uint32_t begins = (uint32_t)(__ballot(mine != UINT32_MAX && (i == 0 || key_of(mine) != key_of(before))) & 0xFFFFu);
  for (int s = 0; begins; ++s) {
    const int first = __ffs(begins) - 1;
    begins &= begins - 1;
    if (s % slots == slot)
      body(__builtin_amdgcn_readlane((int)key_of(mine), first), first, begins ? __ffs(begins) - 1 : rows);
  }
}

// Of each wave's sums of RT tiles of ranks and 16 rows the block's, written to the part's place: rank
// RT c + t of tile t's column c, so that a lane's are in a row.
template <int RT>
__device__ __forceinline__ void write_part(const AdaptArgs& a, int p, int window, int first, int end, int ranks,
                                           const v4f (&sum)[RT], v4f (*join)[RT][kWave]) {
  const int l = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  __syncthreads();
#pragma unroll
  for (int t = 0; t < RT; ++t) join[wave][t][l] = sum[t];
  __syncthreads();
  // wave w takes row 4 (l / 16) + w of each tile
  const int i = l / kTile * 4 + wave, j = ranks + l % kTile * RT;
  if (i < first || i >= end) return;
  float v[RT];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
    v[t] = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) v[t] += ((const float*)&join[w][t][l])[wave];
    if (j + t >= a.r) v[t] = 0.0f;  // not another rank's infinity
  }
  __builtin_memcpy(a.part + ((int64_t)p * a.N + window * kTile + i) * a.padded + j, v, sizeof v);
}

// ------------------------------------------------------------------------------------ forward
// Clauses and weights of one 16-bit type (bits have any) are multiplied as they are, 32 clauses a product,
// each exact in f32; all else as f32, 4 clauses a product.
template <int X, int W>
constexpr bool kHalves = W != YTM_DTYPE_F32 && (X == W || X == YTM_DTYPE_BITS);
template <int X, int W>
constexpr int kChunk = kHalves<X, W> ? 128 : 64;  // clauses that a wave's lanes load at once, in four steps

typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));

template <int W>
__device__ __forceinline__ v4f half_product(v4u x, v4u w, v4f d) {
  if (W == YTM_DTYPE_F16)
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8h, x), __builtin_bit_cast(v8h, w), d, 0, 0, 0);
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8bf, x), __builtin_bit_cast(v8bf, w), d, 0, 0, 0);
}

// Eight 16-bit values at p, of which `left` are there.  ODD: p is at any multiple of 2; lanes that read rows of
// their own take such loads piece by piece (2048 rows of 10007 bfloat16, one pass: 37 us, at multiples of 4 22), so
// the aligned words around them are read, all of which hold some of the eight, and shifted.
template <typename T, bool WHOLE, bool ODD = false>
__device__ __forceinline__ v4u load_halves(const T* p, int left) {
  v4u r;
  if (WHOLE && ODD) {
    const uintptr_t u = (uintptr_t)p;
    const uint32_t shift = (uint32_t)(u & 2) * 8;
    typedef uint32_t v4a __attribute__((ext_vector_type(4), aligned(4)));
    const v4u v = *(const v4a*)(u & ~(uintptr_t)3);
    const uint32_t last = *(const uint32_t*)(u + 14 & ~(uintptr_t)3);
#pragma unroll
    for (int q = 0; q < 4; ++q) r[q] = __builtin_amdgcn_alignbit(q < 3 ? v[(q + 1) % 4] : last, v[q], shift);
    return r;
  }
  if (WHOLE || left >= 8) {
    __builtin_memcpy(&r, p, sizeof r);
    return r;
  }
  uint16_t v[8];
#pragma unroll
  for (int e = 0; e < 8; ++e) {
    v[e] = 0;
    if (e < left) __builtin_memcpy(&v[e], p + e, 2);
  }
#pragma unroll
  for (int q = 0; q < 4; ++q) r[q] = (uint32_t)v[2 * q + 1] << 16 | v[2 * q];
  return r;
}

// Sums over a part of the clauses of 16 rows with 16 RT ranks of a segment's adapter.  Lane l has row l % 16, the
// ranks RT (l % 16) + t and 16 bytes of each 64 of a chunk, so that a load has whole lines of 16 rows; a block's
// waves take chunks in turn, each with the next one's operands on their way.
template <int X, int W, int RT>
__global__ __launch_bounds__(kThreads) void down_kernel(AdaptArgs a) {
  typedef typename Element<W>::type T;
  constexpr int kOwn = kHalves<X, W> ? 8 : 4, kStep = 4 * kOwn;  // clauses of a lane and of the wave in a step
  __shared__ Order order;
  __shared__ v4f join[kWaves][RT][kWave];
  // blocks of the same clauses are on the same XCD where there are 8 or 16 parts, and its L2 has their weights
  // (512 rows, 8 adapters of 20000 x 32 bfloat16: 30 MB read, 58 the other way)
  const int slot = blockIdx.y / a.windows, window = blockIdx.y % a.windows, p = blockIdx.x, ranks = blockIdx.z * RT * kTile;
  const uint32_t* code = order.window(a, window);
  const int l = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t row = row_of(code[l % kTile] == UINT32_MAX ? code[0] : code[l % kTile]);
  segments(code, slot, a.slots, [&](int key, int first, int end) {
    if (key == a.M) return;
    v4f sum[RT];
    const T* down[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      sum[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
      const int j = ranks + l % kTile * RT + t;
      down[t] = (const T*)a.down + key * a.down_adapter + (int64_t)(j < a.r ? j : a.r - 1) * a.down_rank;
    }
    // a chunk's operands, as they are in memory
    struct Operands {
      v4u x[kHalves<X, W> ? 4 : 1], w[kHalves<X, W> ? RT : 1][4];
      uint32_t words[4];
      float fx[kHalves<X, W> ? 1 : 4][4], fw[kHalves<X, W> ? 1 : RT][4][4];
    };
    const auto load = [&](int at, auto all, Operands& o) {
      constexpr bool kWhole = decltype(all)::value;
      const int c = at * kChunk<X, W> + l / kTile * kOwn;
      if constexpr (X == YTM_DTYPE_BITS) {
        constexpr int kWords = kChunk<X, W> / 32;
        const uint32_t* from = (const uint32_t*)a.x + row * a.x_stride + at * kWords;
        if (kWhole) {
          __builtin_memcpy(o.words, from, kWords * 4);
        } else {
#pragma unroll
          for (int i = 0; i < kWords; ++i) {
            const int left = a.C - (at * kWords + i) * 32;
            o.words[i] = left > 0 ? from[i] & (left < 32 ? (1u << left) - 1u : ~0u) : 0u;
          }
        }
      }
      if constexpr (kHalves<X, W>) {
        if constexpr (X != YTM_DTYPE_BITS) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
            o.x[i] = load_halves<T, kWhole>((const T*)a.x + row * a.x_stride + c + kStep * i, a.C - c - kStep * i);
        }
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
          for (int i = 0; i < 4; ++i) o.w[t][i] = load_halves<T, kWhole>(down[t] + c + kStep * i, a.C - c - kStep * i);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if constexpr (X != YTM_DTYPE_BITS) load_clauses<X, 4, kWhole>(a, row, c + kStep * i, o.fx[i]);
#pragma unroll
          for (int t = 0; t < RT; ++t)
            load_floats<4, kWhole>(down[t] + c + kStep * i, a.C - c - kStep * i, o.fw[t][i]);
        }
      }
    };
    const auto multiply = [&](const Operands& o) {
      if constexpr (kHalves<X, W>) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          v4u x = o.x[i];
          if constexpr (X == YTM_DTYPE_BITS) {
            constexpr uint32_t one = W == YTM_DTYPE_F16 ? 0x3C00u : 0x3F80u;
#pragma unroll
            for (int q = 0; q < 4; ++q) {
              const uint32_t two = o.words[i] >> (l / kTile * 8 + 2 * q);
              x[q] = ((two & 1u) | (two & 2u) << 15) * one;
            }
          }
#pragma unroll
          for (int t = 0; t < RT; ++t) sum[t] = half_product<W>(x, o.w[t][i], sum[t]);
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int t = 0; t < RT; ++t) {
              float x;
              if constexpr (X == YTM_DTYPE_BITS)
                x = (float)(o.words[i / 2] >> (i % 2 * 16 + l / kTile * 4 + e) & 1u);
              else
                x = o.fx[i][e];
              sum[t] = product(x, o.fw[t][i][e], sum[t]);
            }
      }
    };
    const int whole = a.C / kChunk<X, W>, last = (p + 1) * a.part_steps < whole ? (p + 1) * a.part_steps : whole;
    int at = p * a.part_steps + wave;
    if (at < last) {
      Operands now;
      load(at, std::true_type{}, now);
      for (; at + kWaves < last; at += kWaves) {
        Operands next;
        load(at + kWaves, std::true_type{}, next);
        loads_first();
        multiply(now);
        now = next;
      }
      multiply(now);
    }
    if (whole * kChunk<X, W> < a.C && whole / a.part_steps == p && whole % kWaves == wave) {
      Operands end_of_row;
      load(whole, std::false_type{}, end_of_row);
      multiply(end_of_row);
    }
    write_part<RT>(a, p, window, first, end, ranks, sum, join);
  });
}

// 64 outputs a wave at a time of 16 rows; f32 operands, since hidden is f32 and there are few products.
// Lane l has output l % 16 of a tile and row l % 16, and four ranks of every 16; it gets sums of four outputs
// in a row of row l % 16.  RANKS: those of a.padded, or the most.
template <int W, int S, int RANKS>
__global__ __launch_bounds__(kThreads) void up_kernel(AdaptArgs a) {
  typedef typename Element<W>::type T;
  typedef typename Element<S>::type In;
  constexpr int kTiles = 4, kOutputs = kTiles * kTile;
  constexpr int kSteps = RANKS > 32 ? 1 : RANKS / kTile;  // of 16 ranks, at once
  constexpr int kGroups = RANKS > 32 ? 1 : kThreads / (kTile * RANKS / 4);
  __shared__ Order order;
  __shared__ __attribute__((aligned(16))) float hidden[kTile][RANKS + 4];
  __shared__ __attribute__((aligned(16))) float group_sums[kGroups > 1 ? kGroups : 1][kGroups > 1 ? kTile : 1][RANKS + 4];
  // Few rows: blocks of the same outputs on the same XCD, which then reads their weights once (48 rows of
  // some 30 adapters, 10000 outputs, rank 16: 12.3 us, 16.0 the other way); many rows: those of the same rows
  // one after the other (4096 rows of 8 adapters, rank 32: 106 us, 182; 512 rows 22.2, where the other way
  // takes 19.6).
  const int apart = a.tiles_first ? (a.tiles + 7) / 8 * 8 : a.windows * a.slots;
  const int tile = a.tiles_first ? blockIdx.x % apart : blockIdx.x / apart;
  const int rows = a.tiles_first ? blockIdx.x / apart : blockIdx.x % apart;
  if (tile >= a.tiles) return;
  const int slot = rows / a.windows, window = rows % a.windows;
  const uint32_t* code = order.window(a, window);
  const int l = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int at = l % kTile, four = l / kTile * 4;
  const int padded = RANKS <= 32 ? RANKS : a.padded;
  segments(code, slot, a.slots, [&](int key, int first, int end) {
    const bool mine = at >= first && at < end, some = key < a.M;
    const int64_t row = row_of(code[mine ? at : first]);
    const T* up = (const T*)a.up + key * a.up_adapter;
    const In* scores = (const In*)a.scores + row * a.stride;
    // whole blocks of 64 outputs and 16 ranks: the scores and the first ranks' weights, as they are in memory
    struct Operands {
      In v[kTiles][4];
      T w[kSteps][kTiles][4];
    };
    const uint32_t lane = (uint32_t)(at * a.up_output + four) * sizeof(T);  // rows are at most 8 MiB apart
    const auto weights = [&](int o0, int j, T (&w)[kTiles][4]) {
#pragma unroll
      for (int t = 0; t < kTiles; ++t)
        __builtin_memcpy(w[t], (const char*)(up + (o0 + t * kTile) * a.up_output + j) + lane, sizeof w[t]);
    };
    const auto load = [&](int o0, Operands& x) {
#pragma unroll
      for (int s = 0; s < kSteps; ++s) weights(o0, s * kTile, x.w[s]);
#pragma unroll
      for (int t = 0; t < kTiles; ++t) __builtin_memcpy(x.v[t], scores + o0 + t * kTile + four, sizeof x.v[t]);
    };
    const auto multiply = [&](int j, const T (&w)[kTiles][4], v4f (&sum)[kTiles]) {
      float h[4];
      __builtin_memcpy(h, &hidden[at][j + four], sizeof h);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int t = 0; t < kTiles; ++t) sum[t] = product(to_float(w[t][e]), h[e], sum[t]);
    };
    const auto finish = [&](int o0, const Operands& x) {
      v4f sum[kTiles];
#pragma unroll
      for (int t = 0; t < kTiles; ++t) sum[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
      for (int s = 0; s < kSteps; ++s) multiply(s * kTile, x.w[s], sum);
      // up to r, a multiple of 16 here, and not to `padded`: what follows a row of up is not its own
      for (int j = kSteps * kTile; RANKS > 32 && j < a.r; j += kTile) {
        T w[kTiles][4];
        weights(o0, j, w);
        multiply(j, w, sum);
      }
      if (!mine) return;
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        float v[4];
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = __builtin_fmaf(a.scale, sum[t][q], to_float(x.v[t][q]));
        store_floats<4>(a.out, row * a.out_stride + o0 + t * kTile + four, a.out_dtype, 4, v);
      }
    };
    // any 16 outputs
    const auto guarded = [&](int o0) {
      v4f sum = v4f{0.0f, 0.0f, 0.0f, 0.0f};
      const int o = o0 + at < a.K ? o0 + at : a.K - 1;
      for (int j = four; some && j < padded; j += kTile) {
        float w[4], h[4];
        load_floats<4>(up + o * a.up_output + j, a.r - j, w);
        __builtin_memcpy(h, &hidden[at][j], sizeof h);
#pragma unroll
        for (int e = 0; e < 4; ++e) sum = product(w[e], h[e], sum);
      }
      if (!mine || o0 + four >= a.K) return;
      float v[4];
      load_floats<4>(scores + o0 + four, a.K - o0 - four, v);
#pragma unroll
      for (int q = 0; q < 4; ++q) v[q] = some ? __builtin_fmaf(a.scale, sum[q], v[q]) : v[q];
      store_floats<4>(a.out, row * a.out_stride + o0 + four, a.out_dtype, a.K - o0 - four, v);
    };
    const int whole = some && a.r % kTile == 0 ? a.K / kOutputs : 0;
    // a block's outputs are in a row
    int block = tile * a.tile_blocks + wave;
    const int past = (tile + 1) * a.tile_blocks, last = (a.K + kOutputs - 1) / kOutputs;
    const int end_block = past < last ? past : last;
    Operands x;
    const bool early = block < whole && block < end_block;  // on their way beside the parts
    if (early) load(block * kOutputs, x);
    loads_first();
    __syncthreads();
    // the parts' sums: four ranks of a row a thread, and where that leaves threads every kGroups-th part
    const int each = kTile * padded / 4;
    for (int i = threadIdx.x; i < each * kGroups; i += kThreads) {
      const int g = i / each, n = i % each / (padded / 4), j = i % (padded / 4) * 4;
      float4 sum{0.0f, 0.0f, 0.0f, 0.0f};
      if (n >= first && n < end && some) {
        const float* from = a.part + ((int64_t)window * kTile + n) * padded + j;
        const int64_t part = (int64_t)a.N * padded;
        for (int p = g; p < a.parts; p += 4 * kGroups) {
          float4 v[4];
#pragma unroll
          for (int q = 0; q < 4; ++q)
            v[q] = *(const float4*)(from + (p + q * kGroups < a.parts ? p + q * kGroups : p) * part);
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (p + q * kGroups < a.parts) sum.x += v[q].x, sum.y += v[q].y, sum.z += v[q].z, sum.w += v[q].w;
        }
      }
      *(float4*)&(kGroups > 1 ? group_sums[g][n][j] : hidden[n][j]) = sum;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < each; i += kThreads) {
      const int n = i / (padded / 4), j = i % (padded / 4) * 4;
      if (kGroups > 1) {
        float4 sum = *(const float4*)&group_sums[0][n][j];
#pragma unroll
        for (int g = 1; g < kGroups; ++g) {
          const float4 v = *(const float4*)&group_sums[g][n][j];
          sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
        }
        *(float4*)&hidden[n][j] = sum;
      }
      if (a.hidden && tile == 0 && n >= first && n < end) {
        float v[4];
        __builtin_memcpy(v, &hidden[n][j], sizeof v);
        store_floats<4>(a.hidden + row_of(code[n]) * a.hidden_stride + j, a.r - j, v);
      }
    }
    __syncthreads();
    if (early)
      for (;;) {
        Operands next;
        const bool more = block + kWaves < whole && block + kWaves < end_block;
        if (more) load((block + kWaves) * kOutputs, next);
        loads_first();
        finish(block * kOutputs, x);
        block += kWaves;
        if (!more) break;
        x = next;
      }
    for (; block < end_block; block += kWaves)
      for (int o0 = block * kOutputs; o0 < a.K && o0 < (block + 1) * kOutputs; o0 += kTile) guarded(o0);
  });
}

// ----------------------------------------------------------------------------------- gradients
// back, a part of the outputs: lane l has row l % 16 and eight outputs in a row of every 32, whose weights of
// ranks RT (l % 16) + t it reads one output after the other.  Gradients and weights of one 16-bit type are
// multiplied as they are.
template <int G, int W, int RT>
__device__ __forceinline__ void back_block(const AdaptArgs& a, int block, int p, int ranks, Order& order,
                                           v4f (*join)[RT][kWave]) {
  typedef typename Element<W>::type T;
  typedef typename Element<G>::type S;
  constexpr bool kHalf = G == W && W != YTM_DTYPE_F32;
  const int slot = block / a.windows, window = block % a.windows;
  const uint32_t* code = order.window(a, window);
  const int l = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t row = row_of(code[l % kTile] == UINT32_MAX ? code[0] : code[l % kTile]);
  const S* grad = (const S*)a.scores + row * a.stride;
  segments(code, slot, a.slots, [&](int key, int first, int end) {
    if (key == a.M) return;
    const int j = ranks + l % kTile * RT;
    const T* up = (const T*)a.up + key * a.up_adapter + j;
    v4f sum[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) sum[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    struct Operands {
      v4u x;
      uint16_t h[kHalf ? 8 : 1][RT];
      float g[kHalf ? 1 : 8], w[kHalf ? 1 : 8][RT];
    };
    const auto load = [&](int step, auto all, auto odd, Operands& v) {
      constexpr bool kWhole = decltype(all)::value;
      const int o = step * 32 + l / kTile * 8;
      if constexpr (kHalf) {
        v.x = load_halves<S, kWhole, decltype(odd)::value>(grad + o, a.K - o);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const T* from = up + (int64_t)(o + e) * a.up_output;
          if (kWhole) {
            __builtin_memcpy(v.h[e], from, sizeof v.h[e]);
          } else {
#pragma unroll
            for (int t = 0; t < RT; ++t) {
              v.h[e][t] = 0;
              if (o + e < a.K && j + t < a.r) __builtin_memcpy(&v.h[e][t], from + t, 2);
            }
          }
        }
      } else {
        load_floats<8, kWhole>(grad + o, a.K - o, v.g);
#pragma unroll
        for (int e = 0; e < 8; ++e)
          load_floats<RT, kWhole>(up + (int64_t)(o + e) * a.up_output, o + e < a.K ? a.r - j : 0, v.w[e]);
      }
    };
    const auto multiply = [&](const Operands& v) {
      if constexpr (kHalf) {
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          v4u w;
#pragma unroll
          for (int q = 0; q < 4; ++q) w[q] = (uint32_t)v.h[2 * q + 1][t] << 16 | v.h[2 * q][t];
          sum[t] = half_product<W>(v.x, w, sum[t]);
        }
      } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int t = 0; t < RT; ++t) sum[t] = product(v.g[e], v.w[e][t], sum[t]);
      }
    };
    // whole steps of whole ranks have the next one's operands on their way
    const int steps = (a.K + 31) / 32, last = (p + 1) * a.part_steps < steps ? (p + 1) * a.part_steps : steps;
    const int whole = ranks + RT * kTile <= a.r ? (last < a.K / 32 ? last : a.K / 32) : 0;
    int step = p * a.part_steps + wave;
    const auto pipeline = [&](auto odd) {
      if (step >= whole) return;
      Operands ring[3];  // two steps' operands are on their way
      load(step, std::true_type{}, odd, ring[0]);
      const int second = step + kWaves < whole ? step + kWaves : step;
      load(second, std::true_type{}, odd, ring[1]);
      for (;; step += kWaves) {
        const int third = step + 2 * kWaves;
        load(third < whole ? third : step, std::true_type{}, odd, ring[2]);
        loads_first();
        multiply(ring[0]);
        if (step + kWaves >= whole) break;
        ring[0] = ring[1];
        ring[1] = ring[2];
      }
      step += kWaves;
    };
    if (kHalf && a.odd)
      pipeline(std::true_type{});
    else
      pipeline(std::false_type{});
    for (; step < last; step += kWaves) {
      Operands now;
      load(step, std::false_type{}, std::false_type{}, now);
      multiply(now);
    }
    write_part<RT>(a, p, window, first, end, ranks, sum, join);
  });
}

__global__ __launch_bounds__(kThreads) void back_join_kernel(AdaptArgs a) {
  const int64_t each = (int64_t)a.N * a.padded;
  for (int64_t i = blockIdx.x * (int64_t)kThreads + threadIdx.x; i < each / 4; i += (int64_t)gridDim.x * kThreads) {
    float4 sum{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
    for (int p = 0; p < a.parts; ++p) {
      const float4 v = ((const float4*)(a.part + p * each))[i];
      sum.x += v.x, sum.y += v.y, sum.z += v.z, sum.w += v.w;
    }
    ((float4*)a.back)[i] = sum;
  }
}

// A gradient's tile of 128 columns (outputs or clauses) and 16 RT ranks: the sum over an adapter's rows of a
// row's value at the column times its value at the rank (hidden or back, f32).  The rows are taken 128 at a
// time: their values at the ranks go through LDS, those at the columns are loaded by the wave that has the
// row, eight columns in a row a lane.
//
// PLANES 0: f32 operands.  Lane l has a row of every four and eight columns, each a product's operand.
// PLANES 3: values at the columns that bfloat16 holds (bits, bfloat16).  Lane l has eight rows of 32, whose
// values are exchanged to eight rows of a column, an operand of 32 rows; the values at the ranks are the
// sum of three bfloat16 (8 + 8 + 8 bits of a float32's fraction), a product each.
constexpr int kColumns = 128, kBatch = 128;
template <int X, int RT, int PLANES>
struct OuterShared {
  // Of a rank's rows, so that neighbouring ranks' are in different banks.  Lanes read every RT-th rank: with RT 2
  // two of them meet in a bank, with RT 4 four, and a float of four in `join` meets three others at any RT.
  static constexpr int kPitch = kBatch + 8;
  static constexpr int kValues = PLANES ? PLANES * RT * kTile * kPitch / 2 : kBatch * (RT * kTile + 4);
  union {
    float values[kValues];
    uint16_t planes[2 * kValues];
    v4f join[kWaves][4][kWave];
  };
};

// The fraction of a f32 as the sum of bfloat16: each cut, not rounded, so that nothing overflows; where the first is
// infinite or NaN the others are zero.
template <int PLANES>
__device__ __forceinline__ void split(float v, uint16_t (&part)[PLANES]) {
  const uint32_t u = __float_as_uint(v);
  const bool finite = (u & 0x7F800000u) != 0x7F800000u;
  part[0] = (uint16_t)((finite || (u & 0x007FFFFFu) == 0u ? u : u | 0x00400000u) >> 16);  // a NaN stays one
  float rest = finite ? v - __uint_as_float(u & 0xFFFF0000u) : 0.0f;
#pragma unroll
  for (int p = 1; p < PLANES; ++p) {
    const uint32_t w = __float_as_uint(rest);
    part[p] = (uint16_t)(w >> 16);
    rest -= __uint_as_float(w & 0xFFFF0000u);
  }
}

// Writes a block's sums total[t][e]: wave w has row 4 (l / 16) + w of each product, of outputs 8 (4 (l / 16) + w) + e
// or of ranks.
template <int RT, bool UP>
__device__ __forceinline__ void store_outer(const AdaptArgs& a, int tile, int key, int ranks, const float (&total)[RT][8]) {
  const int l = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  if constexpr (UP) {
    const int j = ranks + l % kTile * RT;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int o = tile * kColumns + 8 * (l / kTile * 4 + wave) + e;
      float v[RT];
#pragma unroll
      for (int t = 0; t < RT; ++t) v[t] = total[t][e];
      if (o < a.K && j < a.r)
        store_floats<RT>(a.out, key * a.d_up_adapter + o * a.d_up_output + j, a.d_dtype, a.r - j, v);
    }
  } else {
    const int column = tile * kColumns + l % kTile * 8;
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int rank = ranks + (l / kTile * 4 + wave) * RT + t;
      if (rank < a.r && column < a.C)
        store_floats<8>(a.d_down, key * a.d_down_adapter + rank * a.d_down_rank + column, a.d_dtype, a.C - column,
                        total[t]);
    }
  }
}

// The place of a block's partial sums, by slot (two a window), block of ranks and tile.
template <int RT>
__device__ __forceinline__ float* partial_of(float* from, int slot, int ranks, int tiles, int tile, int r) {
  const int64_t blocks = (r + RT * kTile - 1) / (RT * kTile);
  return from + ((slot * blocks + ranks / (RT * kTile)) * tiles + tile) * (RT * 8 * kThreads);
}

// The sums over rows begin .. end - 1 of the order, all of adapter `key`; to the gradient, or to `partial`.
template <int X, int RT, bool UP, int PLANES>
__device__ __forceinline__ void outer_block(const AdaptArgs& a, int tile, int key, int begin, int end, int ranks,
                                            Order& order, OuterShared<X, RT, PLANES>& sh, float* partial) {
  typedef OuterShared<X, RT, PLANES> Shared;
  constexpr int kRanks = RT * kTile;
  const int l = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  v4f sum[RT][8];
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int e = 0; e < 8; ++e) sum[t][e] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  const int column = tile * kColumns + l % kTile * 8, columns = UP ? a.K : a.C;
  const bool whole_tile = (tile + 1) * kColumns <= columns;
  for (int first = begin; first < end; first += kBatch) {
    const int rows = end - first < kBatch ? end - first : kBatch;
    __syncthreads();
    if (a.N > kInline && threadIdx.x < kBatch)  // rows past the last are it
      order.code[threadIdx.x] = a.order[first + ((int)threadIdx.x < rows ? (int)threadIdx.x : rows - 1)];
    __syncthreads();
    const uint32_t* code = a.N > kInline ? order.code : order.code + first;
    // 32 rows a wave: its lane's eight (of four, RANK by RANK, with f32 operands)
    const bool work = wave * 32 < rows;
    int mine[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const int at = wave * 32 + (PLANES ? l / kTile * 8 + i : i * 4 + l / kTile);
      mine[i] = at < rows ? row_of(code[at]) : -1;
    }
    v4u raw[PLANES && X != YTM_DTYPE_BITS ? 8 : 1];
    uint32_t bits[8];
    float v[PLANES ? 1 : 8][8];
    const auto load = [&](auto all, auto odd) {
      constexpr bool kWhole = decltype(all)::value;
      const int last = row_of(code[rows - 1]);
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const bool there = kWhole || mine[i] >= 0;
        const int64_t row = there ? mine[i] : last;
        const int left = there ? columns - column : 0;
        if constexpr (X == YTM_DTYPE_BITS && PLANES) {
          bits[i] = 0u;
          if (kWhole || left > 0)
            bits[i] = ((const uint8_t*)((const uint32_t*)a.x + row * a.x_stride))[column / 8];
          if (!kWhole && left > 0 && left < 8) bits[i] &= (1u << left) - 1u;
        } else if constexpr (PLANES > 0) {
          const bf16* from = UP ? (const bf16*)a.scores + row * a.stride : (const bf16*)a.x + row * a.x_stride;
          raw[i] = load_halves<bf16, kWhole, decltype(odd)::value>(from + column, left);
        } else if constexpr (UP) {
          load_floats<8, kWhole>((const typename Element<X>::type*)a.scores + row * a.stride + column, left, v[i]);
        } else {
          load_clauses<X, 8, kWhole>(a, row, there ? column : a.C, v[i]);
        }
      }
    };
    if (work) {
      if (!whole_tile || wave * 32 + 32 > rows)
        load(std::false_type{}, std::false_type{});
      else if (PLANES > 0 && X == YTM_DTYPE_BF16 && a.odd)
        load(std::true_type{}, std::true_type{});
      else
        load(std::true_type{}, std::false_type{});
    }
    loads_first();
    // the rows' values at the ranks: two threads a row
    {
      const int i = threadIdx.x % kBatch, half = threadIdx.x / kBatch * (kRanks / 2);
      float h[kRanks / 2];
#pragma unroll
      for (int q = 0; q < kRanks / 2; ++q) h[q] = 0.0f;
      if (i < rows) {
        if constexpr (UP) {
          const float* from = a.hidden + row_of(code[i]) * a.hidden_stride + ranks + half;
          if (ranks + kRanks <= a.r) {
            load_floats<kRanks / 2, true>(from, 0, h);
          } else {
#pragma unroll
            for (int q = 0; q < kRanks / 2; ++q) h[q] = ranks + half + q < a.r ? from[q] : 0.0f;
          }
        } else {
          const float* from = a.back + (int64_t)(first + i) * a.padded + ranks + half;
          const int64_t part = (int64_t)a.N * a.padded;
#pragma unroll 4
          for (int p = 0; p < a.back_parts; ++p) {
            float one[kRanks / 2];
            __builtin_memcpy(one, from + p * part, sizeof one);
#pragma unroll
            for (int q = 0; q < kRanks / 2; ++q) h[q] += one[q];
          }
        }
      }
      if constexpr (PLANES > 0) {
#pragma unroll
        for (int q = 0; q < kRanks / 2; ++q) {
          uint16_t part[PLANES > 0 ? PLANES : 1];
          split(h[q], part);
#pragma unroll
          for (int p = 0; p < PLANES; ++p) sh.planes[(p * kRanks + half + q) * Shared::kPitch + i] = part[p];
        }
      } else {
        __builtin_memcpy(&sh.values[i * (kRanks + 4) + half], h, sizeof h);
      }
    }
    __syncthreads();
    if (!work) continue;
    if constexpr (PLANES > 0) {
      v4u h[RT][PLANES > 0 ? PLANES : 1];
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int p = 0; p < PLANES; ++p)
          h[t][p] = *(const v4u*)&sh.planes[(p * kRanks + l % kTile * RT + t) * Shared::kPitch + wave * 32 + l / kTile * 8];
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        v4u x;  // eight rows of column e
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          if constexpr (X == YTM_DTYPE_BITS)
            x[q] = ((bits[2 * q] >> e & 1u) | (bits[2 * q + 1] >> e & 1u) << 16) * 0x3F80u;
          else
            x[q] = __builtin_amdgcn_perm(raw[2 * q + 1][e / 2], raw[2 * q][e / 2], e % 2 ? 0x07060302u : 0x05040100u);
        }
#pragma unroll
        for (int p = PLANES - 1; p >= 0; --p)
#pragma unroll
          for (int t = 0; t < RT; ++t)
            sum[t][e] = UP ? half_product<YTM_DTYPE_BF16>(x, h[t][p], sum[t][e])
                           : half_product<YTM_DTYPE_BF16>(h[t][p], x, sum[t][e]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        float h[RT];
        __builtin_memcpy(h, &sh.values[(wave * 32 + i * 4 + l / kTile) * (kRanks + 4) + l % kTile * RT], sizeof h);
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
          for (int t = 0; t < RT; ++t)
            sum[t][e] = UP ? product(v[i][e], h[t], sum[t][e]) : product(h[t], v[i][e], sum[t][e]);
      }
    }
  }
  float total[RT][8];
#pragma unroll
  for (int t = 0; t < RT; ++t) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (e % 4 == 0) {
        __syncthreads();
#pragma unroll
        for (int q = 0; q < 4; ++q) sh.join[wave][q][l] = sum[t][e + q];
        __syncthreads();
      }
      total[t][e] = 0.0f;
#pragma unroll
      for (int w = 0; w < kWaves; ++w) total[t][e] += ((const float*)&sh.join[w][e % 4][l])[wave];
      if (partial)
        partial[(t * 8 + e) * kThreads + threadIdx.x] = total[t][e];
      else
        total[t][e] *= a.scale;
    }
  }
  if (!partial) store_outer<RT, UP>(a, tile, key, ranks, total);
}

// Block `block` of a gradient: of at most kInline rows a tile of an adapter, all of its rows; of more a tile,
// a window of the order and every slots-th adapter of it, one of whose rows pass the window's ends giving
// partial sums.
template <int X, int RT, bool UP, int PLANES>
__device__ __forceinline__ void outer_blocks(const AdaptArgs& a, int block, int ranks, Order& order,
                                             OuterShared<X, RT, PLANES>& sh) {
  const int tiles = ((UP ? a.K : a.C) + kColumns - 1) / kColumns, tile = block % tiles;
  block /= tiles;
  if (a.N <= kInline) {
    const int key = a.first + block;
    order.make(a);
    const int begin = order.begin(a, key), end = order.begin(a, key + 1);
    outer_block<X, RT, UP, PLANES>(a, tile, key, begin, end, ranks, order, sh, nullptr);
    return;
  }
  const RowWindows& w = UP ? a.up_windows : a.down_windows;
  const int window = block % w.count, from = window * w.rows, to = from + w.rows < a.N ? from + w.rows : a.N;
  const int first = key_of(a.order[from]), last = key_of(a.order[to - 1]);
  for (int key = first + block / w.count; key <= last && key < a.M; key += w.slots) {
    const int begin = order.begin(a, key), end = order.begin(a, key + 1);
    if (begin == end) continue;
    float* partial = nullptr;
    if (begin < from || end > to) partial = partial_of<RT>(w.partial, 2 * window + (begin >= from), ranks, tiles, tile, a.r);
    outer_block<X, RT, UP, PLANES>(a, tile, key, begin < from ? from : begin, end > to ? to : end, ranks, order, sh,
                                   partial);
  }
}

// After both gradients of more than kInline rows: zeros for adapters that no row names, the sums of the
// parts for those that several windows have rows of.
template <int RT, bool UP>
__device__ __forceinline__ void join_block(const AdaptArgs& a, int tile, int tiles, int key, int ranks) {
  const RowWindows& w = UP ? a.up_windows : a.down_windows;
  const int begin = (int)a.order[a.N + key], end = (int)a.order[a.N + key + 1];
  const int first = begin / w.rows, last = (end - 1) / w.rows;
  if (begin < end && first == last) return;
  float total[RT][8] = {};
  if (begin < end)
    for (int window = first; window <= last; ++window) {
      const float* partial = partial_of<RT>(w.partial, 2 * window + (window == first), ranks, tiles, tile, a.r);
#pragma unroll
      for (int t = 0; t < RT; ++t)
#pragma unroll
        for (int e = 0; e < 8; ++e) total[t][e] += partial[(t * 8 + e) * kThreads + threadIdx.x];
    }
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int e = 0; e < 8; ++e) total[t][e] *= a.scale;
  store_outer<RT, UP>(a, tile, key, ranks, total);
}
template <int RT>
__global__ __launch_bounds__(kThreads) void join_kernel(AdaptArgs a) {
  const int ups = (a.K + kColumns - 1) / kColumns, downs = (a.C + kColumns - 1) / kColumns, tile = blockIdx.x;
  for (int key = blockIdx.y; key < a.M; key += gridDim.y) {
    if (tile < ups)
      join_block<RT, true>(a, tile, ups, key, blockIdx.z * RT * kTile);
    else
      join_block<RT, false>(a, tile - ups, downs, key, blockIdx.z * RT * kTile);
  }
}

// Waves that a SIMD holds at once: what the sums of 16 RT ranks, and f32 operands, leave of its registers.  With
// RT 4 they leave too few: 28 bytes of scratch a lane in the gradient of up by f32 and f16 gradients, 36 to 180 in
// that of down (bits 36, bf16 76, f16 156, f32 180); bf16 clause outputs take 12 at smaller RT too.
constexpr int waves_of(int rt, int planes) { return planes ? (rt == 1 ? 4 : rt == 2 ? 3 : 2) : rt == 1 ? 3 : 2; }

template <int G>
constexpr int kGradPlanes = G == YTM_DTYPE_BF16 ? 3 : 0;

// Of at most kInline rows both in one launch: the first blocks make back, the others the gradient of up.
template <int G, int W, int RT>
__global__ __launch_bounds__(kThreads, waves_of(RT, kGradPlanes<G>)) void grad_kernel(AdaptArgs a) {
  __shared__ Order order;
  __shared__ OuterShared<G, RT, kGradPlanes<G>> sh;
  static_assert(sizeof sh.join >= sizeof(v4f[kWaves][RT][kWave]), "");
  const int back = a.windows * a.slots * a.parts, ranks = blockIdx.y * RT * kTile;
  if ((int)blockIdx.x < back) {
    const int p = blockIdx.x % a.parts;
    back_block<G, W, RT>(a, blockIdx.x / a.parts, p, ranks, order, (v4f(*)[RT][kWave])sh.join);
  } else {
    outer_blocks<G, RT, true, kGradPlanes<G>>(a, blockIdx.x - back, ranks, order, sh);
  }
}

// Of more two launches, so that back's blocks are as many as their registers allow (2048 rows of 10007 bfloat16, rank 32:
// together 69 us; apart 20 and 38).
template <int G, int W, int RT>
__global__ __launch_bounds__(kThreads) void back_kernel(AdaptArgs a) {
  __shared__ Order order;
  __shared__ v4f join[kWaves][RT][kWave];
  back_block<G, W, RT>(a, blockIdx.x / a.parts, blockIdx.x % a.parts, blockIdx.y * RT * kTile, order, join);
}
template <int G, int RT>
__global__ __launch_bounds__(kThreads, waves_of(RT, kGradPlanes<G>)) void outputs_kernel(AdaptArgs a) {
  __shared__ Order order;
  __shared__ OuterShared<G, RT, kGradPlanes<G>> sh;
  outer_blocks<G, RT, true, kGradPlanes<G>>(a, blockIdx.x, blockIdx.y * RT * kTile, order, sh);
}

template <int X, int RT, int PLANES>
__global__ __launch_bounds__(kThreads, waves_of(RT, PLANES)) void clauses_kernel(AdaptArgs a) {
  __shared__ Order order;
  __shared__ OuterShared<X, RT, PLANES> sh;
  outer_blocks<X, RT, false, PLANES>(a, blockIdx.x, blockIdx.y * RT * kTile, order, sh);
}

// --------------------------------------------------------------------------------------- host
struct Split {
  int windows, slots, parts, part_steps;
};

// Parts of a sum over `steps` (of `block` rows in a row), so that about 1024 blocks share it, each with a step a
// wave at least, and slots that share a window's segments where there are still few blocks.
Split split_of(int64_t N, int64_t M, int64_t steps, int64_t most_parts) {
  Split s;
  s.windows = (int)((N + kTile - 1) / kTile);
  const int64_t most = steps > kWaves ? (steps + kWaves - 1) / kWaves : 1;
  int64_t parts = 1024 / s.windows;
  parts = parts < 1 ? 1 : parts > most_parts ? most_parts : parts;
  parts = parts < most ? parts : most;
  s.part_steps = (int)((steps + parts - 1) / parts);
  s.part_steps = s.part_steps ? s.part_steps : 1;
  s.parts = steps ? (int)((steps + s.part_steps - 1) / s.part_steps) : 1;
  int64_t slots = 1024 / ((int64_t)s.windows * s.parts);
  int64_t segments = M + 1 < kTile ? M + 1 : kTile;  // of a window, at most
  segments = N < segments ? N : segments;
  slots = slots < 1 ? 1 : slots < segments ? slots : segments;
  s.slots = (int)slots;
  return s;
}
Split down_split(int64_t N, int64_t M, int64_t C, bool halves) {
  const int64_t chunk = halves ? 128 : 64;
  return split_of(N, M, (C + chunk - 1) / chunk, 16);
}
// Few rows: eight parts at most, which the blocks that use back add up themselves.
Split back_split(int64_t N, int64_t M, int64_t K) {
  return split_of(N, M, (K + 31) / 32, N <= kInline ? 8 : 16);
}
bool joins_back(int64_t N, const Split& s) { return N > kInline && s.parts > 1; }

// Windows of a gradient's rows: 256 rows or more, so that about 1024 blocks share them and their sums'
// parts take at most some 64 MB; slots that share the adapters a window has on average.
RowWindows windows_of(int64_t N, int64_t M, int64_t columns, int64_t r) {
  RowWindows w{};
  if (N <= kInline || columns == 0) return w;
  const int64_t ranks = r <= 16 ? 16 : r <= 32 ? 32 : 64;
  const int64_t tiles = (columns + kColumns - 1) / kColumns * ((r + ranks - 1) / ranks);
  int64_t count = (N + 255) / 256;
  const int64_t most = tiles < 1024 ? 1024 / tiles : 1;
  if (count > most) count = most;
  w.rows = (int)((N + count - 1) / count);
  w.count = (int)((N + w.rows - 1) / w.rows);
  const int64_t slots = 2 * (M * w.rows / N);
  w.slots = (int)(slots < 1 ? 1 : slots > 64 ? 64 : slots);
  return w;
}
int64_t partial_bytes(const RowWindows& w, int64_t columns, int64_t r) {
  if (w.count < 2) return 0;  // one window has all of an adapter's rows
  const int64_t ranks = r <= 16 ? 16 : r <= 32 ? 32 : 64;
  return 2 * w.count * ((columns + kColumns - 1) / kColumns) * ((r + ranks - 1) / ranks) * (ranks / 2 * kThreads * 4);
}

int64_t aligned(int64_t bytes) { return (bytes + 15) / 16 * 16; }
int64_t padded_of(int64_t r) { return (r + kTile - 1) / kTile * kTile <= 32 ? (r + kTile - 1) / kTile * kTile
                                                                            : (r + 63) / 64 * 64; }

int rank_tiles(int r) { return r <= 16 ? 1 : r <= 32 ? 2 : 4; }

hipError_t launch_order(const AdaptArgs& a, hipStream_t s) {
  if (a.N <= kInline) return hipSuccess;
  order_kernel<<<(a.N + a.begins + kWave - 1) / kWave, kOrderThreads, 0, s>>>(a);
  return hipGetLastError();
}

template <int X, int W>
hipError_t launch_down(const AdaptArgs& a, hipStream_t s) {
  const int t = rank_tiles(a.r);
  const dim3 grid(a.parts, a.windows * a.slots, (a.r + t * kTile - 1) / (t * kTile));
  switch (t) {
    case 1: down_kernel<X, W, 1><<<grid, kThreads, 0, s>>>(a); break;
    case 2: down_kernel<X, W, 2><<<grid, kThreads, 0, s>>>(a); break;
    default: down_kernel<X, W, 4><<<grid, kThreads, 0, s>>>(a); break;
  }
  return hipGetLastError();
}

template <int W, int S>
hipError_t launch_up(const AdaptArgs& a, dim3 grid, hipStream_t s) {
  switch (a.padded) {
    case 16: up_kernel<W, S, 16><<<grid, kThreads, 0, s>>>(a); break;
    case 32: up_kernel<W, S, 32><<<grid, kThreads, 0, s>>>(a); break;
    default: up_kernel<W, S, kMaxRank><<<grid, kThreads, 0, s>>>(a); break;
  }
  return hipGetLastError();
}

template <int W>
hipError_t launch_adapt(AdaptArgs a, int x_dtype, hipStream_t s) {
  hipError_t e = launch_order(a, s);
  if (e != hipSuccess) return e;
  switch (x_dtype) {
    case YTM_DTYPE_BITS: e = launch_down<YTM_DTYPE_BITS, W>(a, s); break;
    case YTM_DTYPE_F16: e = launch_down<YTM_DTYPE_F16, W>(a, s); break;
    case YTM_DTYPE_BF16: e = launch_down<YTM_DTYPE_BF16, W>(a, s); break;
    default: e = launch_down<YTM_DTYPE_F32, W>(a, s); break;
  }
  if (e != hipSuccess) return e;
  // A block takes so many times 256 outputs that there are about 1024 of them, or 2048 for many rows (4096 rows of 8
  // adapters, rank 32: 106 us, with 1024 126; 48 rows of some 30 adapters, rank 16: 12.3 us, with 2048 13.3).
  a.tiles_first = a.windows < 16;
  const int64_t tiles = a.K > 0 ? (a.K + 255) / 256 : 1, blocks = (int64_t)a.windows * a.slots;
  const int64_t most = a.tiles_first ? 1024 : 2048, each = (tiles * blocks + most - 1) / most;
  a.tiles = (int)((tiles + each - 1) / each);
  a.tile_blocks = (int)(each * kWaves);
  const dim3 grid((unsigned)(blocks * (a.tiles_first ? (a.tiles + 7) / 8 * 8 : a.tiles)));
  switch (a.dtype) {
    case YTM_DTYPE_F16: return launch_up<W, YTM_DTYPE_F16>(a, grid, s);
    case YTM_DTYPE_BF16: return launch_up<W, YTM_DTYPE_BF16>(a, grid, s);
    default: return launch_up<W, YTM_DTYPE_F32>(a, grid, s);
  }
}

// A launch counts its threads in 32 bits: launch(first adapter or 0, blocks) for each of as many launches as
// that takes for the blocks of a gradient.
template <typename Launch>
hipError_t launch_outer(const AdaptArgs& a, int64_t columns, const RowWindows& w, Launch launch) {
  const int64_t tiles = (columns + kColumns - 1) / kColumns, most = tiles ? ((int64_t)1 << 23) / tiles : 1;
  if (a.N > kInline) return launch(0, tiles * w.count * w.slots);
  for (int64_t first = 0; first < a.M; first += most) {
    const hipError_t e = launch((int)first, tiles * (a.M - first < most ? a.M - first : most));
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

template <int G, int W, int RT>
hipError_t launch_many(const AdaptArgs& a, hipStream_t s) {
  const unsigned ranks = (a.r + RT * kTile - 1) / (RT * kTile);
  back_kernel<G, W, RT><<<dim3(a.windows * a.slots * a.parts, ranks), kThreads, 0, s>>>(a);
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess || a.K == 0) return e;
  return launch_outer(a, a.K, a.up_windows, [&](int, int64_t blocks) {
    outputs_kernel<G, RT><<<dim3((unsigned)blocks, ranks), kThreads, 0, s>>>(a);
    return hipGetLastError();
  });
}

template <int G, int W>
hipError_t launch_grad(AdaptArgs a, hipStream_t s) {
  const int t = rank_tiles(a.r);
  if (a.N > kInline) {
    if (t == 1) return launch_many<G, W, 1>(a, s);
    return t == 2 ? launch_many<G, W, 2>(a, s) : launch_many<G, W, 4>(a, s);
  }
  return launch_outer(a, a.K, a.up_windows, [&](int first, int64_t blocks) {
    a.first = first;
    if (first) a.windows = 0;  // back is there
    blocks += (int64_t)a.windows * a.slots * a.parts;
    if (blocks == 0) return hipSuccess;
    const dim3 grid((unsigned)blocks, (a.r + t * kTile - 1) / (t * kTile));
    switch (t) {
      case 1: grad_kernel<G, W, 1><<<grid, kThreads, 0, s>>>(a); break;
      case 2: grad_kernel<G, W, 2><<<grid, kThreads, 0, s>>>(a); break;
      default: grad_kernel<G, W, 4><<<grid, kThreads, 0, s>>>(a); break;
    }
    return hipGetLastError();
  });
}
template <int G>
hipError_t launch_grad_of(const AdaptArgs& a, hipStream_t s) {
  switch (a.w_dtype) {
    case YTM_DTYPE_F16: return launch_grad<G, YTM_DTYPE_F16>(a, s);
    case YTM_DTYPE_BF16: return launch_grad<G, YTM_DTYPE_BF16>(a, s);
    default: return launch_grad<G, YTM_DTYPE_F32>(a, s);
  }
}

template <int X, int PLANES>
hipError_t launch_clauses(AdaptArgs a, hipStream_t s) {
  const int t = rank_tiles(a.r);
  return launch_outer(a, a.C, a.down_windows, [&](int first, int64_t blocks) {
    a.first = first;
    const dim3 grid((unsigned)blocks, (a.r + t * kTile - 1) / (t * kTile));
    switch (t) {
      case 1: clauses_kernel<X, 1, PLANES><<<grid, kThreads, 0, s>>>(a); break;
      case 2: clauses_kernel<X, 2, PLANES><<<grid, kThreads, 0, s>>>(a); break;
      default: clauses_kernel<X, 4, PLANES><<<grid, kThreads, 0, s>>>(a); break;
    }
    return hipGetLastError();
  });
}

hipError_t launch_join(const AdaptArgs& a, hipStream_t s) {
  const int t = rank_tiles(a.r);
  const unsigned tiles = (a.K + kColumns - 1) / kColumns + (a.C + kColumns - 1) / kColumns;
  if (a.N <= kInline || tiles == 0) return hipSuccess;
  const dim3 grid(tiles, a.M < 1024 ? a.M : 1024, (a.r + t * kTile - 1) / (t * kTile));
  switch (t) {
    case 1: join_kernel<1><<<grid, kThreads, 0, s>>>(a); break;
    case 2: join_kernel<2><<<grid, kThreads, 0, s>>>(a); break;
    default: join_kernel<4><<<grid, kThreads, 0, s>>>(a); break;
  }
  return hipGetLastError();
}

hipError_t launch_gradient(AdaptArgs a, int x_dtype, hipStream_t s) {
  hipError_t e = launch_order(a, s);
  if (e != hipSuccess) return e;
  switch (a.dtype) {
    case YTM_DTYPE_F16: e = launch_grad_of<YTM_DTYPE_F16>(a, s); break;
    case YTM_DTYPE_BF16: e = launch_grad_of<YTM_DTYPE_BF16>(a, s); break;
    default: e = launch_grad_of<YTM_DTYPE_F32>(a, s); break;
  }
  if (e == hipSuccess && a.back != a.part) {
    const int64_t blocks = ((int64_t)a.N * a.padded / 4 + kThreads - 1) / kThreads;
    back_join_kernel<<<(unsigned)(blocks < 2048 ? blocks : 2048), kThreads, 0, s>>>(a);
    e = hipGetLastError();
  }
  if (e != hipSuccess) return e;
  if (a.C > 0) switch (x_dtype) {
      case YTM_DTYPE_BITS: e = launch_clauses<YTM_DTYPE_BITS, 3>(a, s); break;
      case YTM_DTYPE_BF16: e = launch_clauses<YTM_DTYPE_BF16, 3>(a, s); break;
      case YTM_DTYPE_F16: e = launch_clauses<YTM_DTYPE_F16, 0>(a, s); break;
      default: e = launch_clauses<YTM_DTYPE_F32, 0>(a, s); break;
    }
  return e == hipSuccess ? launch_join(a, s) : e;
}

int size_of(int dtype) { return dtype == YTM_DTYPE_F32 || dtype == YTM_DTYPE_BITS ? 4 : 2; }

// An operand of M parts, each of `rows` rows of `width` elements: the bytes from a part's first to its last.
Rows parts_of(const void* p, int64_t M, int64_t rows, int64_t width, int64_t part_stride, int64_t stride, int size) {
  if (rows < 1 || width < 1) return Rows{nullptr, 1, 0, 0};
  return rows_of(p, M, (rows > 1 ? (rows - 1) * stride : 0) + width, part_stride, size);
}

constexpr int64_t kMostApart = (int64_t)1 << 40;  // elements, so that no distance passes 64 bits

// What both entries ask of their operands; NULL where it is given, else what is wrong.
const char* wrong_operands(int dtype, int64_t stride, int64_t N, int64_t K, int x_dtype, int64_t x_stride, int64_t C,
                           int64_t down_adapter, int64_t down_rank, int64_t up_adapter, int64_t up_output, int w_dtype,
                           int64_t M, int64_t r, float scale) {
  if (!(scale - scale == 0.0f)) return "scale is finite";
  if (!decode_float(dtype) || !decode_float(w_dtype)) return "scores and adapters are float32, float16 or bfloat16";
  if (x_dtype != YTM_DTYPE_BITS && !decode_float(x_dtype)) return "clause outputs are bits, float32, float16 or bfloat16";
  if (N < 0 || K < 0 || C < 0 || M < 0 || N > kDecodeRows || K > kMaxScores || C > kMaxClauses || M > kMaxAdapters)
    return "at most 65535 rows, 8388608 outputs, 2097120 clauses and 65535 adapters";
  if (r < 1 || r > kMaxRank) return "ranks are 1 to 256";
  const int64_t width = x_dtype == YTM_DTYPE_BITS ? (C + 31) / 32 : C;
  const int64_t apart[] = {stride, x_stride, down_adapter, down_rank, up_adapter, up_output};
  for (int64_t v : apart)
    if (v < 0 || v > kMostApart) return "rows are too far apart";
  if (K > 1 && up_output > kMaxApart / 4) return "rows of up are at most 2097152 elements apart";
  if ((N > 1 && ((stride != 0 && stride < K) || (x_stride != 0 && x_stride < width))) ||
      (r > 1 && down_rank != 0 && down_rank < C) || (K > 1 && up_output != 0 && up_output < r) ||
      (M > 1 && ((down_adapter != 0 && down_adapter < C) || (up_adapter != 0 && up_adapter < r))))
    return "rows overlap";
  return nullptr;
}

int64_t order_bytes(int64_t N, int64_t begins) { return N > kInline ? aligned(4 * (N + begins)) : 0; }

}  // namespace

}  // namespace ytm

using ytm::fail;

extern "C" {

int ytm_adapt_workspace(int64_t N, int64_t C, int64_t M, int64_t r, int64_t* bytes) {
  if (!bytes || N < 0 || C < 0 || M < 0 || r < 1 || N > ytm::kDecodeRows || C > ytm::kMaxClauses ||
      M > ytm::kMaxAdapters || r > ytm::kMaxRank)
    return fail(YTM_EINVAL, "bad adapt_workspace arguments");
  *bytes = 0;
  if (N == 0) return YTM_OK;
  int64_t parts = 1;  // the most of the types'
  for (bool halves : {false, true}) {
    const ytm::Split s = ytm::down_split(N, M, C, halves);
    parts = s.parts > parts ? s.parts : parts;
  }
  *bytes = ytm::order_bytes(N, 0) + parts * N * ytm::padded_of(r) * 4;
  return YTM_OK;
}

int ytm_adapt(const void* scores, int dtype, int64_t stride, int64_t N, int64_t K, const void* x, int x_dtype,
              int64_t x_stride, int64_t C, const void* down, int64_t down_adapter, int64_t down_rank, const void* up,
              int64_t up_adapter, int64_t up_output, int w_dtype, int64_t M, int64_t r, const int32_t* which,
              float scale, float* hidden, int64_t hidden_stride, void* out, int out_dtype, int64_t out_stride,
              void* workspace, int64_t workspace_bytes, void* stream) {
  if (const char* wrong = ytm::wrong_operands(dtype, stride, N, K, x_dtype, x_stride, C, down_adapter, down_rank,
                                              up_adapter, up_output, w_dtype, M, r, scale))
    return fail(YTM_EINVAL, std::string("adapt: ") + wrong);
  if (!ytm::decode_float(out_dtype)) return fail(YTM_EINVAL, "adapt: scores are float32, float16 or bfloat16");
  if (N == 0) return YTM_OK;
  if (!which || (K > 0 && (!scores || !out)) || (M > 0 && ((C > 0 && (!x || !down)) || (K > 0 && !up))))
    return fail(YTM_EINVAL, "bad adapt arguments");
  if (out_stride < 0 || out_stride > ytm::kMostApart || hidden_stride < 0 || hidden_stride > ytm::kMostApart ||
      (N > 1 && (out_stride < K || (hidden && hidden_stride < r))))
    return fail(YTM_EINVAL, "adapt: rows overlap or are too far apart");
  int64_t need = 0;
  if (int rc = ytm_adapt_workspace(N, C, M, r, &need)) return rc;
  if (need > 0 && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
    return fail(YTM_EINVAL, "adapt: the workspace is too small or not at a multiple of 16 bytes");
  const int64_t width = x_dtype == YTM_DTYPE_BITS ? (C + 31) / 32 : C;
  const int size = ytm::size_of(dtype), out_size = ytm::size_of(out_dtype), w_size = ytm::size_of(w_dtype);
  const bool in_place = out == scores && size == out_size && (N == 1 || stride == out_stride);
  const ytm::Rows written[] = {ytm::rows_of(out, N, K, out_stride, out_size),
                               ytm::rows_of(hidden, N, r, hidden_stride, 4), ytm::block_of(workspace, need)};
  const ytm::Rows read[] = {ytm::rows_of(in_place ? nullptr : scores, N, K, stride, size),
                            ytm::rows_of(x, N, width, x_stride, ytm::size_of(x_dtype)),
                            ytm::parts_of(down, M, r, C, down_adapter, down_rank, w_size),
                            ytm::parts_of(up, M, K, r, up_adapter, up_output, w_size), ytm::block_of(which, 4 * N)};
  bool overlap = ytm::share_bytes(written[0], written[1]) || ytm::share_bytes(written[0], written[2]) ||
                 ytm::share_bytes(written[1], written[2]);
  for (const ytm::Rows& w : written)
    for (const ytm::Rows& r : read) overlap |= ytm::share_bytes(w, r);
  if (in_place)  // what else is written must still not lie in the scores
    for (int i = 1; i < 3; ++i) overlap |= ytm::share_bytes(written[i], ytm::rows_of(scores, N, K, stride, size));
  if (overlap) return fail(YTM_EINVAL, "adapt: what is written overlaps what is read, and is not the scores' own place");
  const bool halves = w_dtype != YTM_DTYPE_F32 && (x_dtype == w_dtype || x_dtype == YTM_DTYPE_BITS);
  const ytm::Split split = ytm::down_split(N, M, C, halves);
  ytm::AdaptArgs a{};
  a.scores = scores, a.dtype = dtype, a.stride = stride, a.N = (int)N, a.K = (int)K;
  a.x = x, a.x_stride = x_stride, a.C = (int)C;
  a.down = down, a.down_adapter = down_adapter, a.down_rank = down_rank;
  a.up = up, a.up_adapter = up_adapter, a.up_output = up_output;
  a.M = (int)M, a.r = (int)r, a.w_dtype = w_dtype, a.which = which, a.scale = scale;
  a.hidden = hidden, a.hidden_stride = hidden_stride;
  a.out = out, a.out_dtype = out_dtype, a.out_stride = out_stride;
  a.windows = split.windows, a.slots = split.slots, a.parts = split.parts, a.part_steps = split.part_steps;
  a.padded = (int)ytm::padded_of(r);
  a.order = (uint32_t*)workspace;
  a.part = (float*)((char*)workspace + ytm::order_bytes(N, 0));
  hipStream_t s = (hipStream_t)stream;
  hipError_t e;
  switch (w_dtype) {
    case YTM_DTYPE_F16: e = ytm::launch_adapt<YTM_DTYPE_F16>(a, x_dtype, s); break;
    case YTM_DTYPE_BF16: e = ytm::launch_adapt<YTM_DTYPE_BF16>(a, x_dtype, s); break;
    default: e = ytm::launch_adapt<YTM_DTYPE_F32>(a, x_dtype, s); break;
  }
  if (e != hipSuccess) return fail(YTM_EHIP, std::string("adapt failed: ") + hipGetErrorString(e));
  return YTM_OK;
}

int ytm_adapt_gradient_workspace(int64_t N, int64_t C, int64_t K, int64_t M, int64_t r, int64_t* bytes) {
  if (!bytes || N < 0 || C < 0 || K < 0 || M < 0 || r < 1 || N > ytm::kDecodeRows || C > ytm::kMaxClauses ||
      K > ytm::kMaxScores || M > ytm::kMaxAdapters || r > ytm::kMaxRank)
    return fail(YTM_EINVAL, "bad adapt_gradient_workspace arguments");
  *bytes = 0;
  if (N == 0 || M == 0) return YTM_OK;
  const ytm::Split s = ytm::back_split(N, M, K);
  *bytes = ytm::order_bytes(N, M + 1) + (s.parts + ytm::joins_back(N, s)) * N * ytm::padded_of(r) * 4 +
           ytm::partial_bytes(ytm::windows_of(N, M, K, r), K, r) + ytm::partial_bytes(ytm::windows_of(N, M, C, r), C, r);
  return YTM_OK;
}

int ytm_adapt_gradient(const void* grad, int dtype, int64_t stride, int64_t N, int64_t K, const void* x, int x_dtype,
                       int64_t x_stride, int64_t C, const void* up, int64_t up_adapter, int64_t up_output, int w_dtype,
                       int64_t M, int64_t r, const int32_t* which, float scale, const float* hidden,
                       int64_t hidden_stride, void* d_down, int64_t d_down_adapter, int64_t d_down_rank, void* d_up,
                       int64_t d_up_adapter, int64_t d_up_output, void* workspace, int64_t workspace_bytes,
                       void* stream) {
  return ytm_adapt_gradient_as(grad, dtype, stride, N, K, x, x_dtype, x_stride, C, up, up_adapter, up_output, w_dtype, M,
                               r, which, scale, hidden, hidden_stride, w_dtype, d_down, d_down_adapter, d_down_rank, d_up,
                               d_up_adapter, d_up_output, workspace, workspace_bytes, stream);
}

int ytm_adapt_gradient_as(const void* grad, int dtype, int64_t stride, int64_t N, int64_t K, const void* x, int x_dtype,
                          int64_t x_stride, int64_t C, const void* up, int64_t up_adapter, int64_t up_output,
                          int w_dtype, int64_t M, int64_t r, const int32_t* which, float scale, const float* hidden,
                          int64_t hidden_stride, int d_dtype, void* d_down, int64_t d_down_adapter, int64_t d_down_rank,
                          void* d_up, int64_t d_up_adapter, int64_t d_up_output, void* workspace,
                          int64_t workspace_bytes, void* stream) {
  if (const char* wrong = ytm::wrong_operands(dtype, stride, N, K, x_dtype, x_stride, C, d_down_adapter, d_down_rank,
                                              up_adapter, up_output, w_dtype, M, r, scale))
    return fail(YTM_EINVAL, std::string("adapt_gradient: ") + wrong);
  if (d_dtype != w_dtype && d_dtype != YTM_DTYPE_F32)
    return fail(YTM_EINVAL, "adapt_gradient: gradients are of the adapters' type or float32");
  if (M == 0) return YTM_OK;
  if ((C > 0 && !d_down) || (K > 0 && !d_up) ||
      (N > 0 && (!which || !hidden || (K > 0 && (!grad || !up)) || (C > 0 && !x))))
    return fail(YTM_EINVAL, "bad adapt_gradient arguments");
  const int64_t apart[] = {d_up_adapter, d_up_output, hidden_stride};
  for (int64_t v : apart)
    if (v < 0 || v > ytm::kMostApart) return fail(YTM_EINVAL, "adapt_gradient: rows are too far apart");
  if ((N > 1 && hidden_stride != 0 && hidden_stride < r) || (r > 1 && d_down_rank < C) || (K > 1 && d_up_output < r) ||
      (M > 1 && (d_down_adapter < (r - 1) * d_down_rank + C || (K > 0 && d_up_adapter < (K - 1) * d_up_output + r))))
    return fail(YTM_EINVAL, "adapt_gradient: rows overlap");
  int64_t need = 0;
  if (int rc = ytm_adapt_gradient_workspace(N, C, K, M, r, &need)) return rc;
  if (need > 0 && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
    return fail(YTM_EINVAL, "adapt_gradient: the workspace is too small or not at a multiple of 16 bytes");
  const int64_t width = x_dtype == YTM_DTYPE_BITS ? (C + 31) / 32 : C;
  const int size = ytm::size_of(w_dtype), d_size = ytm::size_of(d_dtype);
  const ytm::Rows written[] = {ytm::parts_of(d_down, M, r, C, d_down_adapter, d_down_rank, d_size),
                               ytm::parts_of(d_up, M, K, r, d_up_adapter, d_up_output, d_size),
                               ytm::block_of(workspace, need)};
  const ytm::Rows read[] = {ytm::rows_of(grad, N, K, stride, ytm::size_of(dtype)),
                            ytm::rows_of(x, N, width, x_stride, ytm::size_of(x_dtype)),
                            ytm::parts_of(up, M, K, r, up_adapter, up_output, size),
                            ytm::rows_of(hidden, N, r, hidden_stride, 4), ytm::block_of(which, 4 * N)};
  bool overlap = ytm::share_bytes(written[0], written[1]) || ytm::share_bytes(written[0], written[2]) ||
                 ytm::share_bytes(written[1], written[2]);
  for (const ytm::Rows& w : written)
    for (const ytm::Rows& r : read) overlap |= ytm::share_bytes(w, r);
  if (overlap) return fail(YTM_EINVAL, "adapt_gradient: what is written overlaps what is read");
  ytm::AdaptArgs a{};
  if (N > 0) {
    const ytm::Split split = ytm::back_split(N, M, K);
    const bool joins = ytm::joins_back(N, split);
    a.windows = split.windows, a.slots = split.slots, a.parts = split.parts, a.part_steps = split.part_steps;
    a.padded = (int)ytm::padded_of(r);
    a.order = (uint32_t*)workspace;
    a.part = (float*)((char*)workspace + ytm::order_bytes(N, M + 1));
    a.back = joins ? a.part + split.parts * N * a.padded : a.part;
    a.back_parts = joins ? 1 : split.parts;
    a.begins = (int)M + 1;
    a.up_windows = ytm::windows_of(N, M, K, r);
    a.down_windows = ytm::windows_of(N, M, C, r);
    a.up_windows.partial = a.back + a.back_parts * N * a.padded;
    a.down_windows.partial = a.up_windows.partial + ytm::partial_bytes(a.up_windows, K, r) / 4;
  }
  a.scores = grad, a.dtype = dtype, a.stride = stride, a.N = (int)N, a.K = (int)K;
  a.x = x, a.x_stride = x_stride, a.C = (int)C;
  a.up = up, a.up_adapter = up_adapter, a.up_output = up_output;
  a.M = (int)M, a.r = (int)r, a.w_dtype = w_dtype, a.d_dtype = d_dtype, a.which = which, a.scale = scale;
  a.hidden = const_cast<float*>(hidden), a.hidden_stride = hidden_stride;
  a.out = d_up, a.d_up_adapter = d_up_adapter, a.d_up_output = d_up_output;
  a.d_down = d_down, a.d_down_adapter = d_down_adapter, a.d_down_rank = d_down_rank;
  const auto odd = [](const void* p, int64_t rows, int64_t stride, int type) {
    return ytm::size_of(type) == 2 && (((uintptr_t)p | (rows > 1 ? stride * 2 : 0)) & 2) != 0;
  };
  a.odd = odd(grad, N, stride, dtype) || odd(x, N, x_stride, x_dtype);
  const hipError_t e = ytm::launch_gradient(a, x_dtype, (hipStream_t)stream);
  if (e != hipSuccess) return fail(YTM_EHIP, std::string("adapt_gradient failed: ") + hipGetErrorString(e));
  return YTM_OK;
}

}  // extern "C"
