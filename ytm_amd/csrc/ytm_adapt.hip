// ytm_adapt.hip -- low-rank adapters of many requests beside the readout, and their gradients: the
// entry points ytm_adapt and ytm_adapt_gradient of include/ytm.h and their gfx950 kernels.
//
//   hidden[n] = down[a] x[n], out[n] = scores[n] + scale * up[a] hidden[n], a = which[n]
//   d_up[a] = scale * sum over n of a of grad[n] hidden[n]^T, back[n] = scale * up[a]^T grad[n],
//   d_down[a] = sum over n of a of back[n] x[n]^T
//
// Rows are taken in the order of their adapters (ties in the order of rows), sixteen of that order,
// a window, at a time: a window's rows of one adapter are a segment, whose weights are read once.
// Sums run on the matrix cores in f32 with f32 operands, into which every type converts exactly; their
// operands are one value a lane, so that products over rows need no transposition.  Sums over
// clauses or outputs that several blocks share are joined in a fixed order.
#include <hip/hip_runtime.h>
#include <stdint.h>

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
  int parts, part_steps;  // of a sum over clauses or outputs
  float* part;            // [parts][N in order][r]
  float* back;            // [N in order][r]
  int32_t* order;         // [N] rows, then [N] keys, of more than kInline rows
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
template <int E, typename T>
__device__ __forceinline__ void load_floats(const T* p, int left, float (&v)[E]) {
  T raw[E];
  if (left >= E) {
    __builtin_memcpy(raw, p, sizeof raw);
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = to_float(raw[e]);
  } else {
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = e < left ? to_float(p[e]) : 0.0f;
  }
}
template <int E>
__device__ __forceinline__ void load_floats(const void* p, int64_t at, int dtype, int left, float (&v)[E]) {
  switch (dtype) {
    case YTM_DTYPE_F16: load_floats<E>((const f16*)p + at, left, v); break;
    case YTM_DTYPE_BF16: load_floats<E>((const bf16*)p + at, left, v); break;
    default: load_floats<E>((const float*)p + at, left, v); break;
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
template <int X, int E>
__device__ __forceinline__ void load_clauses(const AdaptArgs& a, int64_t n, int c, float (&v)[E]) {
  const int left = a.C - c;
  if constexpr (X == YTM_DTYPE_BITS) {
    const uint32_t word = left > 0 ? ((const uint32_t*)a.x)[n * a.x_stride + c / 32] >> c % 32 : 0u;
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = e < left ? (float)(word >> e & 1u) : 0.0f;
  } else {
    load_floats<E>((const typename Element<X>::type*)a.x + n * a.x_stride + c, left, v);
  }
}

__device__ __forceinline__ v4f product(float a, float b, v4f d) {
  return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, d, 0, 0, 0);
}

// ---------------------------------------------------------------------------------- the order
// A row's place among the rows is the number of those of a smaller key, or of the same key before it;
// the key is the row's adapter, M where it has none.
__device__ __forceinline__ int key_of(const AdaptArgs& a, int n) {
  const uint32_t w = (uint32_t)a.which[n];
  return w < (uint32_t)a.M ? (int)w : a.M;
}

__global__ __launch_bounds__(kThreads) void order_kernel(AdaptArgs a) {
  __shared__ int keys[4 * kThreads];
  const int n = blockIdx.x * kThreads + threadIdx.x;
  const int mine = n < a.N ? key_of(a, n) : 0;
  int place = 0;
  for (int first = 0; first < a.N; first += 4 * kThreads) {
    __syncthreads();
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int m = first + q * kThreads + threadIdx.x;
      keys[q * kThreads + threadIdx.x] = m < a.N ? key_of(a, m) : INT32_MAX;
    }
    __syncthreads();
#pragma unroll 8
    for (int m = 0; m < 4 * kThreads; ++m) {
      const int key = keys[m];
      place += key < mine || (key == mine && first + m < n);
    }
  }
  if (n < a.N) {
    a.order[place] = n;
    a.order[a.N + place] = mine;
  }
}

// `count` rows (at most kInline) of the order from `first` on, and their keys.
template <int COUNT>
struct Taken {
  int row[COUNT], key[COUNT];
  int keys[kInline];  // of all rows

  __device__ __forceinline__ void take(const AdaptArgs& a, int first) {
    if (a.N > kInline) {
      for (int i = threadIdx.x; i < COUNT; i += kThreads) {
        const bool there = first + i < a.N;
        row[i] = there ? a.order[first + i] : -1;
        key[i] = there ? a.order[a.N + first + i] : INT32_MAX;
      }
    } else {
      const int n = threadIdx.x;
      const int mine = n < a.N ? key_of(a, n) : INT32_MAX;
      keys[n] = mine;
      for (int i = n; i < COUNT; i += kThreads) {
        row[i] = -1;
        key[i] = INT32_MAX;
      }
      __syncthreads();
      int place = 0;
#pragma unroll 4
      for (int m = 0; m < a.N; ++m) place += keys[m] < mine || (keys[m] == mine && m < n);
      if (n < a.N && place >= first && place < first + COUNT) {
        row[place - first] = n;
        key[place - first] = mine;
      }
    }
    __syncthreads();
  }
};

// Where adapter `key` begins in the order of all rows: the number of smaller keys.
__device__ __forceinline__ int begin_of(const AdaptArgs& a, int key, const int* keys) {
  if (a.N <= kInline) {
    int before = 0;
    for (int m = 0; m < a.N; ++m) before += keys[m] < key;
    return before;
  }
  int low = 0, high = a.N;
  while (low < high) {
    const int mid = (low + high) / 2;
    if (a.order[a.N + mid] < key)
      low = mid + 1;
    else
      high = mid;
  }
  return low;
}

// The segments of a window that block `slot` of `slots` takes: body(key, first place, end).
template <typename Body>
__device__ __forceinline__ void segments(const int* key, int slot, int slots, Body body) {
  for (int i = 0, s = 0; i < kTile && key[i] != INT32_MAX; ++s) {
    int end = i + 1;
    while (end < kTile && key[end] == key[i]) ++end;
    if (s % slots == slot) body(__builtin_amdgcn_readfirstlane(key[i]), i, end);
    i = end;
  }
}

// ------------------------------------------------------------------------------------ forward
// Sums over a part of the clauses of 16 rows with 16 RT ranks of a segment's adapter.  Lane l has row and
// rank l % 16 and eight clauses in a row of every 32, one of them a product; a block's waves take 32 clauses in
// turn and are joined in LDS.
template <int X, int W, int RT>
__global__ __launch_bounds__(kThreads) void down_kernel(AdaptArgs a) {
  typedef typename Element<W>::type T;
  __shared__ Taken<kTile> taken;
  __shared__ v4f join[kWaves - 1][RT][kWave];
  const int slot = blockIdx.x % a.slots, window = blockIdx.x / a.slots, p = blockIdx.y, ranks = blockIdx.z * RT * kTile;
  taken.take(a, window * kTile);
  const int l = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int row = taken.row[l % kTile] < 0 ? taken.row[0] : taken.row[l % kTile];
  segments(taken.key, slot, a.slots, [&](int key, int first, int end) {
    if (key == a.M) return;
    const T* down = (const T*)a.down + key * a.down_adapter;
    v4f sum[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) sum[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    const int steps = (a.C + 31) / 32, last = (p + 1) * a.part_steps < steps ? (p + 1) * a.part_steps : steps;
    for (int step = p * a.part_steps + wave; step < last; step += kWaves) {
      const int c = step * 32 + l / kTile * 8;
      float x[8], w[RT][8];
      load_clauses<X, 8>(a, row, c, x);
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        const int j = ranks + t * kTile + l % kTile;
        load_floats<8>(down + (j < a.r ? j : a.r - 1) * a.down_rank + c, a.C - c, w[t]);
      }
#pragma unroll
      for (int e = 0; e < 8; ++e)
#pragma unroll
        for (int t = 0; t < RT; ++t) sum[t] = product(x[e], w[t][e], sum[t]);
    }
    if (wave > 0)
#pragma unroll
      for (int t = 0; t < RT; ++t) join[wave - 1][t][l] = sum[t];
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        for (int w = 0; w < kWaves - 1; ++w) sum[t] += join[w][t][l];
        const int j = ranks + t * kTile + l % kTile;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int i = l / kTile * 4 + q;
          if (i >= first && i < end && j < a.r) a.part[((int64_t)p * a.N + window * kTile + i) * a.r + j] = sum[t][q];
        }
      }
    }
    __syncthreads();
  });
}

// 64 outputs a wave of 16 rows.  Lane l has output l % 16 of a tile and row l % 16, and four ranks of every
// 16; it gets sums of four outputs in a row of row l % 16.
template <int W>
__global__ __launch_bounds__(kThreads) void up_kernel(AdaptArgs a) {
  typedef typename Element<W>::type T;
  constexpr int kTiles = 4;
  __shared__ Taken<kTile> taken;
  __shared__ float hidden[kTile][kMaxRank + 4];
  const int slot = blockIdx.x % a.slots, window = blockIdx.x / a.slots;
  taken.take(a, window * kTile);
  const int l = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int outputs = (blockIdx.y * kWaves + wave) * kTiles * kTile;
  const int padded = (a.r + kTile - 1) / kTile * kTile;
  segments(taken.key, slot, a.slots, [&](int key, int first, int end) {
    for (int i = threadIdx.x; i < kTile * padded; i += kThreads) {
      const int at = i / padded, j = i % padded;
      float sum = 0.0f;
      if (at >= first && at < end && j < a.r) {
        if (key < a.M)
          for (int p = 0; p < a.parts; ++p) sum += a.part[((int64_t)p * a.N + window * kTile + at) * a.r + j];
        if (a.hidden && blockIdx.y == 0) a.hidden[taken.row[at] * a.hidden_stride + j] = sum;
      }
      hidden[at][j] = sum;
    }
    __syncthreads();
    v4f sum[kTiles];
#pragma unroll
    for (int t = 0; t < kTiles; ++t) sum[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    if (key < a.M) {
      const T* up = (const T*)a.up + key * a.up_adapter;
      for (int j = l / kTile * 4; j < padded; j += kTile) {
        float h[4], w[kTiles][4];
        __builtin_memcpy(h, &hidden[l % kTile][j], sizeof h);
#pragma unroll
        for (int t = 0; t < kTiles; ++t) {
          const int o = outputs + t * kTile + l % kTile;
          load_floats<4>(up + (o < a.K ? o : a.K - 1) * a.up_output + j, o < a.K ? a.r - j : 0, w[t]);
        }
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
          for (int t = 0; t < kTiles; ++t) sum[t] = product(w[t][e], h[e], sum[t]);
      }
    }
    const int at = l % kTile;
    if (at >= first && at < end) {
      const int64_t row = taken.row[at];
#pragma unroll
      for (int t = 0; t < kTiles; ++t) {
        const int o = outputs + t * kTile + l / kTile * 4;
        if (o >= a.K) continue;
        float v[4];
        load_floats<4>(a.scores, row * a.stride + o, a.dtype, a.K - o, v);
#pragma unroll
        for (int q = 0; q < 4; ++q) v[q] = key < a.M ? __builtin_fmaf(a.scale, sum[t][q], v[q]) : v[q];
        store_floats<4>(a.out, row * a.out_stride + o, a.out_dtype, a.K - o, v);
      }
    }
    __syncthreads();
  });
}

// ----------------------------------------------------------------------------------- gradients
// back, a part of the outputs: lane l has row l % 16 and four outputs in a row of every 16, whose weights of
// rank l % 16 it reads one after the other.
template <int W, int RT>
__global__ __launch_bounds__(kThreads) void back_kernel(AdaptArgs a) {
  typedef typename Element<W>::type T;
  __shared__ Taken<kTile> taken;
  __shared__ v4f join[kWaves - 1][RT][kWave];
  const int slot = blockIdx.x % a.slots, window = blockIdx.x / a.slots, p = blockIdx.y, ranks = blockIdx.z * RT * kTile;
  taken.take(a, window * kTile);
  const int l = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int64_t row = taken.row[l % kTile] < 0 ? taken.row[0] : taken.row[l % kTile];
  segments(taken.key, slot, a.slots, [&](int key, int first, int end) {
    if (key == a.M) return;
    const T* up = (const T*)a.up + key * a.up_adapter;
    v4f sum[RT];
#pragma unroll
    for (int t = 0; t < RT; ++t) sum[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    const int steps = (a.K + 15) / 16, last = (p + 1) * a.part_steps < steps ? (p + 1) * a.part_steps : steps;
    for (int step = p * a.part_steps + wave; step < last; step += kWaves) {
      const int o = step * 16 + l / kTile * 4;
      float g[4];
      load_floats<4>(a.scores, row * a.stride + o, a.dtype, a.K - o, g);
#pragma unroll
      for (int e = 0; e < 4; ++e)
#pragma unroll
        for (int t = 0; t < RT; ++t) {
          const int j = ranks + t * kTile + l % kTile;
          const float w = o + e < a.K ? to_float(up[(o + e) * a.up_output + (j < a.r ? j : a.r - 1)]) : 0.0f;
          sum[t] = product(g[e], w, sum[t]);
        }
    }
    if (wave > 0)
#pragma unroll
      for (int t = 0; t < RT; ++t) join[wave - 1][t][l] = sum[t];
    __syncthreads();
    if (wave == 0) {
#pragma unroll
      for (int t = 0; t < RT; ++t) {
        for (int w = 0; w < kWaves - 1; ++w) sum[t] += join[w][t][l];
        const int j = ranks + t * kTile + l % kTile;
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int i = l / kTile * 4 + q;
          if (i >= first && i < end && j < a.r) a.part[((int64_t)p * a.N + window * kTile + i) * a.r + j] = sum[t][q];
        }
      }
    }
    __syncthreads();
  });
}

__global__ __launch_bounds__(kThreads) void back_join_kernel(AdaptArgs a) {
  const int64_t each = (int64_t)a.N * a.r;
  for (int64_t i = blockIdx.x * (int64_t)kThreads + threadIdx.x; i < each; i += (int64_t)gridDim.x * kThreads) {
    float sum = 0.0f;
    for (int p = 0; p < a.parts; ++p) sum += a.part[p * each + i];
    a.back[i] = a.scale * sum;
  }
}

// A gradient's tile of 64 columns (outputs or clauses) and 16 RT ranks: the sum over an adapter's rows of a
// row's value at the column times its value at the rank.  A lane has four columns in a row of one of four
// rows, each of them a product's operand; a block's waves take four rows in turn and are joined in LDS.
template <int X, int RT, bool UP>
__global__ __launch_bounds__(kThreads) void outer_kernel(AdaptArgs a, int w_dtype) {
  __shared__ Taken<kInline> taken;
  __shared__ v4f join[kWaves - 1][RT][4][kWave];
  const int key = blockIdx.y, first_column = blockIdx.x * 64, ranks = blockIdx.z * RT * kTile;
  const int l = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  if (a.N <= kInline) taken.take(a, 0);
  const int begin = begin_of(a, key, taken.keys), end = begin_of(a, key + 1, taken.keys);
  v4f sum[RT][4];
#pragma unroll
  for (int t = 0; t < RT; ++t)
#pragma unroll
    for (int e = 0; e < 4; ++e) sum[t][e] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
  const int column = first_column + l % kTile * 4, columns = UP ? a.K : a.C;
  for (int first = begin + wave * 4; first < end; first += kWaves * 4) {
    const int place = first + l / kTile;
    const bool there = place < end;
    const int at = there ? place : end - 1;
    const int64_t row = a.N <= kInline ? taken.row[at] : a.order[at];
    float v[4];
    if constexpr (UP)
      load_floats<4>(a.scores, row * a.stride + column, a.dtype, there ? columns - column : 0, v);
    else
      load_clauses<X, 4>(a, row, column, v);
#pragma unroll
    for (int t = 0; t < RT; ++t) {
      const int j = ranks + t * kTile + l % kTile;
      float h = 0.0f;
      if (there && j < a.r) h = UP ? a.hidden[row * a.hidden_stride + j] : a.back[(int64_t)at * a.r + j];
#pragma unroll
      for (int e = 0; e < 4; ++e)
        sum[t][e] = UP ? product(v[e], h, sum[t][e]) : product(h, there ? v[e] : 0.0f, sum[t][e]);
    }
  }
  if (wave > 0)
#pragma unroll
    for (int t = 0; t < RT; ++t)
#pragma unroll
      for (int e = 0; e < 4; ++e) join[wave - 1][t][e][l] = sum[t][e];
  __syncthreads();
  if (wave > 0) return;
#pragma unroll
  for (int t = 0; t < RT; ++t) {
#pragma unroll
    for (int e = 0; e < 4; ++e)
      for (int w = 0; w < kWaves - 1; ++w) sum[t][e] += join[w][t][e][l];
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if constexpr (UP) {  // outputs first_column + 4 i + e of product e's row i, rank l % 16
        const int j = ranks + t * kTile + l % kTile;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int o = first_column + 4 * (l / kTile * 4 + q) + e;
          const float v[1] = {a.scale * sum[t][e][q]};
          if (j < a.r && o < a.K) store_floats<1>(a.out, key * a.d_up_adapter + o * a.d_up_output + j, w_dtype, 1, v);
        }
      } else {
        const int j = ranks + t * kTile + l / kTile * 4 + q;
        const float v[4] = {sum[t][0][q], sum[t][1][q], sum[t][2][q], sum[t][3][q]};
        if (j < a.r && column < a.C)
          store_floats<4>(a.d_down, key * a.d_down_adapter + j * a.d_down_rank + column, w_dtype, a.C - column, v);
      }
    }
  }
}

// --------------------------------------------------------------------------------------- host
struct Split {
  int windows, slots, parts, part_steps;
};

// Parts of a sum over `steps`, so that about 512 blocks share it, each with a step a wave at least, and
// slots that share a window's segments where there are still few blocks.
Split split_of(int64_t N, int64_t M, int64_t steps) {
  Split s;
  s.windows = (int)((N + kTile - 1) / kTile);
  const int64_t most = steps > kWaves ? (steps + kWaves - 1) / kWaves : 1;
  int64_t parts = 512 / s.windows;
  parts = parts < 1 ? 1 : parts > 32 ? 32 : parts;
  parts = parts < most ? parts : most;
  s.part_steps = (int)((steps + parts - 1) / parts);
  s.parts = s.part_steps ? (int)((steps + s.part_steps - 1) / s.part_steps) : 1;
  int64_t slots = 2048 / ((int64_t)s.windows * s.parts);
  const int64_t segments = M + 1 < kTile ? M + 1 : kTile;
  slots = slots < 1 ? 1 : slots < segments ? slots : segments;
  s.slots = (int)slots;
  return s;
}

int64_t aligned(int64_t bytes) { return (bytes + 15) / 16 * 16; }

int rank_tiles(int r) { return r <= 16 ? 1 : r <= 32 ? 2 : 4; }

hipError_t launch_order(const AdaptArgs& a, hipStream_t s) {
  if (a.N <= kInline) return hipSuccess;
  order_kernel<<<(a.N + kThreads - 1) / kThreads, kThreads, 0, s>>>(a);
  return hipGetLastError();
}

template <int X, int W>
hipError_t launch_down(const AdaptArgs& a, hipStream_t s) {
  const int t = rank_tiles(a.r);
  const dim3 grid(a.windows * a.slots, a.parts, (a.r + t * kTile - 1) / (t * kTile));
  switch (t) {
    case 1: down_kernel<X, W, 1><<<grid, kThreads, 0, s>>>(a); break;
    case 2: down_kernel<X, W, 2><<<grid, kThreads, 0, s>>>(a); break;
    default: down_kernel<X, W, 4><<<grid, kThreads, 0, s>>>(a); break;
  }
  return hipGetLastError();
}

template <int W>
hipError_t launch_adapt(const AdaptArgs& a, int x_dtype, hipStream_t s) {
  hipError_t e = launch_order(a, s);
  if (e != hipSuccess) return e;
  switch (x_dtype) {
    case YTM_DTYPE_BITS: e = launch_down<YTM_DTYPE_BITS, W>(a, s); break;
    case YTM_DTYPE_F16: e = launch_down<YTM_DTYPE_F16, W>(a, s); break;
    case YTM_DTYPE_BF16: e = launch_down<YTM_DTYPE_BF16, W>(a, s); break;
    default: e = launch_down<YTM_DTYPE_F32, W>(a, s); break;
  }
  if (e != hipSuccess) return e;
  const unsigned tiles = a.K > 0 ? (unsigned)((a.K + 4 * kThreads / 4 - 1) / (4 * kThreads / 4)) : 1;
  up_kernel<W><<<dim3(a.windows * a.slots, tiles), kThreads, 0, s>>>(a);
  return hipGetLastError();
}

template <int X, bool UP>
hipError_t launch_outer(const AdaptArgs& a, int w_dtype, hipStream_t s) {
  const int t = rank_tiles(a.r), columns = UP ? a.K : a.C;
  if (columns == 0) return hipSuccess;
  const dim3 grid((columns + 63) / 64, a.M, (a.r + t * kTile - 1) / (t * kTile));
  switch (t) {
    case 1: outer_kernel<X, 1, UP><<<grid, kThreads, 0, s>>>(a, w_dtype); break;
    case 2: outer_kernel<X, 2, UP><<<grid, kThreads, 0, s>>>(a, w_dtype); break;
    default: outer_kernel<X, 4, UP><<<grid, kThreads, 0, s>>>(a, w_dtype); break;
  }
  return hipGetLastError();
}

template <int W>
hipError_t launch_back(const AdaptArgs& a, hipStream_t s) {
  const int t = rank_tiles(a.r);
  const dim3 grid(a.windows * a.slots, a.parts, (a.r + t * kTile - 1) / (t * kTile));
  switch (t) {
    case 1: back_kernel<W, 1><<<grid, kThreads, 0, s>>>(a); break;
    case 2: back_kernel<W, 2><<<grid, kThreads, 0, s>>>(a); break;
    default: back_kernel<W, 4><<<grid, kThreads, 0, s>>>(a); break;
  }
  hipError_t e = hipGetLastError();
  if (e != hipSuccess) return e;
  const int64_t blocks = ((int64_t)a.N * a.r + kThreads - 1) / kThreads;
  back_join_kernel<<<(unsigned)(blocks < 2048 ? blocks : 2048), kThreads, 0, s>>>(a);
  return hipGetLastError();
}

hipError_t launch_gradient(const AdaptArgs& a, int x_dtype, int w_dtype, hipStream_t s) {
  hipError_t e = launch_order(a, s);
  if (e == hipSuccess && a.N > 0) switch (w_dtype) {
      case YTM_DTYPE_F16: e = launch_back<YTM_DTYPE_F16>(a, s); break;
      case YTM_DTYPE_BF16: e = launch_back<YTM_DTYPE_BF16>(a, s); break;
      default: e = launch_back<YTM_DTYPE_F32>(a, s); break;
    }
  if (e == hipSuccess) e = launch_outer<YTM_DTYPE_BITS, true>(a, w_dtype, s);
  if (e != hipSuccess) return e;
  switch (x_dtype) {
    case YTM_DTYPE_BITS: return launch_outer<YTM_DTYPE_BITS, false>(a, w_dtype, s);
    case YTM_DTYPE_F16: return launch_outer<YTM_DTYPE_F16, false>(a, w_dtype, s);
    case YTM_DTYPE_BF16: return launch_outer<YTM_DTYPE_BF16, false>(a, w_dtype, s);
    default: return launch_outer<YTM_DTYPE_F32, false>(a, w_dtype, s);
  }
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
  if ((N > 1 && ((stride != 0 && stride < K) || (x_stride != 0 && x_stride < width))) ||
      (r > 1 && down_rank != 0 && down_rank < C) || (K > 1 && up_output != 0 && up_output < r) ||
      (M > 1 && ((down_adapter != 0 && down_adapter < C) || (up_adapter != 0 && up_adapter < r))))
    return "rows overlap";
  return nullptr;
}

int64_t order_bytes(int64_t N) { return N > kInline ? aligned(8 * N) : 0; }

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
  const ytm::Split s = ytm::split_of(N, M, (C + 31) / 32);
  *bytes = ytm::order_bytes(N) + s.parts * N * r * 4;
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
  const ytm::Split split = ytm::split_of(N, M, (C + 31) / 32);
  ytm::AdaptArgs a{};
  a.scores = scores, a.dtype = dtype, a.stride = stride, a.N = (int)N, a.K = (int)K;
  a.x = x, a.x_stride = x_stride, a.C = (int)C;
  a.down = down, a.down_adapter = down_adapter, a.down_rank = down_rank;
  a.up = up, a.up_adapter = up_adapter, a.up_output = up_output;
  a.M = (int)M, a.r = (int)r, a.which = which, a.scale = scale;
  a.hidden = hidden, a.hidden_stride = hidden_stride;
  a.out = out, a.out_dtype = out_dtype, a.out_stride = out_stride;
  a.windows = split.windows, a.slots = split.slots, a.parts = split.parts, a.part_steps = split.part_steps;
  a.order = (int32_t*)workspace;
  a.part = (float*)((char*)workspace + ytm::order_bytes(N));
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

int ytm_adapt_gradient_workspace(int64_t N, int64_t K, int64_t M, int64_t r, int64_t* bytes) {
  if (!bytes || N < 0 || K < 0 || M < 0 || r < 1 || N > ytm::kDecodeRows || K > ytm::kMaxScores ||
      M > ytm::kMaxAdapters || r > ytm::kMaxRank)
    return fail(YTM_EINVAL, "bad adapt_gradient_workspace arguments");
  *bytes = 0;
  if (N == 0 || M == 0) return YTM_OK;
  const ytm::Split s = ytm::split_of(N, M, (K + 15) / 16);
  *bytes = ytm::order_bytes(N) + ytm::aligned(s.parts * N * r * 4) + N * r * 4;
  return YTM_OK;
}

int ytm_adapt_gradient(const void* grad, int dtype, int64_t stride, int64_t N, int64_t K, const void* x, int x_dtype,
                       int64_t x_stride, int64_t C, const void* up, int64_t up_adapter, int64_t up_output, int w_dtype,
                       int64_t M, int64_t r, const int32_t* which, float scale, const float* hidden,
                       int64_t hidden_stride, void* d_down, int64_t d_down_adapter, int64_t d_down_rank, void* d_up,
                       int64_t d_up_adapter, int64_t d_up_output, void* workspace, int64_t workspace_bytes,
                       void* stream) {
  if (const char* wrong = ytm::wrong_operands(dtype, stride, N, K, x_dtype, x_stride, C, d_down_adapter, d_down_rank,
                                              up_adapter, up_output, w_dtype, M, r, scale))
    return fail(YTM_EINVAL, std::string("adapt_gradient: ") + wrong);
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
  if (int rc = ytm_adapt_gradient_workspace(N, K, M, r, &need)) return rc;
  if (need > 0 && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
    return fail(YTM_EINVAL, "adapt_gradient: the workspace is too small or not at a multiple of 16 bytes");
  const int64_t width = x_dtype == YTM_DTYPE_BITS ? (C + 31) / 32 : C;
  const int size = ytm::size_of(w_dtype);
  const ytm::Rows written[] = {ytm::parts_of(d_down, M, r, C, d_down_adapter, d_down_rank, size),
                               ytm::parts_of(d_up, M, K, r, d_up_adapter, d_up_output, size),
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
    const ytm::Split split = ytm::split_of(N, M, (K + 15) / 16);
    a.windows = split.windows, a.slots = split.slots, a.parts = split.parts, a.part_steps = split.part_steps;
    a.order = (int32_t*)workspace;
    a.part = (float*)((char*)workspace + ytm::order_bytes(N));
    a.back = (float*)((char*)a.part + ytm::aligned(split.parts * N * r * 4));
  }
  a.scores = grad, a.dtype = dtype, a.stride = stride, a.N = (int)N, a.K = (int)K;
  a.x = x, a.x_stride = x_stride, a.C = (int)C;
  a.up = up, a.up_adapter = up_adapter, a.up_output = up_output;
  a.M = (int)M, a.r = (int)r, a.which = which, a.scale = scale;
  a.hidden = const_cast<float*>(hidden), a.hidden_stride = hidden_stride;
  a.out = d_up, a.d_up_adapter = d_up_adapter, a.d_up_output = d_up_output;
  a.d_down = d_down, a.d_down_adapter = d_down_adapter, a.d_down_rank = d_down_rank;
  const hipError_t e = ytm::launch_gradient(a, x_dtype, w_dtype, (hipStream_t)stream);
  if (e != hipSuccess) return fail(YTM_EHIP, std::string("adapt_gradient failed: ") + hipGetErrorString(e));
  return YTM_OK;
}

}  // extern "C"
