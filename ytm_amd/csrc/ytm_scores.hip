// ytm_scores.hip -- from scores to an answer: scores shaped by history, bias and grammar, and the
// choice of one answer a row.  Entry points of include/ytm.h and their gfx950 kernels.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <cfloat>
#include <cmath>

#include "ytm_decode.h"
#include "ytm_internal.h"

namespace ytm {

namespace {

constexpr int kWave = 64;

// ---------------------------------------------------------------------------- adjust_scores
// Of row n and answer v, with c the times v stands in the row's history from its prompt on, and
// `told` whether it stands anywhere in the history:
//   s = score; told: s = s > 0 ? s / repetition : s * repetition
//   s = s - frequency * c - presence * [c > 0] + bias;  not allowed: -inf
// all in float32, rounded once to the output's type.
struct AdjustArgs {
  const void* scores;
  int64_t stride, V;
  const int32_t* tokens;
  int64_t token_stride, T;
  const int32_t *lengths, *prompt;
  const float *repetition, *frequency, *presence;
  const float* bias;
  int64_t bias_stride;
  const uint32_t* allowed;
  int64_t allowed_stride;
  void* out;
  int64_t out_stride;
};

// A block takes kPacks packs of 16 bytes of scores for each of its threads, and counts its answers'
// occurrences in LDS from the whole of the row's history: integers, so their order does not matter.
// What it reads of scores, bias and grammar is on its way before the history is looked at.
//
// Bound by bytes: 256 x 131072 float32 after 4096 answers each, a bias for all and a grammar a row, 62 us,
// 4.4 TB/s; with few rows by the history's pass (64 x 32001 bfloat16, 2048 answers: 7.9 us of which 2.6
// are bytes) and the launch (1 x 10000: 3.8 us).
constexpr int kAdjustThreads = 256;
constexpr uint32_t kTold = 0x80000000u;  // the answer stands in the prompt

template <typename In, typename Out, int kPacks>
__global__ __launch_bounds__(kAdjustThreads) void adjust_kernel(AdjustArgs a) {
  constexpr int n_ = 16 / sizeof(In);  // scores of a pack
  constexpr int kChunk = kPacks * n_ * kAdjustThreads;
  __shared__ uint32_t counts[kChunk];
  const int64_t n = blockIdx.y;
  const int64_t first = blockIdx.x * (int64_t)kChunk;
  const int here = (int)(a.V - first < kChunk ? a.V - first : kChunk);
  const In* in = (const In*)a.scores + n * a.stride + first;
  Out* out = (Out*)a.out + n * a.out_stride + first;
  const float* bias = a.bias ? a.bias + n * a.bias_stride + first : nullptr;
  const uint32_t* allowed = a.allowed ? a.allowed + n * a.allowed_stride + first / 32 : nullptr;
  In score[kPacks][n_];
  float more[kPacks][n_];
  uint32_t may[kPacks];
#pragma unroll
  for (int p = 0; p < kPacks; ++p) {
    const int i = (p * kAdjustThreads + threadIdx.x) * n_;
    if (i + n_ <= here) {
      __builtin_memcpy(score[p], in + i, sizeof score[p]);
      if (bias) __builtin_memcpy(more[p], bias + i, sizeof more[p]);
    } else {
#pragma unroll
      for (int j = 0; j < n_; ++j) {
        score[p][j] = i + j < here ? in[i + j] : In{};
        if (bias) more[p][j] = i + j < here ? bias[i + j] : 0.0f;
      }
    }
    may[p] = allowed && i < here ? allowed[i / 32] : 0xFFFFFFFFu;
  }
  bool said = false;
  float repetition = 1.0f, frequency = 0.0f, presence = 0.0f;
  if (a.tokens) {
    const int64_t length = a.lengths ? (a.lengths[n] < a.T ? a.lengths[n] : a.T) : a.T;
    const int64_t prompt = a.prompt ? a.prompt[n] : 0;
    const int32_t* tokens = a.tokens + n * a.token_stride;
    if (a.repetition) repetition = a.repetition[n];
    if (a.frequency) frequency = a.frequency[n];
    if (a.presence) presence = a.presence[n];
    for (int i = threadIdx.x; i < kChunk / 4; i += kAdjustThreads) ((uint4*)counts)[i] = uint4{0u, 0u, 0u, 0u};
    __syncthreads();
    for (int64_t at = threadIdx.x; at < length; at += 8 * kAdjustThreads) {
      int32_t t[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) {  // past the end the last entry, which is not counted again
        const int64_t k = at + j * kAdjustThreads;
        t[j] = tokens[k < length ? k : length - 1];
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        const int64_t k = at + j * kAdjustThreads, v = t[j] - first;
        if (k < length && v >= 0 && v < here) {
          said = true;
          if (k >= prompt)
            atomicAdd(&counts[v], 1u);
          else
            atomicOr(&counts[v], kTold);
        }
      }
    }
    said = __syncthreads_or(said);
  }
#pragma unroll
  for (int p = 0; p < kPacks; ++p) {
    const int i = (p * kAdjustThreads + threadIdx.x) * n_;
    if (i >= here) break;
    float s[n_];
#pragma unroll
    for (int j = 0; j < n_; ++j) s[j] = to_float(score[p][j]);
    if (said) {
      uint32_t c[n_];
#pragma unroll
      for (int j = 0; j < n_; j += 4) *(uint4*)(c + j) = *(const uint4*)(counts + i + j);
#pragma unroll
      for (int j = 0; j < n_; ++j)
        if (c[j]) {
          s[j] = s[j] > 0.0f ? s[j] / repetition : s[j] * repetition;
          if (c[j] & ~kTold) {
            s[j] -= frequency * (float)(c[j] & ~kTold);
            s[j] -= presence;
          }
        }
    }
    Out r[n_];
#pragma unroll
    for (int j = 0; j < n_; ++j) {
      if (bias) s[j] += more[p][j];
      r[j] = from_float<Out>(may[p] >> ((i + j) % 32) & 1u ? s[j] : -INFINITY);
    }
    if (i + n_ <= here) {
      __builtin_memcpy(out + i, r, sizeof r);
    } else {
#pragma unroll
      for (int j = 0; j < n_; ++j)
        if (i + j < here) out[i + j] = r[j];
    }
  }
}

// Blocks of 4096 answers count a row's history four (two) times less often than blocks of 1024 (2048 of
// 16 bits), which a few short rows take so that more than a few CUs work.
template <typename In, typename Out>
hipError_t launch_adjust(const AdjustArgs& a, int64_t N, hipStream_t s) {
  constexpr int kMany = sizeof(In);  // packs that make 4096 answers
  const auto blocks = [&](int answers) { return (a.V + answers - 1) / answers; };
  if (N * blocks(4096) >= 256)
    adjust_kernel<In, Out, kMany><<<dim3((unsigned)blocks(4096), (unsigned)N), kAdjustThreads, 0, s>>>(a);
  else if (sizeof(In) == 4)
    adjust_kernel<In, Out, 1><<<dim3((unsigned)blocks(1024), (unsigned)N), kAdjustThreads, 0, s>>>(a);
  else
    adjust_kernel<In, Out, 1><<<dim3((unsigned)blocks(2048), (unsigned)N), kAdjustThreads, 0, s>>>(a);
  return hipGetLastError();
}

template <typename In>
hipError_t launch_adjust_out(int out_dtype, const AdjustArgs& a, int64_t N, hipStream_t s) {
  switch (out_dtype) {
    case YTM_DTYPE_F16: return launch_adjust<In, f16>(a, N, s);
    case YTM_DTYPE_BF16: return launch_adjust<In, bf16>(a, N, s);
    default: return launch_adjust<In, float>(a, N, s);
  }
}

// ----------------------------------------------------------------------------------- choose
// With z = score / temperature (NaN counts as -inf, +inf as the largest float), a row's answers
// in the order of z descending, index ascending: what the filters keep is a first part of that
// order, ended by a cut, the last answer kept.  The answer drawn is the largest z + noise of the
// kept ones.  Masses exp(z - max) are whole numbers of 2^-40, so that sums in any order are the
// same; 2^23 of them stay below 2^63.
//
// A block takes a row.  What it needs of the row depends on the filters:
//  - none: one pass, a running maximum and sum of exponentials beside the largest z + noise;
//  - top_k up to kMaxSeek: the k-th largest of the threads' own maxima over a part of the row is
//    no larger than the k-th largest score, so the scores that reach it hold the first k; they
//    go to a list in LDS in the one pass over the row and are sorted there, and everything else
//    (min_p, top_p, the noise) looks at the list alone;
//  - min_p without top_k: the same with the bound that the row's maximum gives, after a pass for it;
//  - otherwise: a histogram of counts and masses over max - z finds the slice of 1/64 in which the
//    cut lies, and that slice's answers, sorted, the cut;
//  - where a list overflows (thousands of equal scores): the cut's key eight bits at a time, from
//    histograms over the whole row.
//
// 256 x 131072 float32 with noise: no filter 67 us (4.0 TB/s), top_k 62 (the noise of what is dropped is
// not read), all three 86 to 98 over several cards, min_p alone 160 and top_p alone 174, where most of a
// row passes the bound and goes through the histogram.  With filters a row's steps (bound, pass, list,
// sort, cuts, draw) follow one another, and most read little: 64 x 32001 bfloat16 takes 21 us, of which
// its 64 KB a row are two.  1 x 10000 without filters 5.7 us, three waits for memory and the block's joins.
// Rows of ties: 64 x 4096 scores of about 60 whole numbers 22 us, 64 x 32001, whose lists overflow, 61.
struct ChooseArgs {
  const void* scores;
  int64_t stride;
  int V;
  const float* temperature;
  const int32_t* top_k;
  const float *top_p, *min_p;
  const float* noise;
  int64_t noise_stride;
  int32_t* tokens;
  float* logprobs;
  int64_t first;     // row of the launch's first block
  int slices, each;  // of a row, and scores in one (0: rows are not sliced)
  struct Slice* found;
};

typedef unsigned long long u64;

constexpr int kChooseThreads = 1024;
constexpr int kChooseWaves = kChooseThreads / kWave;
constexpr int kDigits = 256;
constexpr float kMass = 1099511627776.0f;  // 2^40
template <typename In>
constexpr int kPack = 16 / sizeof(In);  // scores of a 16-byte load
template <typename In>
constexpr int kRound = kPack<In> * kChooseThreads;
constexpr int kList = 4096;
constexpr int kSub = 1024;  // answers of a slice of the histogram
constexpr int kSmall = 256;    // entries that one wave sorts in registers
constexpr int kMaxSeek = 256;  // a quarter of the threads, so that few of the largest share a thread
constexpr int kBins = 2048;
constexpr float kBinsPerUnit = 64.0f;

// Floats as whole numbers of the same order (no -0.0, no NaN).
__device__ __forceinline__ uint32_t key_of(float z) {
  const uint32_t u = __float_as_uint(z);
  return u ^ (u >> 31 ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xFFFFFFFFu));
}
constexpr uint32_t kNone = 0x007FFFFFu;  // key of -inf

// score / t: the product with the reciprocal, corrected by its remainder, which rounds as the division
// does (but for quotients below the normal floats) in half its instructions; t of a row is the
// same for all its scores, so the reciprocal is made once.
__device__ __forceinline__ float scaled(float score, float t) {
  const float r = 1.0f / t, q = score * r;
  const float c = __builtin_fmaf(__builtin_fmaf(-q, t, score), r, q);
  const float z = c == c ? c : q;  // infinities have no remainder
  return (z != z ? -INFINITY : fminf(z, FLT_MAX)) + 0.0f;
}

template <typename In>
struct Row {
  const In* in;
  float t;
  __device__ __forceinline__ float operator()(int i) const { return scaled(to_float(in[i]), t); }
};

// exp(x) for x <= 0 as 2^(x log2 e), the rounding of that product put back: within two units in the last
// place, 0 below 2^-126.
__device__ __forceinline__ float exp_of(float x) {
  const float y = x * 1.44269502f;
  const float rest = __builtin_fmaf(x, 1.92596299e-8f, __builtin_fmaf(x, 1.44269502f, -y));
  const float e = __builtin_amdgcn_exp2f(y);
  return y > -INFINITY ? __builtin_fmaf(e, rest * 0.693147182f, e) : 0.0f;
}

__device__ __forceinline__ u64 mass_of(float z, float best) {
  const float e = exp_of(z - best) * 256.0f;  // the upper 8 of 40 bits, then the lower 32
  const uint32_t high = (uint32_t)e;
  return (u64)high << 32 | (uint32_t)((e - (float)high) * 4294967296.0f);
}

__device__ __forceinline__ u64 drawn_of(float z, int i, const float* noise) {
  float y = noise ? z + noise[i] : z;
  y = y >= -FLT_MAX ? y + 0.0f : -FLT_MAX;
  return (u64)key_of(y) << 32 | (uint32_t)~i;
}

// P elements of a row from element i on, as they are in memory: loads that need no alignment
// and no branch, so that several are on their way at once.  A pack that would pass the row's end
// V is taken from V - P, and the elements before i are not its own.
template <typename In, int P>
struct Pack {
  uint32_t raw[P * sizeof(In) / 4];  // not In[P]: 16-bit elements would take a register each
  __device__ __forceinline__ int load(const In* in, int i, int V) {
    const int at = i + P <= V ? i : V - P;
    if (V >= P) {
      __builtin_memcpy(raw, in + at, sizeof raw);
    } else {
      In e[P];
#pragma unroll
      for (int j = 0; j < P; ++j) e[j] = at + j >= 0 ? in[at + j] : In{};
      __builtin_memcpy(raw, e, sizeof raw);
    }
    return at;
  }
  __device__ __forceinline__ float value(int j) const {
    if constexpr (sizeof(In) == 4)
      return __uint_as_float(raw[j]);
    else
      return to_float(__builtin_bit_cast(In, (uint16_t)(raw[j / 2] >> (16 * (j % 2)))));
  }
  // the elements as floats, `past` for those not the pack's own
  __device__ __forceinline__ void values(int i, int at, float past, float (&v)[P]) const {
#pragma unroll
    for (int j = 0; j < P; ++j) v[j] = value(j);
    if (at != i) {
#pragma unroll
      for (int j = 0; j < P; ++j) v[j] = at + j >= i && at + j >= 0 ? v[j] : past;
    }
  }
};

// f(first index, values) for this thread's packs of elements 0 .. end - 1, -inf where there are
// none; `end` the row's length V or a multiple of kRound.  U packs are loaded before the first is
// looked at.
template <int U, typename In, typename F>
__device__ __forceinline__ void each_pack(const In* in, int V, int end, F f) {
  constexpr int P = kPack<In>;
  for (int first = P * threadIdx.x; first < end; first += U * kRound<In>) {
    Pack<In, P> pack[U];
    int at[U];
#pragma unroll
    for (int u = 0; u < U; ++u) at[u] = pack[u].load(in, first + u * kRound<In>, V);
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float v[P];
      pack[u].values(first + u * kRound<In>, at[u], -INFINITY, v);
      f(at[u], v);
    }
  }
}

template <int P>
__device__ __forceinline__ float most(const float (&v)[P]) {  // NaN only where all are
  float m = v[0];
#pragma unroll
  for (int j = 1; j < P; ++j) m = fmaxf(m, v[j]);
  return m;
}

// ---- sums, maxima and exchanges of a wave in registers (data-parallel moves between lanes)
template <int CTRL, int ROWS>
__device__ __forceinline__ u64 moved(u64 v) {  // 0 where no lane's value moves to
  const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)v, CTRL, ROWS, 0xF, true);
  const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(v >> 32), CTRL, ROWS, 0xF, true);
  return (u64)hi << 32 | lo;
}
// Inclusive scans: 1, 2, 4 and 8 lanes up within rows of 16, then the last of a row to the next
// row and the last of the lower half to the upper.
template <typename Op>
__device__ __forceinline__ u64 wave_scan(u64 v, Op op) {
  v = op(v, moved<0x111, 0xF>(v));
  v = op(v, moved<0x112, 0xF>(v));
  v = op(v, moved<0x114, 0xF>(v));
  v = op(v, moved<0x118, 0xF>(v));
  v = op(v, moved<0x142, 0xA>(v));
  v = op(v, moved<0x143, 0xC>(v));
  return v;
}
struct Add {
  __device__ __forceinline__ u64 operator()(u64 a, u64 b) const { return a + b; }
};
struct Max {
  __device__ __forceinline__ u64 operator()(u64 a, u64 b) const { return a > b ? a : b; }
};
__device__ __forceinline__ u64 lane_value(u64 v, int lane) {  // uniform lane
  const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)v, lane);
  const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(v >> 32), lane);
  return (u64)hi << 32 | lo;
}
template <typename Op>
__device__ __forceinline__ u64 wave_all(u64 v, Op op) {
  return lane_value(wave_scan(v, op), kWave - 1);
}
// The value of lane l ^ M.
template <int M>
__device__ __forceinline__ uint32_t across(uint32_t v) {
  if constexpr (M == 1) return __builtin_amdgcn_mov_dpp((int)v, 0xB1, 0xF, 0xF, true);
  if constexpr (M == 2) return __builtin_amdgcn_mov_dpp((int)v, 0x4E, 0xF, 0xF, true);
  if constexpr (M == 4)  // mirrored in eight, then in four
    return __builtin_amdgcn_mov_dpp(__builtin_amdgcn_mov_dpp((int)v, 0x141, 0xF, 0xF, true), 0x1B, 0xF, 0xF, true);
  if constexpr (M == 8) return __builtin_amdgcn_mov_dpp((int)v, 0x128, 0xF, 0xF, true);
  if constexpr (M == 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(v, v, false, false);
    return threadIdx.x & 16 ? r[0] : r[1];
  }
  const auto r = __builtin_amdgcn_permlane32_swap(v, v, false, false);
  return threadIdx.x & 32 ? r[0] : r[1];
}
template <int M>
__device__ __forceinline__ u64 across64(u64 v) {
  return (u64)across<M>((uint32_t)(v >> 32)) << 32 | across<M>((uint32_t)v);
}

// The last answer kept: all of a larger key are, and of its own key those up to its index.
struct Cut {
  uint32_t key;
  int last;
  __device__ __forceinline__ bool keeps(uint32_t key_, int i) const { return key_ > key || (key_ == key && i <= last); }
};

struct ChooseShared {
  u64 list[kList];
  u64 sub[kSub];
  u64 mass[kBins];
  uint32_t count[kBins];
  u64 part[kChooseWaves];
  double sums[kChooseWaves];
  uint32_t tops[kChooseWaves];
  u64 above, in;
  uint32_t listed;
  int digit;
  int found;
};

// Of the waves' values in sh.part, those of the first `waves` (uniform).
template <typename Op>
__device__ __forceinline__ u64 parts_all(int waves, ChooseShared& sh, Op op) {
  const int l = threadIdx.x % kWave;
  static_assert(kChooseWaves == 16, "a row of lanes");
  u64 v = l < waves ? sh.part[l % kChooseWaves] : 0;
  v = op(v, moved<0x111, 0xF>(v));
  v = op(v, moved<0x112, 0xF>(v));
  v = op(v, moved<0x114, 0xF>(v));
  v = op(v, moved<0x118, 0xF>(v));
  return lane_value(v, kChooseWaves - 1);
}

template <typename Op>
__device__ __forceinline__ u64 block_all(u64 v, ChooseShared& sh, Op op) {
  v = wave_scan(v, op);
  __syncthreads();
  if (threadIdx.x % kWave == kWave - 1) sh.part[threadIdx.x / kWave] = v;
  __syncthreads();
  return parts_all(kChooseWaves, sh, op);
}
__device__ __forceinline__ u64 block_max(u64 v, ChooseShared& sh) { return block_all(v, sh, Max()); }
__device__ __forceinline__ u64 block_sum(u64 v, ChooseShared& sh) { return block_all(v, sh, Add()); }

// Sum of the v of this thread and those before it.
__device__ __forceinline__ u64 block_upto(u64 v, ChooseShared& sh) {
  v = wave_scan(v, Add());
  __syncthreads();
  if (threadIdx.x % kWave == kWave - 1) sh.part[threadIdx.x / kWave] = v;
  __syncthreads();
  return v + parts_all(__builtin_amdgcn_readfirstlane(threadIdx.x / kWave), sh, Add());
}

// The first wave finds the highest bin at which the bins from the top on (bin 0 first where
// RISING), after `before`, reach `target`; sh.digit is it or -1, sh.above what comes before it,
// sh.in what it holds.
template <int BINS, bool RISING, typename T>
__device__ __forceinline__ void find_bin(const T* bins, u64 before, u64 target, ChooseShared& sh) {
  __syncthreads();
  if (threadIdx.x < kWave) {
    constexpr int kEach = BINS / kWave;
    const auto at = [&](int j) { return (u64)bins[RISING ? j : BINS - 1 - j]; };
    u64 own = 0;
#pragma unroll 4
    for (int j = 0; j < kEach; ++j) own += at(kEach * threadIdx.x + j);
    const u64 upto = wave_scan(own, Add());
    const u64 reached = __ballot(before + upto >= target);
    if (threadIdx.x == 0) sh.digit = -1;
    if (reached && (int)threadIdx.x == __ffsll(reached) - 1) {
      u64 sum = before + upto - own;
      int j = kEach * threadIdx.x;
      while (sum + at(j) < target) sum += at(j++);
      sh.digit = RISING ? j : BINS - 1 - j;
      sh.above = sum;
      sh.in = at(j);
    }
  }
  __syncthreads();
}

// Index of the r-th (from 1) answer of key `key`, in index order.
template <typename In>
__device__ __forceinline__ int tie_index(const Row<In>& row, int V, uint32_t key, int r, ChooseShared& sh) {
  int seen = 0;
  if (threadIdx.x == 0) sh.found = V - 1;
  for (int first = 0; first < V; first += kChooseThreads) {
    const int i = first + threadIdx.x;
    const bool tie = i < V && key_of(row(i)) == key;
    const u64 mine = __ballot(tie);
    __syncthreads();
    if (threadIdx.x % kWave == 0) sh.part[threadIdx.x / kWave] = __popcll(mine);
    __syncthreads();
    int before = seen;
    for (int w = 0; w < kChooseWaves; ++w) {
      if (w < (int)threadIdx.x / kWave) before += (int)sh.part[w];
      seen += (int)sh.part[w];
    }
    before += __popcll(mine & ((1ull << (threadIdx.x % kWave)) - 1));
    if (tie && before + 1 == r) sh.found = i;
    if (seen >= r) break;
  }
  __syncthreads();
  return sh.found;
}

// Moves the cut up to the first answer at which the answers kept so far, counted (MASS false) or
// weighed, reach `target`; leaves it where they never do.  The key is found eight bits at a time
// from a histogram.
template <bool MASS, typename In>
__device__ __forceinline__ void raise_cut(const Row<In>& row, int V, float best, u64 target, Cut& cut, ChooseShared& sh) {
  uint32_t prefix = 0u, mask = 0u;
  u64 above = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < kDigits; i += kChooseThreads) sh.mass[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < V; i += kChooseThreads) {
      const float z = row(i);
      const uint32_t key = key_of(z);
      if (cut.keeps(key, i) && (key & mask) == prefix)
        atomicAdd(&sh.mass[key >> shift & 255u], MASS ? mass_of(z, best) : 1ull);
    }
    find_bin<kDigits, false>(sh.mass, above, target, sh);
    if (sh.digit < 0) return;
    above = sh.above;
    prefix |= (uint32_t)sh.digit << shift;
    mask |= 255u << shift;
  }
  // `above` comes before the answers of key `prefix`, which have `in` together
  const u64 need = target - above;
  const u64 each = MASS ? mass_of(value_of(prefix), best) : 1ull;
  const u64 in = sh.in;
  int last = prefix == cut.key ? cut.last : V - 1;
  if (each && need + each <= in) {  // some of them are left out
    const u64 r = (need + each - 1) / each;
    last = tie_index(row, V, prefix, (int)(r < 1 ? 1 : r), sh);
  }
  cut.key = prefix;
  cut.last = last;
  __syncthreads();
}

// target of a cut by mass: the first answer at which masses add up to it is the last kept.
__device__ __forceinline__ u64 share_of(float p, u64 total) {
  const double target = ceil((double)p * (double)total);
  return target > 1.0 ? (u64)target : 1ull;
}

__device__ __forceinline__ void answer(const ChooseArgs& a, int64_t n, u64 drawn, float z, float best, u64 mass) {
  if (threadIdx.x == 0) {
    a.tokens[n] = (int)~(uint32_t)drawn;
    a.logprobs[n] = (z - best) - logf((float)mass * (1.0f / kMass));
  }
}
__device__ __forceinline__ void no_answer(const ChooseArgs& a, int64_t n) {
  if (threadIdx.x == 0) {
    a.tokens[n] = -1;
    a.logprobs[n] = -INFINITY;
  }
}

// Sorts list[0 .. size) (size a power of two from 128 on) descending.  A wave's pairs at
// distances up to 64 lie in 128 places of its own, so the block waits only at longer ones.
__device__ __forceinline__ void sort_list(u64* list, int size) {
  for (int k = 2; k <= size; k <<= 1)
    for (int j = k >> 1; j; j >>= 1) {
      if (j >= kWave || j == k >> 1) __syncthreads();
      for (int p = threadIdx.x; p < size / 2; p += kChooseThreads) {
        const int i = 2 * p - (p & (j - 1));
        const u64 x = list[i], y = list[i + j];
        if ((x < y) == ((i & k) == 0)) {
          list[i] = y;
          list[i + j] = x;
        }
      }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
  __syncthreads();
}

// Sorts a list's `count` entries (descending; zeros follow them).
__device__ __forceinline__ void order_list(u64* list, int count) {
  int size = 2 * kWave;
  while (size < count) size <<= 1;
  __syncthreads();
  for (int i = count + threadIdx.x; i < size; i += kChooseThreads) list[i] = 0;
  sort_list(list, size);
}

// One step of a bitonic sort (descending) of 4 x 64 values, value 4 l + r being register r of lane l:
// pairs at distance J within runs of K that go down and up in turn.
template <int K, int J>
__device__ __forceinline__ void sort_step(u64 (&v)[4], int l) {
  if constexpr (J >= 4) {
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      const u64 o = across64<J / 4>(v[r]);
      const bool larger = ((4 * l & J) == 0) == ((4 * l & K) == 0);  // this place takes the larger
      v[r] = (o > v[r]) == larger ? o : v[r];
    }
  } else {
#pragma unroll
    for (int r = 0; r < 4; ++r)
      if ((r & J) == 0) {
        const bool down = ((4 * l + r) & K) == 0;
        const u64 x = v[r], y = v[r | J];
        const bool swap = (x < y) == down;
        v[r] = swap ? y : x;
        v[r | J] = swap ? x : y;
      }
  }
  if constexpr (J > 1) sort_step<K, J / 2>(v, l);
}
template <int K>
__device__ __forceinline__ void sort_runs(u64 (&v)[4], int l) {
  if constexpr (K > 2) sort_runs<K / 2>(v, l);
  sort_step<K, K / 2>(v, l);
}

// The largest z of a part of a row, the sum of exp(z - it), the largest z + noise with its index
// (0: no z above -inf).
struct All {
  float best;
  double sum;
  u64 drawn;
};

// Every answer may be drawn: what a block finds of answers begin .. end - 1, sum in thread 0 alone.
// Sums are kept in double: a float's would lose what many small terms add up to.
template <typename In>
__device__ __forceinline__ All all_of(const ChooseArgs& a, int64_t n, const Row<In>& row, int begin, int end,
                                      ChooseShared& sh) {
  const float* noise = a.noise ? a.noise + n * a.noise_stride + begin : nullptr;
  const In* in = row.in + begin;
  const int V = end - begin;
  float top = -INFINITY;
  double sum = 0.0;
  u64 drawn = 0;
  constexpr int P = kPack<In>;
  for (int first = P * threadIdx.x; first < V; first += 2 * kRound<In>) {
    Pack<In, P> score[2];
    Pack<float, P> more[2];
    int at[2];
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      at[u] = score[u].load(in, first + u * kRound<In>, V);
      if (noise) more[u].load(noise, first + u * kRound<In>, V);
    }
#pragma unroll
    for (int u = 0; u < 2; ++u) {
      float z[P], g[P];
      score[u].values(first + u * kRound<In>, at[u], -INFINITY, z);
      if (noise) more[u].values(first + u * kRound<In>, at[u], 0.0f, g);
#pragma unroll
      for (int j = 0; j < P; ++j) z[j] = scaled(z[j], row.t);
      const float here = most(z);
      if (here > top) {
        sum *= (double)expf(top - here);  // 0 the first time
        top = here;
      }
      if (top == -INFINITY) continue;
      float part = 0.0f;
#pragma unroll
      for (int j = 0; j < P; ++j) {
        part += exp_of(z[j] - top);
        float y = noise ? z[j] + g[j] : z[j];
        y = y >= -FLT_MAX ? y + 0.0f : -FLT_MAX;
        const u64 d = z[j] > -INFINITY ? (u64)key_of(y) << 32 | (uint32_t)~(begin + at[u] + j) : 0;
        drawn = d > drawn ? d : drawn;
      }
      sum += (double)part;
    }
  }
  // the largest z of all and the largest z + noise, then the sums against it, in lanes' and waves' order
  drawn = wave_scan(drawn, Max());
  const u64 high = wave_scan(key_of(top), Max());
  if (threadIdx.x % kWave == kWave - 1) {
    sh.part[threadIdx.x / kWave] = drawn;
    sh.tops[threadIdx.x / kWave] = (uint32_t)high;
  }
  __syncthreads();
  drawn = parts_all(kChooseWaves, sh, Max());
  const int l = threadIdx.x % kWave;
  const float best = value_of((uint32_t)wave_all(sh.tops[l % kChooseWaves], Max()));
  sum *= top > -INFINITY ? (double)expf(top - best) : 0.0;
  for (int d = 1; d < kWave; d <<= 1) sum += __shfl_xor(sum, d);
  if (l == 0) sh.sums[threadIdx.x / kWave] = sum;
  __syncthreads();
  if (threadIdx.x == 0) {
    sum = 0.0;
    for (int w = 0; w < kChooseWaves; ++w) sum += sh.sums[w];
  }
  return All{best, sum, drawn};
}

// Thread 0 writes the answer.
template <typename In>
__device__ __forceinline__ void from_all(const ChooseArgs& a, int64_t n, const Row<In>& row, const All& all) {
  if (all.drawn == 0) return no_answer(a, n);
  if (threadIdx.x == 0) {
    const int i = (int)~(uint32_t)all.drawn;
    a.tokens[n] = i;
    a.logprobs[n] = (row(i) - all.best) - logf((float)all.sum);
  }
}

// The answer from a histogram over max - z: the slice in which a cut lies, and that slice's answers,
// sorted, the cut.  each(least, few, f) calls f(z, index) for this thread's answers, those of a z below
// `least` not for certain; `few`: not many are above it.  False, with nothing written, where a slice
// holds more than kSub.
template <typename In, typename Each>
__device__ __forceinline__ bool from_bins(const ChooseArgs& a, int64_t n, const Row<In>& row, Each each, float best,
                                          int k, float p, Cut cut, ChooseShared& sh) {
  const auto bin_of = [&](float z) { return (int)fminf((best - z) * kBinsPerUnit, (float)(kBins - 1)); };
  for (int i = threadIdx.x; i < kBins; i += kChooseThreads) {
    sh.mass[i] = 0;
    sh.count[i] = 0;
  }
  __syncthreads();
  const bool counted = k > 0;
  const float lightest = best - 28.0f;  // from here on masses are below 2^-40, none
  uint32_t rest = 0;                    // answers of the last slice, which may be nearly all
  const float floor = value_of(cut.key);
  const bool bounded = cut.key > kNone + 1u;
  each(counted ? floor : fmaxf(floor, lightest), bounded, [&](float z, int) {
    if (key_of(z) < cut.key) return;
    const int b = bin_of(z);
    const u64 m = mass_of(z, best);
    if (m) atomicAdd(&sh.mass[b], m);
    if (counted) {
      if (b == kBins - 1)
        ++rest;
      else
        atomicAdd(&sh.count[b], 1u);
    }
  });
  if (counted && rest) atomicAdd(&sh.count[kBins - 1], rest);
  const float* noise = a.noise ? a.noise + n * a.noise_stride : nullptr;
  u64 total = 0;  // of what top_k leaves
  u64 drawn = 0, sum = 0;
  int listed = -1, count = 0;  // the slice in the list
  // puts the answers of slice b into sh.sub in their order, and the largest z + noise of those before it
  // into `drawn`; whether they fit
  const auto gather = [&](int b) {
    __syncthreads();
    if (threadIdx.x == 0) sh.listed = 0;
    __syncthreads();
    drawn = 0;
    each(b < kBins - 1 ? fmaxf(floor, best - (float)(b + 2) / kBinsPerUnit) : floor, b < kBins - 1 || bounded,
         [&](float z, int i) {
      if (key_of(z) < cut.key) return;
      const int at = bin_of(z);
      if (at == b) {
        const uint32_t place = atomicAdd(&sh.listed, 1u);
        if (place < kSub) sh.sub[place] = (u64)key_of(z) << 32 | (uint32_t)~i;
      }
      if (at < b) {
        const u64 d = drawn_of(z, i, noise);
        drawn = d > drawn ? d : drawn;
      }
    });
    __syncthreads();
    listed = b;
    count = (int)sh.listed;
    if (count > kSub) return false;
    if (count <= kSmall) {  // one wave, in registers
      if (threadIdx.x < kWave) {
        u64 v[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) v[r] = r * kWave + (int)threadIdx.x < count ? sh.sub[r * kWave + threadIdx.x] : 0;
        sort_runs<kSmall>(v, threadIdx.x);
#pragma unroll
        for (int r = 0; r < 4; ++r) sh.sub[4 * threadIdx.x + r] = v[r];
      }
      __syncthreads();
    } else {
      order_list(sh.sub, count);
    }
    return true;
  };
  // the number of the first `among` of them whose masses reach `target` (all where they never do), and their sum
  const auto upto = [&](int among, u64 target) {
    const int i = threadIdx.x;
    static_assert(kSub <= kChooseThreads, "");
    const u64 mass = i < among ? mass_of(value_of((uint32_t)(sh.sub[i] >> 32)), best) : 0;
    const u64 up = block_upto(mass, sh);
    const bool keep = i < among && up - mass < target;
    sum = block_sum(keep ? mass : 0, sh);
    return (int)block_sum(keep ? 1 : 0, sh);
  };
  int kept = 0;  // of the list
  u64 above = 0;
  int end = kBins;  // slices from here on are left out
  sh.digit = -1;
  if (counted) find_bin<kBins, true>(sh.count, 0, (u64)k, sh);
  __syncthreads();
  if (sh.digit >= 0) {
    end = sh.digit;
    const int r = k - (int)sh.above;
    if (!gather(end)) return false;
    u64 m = 0;
    for (int i = threadIdx.x; i < end; i += kChooseThreads) m += sh.mass[i];
    above = block_sum(m, sh);
    kept = upto(r, ~0ull);
    total = above + sum;
  } else {
    u64 m = 0;
    for (int i = threadIdx.x; i < kBins; i += kChooseThreads) m += sh.mass[i];
    total = block_sum(m, sh);
  }
  if (p < 1.0f) {
    const u64 target = share_of(p, total);
    find_bin<kBins, true>(sh.mass, 0, target, sh);
    const int b = sh.digit;
    if (b >= 0 && b < end) {  // in a slice that top_k leaves whole
      above = sh.above;
      if (!gather(b)) return false;
      kept = upto(count, target - above);
    } else if (listed >= 0) {
      kept = upto(kept, target - above);
    }
  }
  if (listed < 0) {  // nothing is cut off
    gather(kBins);
    above = total;
    sum = 0;
  }
  if ((int)threadIdx.x < kept) {
    const u64 e = sh.sub[threadIdx.x];
    const u64 d = drawn_of(value_of((uint32_t)(e >> 32)), (int)~(uint32_t)e, noise);
    drawn = d > drawn ? d : drawn;
  }
  drawn = block_max(drawn, sh);
  answer(a, n, drawn, row((int)~(uint32_t)drawn), best, above + sum);
  return true;
}

// A row's filters, as every path below takes them: a bound that is not a number is none.
struct Filters {
  float t, p, min;
  int k;
  bool bounded, seek;  // min_p holds; top_k is sought by a bound

  __device__ __forceinline__ Filters(const ChooseArgs& a, int64_t n) {
    t = a.temperature ? a.temperature[n] : 1.0f;
    k = a.top_k ? a.top_k[n] : 0;
    if (t <= 0.0f) {
      t = 1.0f;
      k = 1;
    }
    t = fmaxf(t, FLT_MIN);  // a smaller one has no reciprocal; a NaN too becomes it
    min = a.min_p ? a.min_p[n] : 0.0f;
    if (min > 1.0f) {  // not even the first answer reaches it, which alone is kept all the same
      min = 0.0f;
      k = 1;
    }
    if (k >= a.V) k = 0;
    p = a.top_p && a.top_p[n] < 1.0f ? a.top_p[n] : 1.0f;
    bounded = min > 0.0f;
    seek = k > 0 && k <= kMaxSeek;
  }
  __device__ __forceinline__ bool none() const { return k <= 0 && p >= 1.0f && !bounded; }
};

// The answer from a list (of key of score, ~index) that holds every answer the filters may keep:
// from a histogram over it, or from the whole list sorted where a slice holds too many.
template <typename In>
__device__ __forceinline__ void from_list(const ChooseArgs& a, int64_t n, const Row<In>& row, int count,
                                          const Filters& filters, ChooseShared& sh) {
  const int k = filters.k;
  const float p = filters.p;
  u64 first = 0;
  for (int i = threadIdx.x; i < count; i += kChooseThreads) {
    const u64 e = sh.list[i];
    const u64 z = (u64)key_of(scaled(value_of((uint32_t)(e >> 32)), row.t)) << 32 | (uint32_t)e;
    sh.list[i] = z;
    first = z > first ? z : first;
  }
  const uint32_t top = (uint32_t)(block_max(first, sh) >> 32);
  if (top <= kNone) return no_answer(a, n);
  const float best = value_of(top);
  uint32_t least = kNone + 1u;
  if (filters.bounded) {
    const uint32_t key = key_of(best + logf(filters.min) + 0.0f);
    if (key > least) least = key;
  }
  const auto each = [&](float, bool, auto f) {
    for (int i = threadIdx.x; i < count; i += kChooseThreads)
      f(value_of((uint32_t)(sh.list[i] >> 32)), (int)~(uint32_t)sh.list[i]);
  };
  if (from_bins(a, n, row, each, best, k, p, Cut{least, a.V - 1}, sh)) return;
  order_list(sh.list, count);
  if (k > 0 && k < count) count = k;
  const float* noise = a.noise ? a.noise + n * a.noise_stride : nullptr;
  u64 total = 0, drawn = 0, sum = 0;
  for (int i = threadIdx.x; i < count; i += kChooseThreads) {
    const uint32_t key = (uint32_t)(sh.list[i] >> 32);
    if (key >= least) total += mass_of(value_of(key), best);
  }
  total = block_sum(total, sh);
  const u64 target = p >= 1.0f ? ~0ull : share_of(p, total);
  u64 before = 0;
  for (int first = 0; first < count; first += kChooseThreads) {
    const int i = first + threadIdx.x;
    const u64 e = i < count ? sh.list[i] : 0;
    const uint32_t key = (uint32_t)(e >> 32);
    const u64 mass = key >= least ? mass_of(value_of(key), best) : 0;
    const u64 upto = before + block_upto(mass, sh);
    if (key >= least && (upto - mass < target || i == 0)) {
      sum += mass;
      const u64 d = drawn_of(value_of(key), (int)~(uint32_t)e, noise);
      drawn = d > drawn ? d : drawn;
    }
    if (first + kChooseThreads < count) {  // what this round holds
      __syncthreads();
      if (threadIdx.x == kChooseThreads - 1) sh.above = upto;
      __syncthreads();
      before = sh.above;
    }
  }
  sum = block_sum(sum, sh);
  drawn = block_max(drawn, sh);
  const int at = (int)~(uint32_t)drawn;
  // z of the answer drawn: its noise taken off again would not be exact
  for (int i = threadIdx.x; i < count; i += kChooseThreads)
    if ((uint32_t)~sh.list[i] == (uint32_t)at) sh.tops[0] = (uint32_t)(sh.list[i] >> 32);
  __syncthreads();
  answer(a, n, drawn, value_of(sh.tops[0]), best, sum);
}

// Passes over the whole row for each step: right for every row, and what is left for lists
// that overflow.
template <typename In>
__device__ __forceinline__ void from_row(const ChooseArgs& a, int64_t n, const Row<In>& row, float best, int k, float p, Cut cut,
                         ChooseShared& sh) {
  const int V = a.V;
  if (k > 0 && k < V) raise_cut<false>(row, V, best, (u64)k, cut, sh);
  if (p < 1.0f) {
    u64 m = 0;
    for (int i = threadIdx.x; i < V; i += kChooseThreads) {
      const float z = row(i);
      if (cut.keeps(key_of(z), i)) m += mass_of(z, best);
    }
    raise_cut<true>(row, V, best, share_of(p, block_sum(m, sh)), cut, sh);
  }
  const float* noise = a.noise ? a.noise + n * a.noise_stride : nullptr;
  u64 m = 0, drawn = 0;
  for (int i = threadIdx.x; i < V; i += kChooseThreads) {
    const float z = row(i);
    if (!cut.keeps(key_of(z), i)) continue;
    m += mass_of(z, best);
    const u64 d = drawn_of(z, i, noise);
    drawn = d > drawn ? d : drawn;
  }
  m = block_sum(m, sh);
  drawn = block_max(drawn, sh);
  answer(a, n, drawn, row((int)~(uint32_t)drawn), best, m);
}

// A score from which on z may equal that of one at `score`: two scores' quotients by t are
// equal only within a rounding of them, below the smallest normal float or at the largest.
__device__ __forceinline__ float with_equals(float score, float t) {
  score = fminf(score, FLT_MAX);
  const float lower = score - fabsf(score) * 0x1p-22f - t * 0x1p-124f;
  return t < 1.0f ? fminf(lower, FLT_MAX * t * (1.0f - 0x1p-20f)) : lower;
}

// Marks, a bit an element, of this thread's packs of kWords x kPacks rounds from `start` on: those of
// `least` or more.  No branch on what they are; the next four packs are on their way while four are
// looked at.
template <typename In>
struct Marks {
  static constexpr int P = kPack<In>, kWords = 4, kPacks = 32 / P;  // packs to a word of marks
  static constexpr int kSpan = kWords * kPacks * kRound<In>;
  uint32_t word[kWords];

  __device__ __forceinline__ void make(const In* in, int V, int start, float least, float& top) {
    constexpr int kAtOnce = sizeof(In) == 4 ? 4 : 2, kSteps = kWords * kPacks / kAtOnce;
    Pack<In, P> pack[2][kAtOnce];
    int at[2][kAtOnce];
    const auto load = [&](int step) {
#pragma unroll
      for (int u = 0; u < kAtOnce; ++u)
        at[step % 2][u] = pack[step % 2][u].load(in, index(start, step * kAtOnce + u), V);
    };
    load(0);
#pragma unroll
    for (int w = 0; w < kWords; ++w) word[w] = 0;
#pragma unroll
    for (int step = 0; step < kSteps; ++step) {
      if (start + step * kAtOnce * kRound<In> < V) {
        if (step + 1 < kSteps) load(step + 1);
        uint32_t m = 0;
#pragma unroll
        for (int u = 0; u < kAtOnce; ++u) {
          float v[P];
          pack[step % 2][u].values(index(start, step * kAtOnce + u), at[step % 2][u], -INFINITY, v);
#pragma unroll
          for (int j = 0; j < P; ++j) m = m * 2 + (v[j] >= least ? 1u : 0u);
          top = fmaxf(top, most(v));
        }
        word[step * kAtOnce / kPacks] |= m << (32 - P * kAtOnce * (step % (kPacks / kAtOnce) + 1));
      }
    }
  }
  __device__ __forceinline__ static int index(int start, int pack) {
    return start + pack * kRound<In> + P * (int)threadIdx.x;
  }
  // f(index) of the marked elements
  template <typename F>
  __device__ __forceinline__ void each(int V, int start, F f) const {
#pragma unroll
    for (int w = 0; w < kWords; ++w)
      for (uint32_t m = word[w]; m;) {
        const int b = __clz(m);  // pack b / P of the word, its element b % P
        m &= ~(0x80000000u >> b);
        const int i = index(start, w * kPacks + b / P);
        f((i + P <= V ? i : V - P) + b % P);
      }
  }
};

// Lists the row's scores from `least` on (those above -inf) in an order of threads; whether they
// fit.  They are marked first and read again once each thread knows its place in the list: few reach
// `least`.  `top` is raised to the largest score this thread has seen.
template <typename In>
__device__ __forceinline__ bool list_from(const In* in, int V, float least, float& top, ChooseShared& sh) {
  uint32_t listed = 0;
  bool fits = true;
  least = fmaxf(least, -FLT_MAX);  // nothing where it is NaN: the largest is what is left of both
  for (int start = 0; start < V; start += Marks<In>::kSpan) {
    Marks<In> marks;
    marks.make(in, V, start, least, top);
    uint32_t own = 0;
#pragma unroll
    for (int w = 0; w < Marks<In>::kWords; ++w) own += __popc(marks.word[w]);
    const uint32_t upto = (uint32_t)block_upto(own, sh);
    uint32_t place = listed + upto - own;
    __syncthreads();
    if (threadIdx.x == kChooseThreads - 1) sh.listed = upto;
    __syncthreads();
    listed += sh.listed;
    if (listed > kList) {  // what is left is looked at for its largest score alone
      fits = false;
      continue;
    }
    marks.each(V, start, [&](int e) {
      sh.list[place++] = (u64)key_of(to_float(in[e]) + 0.0f) << 32 | (uint32_t)~e;
    });
  }
  __syncthreads();
  if (threadIdx.x == 0) sh.listed = listed;
  __syncthreads();
  return fits;
}

// The largest of this thread's packs over the row's first `rounds` rounds.
template <typename In>
__device__ __forceinline__ float own_most(const In* in, int V, int rounds) {
  float top = -INFINITY;
  each_pack<32 / kPack<In>>(in, V, V < (int64_t)rounds * kRound<In> ? V : rounds * kRound<In>,
                            [&](int, auto& v) { top = fmaxf(top, most(v)); });
  return top;
}

// A key no larger than the k-th largest of the threads' keys: its upper 16 bits.
__device__ __forceinline__ uint32_t kth_of(uint32_t own, int k, ChooseShared& sh) {
  uint32_t prefix = 0u;
  u64 above = 0;
  for (int shift = 24; shift >= 16; shift -= 8) {
    for (int i = threadIdx.x; i < kDigits; i += kChooseThreads) sh.count[i] = 0;
    __syncthreads();
    if (shift == 24 || own >> 24 == prefix >> 24) atomicAdd(&sh.count[own >> shift & 255u], 1u);
    find_bin<kDigits, false>(sh.count, above, (u64)k, sh);
    prefix |= (uint32_t)sh.digit << shift;
    above = sh.above;
    __syncthreads();
  }
  return prefix;
}

// Leaves out of a list what the same bound over the list itself leaves out; the new length.
__device__ __forceinline__ int shorten_list(int count, float t, int k, ChooseShared& sh) {
  constexpr int kEach = kList / kChooseThreads;
  u64 own[kEach];
  u64 most_ = 0;
#pragma unroll
  for (int j = 0; j < kEach; ++j) {
    const int i = j * kChooseThreads + threadIdx.x;
    own[j] = i < count ? sh.list[i] : 0;
    most_ = own[j] > most_ ? own[j] : most_;
  }
  const uint32_t bound = kth_of((uint32_t)(most_ >> 32), k, sh);
  const uint32_t least = bound > kNone ? key_of(with_equals(value_of(bound), t) + 0.0f) : 0u;
  uint32_t keep = 0;
#pragma unroll
  for (int j = 0; j < kEach; ++j) keep += own[j] && (uint32_t)(own[j] >> 32) >= least;
  const uint32_t upto = (uint32_t)block_upto(keep, sh);  // the list has been read by then
  uint32_t place = upto - keep;
#pragma unroll
  for (int j = 0; j < kEach; ++j)
    if (own[j] && (uint32_t)(own[j] >> 32) >= least) sh.list[place++] = own[j];
  if (threadIdx.x == kChooseThreads - 1) sh.listed = upto;
  __syncthreads();
  return (int)sh.listed;
}

// from_list for up to kSmall entries: one wave, in registers, without a barrier.
__device__ __forceinline__ void from_small(const ChooseArgs& a, int64_t n, int count, const Filters& filters,
                                           ChooseShared& sh) {
  if (threadIdx.x >= kWave) return;
  const float t = filters.t, p = filters.p;
  const int k = filters.k;
  const int l = threadIdx.x;
  u64 v[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const int i = r * kWave + l;
    v[r] = i < count ? sh.list[i] : 0;
    if (v[r]) v[r] = (u64)key_of(scaled(value_of((uint32_t)(v[r] >> 32)), t)) << 32 | (uint32_t)v[r];
  }
  sort_runs<kSmall>(v, l);
  const uint32_t top = (uint32_t)(lane_value(v[0], 0) >> 32);
  if (top <= kNone) return no_answer(a, n);
  const float best = value_of(top);
  uint32_t least = kNone + 1u;
  if (filters.bounded) {
    const uint32_t key = key_of(best + logf(filters.min) + 0.0f);
    if (key > least) least = key;
  }
  const float* noise = a.noise ? a.noise + n * a.noise_stride : nullptr;
  u64 mass[4], own = 0;
  bool in[4];
  float z[4], g[4];
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    in[r] = (uint32_t)(v[r] >> 32) >= least && (k <= 0 || 4 * l + r < k);
    z[r] = value_of((uint32_t)(v[r] >> 32));
    g[r] = noise && in[r] ? noise[(int)~(uint32_t)v[r]] : 0.0f;
    mass[r] = in[r] ? mass_of(z[r], best) : 0;
    own += mass[r];
  }
  const u64 upto = wave_scan(own, Add());
  const u64 target = p >= 1.0f ? ~0ull : share_of(p, lane_value(upto, kWave - 1));
  u64 before = upto - own, sum = 0, drawn = 0;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    if (in[r] && (before < target || (l == 0 && r == 0))) {
      sum += mass[r];
      float y = noise ? z[r] + g[r] : z[r];
      y = y >= -FLT_MAX ? y + 0.0f : -FLT_MAX;
      const u64 d = (u64)key_of(y) << 32 | (uint32_t)v[r];
      drawn = d > drawn ? d : drawn;
    }
    before += mass[r];
  }
  sum = wave_all(sum, Add());
  drawn = wave_all(drawn, Max());
#pragma unroll
  for (int r = 0; r < 4; ++r)  // the lane whose answer it is
    if (in[r] && (uint32_t)v[r] == (uint32_t)drawn) {
      a.tokens[n] = (int)~(uint32_t)drawn;
      a.logprobs[n] = (z[r] - best) - logf((float)sum * (1.0f / kMass));
    }
}

// Lists what may be kept of `V` scores (a row, or a slice, whose k-th largest and largest are no larger
// than the row's), with a bound from their first `rounds` rounds; whether it fits.
template <typename In>
__device__ __forceinline__ bool list_kept(const In* in, int V, int rounds, const Filters& f, float& own,
                                          ChooseShared& sh) {
  own = own_most(in, V, rounds);
  float least;
  if (f.seek) {
    const uint32_t bound = kth_of(key_of(own + 0.0f), f.k, sh);
    least = bound > kNone ? with_equals(value_of(bound), f.t) : -INFINITY;
  } else {
    const float z = scaled(value_of((uint32_t)block_max(key_of(own + 0.0f), sh)), f.t);
    least = with_equals((z + logf(f.min)) * f.t, f.t);
  }
  return list_from(in, V, least, own, sh);
}

// A CU reads about 40 GB/s here whatever is on its way, so a long row alone takes 13 us per 512 KB:
// where rows are few, slices of them go to blocks of their own, which leave for the row's block
// what they list (`count` entries; more than kSliceList, or a row whose filters no list serves: -1)
// or, without filters, what all_of finds.
constexpr int kSliceList = 512;
struct Slice {
  int count;
  float best;
  double sum;
  u64 drawn;
  u64 list[kSliceList];
};

template <typename In>
__global__ __launch_bounds__(kChooseThreads) __attribute__((amdgpu_waves_per_eu(4, 4))) void slice_kernel(
    ChooseArgs a) {
  __shared__ ChooseShared sh;
  const int64_t n = blockIdx.y;
  const int begin = blockIdx.x * a.each, end = begin + a.each < a.V ? begin + a.each : a.V;
  const Filters f(a, n);
  const Row<In> row{(const In*)a.scores + n * a.stride, f.t};
  Slice& to = a.found[n * a.slices + blockIdx.x];
  if (f.none()) {
    const All all = all_of(a, n, row, begin, end, sh);
    if (threadIdx.x == 0) {
      to.best = all.best;
      to.sum = all.sum;
      to.drawn = all.drawn;
    }
    return;
  }
  int count = -1;
  if (f.seek || f.bounded) {
    float own;
    const int rounds = (end - begin + kRound<In> - 1) / kRound<In>;
    if (list_kept(row.in + begin, end - begin, rounds, f, own, sh) && sh.listed <= kSliceList) {
      count = (int)sh.listed;
      for (int i = threadIdx.x; i < count; i += kChooseThreads) to.list[i] = sh.list[i] - (uint32_t)begin;  // ~index
    }
  }
  if (threadIdx.x == 0) to.count = count;
}

template <typename In>
__global__ __launch_bounds__(kChooseThreads) __attribute__((amdgpu_waves_per_eu(4, 4))) void choose_kernel(
    ChooseArgs a) {
  __shared__ ChooseShared sh;
  const int64_t n = a.first + blockIdx.x;
  const int V = a.V;
  const Filters filters(a, n);
  const float t = filters.t, p = filters.p;
  const int k = filters.k;
  const bool bounded = filters.bounded;
  const Row<In> row{(const In*)a.scores + n * a.stride, t};
  const Slice* slices = a.found + n * a.slices;
  const auto from_entries = [&](int count) {
    if (filters.seek && count > kSmall) count = shorten_list(count, t, k, sh);
    return count <= kSmall ? from_small(a, n, count, filters, sh) : from_list(a, n, row, count, filters, sh);
  };
  if (filters.none()) {
    if (a.slices == 0) return from_all(a, n, row, all_of(a, n, row, 0, V, sh));
    if (threadIdx.x >= kWave) return;
    const int l = threadIdx.x;  // a slice a lane
    const bool real = l < a.slices;
    const u64 drawn = wave_all(real ? slices[l].drawn : 0, Max());
    const float top = real ? slices[l].best : -INFINITY;
    const float best = value_of((uint32_t)wave_all(key_of(top), Max()));
    double sum = top > -INFINITY ? slices[l].sum * (double)expf(top - best) : 0.0;
    for (int d = 1; d < kWave; d <<= 1) sum += __shfl_xor(sum, d);
    return from_all(a, n, row, All{best, sum, drawn});
  }
  float own = -INFINITY;
  if (a.slices > 0 && (filters.seek || bounded)) {
    const int l = threadIdx.x % kWave;
    const int mine = l < a.slices ? slices[l].count : 0;
    const u64 upto = wave_scan(mine > 0 ? mine : 0, Add());
    const int count = (int)lane_value(upto, kWave - 1);
    if (!__any(mine < 0) && count <= kList) {
      for (int s = threadIdx.x / kWave; s < a.slices; s += kChooseWaves) {
        const int many = __builtin_amdgcn_readlane(mine, s), to = (int)lane_value(upto, s) - many;
        for (int i = l; i < many; i += kWave) sh.list[to + i] = slices[s].list[i];
      }
      __syncthreads();
      return from_entries(count);
    }
  }
  if (filters.seek || bounded) {
    const int rounds = (V + kRound<In> - 1) / kRound<In>;
    if (list_kept(row.in, V, (rounds + 3) / 4, filters, own, sh)) return from_entries((int)sh.listed);
  } else {
    own = own_most(row.in, V, (V + kRound<In> - 1) / kRound<In>);
  }
  const float best = scaled(value_of((uint32_t)block_max(key_of(own + 0.0f), sh)), t);
  if (best == -INFINITY) return no_answer(a, n);
  Cut cut{kNone + 1u, V - 1};
  if (bounded) {
    const uint32_t key = key_of(best + logf(filters.min) + 0.0f);
    if (key > cut.key) cut.key = key;
  }
  // Where a bound leaves few scores, the threads mark them and go through their marks: every lane
  // of a wave would wait for those few otherwise.
  const auto each = [&](float least, bool few, auto f) {
    const float from = least > -INFINITY ? with_equals(least * t, t) : -FLT_MAX;
    if (few) {
      for (int start = 0; start < V; start += Marks<In>::kSpan) {
        Marks<In> marks;
        float unused = -INFINITY;
        marks.make(row.in, V, start, fmaxf(from, -FLT_MAX), unused);
        marks.each(V, start, [&](int e) { f(row(e), e); });
      }
      return;
    }
    each_pack<16 / kPack<In>>(row.in, V, V, [&](int i, auto& v) {
#pragma unroll
      for (int j = 0; j < kPack<In>; ++j)
        if (v[j] >= from) f(scaled(v[j], t), i + j);
    });
  };
  if ((k > 0 || p < 1.0f) && from_bins(a, n, row, each, best, k, p, cut, sh)) return;
  __syncthreads();
  from_row(a, n, row, best, k, p, cut, sh);
}

// A row a block.  A launch counts its threads in 32 bits, and one of more leaves blocks out without an
// error, so more rows than that take several.
template <typename In>
hipError_t launch_choose(ChooseArgs a, int64_t N, hipStream_t s) {
  if (a.slices) {
    slice_kernel<In><<<dim3(a.slices, (unsigned)N), kChooseThreads, 0, s>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  constexpr int64_t kMost = UINT32_MAX / kChooseThreads;
  for (a.first = 0; a.first < N; a.first += kMost) {
    choose_kernel<In><<<(unsigned)(N - a.first < kMost ? N - a.first : kMost), kChooseThreads, 0, s>>>(a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
  }
  return hipSuccess;
}

// Slices of each row: none where a row has less than 128 KB or the rows alone take more than a quarter
// of the 256 CUs, else 32 KB each, up to 16 (16 lists of the largest top_k sought fit one of kList).
// 131072 float32 with noise, us, 16 and 64 rows in slices and 65 rows a block each: no filter 17, 35 and 46;
// top_k 21, 48 and 45; all three filters 38, 105 and 45.  A row whose min_p leaves more than a slice's list
// holds has its slices read in vain, and so do rows of min_p alone (29, 147 and 114): up to a few dozen
// rows slices are the faster side, at 64 only without filters.
int slices_of(int size, int64_t N, int64_t V) {
  if (V * size < 128 * 1024 || N > 64) return 0;
  const int64_t slices = (V * size + 32 * 1024 - 1) / (32 * 1024);
  return slices < 16 ? (int)slices : 16;
}

}  // namespace

}  // namespace ytm

using ytm::fail;

extern "C" {

int ytm_adjust_scores(const void* scores, int dtype, int64_t stride, int64_t N, int64_t V, const int32_t* tokens,
                      int64_t token_stride, int64_t T, const int32_t* lengths, const int32_t* prompt,
                      const float* repetition, const float* frequency, const float* presence, const float* bias,
                      int64_t bias_stride, const uint32_t* allowed, int64_t allowed_stride, void* out, int out_dtype,
                      int64_t out_stride, void* stream) {
  if (!ytm::decode_float(dtype) || !ytm::decode_float(out_dtype))
    return fail(YTM_EINVAL, "scores are float32, float16 or bfloat16");
  if (N < 0 || V < 0 || T < 0 || N > ytm::kDecodeRows || V > ytm::kMaxScores)
    return fail(YTM_EINVAL, "adjust_scores takes at most 65535 rows of 8388608 scores");
  if (T > INT32_MAX)  // the top bit of an answer's count says that it was given
    return fail(YTM_EINVAL, "adjust_scores takes a history of at most 2147483647 answers");
  if (N == 0 || V == 0) return YTM_OK;
  if (!scores || !out || (T > 0 && !tokens)) return fail(YTM_EINVAL, "bad adjust_scores arguments");
  if ((N > 1 && ((stride != 0 && stride < V) || out_stride < V)) ||
      (tokens && N > 1 && token_stride != 0 && token_stride < T) ||
      (bias && bias_stride != 0 && N > 1 && bias_stride < V) ||
      (allowed && allowed_stride != 0 && N > 1 && allowed_stride < (V + 31) / 32))
    return fail(YTM_EINVAL, "adjust_scores: rows overlap");
  const int size = dtype == YTM_DTYPE_F32 ? 4 : 2, out_size = out_dtype == YTM_DTYPE_F32 ? 4 : 2;
  // a block reads its own part of these before it writes it
  const auto in_place = [&](const void* p, int64_t distance, int bytes) {
    return out == p && out_size == bytes && (N == 1 || distance == out_stride);
  };
  const ytm::Rows written = ytm::rows_of(out, N, V, out_stride, out_size);
  const ytm::Rows read[] = {ytm::rows_of(in_place(scores, stride, size) ? nullptr : scores, N, V, stride, size),
                            ytm::rows_of(in_place(bias, bias_stride, 4) ? nullptr : bias, N, V, bias_stride, 4),
                            ytm::rows_of(tokens, N, T, token_stride, 4),
                            ytm::rows_of(allowed, N, (V + 31) / 32, allowed_stride, 4),
                            ytm::block_of(lengths, 4 * N), ytm::block_of(prompt, 4 * N),
                            ytm::block_of(repetition, 4 * N), ytm::block_of(frequency, 4 * N),
                            ytm::block_of(presence, 4 * N)};
  for (const ytm::Rows& r : read)
    if (ytm::share_bytes(written, r))
      return fail(YTM_EINVAL, "adjust_scores: out overlaps an input, and is not the scores' or the bias's own place");
  ytm::AdjustArgs a{scores, stride, V, T > 0 ? tokens : nullptr, token_stride, T, lengths, prompt, repetition,
                    frequency, presence, bias, bias_stride, allowed, allowed_stride, out, out_stride};
  hipStream_t s = (hipStream_t)stream;
  hipError_t e;
  switch (dtype) {
    case YTM_DTYPE_F16: e = ytm::launch_adjust_out<ytm::f16>(out_dtype, a, N, s); break;
    case YTM_DTYPE_BF16: e = ytm::launch_adjust_out<ytm::bf16>(out_dtype, a, N, s); break;
    default: e = ytm::launch_adjust_out<float>(out_dtype, a, N, s); break;
  }
  if (e != hipSuccess) return fail(YTM_EHIP, std::string("adjust_scores failed: ") + hipGetErrorString(e));
  return YTM_OK;
}

int ytm_choose_workspace(int dtype, int64_t N, int64_t V, int64_t* bytes) {
  if (!bytes || !ytm::decode_float(dtype) || N < 0 || N > INT32_MAX || V < 0 || V > ytm::kMaxScores)
    return fail(YTM_EINVAL, "bad choose_workspace arguments");
  *bytes = N * ytm::slices_of(dtype == YTM_DTYPE_F32 ? 4 : 2, N, V) * (int64_t)sizeof(ytm::Slice);
  return YTM_OK;
}

int ytm_choose(const void* scores, int dtype, int64_t stride, int64_t N, int64_t V, const float* temperature,
               const int32_t* top_k, const float* top_p, const float* min_p, const float* noise, int64_t noise_stride,
               int32_t* tokens, float* logprobs, void* workspace, int64_t workspace_bytes, void* stream) {
  if (!ytm::decode_float(dtype)) return fail(YTM_EINVAL, "scores are float32, float16 or bfloat16");
  if (N < 0 || V < 0 || N > INT32_MAX || V > ytm::kMaxScores)
    return fail(YTM_EINVAL, "choose takes at most 2147483647 rows of 8388608 scores");
  if (N == 0) return YTM_OK;
  if ((V > 0 && !scores) || !tokens || !logprobs) return fail(YTM_EINVAL, "bad choose arguments");
  if (N > 1 && ((stride != 0 && stride < V) || (noise && noise_stride != 0 && noise_stride < V)))
    return fail(YTM_EINVAL, "choose: rows overlap");
  int64_t need = 0;
  if (int rc = ytm_choose_workspace(dtype, N, V, &need)) return rc;
  if (need > 0 && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
    return fail(YTM_EINVAL, "choose: the workspace is too small or not at a multiple of 16 bytes");
  const ytm::Rows written[] = {ytm::block_of(tokens, 4 * N), ytm::block_of(logprobs, 4 * N),
                               ytm::block_of(workspace, need)};
  const ytm::Rows read[] = {ytm::rows_of(scores, N, V, stride, dtype == YTM_DTYPE_F32 ? 4 : 2),
                            ytm::rows_of(noise, N, V, noise_stride, 4), ytm::block_of(temperature, 4 * N),
                            ytm::block_of(top_k, 4 * N), ytm::block_of(top_p, 4 * N), ytm::block_of(min_p, 4 * N)};
  bool overlap = ytm::share_bytes(written[0], written[1]) || ytm::share_bytes(written[0], written[2]) ||
                 ytm::share_bytes(written[1], written[2]);
  for (const ytm::Rows& w : written)
    for (const ytm::Rows& r : read) overlap |= ytm::share_bytes(w, r);
  if (overlap) return fail(YTM_EINVAL, "choose: what is written overlaps what is read");
  const int slices = ytm::slices_of(dtype == YTM_DTYPE_F32 ? 4 : 2, N, V);
  const ytm::ChooseArgs a{scores, stride, (int)V, temperature, top_k, top_p, min_p, noise, noise_stride, tokens, logprobs,
                          0, slices, slices ? (int)((V + slices - 1) / slices) : 0, (ytm::Slice*)workspace};
  hipStream_t s = (hipStream_t)stream;
  hipError_t e;
  switch (dtype) {
    case YTM_DTYPE_F16: e = ytm::launch_choose<ytm::f16>(a, N, s); break;
    case YTM_DTYPE_BF16: e = ytm::launch_choose<ytm::bf16>(a, N, s); break;
    default: e = ytm::launch_choose<float>(a, N, s); break;
  }
  if (e != hipSuccess) return fail(YTM_EHIP, std::string("choose failed: ") + hipGetErrorString(e));
  return YTM_OK;
}

}  // extern "C"
