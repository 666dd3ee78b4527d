// ytm_losses.hip -- losses of a model's answers with the gradient of the scores: the entry points
// ytm_policy_loss and ytm_preference_loss of include/ytm.h and their gfx950 kernels.
//
// With z = score / temperature, p = softmax(z) over a row and lp = log p of the row's answer t, both losses
// reach the scores through lp alone:
//
//   d loss / d score[v] = c / temperature * ((v == t) - p[v]),  c = d loss / d lp
//
// so a row is read for its sum of exp(z), relative to one of its scores, c is found, and the row is written from what
// the threads still hold of it, or, where c needs other rows or the row is longer, read again.  Both are bound by
// memory: 1024 rows of 131072 bfloat16 126 us, 4.3 TB/s, with the exponentials made twice at a third of the
// vector units' time.
#include <hip/hip_runtime.h>
#include <float.h>
#include <stdint.h>

#include <type_traits>

#include "ytm_decode.h"
#include "ytm_internal.h"

namespace ytm {

namespace {

constexpr int kWave = 64;
constexpr int kMaxWaves = 8;  // of a block
constexpr int kMaxSlices = 32;
constexpr float kLog2e = 1.44269504088896340736f;

struct LossArgs {
  const void* scores;
  int64_t stride;
  int N, V;
  const int32_t* tokens;
  const float* temperature;
  // policy
  const float *old, *advantages, *reference, *weights;
  float kl, low, high;
  // preference
  const int32_t* starts;
  const float* sequence_reference;
  float beta, smoothing;
  int pairs;
  float *losses, *logprobs;
  void* grad;
  int64_t grad_stride;
  int slices, slice;  // a row's blocks, each of so many scores
  float2* stats;      // [N][slices]: maximum, sum
  float* at;          // [N]: the answer's score
  float* slope;       // [N]: c, of preferences
};

// A score that is NaN counts as -inf, one of +inf as the largest float: the median of three, which is the least of
// the others beside a NaN.  (The compiler would make a minimum of it, which is not, if it knew the -inf.)
__device__ __forceinline__ float score_of(float v) {
  float least = -INFINITY;
  asm("" : "+s"(least));
  return __builtin_amdgcn_fmed3f(v, least, FLT_MAX);
}
template <typename In>
__device__ __forceinline__ float score_of(In v) {
  return score_of(to_float(v));
}

// 2^x, to one unit in its last place; what is less than the smallest normal float is 0.
__device__ __forceinline__ float power(float x) { return __builtin_amdgcn_exp2f(x); }

// 1 / temperature as choose() takes it: 0 or less counts as 1, less than the smallest normal float or NaN as that,
// and an infinite one as the largest float, beside which a score of -inf stays -inf.
__device__ __forceinline__ float cooling(const LossArgs& a, int n) {
  if (!a.temperature) return 1.0f;
  const float t = a.temperature[n];
  return t <= 0.0f ? 1.0f : 1.0f / (t >= FLT_MIN ? fminf(t, FLT_MAX) : FLT_MIN);
}

// Of some of a row's scores: one of them, or near them, and their sum of exp((score - it) / temperature), in powers of
// two; -inf and 0 where none is above -inf.
struct Stats {
  float max, sum;
  __device__ __forceinline__ void add(const Stats& o, float scale) {
    if (o.max == -INFINITY) return;
    if (o.max > max) {
      sum = max == -INFINITY ? o.sum : sum * power((max - o.max) * scale) + o.sum;
      max = o.max;
    } else {
      sum += o.sum * power((o.max - max) * scale);
    }
  }
};

// A thread's part of a row: R times 16 bytes, as they are in memory, every thread's one after the other; past
// the last score -inf.  All are asked for before the first is used, and a row that fits is read
// once.
constexpr float kWholes = 0x1p22f;  // whole numbers below it are exact, and their neighbours a quarter apart
template <typename In>
constexpr int kEach = 16 / sizeof(In);
template <typename In>
constexpr uint32_t kNothing = 0xFF800000u;
template <>
constexpr uint32_t kNothing<f16> = 0xFC00u;
template <>
constexpr uint32_t kNothing<bf16> = 0xFF80u;
__device__ __forceinline__ float half_of(uint32_t u, int i, f16) {
  return (float)__builtin_bit_cast(f16, (uint16_t)(i ? u >> 16 : u));
}
__device__ __forceinline__ float half_of(uint32_t u, int i, bf16) {
  return __uint_as_float(i ? u & 0xFFFF0000u : u << 16);
}
__device__ __forceinline__ float half_of(uint32_t u, int, float) { return __uint_as_float(u); }

template <typename In, int R>
struct Part {
  static constexpr int E = kEach<In>, kPerWord = E / 4;
  uint32_t v[R][4];

  // from the uniform score `first` on, up to `last`
  __device__ __forceinline__ void load(const In* row, int first, int last) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      const int from = first + r * (int)blockDim.x * E, i = from + (int)threadIdx.x * E;
      if (from + (int)blockDim.x * E <= last) {
        __builtin_memcpy(v[r], row + i, sizeof v[r]);
      } else {
        uint32_t one[E];
#pragma unroll
        for (int e = 0; e < E; ++e) {
          one[e] = kNothing<In>;
          if (i + e < last) {
            In at = row[i + e];
            one[e] = 0u;
            __builtin_memcpy(&one[e], &at, sizeof at);
          }
        }
#pragma unroll
        for (int q = 0; q < 4; ++q) v[r][q] = kPerWord == 1 ? one[q] : one[2 * q] | one[2 * q + 1] << 16;
      }
    }
    __builtin_amdgcn_sched_barrier(0);
  }
  __device__ __forceinline__ float score(int r, int e) const {
    return score_of(half_of(v[r][e / kPerWord], e % kPerWord, In{}));
  }
  // Scores are made from what is in memory each time that they are used: kept, they would not fit the registers.
  __device__ __forceinline__ void again() {
#pragma unroll
    for (int r = 0; r < R; ++r)
#pragma unroll
      for (int q = 0; q < 4; ++q) asm volatile("" : "+v"(v[r][q]));
  }
  // whether any thread has scores in place r
  __device__ __forceinline__ static bool has(int r, int first, int last) { return first + r * (int)blockDim.x * E < last; }

  // The sum is made relative to the largest of the thread's first few scores, or to 0, in one pass: each exponent is
  // score * scale less a whole number near that score's, rounded once beside the rounding that all share in scale,
  // and the power to that whole number comes as one more factor.  (Of all gradients of 64 rows of 10000 scores of
  // deviation 3 the mean error is 6.9 units of 2^-24 and the largest 32; of differences to the maximum, powers and
  // a quotient, each rounded, 9.0 and 48.)  Where that is not good enough (a NaN, an
  // infinity, scores far above, whose exponents have fewer bits of fraction, or all far below: a sum above 2^24 or
  // below 2^-24), relative to the largest.
  __device__ __forceinline__ Stats stats(int first, int last, float scale) {
    float near = -INFINITY;
#pragma unroll
    for (int e = 0; e < E; ++e) near = fmaxf(near, half_of(v[0][e / kPerWord], e % kPerWord, In{}));
    near = near == -INFINITY ? 0.0f : near;
    const float whole = rintf(near * scale);
    float sum[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (has(r, first, last)) {
#pragma unroll
        for (int e = 0; e < E; ++e)
          sum[e % 4] += power(__builtin_fmaf(half_of(v[r][e / kPerWord], e % kPerWord, In{}), scale, -whole));
      }
    Stats s{near, ((sum[0] + sum[1]) + (sum[2] + sum[3])) * power(__builtin_fmaf(-near, scale, whole))};
    again();
    if (s.sum > 0x1p-24f && s.sum < 0x1p24f && fabsf(whole) < kWholes) return s;
    s = Stats{-INFINITY, 0.0f};
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (has(r, first, last)) {
#pragma unroll
        for (int e = 0; e < E; ++e) s.max = fmaxf(s.max, score(r, e));
      }
    again();
    if (s.max == -INFINITY) return s;
#pragma unroll
    for (int r = 0; r < R; ++r)
      if (has(r, first, last)) {
#pragma unroll
        for (int e = 0; e < E; ++e) s.sum += power((score(r, e) - s.max) * scale);
      }
    again();
    return s;
  }
};

// Of the scores first .. last - 1 of a row, each thread's own, part after part.
template <typename In, int R>
__device__ __forceinline__ Stats own_stats(const In* row, int first, int last, float scale) {
  Stats s{-INFINITY, 0.0f};
  if (first >= last) return s;
  const int step = R * (int)blockDim.x * kEach<In>;
  Part<In, R> now;
  now.load(row, first, last);
  for (; first + step < last; first += step) {  // the next part is on its way
    Part<In, R> next;
    next.load(row, first + step, last);
    s.add(now.stats(first, last, scale), scale);
    now = next;
  }
  s.add(now.stats(first, last, scale), scale);
  return s;
}

// Of all threads of the block, to all of them, in a fixed order.
__device__ __forceinline__ Stats block_stats(Stats s, float scale, Stats* part) {
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const Stats o{__shfl_xor(s.max, d), __shfl_xor(s.sum, d)};
    s.add(o, scale);
  }
  if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = s;
  __syncthreads();
  Stats all = part[0];
  for (int w = 1; w < (int)blockDim.x / kWave; ++w) all.add(part[w], scale);
  return all;
}

template <typename In, int THREADS, int R>
__global__ __launch_bounds__(THREADS) void stats_kernel(LossArgs a) {
  __shared__ Stats part[THREADS / kWave];
  const int n = blockIdx.y, slice = blockIdx.x;
  const In* row = (const In*)a.scores + n * a.stride;
  const int first = slice * a.slice, last = first + a.slice < a.V ? first + a.slice : a.V;
  const float scale = cooling(a, n) * kLog2e;
  const Stats s = block_stats(own_stats<In, R>(row, first, last, scale), scale, part);
  if (threadIdx.x != 0) return;
  a.stats[(int64_t)n * a.slices + slice] = float2{s.max, s.sum};
  const int t = a.tokens[n];
  if (t >= first && t < last) a.at[n] = score_of(row[t]);
  if (slice == 0 && a.slope) a.slope[n] = 0.0f;
}

// What a row's answer comes to.
struct Answer {
  Stats all;
  bool there;  // an answer, of a score above -inf
  float lp, cooling;
};

__device__ __forceinline__ Answer answer_of(const LossArgs& a, int n, float z, const Stats& all) {
  Answer r;
  const int t = a.tokens[n];
  r.all = all;
  r.cooling = cooling(a, n);
  r.there = t >= 0 && t < a.V && z > -INFINITY;
  r.lp = 0.0f;
  if (r.there) r.lp = (float)(((double)z - (double)all.max) * (double)r.cooling - log((double)all.sum));
  return r;
}

__device__ __forceinline__ Answer answer_of(const LossArgs& a, int n) {
  const float scale = cooling(a, n) * kLog2e;
  Stats all{-INFINITY, 0.0f};
  for (int s = 0; s < a.slices; ++s) {
    const float2 v = a.stats[(int64_t)n * a.slices + s];
    all.add(Stats{v.x, v.y}, scale);
  }
  const int t = a.tokens[n];
  return answer_of(a, n, t >= 0 && t < a.V ? a.at[n] : -INFINITY, all);
}

// The policy loss of a row and its derivative by lp; 0 where its weight is, whatever fills such a row.
struct Loss {
  float value, slope;
};
__device__ __forceinline__ Loss policy(const LossArgs& a, int n, const Answer& r) {
  const float w = a.weights ? a.weights[n] : 1.0f / (float)a.N, adv = a.advantages[n];
  if (!r.there || w == 0.0f) return Loss{0.0f, 0.0f};
  const float ratio = expf(r.lp - a.old[n]);
  // an advantage of 0 makes nothing of a ratio past float32; what is NaN makes the comparison false and goes on
  const float free = adv == 0.0f && ratio == INFINITY ? 0.0f : ratio * adv;
  const float held = fminf(fmaxf(ratio, a.low), a.high) * adv;
  const bool outside = free > held;
  float value = outside ? -held : -free, slope = outside ? 0.0f : -free;
  if (a.kl != 0.0f) {
    const float far = a.reference[n] - r.lp, up = expm1f(far);
    value += a.kl * (up - far);
    slope -= a.kl * up;
  }
  return Loss{w * value, w * slope};
}

// Two values to the gradient's type.
typedef float v2f __attribute__((ext_vector_type(2)));
typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
template <typename Out>
__device__ __forceinline__ void to_out(float a, float b, Out* to) {
  to[0] = from_float<Out>(a), to[1] = from_float<Out>(b);
}
template <>
__device__ __forceinline__ void to_out<bf16>(float a, float b, bf16* to) {
  const v2bf v = __builtin_convertvector((v2f{a, b}), v2bf);
  __builtin_memcpy(to, &v, 4);
}

// The gradient of a row's scores first .. last - 1, of which `part` holds the first (whole: all); c is 0 where
// the row takes no part.
struct Slope {
  float by, each, max, scale, whole;
  int t;
  bool any, far;  // far: an exponent is no float's, and only differences are
  __device__ __forceinline__ Slope(const LossArgs& a, int n, const Answer& r, float c) {
    any = r.there && c != 0.0f;
    by = any ? c * r.cooling : 0.0f;
    each = any ? -by / r.all.sum : 0.0f;
    max = r.all.max, scale = r.cooling * kLog2e, t = a.tokens[n];
    whole = rintf(max * scale);
    far = !(fabsf(whole) < kWholes);
    if (!far) each *= power(__builtin_fmaf(-max, scale, whole));
  }
};
template <typename In, typename Out, int R>
__device__ __forceinline__ void write_part(const Part<In, R>& part, const Slope& s, Out* to, int first, int last) {
  constexpr int E = kEach<In>;
#pragma unroll
  for (int r = 0; r < R; ++r) {
    const int from = first + r * (int)blockDim.x * E, i = from + (int)threadIdx.x * E;
    if (!Part<In, R>::has(r, first, last)) continue;
    float v[E];
    if (s.any) {
      if (s.far) {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = s.each * power((part.score(r, e) - s.max) * s.scale);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = s.each * power(__builtin_fmaf(part.score(r, e), s.scale, -s.whole));
      }
      if (s.t >= i && s.t < i + E) {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] += i + e == s.t ? s.by : 0.0f;
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = 0.0f;
    }
    Out out[E];
#pragma unroll
    for (int e = 0; e < E; e += 2) to_out<Out>(v[e], v[e + 1], out + e);
    if (from + (int)blockDim.x * E <= last) {
      __builtin_memcpy(to + i, out, sizeof out);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (i + e < last) to[i + e] = out[e];
    }
  }
}
template <typename In, typename Out, int R>
__device__ __forceinline__ void write_grad(const LossArgs& a, int n, int first, int last, const Slope& s) {
  const In* row = (const In*)a.scores + n * a.stride;
  Out* to = (Out*)a.grad + n * a.grad_stride;
  for (int from = first; from < last; from += R * (int)blockDim.x * kEach<In>) {
    Part<In, R> part;
    if (s.any) part.load(row, from, last);
    write_part<In, Out, R>(part, s, to, from, last);
  }
}

// A pair of sequences: their rows and log probabilities, made by the whole block, the loss, and its derivative by
// the log probability of the first.
struct Pair {
  int begin[2], end[2];
  double said[2];
  float loss, slope;
  __device__ __forceinline__ Pair(const LossArgs& a, int pair, double (*part)[kMaxWaves]) {
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      begin[side] = a.starts[2 * pair + side];
      end[side] = a.starts[2 * pair + side + 1];
      begin[side] = begin[side] < 0 ? 0 : begin[side];
      end[side] = end[side] > a.N ? a.N : end[side];
    }
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      double sum = 0.0;
      for (int64_t n = begin[side] + (int64_t)threadIdx.x; n < end[side]; n += blockDim.x)
        sum += (double)answer_of(a, (int)n).lp;
#pragma unroll
      for (int d = 1; d < kWave; d <<= 1) sum += __shfl_xor(sum, d);
      if (threadIdx.x % kWave == 0) part[side][threadIdx.x / kWave] = sum;
    }
    __syncthreads();
#pragma unroll
    for (int side = 0; side < 2; ++side) {
      said[side] = 0.0;
      for (int w = 0; w < (int)blockDim.x / kWave; ++w) said[side] += part[side][w];
    }
    const float* ref = a.sequence_reference + 2 * pair;
    const float m = (float)((double)a.beta * ((said[0] - (double)ref[0]) - (said[1] - (double)ref[1])));
    const float small = expf(-fabsf(m));  // softplus(m) = max(m, 0) + log(1 + exp(-|m|)), sigmoid(m) alike
    const float share = 1.0f / (float)a.pairs, log1 = log1pf(small);
    const float won = (m >= 0.0f ? 1.0f : small) / (1.0f + small), lost = (m >= 0.0f ? small : 1.0f) / (1.0f + small);
    slope = share * a.beta * (a.smoothing * won - (1.0f - a.smoothing) * lost);
    // what has no part may be infinite
    const float right = a.smoothing == 1.0f ? 0.0f : (1.0f - a.smoothing) * (fmaxf(-m, 0.0f) + log1);
    const float wrong = a.smoothing == 0.0f ? 0.0f : a.smoothing * (fmaxf(m, 0.0f) + log1);
    loss = share * (right + wrong);
  }
  __device__ __forceinline__ void write(const LossArgs& a, int pair) const {
    if (threadIdx.x != 0) return;
    a.losses[pair] = loss;
    a.logprobs[2 * pair] = (float)said[0];
    a.logprobs[2 * pair + 1] = (float)said[1];
  }
};

constexpr int kPairThreads = 256;
__global__ __launch_bounds__(kPairThreads) void pair_kernel(LossArgs a) {
  __shared__ double part[2][kMaxWaves];
  const Pair pair(a, blockIdx.x, part);
  pair.write(a, blockIdx.x);
#pragma unroll
  for (int side = 0; side < 2; ++side)
    for (int64_t n = pair.begin[side] + (int64_t)threadIdx.x; n < pair.end[side]; n += kPairThreads)
      a.slope[n] = side ? -pair.slope : pair.slope;
}

// Row n's sequence: the last that begins at or before it; 2 pairs or -1 where it is in none.
__device__ __forceinline__ int sequence_of(const LossArgs& a, int n, int* count) {
  int before = 0;
  for (int i = threadIdx.x; i < 2 * a.pairs + 1; i += blockDim.x) before += a.starts[i] <= n;
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) before += __shfl_xor(before, d);
  if (threadIdx.x % kWave == 0) count[threadIdx.x / kWave] = before;
  __syncthreads();
  int all = 0;
  for (int w = 0; w < (int)blockDim.x / kWave; ++w) all += count[w];
  return __builtin_amdgcn_readfirstlane(all) - 1;
}

// A slice of a row, after stats_kernel.  What its loss is to it: a policy's, that of a preference after pair_kernel,
// or that of a preference whose pair each of its blocks looks at itself, with a block more for each pair.
enum Kind { kPolicy, kPreference, kFewPreferences };
template <typename In, typename Out, Kind KIND, int THREADS, int R>
__global__ __launch_bounds__(THREADS) void grad_kernel(LossArgs a) {
  const int n = blockIdx.y, first = blockIdx.x * a.slice, last = first + a.slice < a.V ? first + a.slice : a.V;
  float c = 0.0f;
  if constexpr (KIND == kFewPreferences) {
    __shared__ double part[2][kMaxWaves];
    __shared__ int count[kMaxWaves];
    if (n >= a.N) {
      if (blockIdx.x == 0) Pair(a, n - a.N, part).write(a, n - a.N);
      return;
    }
    const int sequence = sequence_of(a, n, count);
    if (sequence >= 0 && sequence < 2 * a.pairs) {
      const Pair pair(a, sequence / 2, part);
      c = sequence % 2 ? -pair.slope : pair.slope;
    }
  }
  const Answer r = answer_of(a, n);
  if constexpr (KIND == kPolicy) {
    const Loss loss = policy(a, n, r);
    c = loss.slope;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      a.losses[n] = loss.value;
      a.logprobs[n] = r.lp;
    }
  } else if constexpr (KIND == kPreference) {
    c = a.slope[n];
  }
  write_grad<In, Out, R>(a, n, first, last, Slope(a, n, r, c));
}

// A policy loss's whole row; ONCE: it is in the threads' registers from its one reading to its gradient.
template <typename In, typename Out, int THREADS, int R, bool ONCE>
__global__ __launch_bounds__(THREADS) void policy_kernel(LossArgs a) {
  __shared__ Stats part[THREADS / kWave];
  const int n = blockIdx.x;
  const In* row = (const In*)a.scores + n * a.stride;
  const int t = a.tokens[n];
  const float scale = cooling(a, n) * kLog2e;
  const float z = t >= 0 && t < a.V ? score_of(row[t]) : -INFINITY;
  Part<In, R> held;
  Stats own;
  if (ONCE) {
    held.load(row, 0, a.V);
    own = held.stats(0, a.V, scale);
  } else {
    own = own_stats<In, R>(row, 0, a.V, scale);
  }
  const Answer r = answer_of(a, n, z, block_stats(own, scale, part));
  const Loss loss = policy(a, n, r);
  if (threadIdx.x == 0) {
    a.losses[n] = loss.value;
    a.logprobs[n] = r.lp;
  }
  const Slope s(a, n, r, loss.slope);
  if (ONCE)
    write_part<In, Out, R>(held, s, (Out*)a.grad + n * a.grad_stride, 0, a.V);
  else
    write_grad<In, Out, R>(a, n, 0, a.V, s);
}

// --------------------------------------------------------------------------------------- host
// launch(threads, 16 bytes that each has of a row at once, whether that is all of it): the fewest that hold
// the row, up to 256 KB, half of a CU's registers.
template <typename In, typename Launch>
hipError_t shaped(int64_t scores, Launch launch) {
  const int64_t pieces = (scores + kEach<In> - 1) / kEach<In>;
  const std::integral_constant<int, 64> one{};
  const std::integral_constant<int, 256> four{};
  const std::integral_constant<int, 512> eight{};
  const std::integral_constant<int, 4> few{};
  const std::integral_constant<int, 16> some{};
  const std::integral_constant<int, 32> many{};
  if (pieces <= 64 * 4) return launch(one, few, std::true_type{});
  if (pieces <= 256 * 4) return launch(four, few, std::true_type{});
  if (pieces <= 256 * 16) return launch(four, some, std::true_type{});
  if (pieces <= 512 * 16) return launch(eight, some, std::true_type{});
  if (pieces <= 512 * 32) return launch(eight, many, std::true_type{});
  return launch(eight, some, std::false_type{});
}

// Slices of a row: rows alone fill the 256 CUs, or a slice would have less than 8192 scores; a row of fewer than 32768
// is one block's.
int slices_of(int64_t N, int64_t V) {
  int64_t slices = N > 0 && V >= 32768 ? 512 / N : 1;
  if (slices > V / 8192) slices = V / 8192;
  return slices < 1 ? 1 : slices > kMaxSlices ? kMaxSlices : (int)slices;
}

// Whether each row's block finds its pair's loss by itself, which saves a launch.
bool few_pairs(int64_t N, int64_t pairs) { return N <= 256 && pairs <= 128; }

int64_t workspace_bytes_of(int64_t N, int64_t slices) { return N * (slices * 8 + 8); }

template <typename In, typename Out, bool POLICY>
hipError_t launch_loss(const LossArgs& a, hipStream_t s) {
  if (POLICY && a.slices == 1)
    return shaped<In>(a.V, [&](auto threads, auto r, auto once) {
      constexpr int T = decltype(threads)::value, R = decltype(r)::value;
      policy_kernel<In, Out, T, R, decltype(once)::value><<<a.N, T, 0, s>>>(a);
      return hipGetLastError();
    });
  const dim3 grid(a.slices, a.N);
  return shaped<In>(a.slice, [&](auto threads, auto r, auto) {
    constexpr int T = decltype(threads)::value, R = decltype(r)::value;
    stats_kernel<In, T, 4><<<grid, T, 0, s>>>(a);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    constexpr int G = R > 8 ? 8 : R;  // nothing is kept: fewer registers, more blocks
    if (POLICY) {
      grad_kernel<In, Out, kPolicy, T, G><<<grid, T, 0, s>>>(a);
    } else if (few_pairs(a.N, a.pairs)) {
      grad_kernel<In, Out, kFewPreferences, T, G><<<dim3(a.slices, a.N + a.pairs), T, 0, s>>>(a);
    } else {
      pair_kernel<<<a.pairs, kPairThreads, 0, s>>>(a);
      e = hipGetLastError();
      if (e != hipSuccess) return e;
      grad_kernel<In, Out, kPreference, T, G><<<grid, T, 0, s>>>(a);
    }
    return hipGetLastError();
  });
}

template <typename In, bool POLICY>
hipError_t launch_loss_out(int grad_dtype, const LossArgs& a, hipStream_t s) {
  switch (grad_dtype) {
    case YTM_DTYPE_F16: return launch_loss<In, f16, POLICY>(a, s);
    case YTM_DTYPE_BF16: return launch_loss<In, bf16, POLICY>(a, s);
    default: return launch_loss<In, float, POLICY>(a, s);
  }
}
template <bool POLICY>
hipError_t launch_loss_in(int dtype, int grad_dtype, const LossArgs& a, hipStream_t s) {
  switch (dtype) {
    case YTM_DTYPE_F16: return launch_loss_out<f16, POLICY>(grad_dtype, a, s);
    case YTM_DTYPE_BF16: return launch_loss_out<bf16, POLICY>(grad_dtype, a, s);
    default: return launch_loss_out<float, POLICY>(grad_dtype, a, s);
  }
}

// What both entries ask; NULL where it is given, else what is wrong.
const char* wrong_scores(const void* scores, int dtype, int64_t stride, int64_t N, int64_t V, const int32_t* tokens,
                         const void* grad, int grad_dtype, int64_t grad_stride) {
  if (!decode_float(dtype) || !decode_float(grad_dtype)) return "scores and gradients are float32, float16 or bfloat16";
  if (N < 0 || V < 0 || N > kDecodeRows || V > kMaxScores) return "at most 65535 rows of 8388608 scores";
  if (N > 0 && (!tokens || (V > 0 && (!scores || !grad)))) return "an operand is missing";
  if (N > 1 && ((stride != 0 && stride < V) || grad_stride < V)) return "rows overlap";
  return nullptr;
}

// Whether what is written (the gradient, two arrays, the workspace) shares memory with what is read or with
// each other.
bool overlapping(const LossArgs& a, int dtype, int grad_dtype, int64_t losses, int64_t logprobs, const void* workspace,
                 int64_t need) {
  const int size = dtype == YTM_DTYPE_F32 ? 4 : 2, grad_size = grad_dtype == YTM_DTYPE_F32 ? 4 : 2;
  const bool in_place = a.grad == a.scores && size == grad_size && (a.N == 1 || a.stride == a.grad_stride);
  const Rows scores = rows_of(a.scores, a.N, a.V, a.stride, size);
  const Rows written[] = {rows_of(a.grad, a.N, a.V, a.grad_stride, grad_size), block_of(a.losses, 4 * losses),
                          block_of(a.logprobs, 4 * logprobs), block_of(workspace, need)};
  const int64_t rows = 4 * (int64_t)a.N;
  const Rows read[] = {block_of(a.tokens, rows), block_of(a.temperature, rows), block_of(a.old, rows),
                       block_of(a.advantages, rows), block_of(a.reference, rows), block_of(a.weights, rows),
                       block_of(a.starts, 8 * (int64_t)a.pairs + 4),
                       block_of(a.sequence_reference, 8 * (int64_t)a.pairs)};
  for (int i = 0; i < 4; ++i) {
    if (!(i == 0 && in_place) && share_bytes(written[i], scores)) return true;
    for (const Rows& r : read)
      if (share_bytes(written[i], r)) return true;
    for (int j = 0; j < i; ++j)
      if (share_bytes(written[i], written[j])) return true;
  }
  return false;
}

}  // namespace

}  // namespace ytm

using ytm::fail;

extern "C" {

int ytm_policy_loss_workspace(int64_t N, int64_t V, int64_t* bytes) {
  if (!bytes || N < 0 || V < 0 || N > ytm::kDecodeRows || V > ytm::kMaxScores)
    return fail(YTM_EINVAL, "bad policy_loss_workspace arguments");
  const int slices = ytm::slices_of(N, V);
  *bytes = slices > 1 ? ytm::workspace_bytes_of(N, slices) : 0;
  return YTM_OK;
}

int ytm_policy_loss(const void* scores, int dtype, int64_t stride, int64_t N, int64_t V, const int32_t* tokens,
                    const float* old, const float* advantages, const float* reference, float kl, float low, float high,
                    const float* weights, const float* temperature, float* losses, float* logprobs, void* grad,
                    int grad_dtype, int64_t grad_stride, void* workspace, int64_t workspace_bytes, void* stream) {
  if (const char* wrong = ytm::wrong_scores(scores, dtype, stride, N, V, tokens, grad, grad_dtype, grad_stride))
    return fail(YTM_EINVAL, std::string("policy_loss: ") + wrong);
  if (N == 0) return YTM_OK;
  if (!old || !advantages || !losses || !logprobs || (kl != 0.0f && !reference))
    return fail(YTM_EINVAL, "policy_loss: an operand is missing");
  if (!(kl >= 0.0f) || !(low >= 0.0f) || !(low <= 1.0f) || !(high >= 0.0f))
    return fail(YTM_EINVAL, "policy_loss: kl is 0 or more, the clip's bounds 0 or more, the lower one at most 1");
  int64_t need = 0;
  if (int rc = ytm_policy_loss_workspace(N, V, &need)) return rc;
  if (need > 0 && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
    return fail(YTM_EINVAL, "policy_loss: the workspace is too small or not at a multiple of 16 bytes");
  ytm::LossArgs a{};
  a.scores = scores, a.stride = stride, a.N = (int)N, a.V = (int)V, a.tokens = tokens, a.temperature = temperature;
  a.old = old, a.advantages = advantages, a.reference = kl != 0.0f ? reference : nullptr, a.weights = weights;
  a.kl = kl, a.low = 1.0f - low, a.high = 1.0f + high;
  a.losses = losses, a.logprobs = logprobs, a.grad = grad, a.grad_stride = grad_stride;
  if (ytm::overlapping(a, dtype, grad_dtype, N, N, workspace, need))
    return fail(YTM_EINVAL, "policy_loss: what is written overlaps what is read, and is not the scores' own place");
  a.slices = ytm::slices_of(N, V);
  a.slice = (int)((V + a.slices - 1) / a.slices);
  a.stats = (float2*)workspace;
  a.at = (float*)((char*)workspace + N * a.slices * 8);
  const hipError_t e = ytm::launch_loss_in<true>(dtype, grad_dtype, a, (hipStream_t)stream);
  if (e != hipSuccess) return fail(YTM_EHIP, std::string("policy_loss failed: ") + hipGetErrorString(e));
  return YTM_OK;
}

int ytm_preference_loss_workspace(int64_t N, int64_t V, int64_t* bytes) {
  if (!bytes || N < 0 || V < 0 || N > ytm::kDecodeRows || V > ytm::kMaxScores)
    return fail(YTM_EINVAL, "bad preference_loss_workspace arguments");
  *bytes = ytm::workspace_bytes_of(N, ytm::slices_of(N, V));
  return YTM_OK;
}

int ytm_preference_loss(const void* scores, int dtype, int64_t stride, int64_t N, int64_t V, const int32_t* tokens,
                        const int32_t* starts, int64_t pairs, const float* reference, float beta, float smoothing,
                        const float* temperature, float* losses, float* logprobs, void* grad, int grad_dtype,
                        int64_t grad_stride, void* workspace, int64_t workspace_bytes, void* stream) {
  if (const char* wrong = ytm::wrong_scores(scores, dtype, stride, N, V, tokens, grad, grad_dtype, grad_stride))
    return fail(YTM_EINVAL, std::string("preference_loss: ") + wrong);
  if (pairs < 1 || pairs > ytm::kDecodeRows) return fail(YTM_EINVAL, "preference_loss takes 1 to 65535 pairs");
  if (!starts || !reference || !losses || !logprobs) return fail(YTM_EINVAL, "preference_loss: an operand is missing");
  if (!(beta - beta == 0.0f) || !(smoothing >= 0.0f && smoothing <= 1.0f))
    return fail(YTM_EINVAL, "preference_loss: beta is finite, smoothing between 0 and 1");
  int64_t need = 0;
  if (int rc = ytm_preference_loss_workspace(N, V, &need)) return rc;
  if (need > 0 && (!workspace || workspace_bytes < need || (uintptr_t)workspace % 16))
    return fail(YTM_EINVAL, "preference_loss: the workspace is too small or not at a multiple of 16 bytes");
  ytm::LossArgs a{};
  a.scores = scores, a.stride = stride, a.N = (int)N, a.V = (int)V, a.tokens = tokens, a.temperature = temperature;
  a.starts = starts, a.sequence_reference = reference, a.beta = beta, a.smoothing = smoothing, a.pairs = (int)pairs;
  a.losses = losses, a.logprobs = logprobs, a.grad = grad, a.grad_stride = grad_stride;
  if (ytm::overlapping(a, dtype, grad_dtype, pairs, 2 * pairs, workspace, need))
    return fail(YTM_EINVAL, "preference_loss: what is written overlaps what is read, and is not the scores' own place");
  a.slices = ytm::slices_of(N, V);
  a.slice = (int)((V + a.slices - 1) / a.slices);
  a.stats = (float2*)workspace;
  a.at = (float*)((char*)workspace + N * a.slices * 8);
  a.slope = a.at + N;
  hipStream_t s = (hipStream_t)stream;
  hipError_t e;
  if (N == 0) {
    ytm::pair_kernel<<<a.pairs, ytm::kPairThreads, 0, s>>>(a);
    e = hipGetLastError();
  } else {
    e = ytm::launch_loss_in<false>(dtype, grad_dtype, a, s);
  }
  if (e != hipSuccess) return fail(YTM_EHIP, std::string("preference_loss failed: ") + hipGetErrorString(e));
  return YTM_OK;
}

}  // extern "C"
