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

constexpr int kAdjustThreads = 256;
constexpr int kChunk = 4096;            // answers of a block
constexpr uint32_t kTold = 0x80000000u; // the answer stands in the prompt

template <typename In, typename Out>
__global__ __launch_bounds__(kAdjustThreads) void adjust_kernel(AdjustArgs a) {
  __shared__ uint32_t counts[kChunk];
  const int64_t n = blockIdx.y;
  const int64_t first = blockIdx.x * (int64_t)kChunk;
  const int here = (int)(a.V - first < kChunk ? a.V - first : kChunk);
  if (a.tokens) {
    for (int i = threadIdx.x; i < kChunk; i += kAdjustThreads) counts[i] = 0u;
    __syncthreads();
    const int64_t length = a.lengths ? (a.lengths[n] < a.T ? a.lengths[n] : a.T) : a.T;
    const int64_t prompt = a.prompt ? a.prompt[n] : 0;
    const int32_t* tokens = a.tokens + n * a.token_stride;
    for (int64_t i = threadIdx.x; i < length; i += kAdjustThreads) {
      const int64_t at = tokens[i] - first;
      if (at >= 0 && at < here) {
        if (i >= prompt)
          atomicAdd(&counts[at], 1u);
        else
          atomicOr(&counts[at], kTold);
      }
    }
    __syncthreads();
  }
  const float repetition = a.repetition ? a.repetition[n] : 1.0f;
  const float frequency = a.frequency ? a.frequency[n] : 0.0f, presence = a.presence ? a.presence[n] : 0.0f;
  const In* in = (const In*)a.scores + n * a.stride + first;
  Out* out = (Out*)a.out + n * a.out_stride + first;
  const float* bias = a.bias ? a.bias + n * a.bias_stride + first : nullptr;
  const uint32_t* allowed = a.allowed ? a.allowed + n * a.allowed_stride + first / 32 : nullptr;
  for (int i = threadIdx.x; i < here; i += kAdjustThreads) {
    float s = to_float(in[i]);
    const uint32_t c = a.tokens ? counts[i] : 0u;
    if (c) {
      s = s > 0.0f ? s / repetition : s * repetition;
      if (c & ~kTold) {
        s -= frequency * (float)(c & ~kTold);
        s -= presence;
      }
    }
    if (bias) s += bias[i];
    if (allowed && !(allowed[i / 32] >> (i % 32) & 1u)) s = -INFINITY;
    out[i] = from_float<Out>(s);
  }
}

template <typename In, typename Out>
hipError_t launch_adjust(const AdjustArgs& a, int64_t N, hipStream_t s) {
  const dim3 grid((unsigned)((a.V + kChunk - 1) / kChunk), (unsigned)N);
  adjust_kernel<In, Out><<<grid, kAdjustThreads, 0, s>>>(a);
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
};

constexpr int kChooseThreads = 1024;
constexpr int kChooseWaves = kChooseThreads / kWave;
constexpr int kDigits = 256;
constexpr float kMass = 1099511627776.0f;  // 2^40

// Floats as whole numbers of the same order (no -0.0, no NaN).
__device__ __forceinline__ uint32_t key_of(float z) {
  const uint32_t u = __float_as_uint(z);
  return u ^ (u >> 31 ? 0xFFFFFFFFu : 0x80000000u);
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key ^ (key >> 31 ? 0x80000000u : 0xFFFFFFFFu));
}
constexpr uint32_t kNone = 0x007FFFFFu;  // key of -inf

template <typename In>
struct Row {
  const In* in;
  float t;
  __device__ __forceinline__ float operator()(int i) const {
    float z = to_float(in[i]) / t;
    z = z != z ? -INFINITY : fminf(z, FLT_MAX);
    return z + 0.0f;
  }
};

__device__ __forceinline__ unsigned long long mass_of(float z, float best) {
  return (unsigned long long)(expf(z - best) * kMass);
}

// The last answer kept: all of a larger key are, and of its own key those up to its index.
struct Cut {
  uint32_t key;
  int last;
  __device__ __forceinline__ bool keeps(uint32_t key_, int i) const { return key_ > key || (key_ == key && i <= last); }
};

struct ChooseShared {
  unsigned long long hist[kDigits];
  unsigned long long part[kChooseWaves];
  unsigned long long above, in;
  int digit;
  int found;
};

__device__ __forceinline__ unsigned long long block_max(unsigned long long v, ChooseShared& sh) {
  for (int d = 32; d; d >>= 1) {
    const unsigned long long o = __shfl_xor(v, d);
    v = o > v ? o : v;
  }
  __syncthreads();
  if (threadIdx.x % kWave == 0) sh.part[threadIdx.x / kWave] = v;
  __syncthreads();
  for (int w = 0; w < kChooseWaves; ++w) v = sh.part[w] > v ? sh.part[w] : v;
  return v;
}

__device__ __forceinline__ unsigned long long block_sum(unsigned long long v, ChooseShared& sh) {
  for (int d = 32; d; d >>= 1) v += __shfl_xor(v, d);
  __syncthreads();
  if (threadIdx.x % kWave == 0) sh.part[threadIdx.x / kWave] = v;
  __syncthreads();
  v = 0;
  for (int w = 0; w < kChooseWaves; ++w) v += sh.part[w];
  return v;
}

// Index of the r-th (from 1) answer of key `key`, in index order.
template <typename In>
__device__ int tie_index(const Row<In>& row, int V, uint32_t key, int r, ChooseShared& sh) {
  int seen = 0;
  if (threadIdx.x == 0) sh.found = V - 1;
  for (int first = 0; first < V; first += kChooseThreads) {
    const int i = first + threadIdx.x;
    const bool tie = i < V && key_of(row(i)) == key;
    const unsigned long long mine = __ballot(tie);
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
__device__ void raise_cut(const Row<In>& row, int V, float best, unsigned long long target, Cut& cut,
                          ChooseShared& sh) {
  uint32_t prefix = 0u, mask = 0u;
  unsigned long long above = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    for (int i = threadIdx.x; i < kDigits; i += kChooseThreads) sh.hist[i] = 0;
    __syncthreads();
    for (int i = threadIdx.x; i < V; i += kChooseThreads) {
      const float z = row(i);
      const uint32_t key = key_of(z);
      if (cut.keeps(key, i) && (key & mask) == prefix)
        atomicAdd(&sh.hist[key >> shift & 255u], MASS ? mass_of(z, best) : 1ull);
    }
    __syncthreads();
    if (threadIdx.x < kWave) {  // lane l takes the digits 255 - 4 l and the three below
      unsigned long long own = 0;
      for (int j = 0; j < 4; ++j) own += sh.hist[kDigits - 1 - 4 * threadIdx.x - j];
      unsigned long long upto = own;
      for (int d = 1; d < kWave; d <<= 1) {
        const unsigned long long o = __shfl_up(upto, d);
        if ((int)threadIdx.x >= d) upto += o;
      }
      const unsigned long long reached = __ballot(above + upto >= target);
      if (threadIdx.x == 0) sh.digit = -1;
      if (reached && (int)threadIdx.x == __ffsll(reached) - 1) {
        unsigned long long sum = above + upto - own;
        int j = kDigits - 1 - 4 * threadIdx.x;
        while (sum + sh.hist[j] < target) sum += sh.hist[j--];
        sh.digit = j;
        sh.above = sum;
        sh.in = sh.hist[j];
      }
    }
    __syncthreads();
    if (sh.digit < 0) return;
    above = sh.above;
    prefix |= (uint32_t)sh.digit << shift;
    mask |= 255u << shift;
  }
  // `above` comes before the answers of key `prefix`, which have `in` together
  const unsigned long long need = target - above;
  const unsigned long long each = MASS ? mass_of(value_of(prefix), best) : 1ull;
  const unsigned long long in = sh.in;
  int last = prefix == cut.key ? cut.last : V - 1;
  if (each && need + each <= in) {  // some of them are left out
    const unsigned long long r = (need + each - 1) / each;
    last = tie_index(row, V, prefix, (int)(r < 1 ? 1 : r), sh);
  }
  cut.key = prefix;
  cut.last = last;
  __syncthreads();
}

template <typename In>
__global__ __launch_bounds__(kChooseThreads) void choose_kernel(ChooseArgs a) {
  __shared__ ChooseShared sh;
  const int64_t n = blockIdx.x;
  const int V = a.V;
  float t = a.temperature ? a.temperature[n] : 1.0f;
  int k = a.top_k ? a.top_k[n] : 0;
  if (t <= 0.0f) {
    t = 1.0f;
    k = 1;
  }
  const Row<In> row{(const In*)a.scores + n * a.stride, t};
  unsigned long long v = 0;
  for (int i = threadIdx.x; i < V; i += kChooseThreads) {
    const unsigned long long key = key_of(row(i));
    v = key > v ? key : v;
  }
  const uint32_t top = (uint32_t)block_max(v, sh);
  if (top <= kNone) {
    if (threadIdx.x == 0) {
      a.tokens[n] = -1;
      a.logprobs[n] = -INFINITY;
    }
    return;
  }
  const float best = value_of(top);
  Cut cut{kNone + 1u, V - 1};
  if (a.min_p && a.min_p[n] > 0.0f) {
    const float least = best + logf(a.min_p[n]);
    const uint32_t key = key_of((least <= best ? least : best) + 0.0f);
    if (key > cut.key) cut.key = key;
  }
  if (k > 0 && k < V) raise_cut<false>(row, V, best, (unsigned long long)k, cut, sh);
  if (a.top_p && !(a.top_p[n] >= 1.0f)) {
    unsigned long long m = 0;
    for (int i = threadIdx.x; i < V; i += kChooseThreads) {
      const float z = row(i);
      if (cut.keeps(key_of(z), i)) m += mass_of(z, best);
    }
    const double target = ceil((double)a.top_p[n] * (double)block_sum(m, sh));
    raise_cut<true>(row, V, best, target > 1.0 ? (unsigned long long)target : 1ull, cut, sh);
  }
  const float* noise = a.noise ? a.noise + n * a.noise_stride : nullptr;
  unsigned long long m = 0, drawn = 0;
  for (int i = threadIdx.x; i < V; i += kChooseThreads) {
    const float z = row(i);
    if (!cut.keeps(key_of(z), i)) continue;
    m += mass_of(z, best);
    float y = noise ? z + noise[i] : z;
    y = y >= -FLT_MAX ? y + 0.0f : -FLT_MAX;
    const unsigned long long w = (unsigned long long)key_of(y) << 32 | (uint32_t)~i;
    drawn = w > drawn ? w : drawn;
  }
  m = block_sum(m, sh);
  drawn = block_max(drawn, sh);
  if (threadIdx.x == 0) {
    const int i = (int)~(uint32_t)drawn;
    a.tokens[n] = i;
    a.logprobs[n] = (row(i) - best) - logf((float)m * (1.0f / kMass));
  }
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
  if (N == 0 || V == 0) return YTM_OK;
  if (!scores || !out || (T > 0 && !tokens)) return fail(YTM_EINVAL, "bad adjust_scores arguments");
  if ((N > 1 && (stride < V || out_stride < V)) || (tokens && N > 1 && token_stride < T) ||
      (bias && bias_stride != 0 && N > 1 && bias_stride < V) ||
      (allowed && allowed_stride != 0 && N > 1 && allowed_stride < (V + 31) / 32))
    return fail(YTM_EINVAL, "adjust_scores: rows overlap");
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

int ytm_choose(const void* scores, int dtype, int64_t stride, int64_t N, int64_t V, const float* temperature,
               const int32_t* top_k, const float* top_p, const float* min_p, const float* noise, int64_t noise_stride,
               int32_t* tokens, float* logprobs, void* stream) {
  if (!ytm::decode_float(dtype)) return fail(YTM_EINVAL, "scores are float32, float16 or bfloat16");
  if (N < 0 || V < 0 || N > INT32_MAX || V > ytm::kMaxScores)
    return fail(YTM_EINVAL, "choose takes at most 8388608 scores a row");
  if (N == 0) return YTM_OK;
  if ((V > 0 && !scores) || !tokens || !logprobs) return fail(YTM_EINVAL, "bad choose arguments");
  if (N > 1 && (stride < V || (noise && noise_stride != 0 && noise_stride < V)))
    return fail(YTM_EINVAL, "choose: rows overlap");
  ytm::ChooseArgs a{scores, stride, (int)V, temperature, top_k, top_p, min_p, noise, noise_stride, tokens, logprobs};
  hipStream_t s = (hipStream_t)stream;
  switch (dtype) {
    case YTM_DTYPE_F16: ytm::choose_kernel<ytm::f16><<<(unsigned)N, ytm::kChooseThreads, 0, s>>>(a); break;
    case YTM_DTYPE_BF16: ytm::choose_kernel<ytm::bf16><<<(unsigned)N, ytm::kChooseThreads, 0, s>>>(a); break;
    default: ytm::choose_kernel<float><<<(unsigned)N, ytm::kChooseThreads, 0, s>>>(a); break;
  }
  const hipError_t e = hipGetLastError();
  if (e != hipSuccess) return fail(YTM_EHIP, std::string("choose failed: ") + hipGetErrorString(e));
  return YTM_OK;
}

}  // extern "C"
