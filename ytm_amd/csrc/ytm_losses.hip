// ytm_losses.hip -- losses of a model's answers with the gradient of the scores: the entry points
// ytm_policy_loss and ytm_preference_loss of include/ytm.h and their gfx950 kernels.
//
// With z = score / temperature, p = softmax(z) over a row and lp = log p of the row's answer t, both losses
// reach the scores through lp alone:
//
//   d loss / d score[v] = c / temperature * ((v == t) - p[v]),  c = d loss / d lp
//
// so a row is read for its maximum and its sum of exp(z - max) (one pass, rescaled where the maximum
// grows), c is found, and the row is read again where it is written.
#include <hip/hip_runtime.h>
#include <float.h>
#include <stdint.h>

#include "ytm_decode.h"
#include "ytm_internal.h"

namespace ytm {

namespace {

constexpr int kWave = 64;
constexpr int kMaxThreads = 1024;
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

// A score that is NaN counts as -inf, one of +inf as the largest float.
template <typename In>
__device__ __forceinline__ float score_of(In v) {
  const float s = to_float(v);
  return s != s ? -INFINITY : fminf(s, FLT_MAX);
}

// 1 / temperature as choose() takes it: 0 or less counts as 1, less than the smallest normal float or NaN as that.
__device__ __forceinline__ float cooling(const LossArgs& a, int n) {
  if (!a.temperature) return 1.0f;
  const float t = a.temperature[n];
  return t <= 0.0f ? 1.0f : 1.0f / (t >= FLT_MIN ? t : FLT_MIN);
}

// A row's maximum and its sum of exp((score - maximum) / temperature), in powers of two.
struct Stats {
  float max, sum;
  __device__ __forceinline__ void add(const Stats& o, float scale) {
    if (o.max == -INFINITY) return;
    if (o.max > max) {
      sum = sum * exp2f((max - o.max) * scale) + o.sum;  // max may be -inf, sum is 0 then
      max = o.max;
    } else {
      sum += o.sum * exp2f((o.max - max) * scale);
    }
  }
};

template <int E, typename T>
__device__ __forceinline__ void load_scores(const T* p, float (&v)[E]) {
  T raw[E];
  __builtin_memcpy(raw, p, sizeof raw);
#pragma unroll
  for (int e = 0; e < E; ++e) v[e] = score_of(raw[e]);
}

// Of the scores first .. last - 1 of a row, each thread's own.
template <typename In>
__device__ __forceinline__ Stats own_stats(const In* row, int first, int last, float scale) {
  constexpr int E = 16 / sizeof(In);
  Stats s{-INFINITY, 0.0f};
  for (int i = first + threadIdx.x * E; i < last; i += blockDim.x * E) {
    float v[E];
    if (i + E <= last) {
      load_scores<E>(row + i, v);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = i + e < last ? score_of(row[i + e]) : -INFINITY;
    }
    float max = v[0];
#pragma unroll
    for (int e = 1; e < E; ++e) max = fmaxf(max, v[e]);
    if (max == -INFINITY) continue;
    if (max > s.max) {
      s.sum *= exp2f((s.max - max) * scale);
      s.max = max;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) s.sum += exp2f((v[e] - s.max) * scale);
  }
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

template <typename In>
__global__ __launch_bounds__(kMaxThreads) void stats_kernel(LossArgs a) {
  __shared__ Stats part[kMaxThreads / kWave];
  const int n = blockIdx.y, slice = blockIdx.x;
  const In* row = (const In*)a.scores + n * a.stride;
  const int first = slice * a.slice, last = first + a.slice < a.V ? first + a.slice : a.V;
  const float scale = cooling(a, n) * kLog2e;
  const Stats s = block_stats(own_stats(row, first, last, scale), scale, part);
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
  if (r.there) r.lp = (float)((double)(z - all.max) * (double)r.cooling - log((double)all.sum));
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

// The policy loss of a row and its derivative by lp.
struct Loss {
  float value, slope;
};
__device__ __forceinline__ Loss policy(const LossArgs& a, int n, const Answer& r) {
  if (!r.there) return Loss{0.0f, 0.0f};
  const float w = a.weights ? a.weights[n] : 1.0f / (float)a.N, adv = a.advantages[n];
  const float ratio = expf(r.lp - a.old[n]);
  const float free = ratio * adv, held = fminf(fmaxf(ratio, a.low), a.high) * adv;
  float value = -fminf(free, held), slope = free <= held ? -free : 0.0f;
  if (a.kl != 0.0f) {
    const float far = a.reference[n] - r.lp, up = expm1f(far);
    value += a.kl * (up - far);
    slope -= a.kl * up;
  }
  return Loss{w * value, w * slope};
}

// The gradient of a row's scores first .. last - 1; c is 0 where the row takes no part.
template <typename In, typename Out>
__device__ __forceinline__ void write_grad(const LossArgs& a, int n, int first, int last, const Answer& r, float c) {
  constexpr int E = 8;
  const In* row = (const In*)a.scores + n * a.stride;
  Out* to = (Out*)a.grad + n * a.grad_stride;
  const int t = a.tokens[n];
  const bool any = r.there && c != 0.0f;
  const float by = any ? c * r.cooling : 0.0f, each = any ? -by / r.all.sum : 0.0f, scale = r.cooling * kLog2e;
  for (int i = first + threadIdx.x * E; i < last; i += blockDim.x * E) {
    float v[E];
    const bool whole = i + E <= last;
    if (!any) {
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = 0.0f;
    } else {
      if (whole) {
        load_scores<E>(row + i, v);
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] = i + e < last ? score_of(row[i + e]) : -INFINITY;
      }
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] = each * exp2f((v[e] - r.all.max) * scale) + (i + e == t ? by : 0.0f);
    }
    Out raw[E];
#pragma unroll
    for (int e = 0; e < E; ++e) raw[e] = from_float<Out>(v[e]);
    if (whole) {
      __builtin_memcpy(to + i, raw, sizeof raw);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (i + e < last) to[i + e] = raw[e];
    }
  }
}

// A slice of a row, after stats_kernel, and after pair_kernel for preferences.
template <typename In, typename Out, bool POLICY>
__global__ __launch_bounds__(kMaxThreads) void grad_kernel(LossArgs a) {
  const int n = blockIdx.y, first = blockIdx.x * a.slice, last = first + a.slice < a.V ? first + a.slice : a.V;
  const Answer r = answer_of(a, n);
  float c;
  if (POLICY) {
    const Loss loss = policy(a, n, r);
    c = loss.slope;
    if (blockIdx.x == 0 && threadIdx.x == 0) {
      a.losses[n] = loss.value;
      a.logprobs[n] = r.lp;
    }
  } else {
    c = a.slope[n];
  }
  write_grad<In, Out>(a, n, first, last, r, c);
}

// A policy loss's whole row.
template <typename In, typename Out>
__global__ __launch_bounds__(kMaxThreads) void policy_kernel(LossArgs a) {
  __shared__ Stats part[kMaxThreads / kWave];
  const int n = blockIdx.x;
  const In* row = (const In*)a.scores + n * a.stride;
  const int t = a.tokens[n];
  const float scale = cooling(a, n) * kLog2e;
  const float z = t >= 0 && t < a.V ? score_of(row[t]) : -INFINITY;
  const Stats all = block_stats(own_stats(row, 0, a.V, scale), scale, part);
  const Answer r = answer_of(a, n, z, all);
  const Loss loss = policy(a, n, r);
  if (threadIdx.x == 0) {
    a.losses[n] = loss.value;
    a.logprobs[n] = r.lp;
  }
  write_grad<In, Out>(a, n, 0, a.V, r, loss.slope);
}

// A pair of sequences a block: their log probabilities, the loss, and its derivative for their rows.
constexpr int kPairThreads = 256;
__global__ __launch_bounds__(kPairThreads) void pair_kernel(LossArgs a) {
  __shared__ double part[2][kPairThreads / kWave];
  const int pair = blockIdx.x;
  int begin[2], end[2];
  double said[2];
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    begin[side] = a.starts[2 * pair + side];
    end[side] = a.starts[2 * pair + side + 1];
    begin[side] = begin[side] < 0 ? 0 : begin[side];
    end[side] = end[side] > a.N ? a.N : end[side];
    double sum = 0.0;
    for (int64_t n = begin[side] + (int64_t)threadIdx.x; n < end[side]; n += kPairThreads)
      sum += (double)answer_of(a, (int)n).lp;
#pragma unroll
    for (int d = 1; d < kWave; d <<= 1) sum += __shfl_xor(sum, d);
    if (threadIdx.x % kWave == 0) part[side][threadIdx.x / kWave] = sum;
  }
  __syncthreads();
#pragma unroll
  for (int side = 0; side < 2; ++side) {
    said[side] = 0.0;
    for (int w = 0; w < kPairThreads / kWave; ++w) said[side] += part[side][w];
  }
  const float* ref = a.sequence_reference + 2 * pair;
  const float m = (float)((double)a.beta * ((said[0] - (double)ref[0]) - (said[1] - (double)ref[1])));
  const float small = expf(-fabsf(m));  // softplus(m) = max(m, 0) + log(1 + exp(-|m|)), sigmoid(m) alike
  const float share = 1.0f / (float)a.pairs;
  const float won = (m >= 0.0f ? 1.0f : small) / (1.0f + small), lost = (m >= 0.0f ? small : 1.0f) / (1.0f + small);
  const float c = share * a.beta * (a.smoothing * won - (1.0f - a.smoothing) * lost);
  if (threadIdx.x == 0) {
    const float log1 = log1pf(small);
    a.losses[pair] =
        share * ((1.0f - a.smoothing) * (fmaxf(-m, 0.0f) + log1) + a.smoothing * (fmaxf(m, 0.0f) + log1));
    a.logprobs[2 * pair] = (float)said[0];
    a.logprobs[2 * pair + 1] = (float)said[1];
  }
#pragma unroll
  for (int side = 0; side < 2; ++side)
    for (int64_t n = begin[side] + (int64_t)threadIdx.x; n < end[side]; n += kPairThreads)
      a.slope[n] = side ? -c : c;
}

// --------------------------------------------------------------------------------------- host
int threads_of(int64_t scores) { return scores <= 1024 ? 64 : scores <= 16384 ? 256 : 1024; }

// Slices of a row: rows alone fill the 256 CUs, or a slice would have less than 4096 scores.
int slices_of(int64_t N, int64_t V) {
  int64_t slices = N > 0 ? 512 / N : 1;
  if (slices > V / 4096) slices = V / 4096;
  return slices < 1 ? 1 : slices > kMaxSlices ? kMaxSlices : (int)slices;
}

int64_t workspace_bytes_of(int64_t N, int64_t slices) { return N * (slices * 8 + 8); }

template <typename In, typename Out, bool POLICY>
hipError_t launch_loss(LossArgs a, hipStream_t s) {
  if (POLICY && a.slices == 1) {
    policy_kernel<In, Out><<<a.N, threads_of(a.V), 0, s>>>(a);
    return hipGetLastError();
  }
  const dim3 grid(a.slices, a.N);
  const int threads = threads_of(a.slice);
  stats_kernel<In><<<grid, threads, 0, s>>>(a);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && !POLICY) {
    pair_kernel<<<a.pairs, kPairThreads, 0, s>>>(a);
    e = hipGetLastError();
  }
  if (e != hipSuccess) return e;
  grad_kernel<In, Out, POLICY><<<grid, threads, 0, s>>>(a);
  return hipGetLastError();
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
