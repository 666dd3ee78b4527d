// ytm_adamw.hip -- an AdamW step over many tensors at once: the entry points ytm_adamw_table and
// ytm_adamw of include/ytm.h and their gfx950 kernels.
//
//   m = beta1 m + (1 - beta1) g, v = beta2 v + (1 - beta2) g^2
//   p = (1 - rate decay) p - rate / (1 - beta1^k) m / (sqrt(v) / sqrt(1 - beta2^k) + eps)
//
// in f32 in this order of operations, each rounded, from states in f32, or in 8 bits: E4M3 floats with a power of two
// for each 256 elements, m itself and v as its root.  What is stored in fewer bits is rounded up or
// down at random with the chances that keep its mean: a step of 1 - beta2 of the state is less than
// half the distance of two codes, so that the nearest one would stay for ever.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "ytm_decode.h"
#include "ytm_internal.h"

namespace ytm {

namespace {

constexpr int kWave = 64;
constexpr int kThreads = 256;
constexpr int kBlock = 256;    // elements of a state in 8 bits that share a scale
constexpr int kChunk = 4096;   // elements of a workgroup
constexpr int kEach = 4;       // elements of a thread, in a row
static_assert(kEach * kWave == kBlock, "a wave finds a scale");

// What a tensor's workgroups take from the number of its step; `active` 0: it takes no step.
struct Step {
  float beta1, rest1, beta2, rest2, keep, rate, cool, eps;
  uint32_t key;
  int32_t active;
};

// One of the tensors, as it is in the table.
struct Tensor {
  void* parameter;
  const void* gradient;
  void *first, *second;
  float *first_scales, *second_scales;
  int64_t count;
  uint64_t place;  // of its first element among all tensors', each a multiple of kBlock long
  int32_t parameter_dtype, gradient_dtype;
  Step step;
};

// A workgroup's tensor and its elements' number in it, in chunks.
struct Chunk {
  int32_t tensor, chunk;
};
static_assert(sizeof(Tensor) % 16 == 0 && sizeof(Chunk) == 8, "");

// Murmur3's finaliser (Appleby): every bit of the result depends on every bit of h.
__device__ __forceinline__ uint32_t mixed(uint32_t h) {
  h ^= h >> 16;
  h *= 0x85EBCA6Bu;
  h ^= h >> 13;
  h *= 0xC2B2AE35u;
  return h ^ h >> 16;
}

// Counts the steps of the tensors that take one, and what follows from it, in double.
__global__ __launch_bounds__(kThreads) void step_kernel(Tensor* tensors, int n, int64_t* steps, const uint8_t* active,
                                                        double rate, const float* rate_at, double beta1, double beta2,
                                                        double eps, double decay, uint32_t seed) {
  const int i = blockIdx.x * kThreads + threadIdx.x;
  if (i >= n) return;
  Step s{};
  s.active = !active || active[i] != 0;
  if (s.active) {
    const int64_t k = ++steps[i];
    if (rate_at) rate = *rate_at;
    s.beta1 = (float)beta1, s.rest1 = (float)(1.0 - beta1), s.beta2 = (float)beta2, s.rest2 = (float)(1.0 - beta2);
    s.keep = (float)(1.0 - rate * decay);
    s.rate = (float)(rate / (1.0 - pow(beta1, (double)k)));
    s.cool = (float)(1.0 / sqrt(1.0 - pow(beta2, (double)k)));
    s.eps = (float)eps;
    s.key = mixed(mixed((uint32_t)k) ^ seed);
  }
  tensors[i].step = s;
}

// Random bits of element `place` in this step: 16 for each state, 16 for the parameter.
struct Chances {
  float first, second, parameter;
};
__device__ __forceinline__ Chances chances_of(uint64_t place, uint32_t key) {
  const uint32_t a = mixed((uint32_t)place ^ key ^ (uint32_t)(place >> 32) * 0xC2B2AE35u), b = a * 0x9E3779B9u;
  constexpr float k = 1.0f / 65536.0f;
  return Chances{(float)(a & 0xFFFFu) * k, (float)(a >> 16) * k, (float)(b >> 16) * k};
}

// The distance of the numbers of `fraction` bits and of at least 2^least at x >= 0, and its reciprocal.
__device__ __forceinline__ void step_of(float x, int fraction, int least, float& step, float& inverse) {
  int e = (int)(__float_as_uint(x) >> 23) - 127;
  e = e < least ? least : e;
  step = ldexpf(1.0f, e - fraction);
  inverse = ldexpf(1.0f, fraction - e);
}

// x to a number of `fraction` bits and at least 2^least: down, or up with the chance of what is cut off.
__device__ __forceinline__ float drawn_to(float x, float chance, int fraction, int least) {
  float step, inverse;
  step_of(fabsf(x), fraction, least, step, inverse);
  return copysignf(floorf(fabsf(x) * inverse + chance) * step, x);
}

__device__ __forceinline__ float stored(float v, float, float) { return v; }
__device__ __forceinline__ f16 stored(float v, float chance, f16) {
  return (f16)(v - v == 0.0f ? drawn_to(v, chance, 10, -14) : v);
}
__device__ __forceinline__ bf16 stored(float v, float chance, bf16) {
  return from_float<bf16>(v - v == 0.0f ? drawn_to(v, chance, 7, -126) : v);
}

template <typename T>
__device__ __forceinline__ void load_each(const T* p, int left, float (&v)[kEach]) {
  T raw[kEach];
  if (left >= kEach) {
    __builtin_memcpy(raw, p, sizeof raw);
#pragma unroll
    for (int e = 0; e < kEach; ++e) v[e] = to_float(raw[e]);
  } else {
#pragma unroll
    for (int e = 0; e < kEach; ++e) v[e] = e < left ? to_float(p[e]) : 0.0f;
  }
}
template <typename T>
__device__ __forceinline__ void store_each(T* p, int left, const T (&v)[kEach]) {
  if (left >= kEach) {
    __builtin_memcpy(p, v, sizeof v);
  } else {
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      if (e < left) p[e] = v[e];
  }
}

// An E4M3 float (sign, four bits of exponent, three of fraction; 2^-9 the least, 448 the largest, 127 a
// NaN) of a number that is one, and back.
__device__ __forceinline__ uint8_t code_of(float v) {
  const uint32_t sign = __float_as_uint(v) >> 24 & 0x80u;
  const float x = fabsf(v);
  if (!(x <= 448.0f)) return (uint8_t)(sign | 0x7Fu);
  if (x < 0.015625f) return (uint8_t)(sign | (uint32_t)(x * 512.0f));
  return (uint8_t)(sign | ((__float_as_uint(x) >> 20) - (120u << 3)));
}
__device__ __forceinline__ float value_of(uint8_t c) {
  const uint32_t m = c & 0x7Fu;
  const float x = m == 0x7Fu ? __uint_as_float(0x7FC00000u)
                  : m < 8    ? (float)m * (1.0f / 512.0f)
                             : __uint_as_float((m + (120u << 3)) << 20);
  return c & 0x80u ? -x : x;
}

// The exponent of a block's scale: 2^e 448 is the least such number that its largest magnitude does not
// pass, and at least 2^-98, so that no product leaves what float32 holds.  What is not finite has no part.
__device__ __forceinline__ int exponent_of(const float (&v)[kEach]) {
  uint32_t most = 0;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const uint32_t u = __float_as_uint(v[e]) & 0x7FFFFFFFu;
    if (u < 0x7F800000u && u > most) most = u;
  }
#pragma unroll
  for (int d = 1; d < kWave; d <<= 1) {
    const uint32_t o = __shfl_xor(most, d);
    most = o > most ? o : most;
  }
  const int bits = (int)((most + 0x1FFFFFu) >> 23);
  return (bits < 37 ? 37 : bits) - 135;
}

template <int BITS, typename P, typename G>
__device__ __forceinline__ void update(const Tensor& t, const Step& s, int64_t i, int left) {
  float p[kEach], g[kEach], m[kEach], v[kEach], root[kEach];
  load_each((const P*)t.parameter + i, left, p);
  load_each((const G*)t.gradient + i, left, g);
  if (BITS == 32) {
    load_each((const float*)t.first + i, left, m);
    load_each((const float*)t.second + i, left, v);
  } else {
    uint8_t c[2][kEach] = {};
    float scale[2] = {0.0f, 0.0f};
    if (left > 0) {
      scale[0] = t.first_scales[i / kBlock];
      scale[1] = t.second_scales[i / kBlock];
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const uint8_t* from = (const uint8_t*)(q ? t.second : t.first) + i;
        if (left >= kEach) {
          __builtin_memcpy(c[q], from, kEach);
        } else {
#pragma unroll
          for (int e = 0; e < kEach; ++e)
            if (e < left) c[q][e] = from[e];
        }
      }
    }
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      m[e] = value_of(c[0][e]) * scale[0];
      v[e] = value_of(c[1][e]) * scale[1];
      v[e] *= v[e];
    }
  }
  P out[kEach];
  Chances chance[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    m[e] = s.beta1 * m[e] + s.rest1 * g[e];
    v[e] = s.beta2 * v[e] + s.rest2 * (g[e] * g[e]);
    root[e] = sqrtf(v[e]);
    if (BITS == 8 || sizeof(P) == 2) chance[e] = chances_of(t.place + i + e, s.key);
    const float next = p[e] * s.keep - s.rate * m[e] / (root[e] * s.cool + s.eps);
    out[e] = stored(next, chance[e].parameter, P{});
  }
  store_each((P*)t.parameter + i, left, out);
  if (BITS == 32) {
    store_each((float*)t.first + i, left, m);
    store_each((float*)t.second + i, left, v);
    return;
  }
  uint8_t c[2][kEach];
  const int e1 = exponent_of(m), e2 = exponent_of(root);
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    c[0][e] = m[e] - m[e] == 0.0f ? code_of(drawn_to(ldexpf(m[e], -e1), chance[e].first, 3, -6)) : (uint8_t)0x7F;
    // v between the squares of two codes: up with the chance that keeps its mean; above zero it stays above
    const float x = ldexpf(root[e], -e2);
    float step, inverse;
    step_of(x, 3, -6, step, inverse);
    const float low = floorf(x * inverse) * step, high = low + step;
    const bool up = x * x - low * low > chance[e].second * (high * high - low * low) || (low == 0.0f && x > 0.0f);
    c[1][e] = x - x == 0.0f ? code_of(up ? high : low) : (uint8_t)0x7F;
  }
  store_each((uint8_t*)t.first + i, left, c[0]);
  store_each((uint8_t*)t.second + i, left, c[1]);
  if (i % kBlock == 0 && left > 0) {
    t.first_scales[i / kBlock] = ldexpf(1.0f, e1);
    t.second_scales[i / kBlock] = ldexpf(1.0f, e2);
  }
}

template <int BITS, typename P, typename G>
__device__ __forceinline__ void update_chunk(const Tensor& t, const Step& s, int64_t first) {
  for (int64_t i = first + threadIdx.x * kEach; i < first + kChunk; i += kThreads * kEach) {
    // a wave goes on together: its lanes share a scale
    if (i - threadIdx.x % kWave * kEach >= t.count) return;
    const int64_t left = t.count - i;
    update<BITS, P, G>(t, s, i, left < 0 ? 0 : left > kEach ? kEach : (int)left);
  }
}

template <int BITS, typename P>
__device__ __forceinline__ void update_gradient(const Tensor& t, const Step& s, int64_t first) {
  if (t.gradient_dtype == YTM_DTYPE_F32)
    update_chunk<BITS, P, float>(t, s, first);
  else
    update_chunk<BITS, P, P>(t, s, first);
}

template <int BITS>
__global__ __launch_bounds__(kThreads) void adamw_kernel(const Tensor* tensors, const Chunk* chunks) {
  const Chunk c = chunks[blockIdx.x];
  const Tensor t = tensors[c.tensor];
  const Step& s = t.step;
  if (!s.active) return;
  const int64_t first = (int64_t)c.chunk * kChunk;
  switch (t.parameter_dtype) {
    case YTM_DTYPE_F16: update_gradient<BITS, f16>(t, s, first); break;
    case YTM_DTYPE_BF16: update_gradient<BITS, bf16>(t, s, first); break;
    default: update_gradient<BITS, float>(t, s, first); break;
  }
}

constexpr int64_t kMaxTensors = 1 << 24;
// Chunks of a table, whose workgroups' threads one launch counts in 32 bits: 68 G elements.
constexpr int64_t kMaxChunks = UINT32_MAX / kThreads;

}  // namespace

}  // namespace ytm

using ytm::fail;

extern "C" {

int ytm_adamw_table(const ytm_adamw_tensor* tensors, int64_t n, int bits, void* table, int64_t* bytes,
                    int64_t* chunks) {
  if (!bytes || !chunks || n < 0 || n > ytm::kMaxTensors || (n > 0 && !tensors) || (bits != 8 && bits != 32))
    return fail(YTM_EINVAL, "bad adamw_table arguments: at most 16777216 tensors, states of 8 or 32 bits");
  int64_t total = 0;
  for (int64_t i = 0; i < n; ++i) {
    const ytm_adamw_tensor& t = tensors[i];
    if (t.count < 0 || t.count > INT64_MAX / 64) return fail(YTM_EINVAL, "adamw: a tensor's size");
    if (!ytm::decode_float(t.parameter_dtype) ||
        (t.gradient_dtype != t.parameter_dtype && t.gradient_dtype != YTM_DTYPE_F32))
      return fail(YTM_EINVAL, "adamw: parameters are float32, float16 or bfloat16, gradients of the same type or float32");
    if (t.count > 0 && (!t.parameter || !t.gradient || !t.first || !t.second ||
                        (bits == 8 && (!t.first_scales || !t.second_scales))))
      return fail(YTM_EINVAL, "adamw: an operand is missing");
    total += (t.count + ytm::kChunk - 1) / ytm::kChunk;
    if (total > ytm::kMaxChunks) return fail(YTM_EINVAL, "adamw: the tensors have more elements than one step takes");
  }
  *chunks = total;
  *bytes = n * (int64_t)sizeof(ytm::Tensor) + total * (int64_t)sizeof(ytm::Chunk);
  if (!table) return YTM_OK;
  ytm::Tensor* to = (ytm::Tensor*)table;
  ytm::Chunk* chunk = (ytm::Chunk*)(to + n);
  uint64_t place = 0;
  for (int64_t i = 0; i < n; ++i) {
    const ytm_adamw_tensor& t = tensors[i];
    to[i] = ytm::Tensor{t.parameter, t.gradient, t.first, t.second, t.first_scales, t.second_scales, t.count, place,
                        t.parameter_dtype, t.gradient_dtype, ytm::Step{}};
    place += (uint64_t)((t.count + ytm::kBlock - 1) / ytm::kBlock * ytm::kBlock);
    for (int64_t c = 0; c * ytm::kChunk < t.count; ++c) *chunk++ = ytm::Chunk{(int32_t)i, (int32_t)c};
  }
  return YTM_OK;
}

int ytm_adamw(void* table, int64_t n, int64_t chunks, int bits, int64_t* steps, const uint8_t* active, double rate,
              const float* rate_at, double beta1, double beta2, double eps, double decay, uint32_t seed, void* stream) {
  if (n < 0 || n > ytm::kMaxTensors || chunks < 0 || chunks > ytm::kMaxChunks || (bits != 8 && bits != 32))
    return fail(YTM_EINVAL, "bad adamw arguments");
  if (!(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(eps >= 0.0))
    return fail(YTM_EINVAL, "adamw: betas are 0 or more and below 1, eps is 0 or more");
  if (n == 0) return YTM_OK;
  if (!table || (uintptr_t)table % 16 || !steps) return fail(YTM_EINVAL, "bad adamw arguments");
  ytm::Tensor* tensors = (ytm::Tensor*)table;
  const ytm::Chunk* of = (const ytm::Chunk*)(tensors + n);
  hipStream_t s = (hipStream_t)stream;
  ytm::step_kernel<<<(unsigned)((n + ytm::kThreads - 1) / ytm::kThreads), ytm::kThreads, 0, s>>>(
      tensors, (int)n, steps, active, rate, rate_at, beta1, beta2, eps, decay, seed);
  hipError_t e = hipGetLastError();
  if (e == hipSuccess && chunks > 0) {
    if (bits == 8)
      ytm::adamw_kernel<8><<<(unsigned)chunks, ytm::kThreads, 0, s>>>(tensors, of);
    else
      ytm::adamw_kernel<32><<<(unsigned)chunks, ytm::kThreads, 0, s>>>(tensors, of);
    e = hipGetLastError();
  }
  if (e != hipSuccess) return fail(YTM_EHIP, std::string("adamw failed: ") + hipGetErrorString(e));
  return YTM_OK;
}

}  // extern "C"
