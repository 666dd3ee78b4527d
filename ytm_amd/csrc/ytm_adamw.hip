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
//
// Bound by memory: 62.1 M bfloat16 parameters with f32 states (1.37 GB) 269 us, 5.1 TB/s.  With states in 8 bits the
// coding takes 72% of the vector units' time: 21.1 M f32 parameters (339 MB) 75 us, 4.5 TB/s; in f32 (592 MB) 120.
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

__device__ double power(double x, int64_t k) {
  double r = 1.0;
  for (; k > 0; k >>= 1, x *= x)
    if (k & 1) r *= x;
  return r;
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
    s.rate = (float)(rate / (1.0 - power(beta1, k)));
    s.cool = (float)(1.0 / sqrt(1.0 - power(beta2, k)));
    s.eps = (float)eps;
    s.key = mixed(mixed((uint32_t)k) ^ seed);
  }
  tensors[i].step = s;
}

// Random bits of element `place` + e (of four in a row, the first a multiple of four) in this step, 16 for
// each state and for the parameter.
struct Chances {
  uint32_t first, second, parameter;
};
__device__ __forceinline__ Chances chances_of(uint64_t place, int e, uint32_t key) {
  const uint32_t a = mixed((uint32_t)place + e ^ key ^ (uint32_t)(place >> 32) * 0xC2B2AE35u), b = a * 0x9E3779B9u;
  return Chances{a & 0xFFFFu, a >> 16, b >> 16};
}
__device__ __forceinline__ float share_of(uint32_t chance) { return (float)chance * (1.0f / 65536.0f); }

// x to a number of `fraction` bits and at least 2^least: down, or up with the chance of what is cut off.
__device__ __forceinline__ float drawn_to(float x, uint32_t chance, int fraction, int least) {
  int e = (int)(__float_as_uint(x) >> 23 & 255u) - 127;
  e = e < least ? least : e;
  const float up = floorf(ldexpf(fabsf(x), fraction - e) + share_of(chance));
  return copysignf(ldexpf(up, e - fraction), x);
}

__device__ __forceinline__ float stored(float v, uint32_t, float) { return v; }
__device__ __forceinline__ f16 stored(float v, uint32_t chance, f16) {
  return (f16)(v - v == 0.0f ? drawn_to(v, chance, 10, -14) : v);
}
// A bfloat16 is a float's upper half, subnormal numbers too: what the sum carries into it.
__device__ __forceinline__ bf16 stored(float v, uint32_t chance, bf16) {
  return v - v == 0.0f ? bf16{(uint16_t)(__float_as_uint(v) + chance >> 16)} : from_float<bf16>(v);
}

// Addresses from a table: of device memory, at a multiple of an element's size.
#define YTM_DEVICE __attribute__((address_space(1)))
template <typename T>
__device__ __forceinline__ YTM_DEVICE T* device(const void* p) {
  return (YTM_DEVICE T*)p;
}
template <int BYTES>
struct Four;  // elements
template <>
struct Four<1> {
  typedef uint8_t one;
  typedef uint32_t type __attribute__((aligned(1)));
};
template <>
struct Four<2> {
  typedef uint16_t one;
  typedef uint32_t type __attribute__((ext_vector_type(2), aligned(2)));
};
template <>
struct Four<4> {
  typedef uint32_t one;
  typedef uint32_t type __attribute__((ext_vector_type(4), aligned(4)));
};

template <typename T>
__device__ __forceinline__ void load_raw(YTM_DEVICE T* p, int left, T (&raw)[kEach]) {
  typedef typename Four<sizeof(T)>::one One;
  if (left >= kEach) {
    const auto v = *(YTM_DEVICE typename Four<sizeof(T)>::type*)p;
    __builtin_memcpy(raw, &v, sizeof raw);
  } else {
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      One v = 0;
      if (e < left) v = ((YTM_DEVICE One*)p)[e];
      __builtin_memcpy(&raw[e], &v, sizeof v);
    }
  }
}
template <typename T>
__device__ __forceinline__ void load_each(YTM_DEVICE T* p, int left, float (&v)[kEach]) {
  T raw[kEach];
  load_raw(p, left, raw);
#pragma unroll
  for (int e = 0; e < kEach; ++e) v[e] = to_float(raw[e]);
}
template <typename T>
__device__ __forceinline__ void store_each(YTM_DEVICE T* p, int left, const T (&v)[kEach]) {
  typedef typename Four<sizeof(T)>::one One;
  typename Four<sizeof(T)>::type all;
  __builtin_memcpy(&all, v, sizeof v);
  if (left >= kEach) {
    *(YTM_DEVICE typename Four<sizeof(T)>::type*)p = all;
  } else {
    One one[kEach];
    __builtin_memcpy(one, v, sizeof v);
#pragma unroll
    for (int e = 0; e < kEach; ++e)
      if (e < left) ((YTM_DEVICE One*)p)[e] = one[e];
  }
}

// Four E4M3 floats (sign, four bits of exponent, three of fraction; 2^-9 the least, 448 the largest, 127 a NaN).
__device__ __forceinline__ void values_of(const uint8_t (&from)[kEach], float (&v)[kEach]) {
  uint32_t codes;
  __builtin_memcpy(&codes, from, sizeof codes);
  const auto low = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, false);
  const auto high = __builtin_amdgcn_cvt_pk_f32_fp8((int)codes, true);
  v[0] = low[0], v[1] = low[1], v[2] = high[0], v[3] = high[1];
}

// Codes of a magnitude x up to 448: that below it, and whether it is one of the equally spaced ones near 0.  A normal
// one's bits are the float's from its third of fraction on, less 120 of exponent.
constexpr float kNormal = 0.015625f;
__device__ __forceinline__ uint32_t normal_code(uint32_t bits) { return (bits >> 20) - (120u << 3); }

// Down, or up with the chance of what is cut off.
__device__ __forceinline__ uint32_t first_code(float m, uint32_t chance) {
  const uint32_t u = __float_as_uint(m), x = u & 0x7FFFFFFFu;
  const uint32_t normal = normal_code(x + (chance << 4));
  const uint32_t small = (uint32_t)(__uint_as_float(x) * 512.0f + share_of(chance));
  const uint32_t code = __uint_as_float(x) < kNormal ? small : normal;
  return x < 0x7F800000u ? code | u >> 24 & 0x80u : 0x7Fu;
}

// x is the root of a number between the squares of two codes: up with the chance that keeps the square's mean;
// above zero it stays above.
__device__ __forceinline__ uint32_t second_code(float x, uint32_t chance) {
  const uint32_t u = __float_as_uint(x);
  const bool tiny = x < kNormal;
  const uint32_t code = tiny ? (uint32_t)(x * 512.0f) : normal_code(u);
  const float low = tiny ? (float)code * (1.0f / 512.0f) : __uint_as_float(u & 0xFFF00000u);
  const float step = tiny ? 1.0f / 512.0f : __uint_as_float((u & 0x7F800000u) - (3u << 23)), high = low + step;
  const bool up = x * x - low * low > share_of(chance) * (high * high - low * low) || (code == 0u && x > 0.0f);
  return u < 0x7F800000u ? code + up : 0x7Fu;
}

// The roots of v >= 0: an estimate of 1 / root to a unit in its last place and one step to the root
// nearest to v; outside the normal floats the library's.
__device__ __forceinline__ void roots_of(const float (&v)[kEach], float (&root)[kEach]) {
  bool normal = true;
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const float y = __builtin_amdgcn_rsqf(v[e]), s = v[e] * y;
    root[e] = __builtin_fmaf(__builtin_fmaf(-s, s, v[e]), 0.5f * y, s);
    normal &= v[e] >= 0x1p-126f && v[e] < INFINITY;
  }
  if (normal) return;
#pragma unroll 1
  for (int e = 0; e < kEach; ++e) {
    float one = 0.0f;
#pragma unroll
    for (int q = 0; q < kEach; ++q) one = q == e ? v[q] : one;
    one = sqrtf(one);
#pragma unroll
    for (int q = 0; q < kEach; ++q) root[q] = q == e ? one : root[q];
  }
}

// Exponents of a block's two scales: 2^e 448 is the least such number that its largest magnitude does not
// pass, at least 2^-98, so that no product leaves what float32 holds, and of roots at least 2^-54, so that the square
// of the least code, 2^-9 of it, is a normal float and not 0 (a block of zeros alone has 2^-98).  What is not finite
// has no part.
typedef uint16_t v2h __attribute__((ext_vector_type(2)));
template <int CONTROL>
__device__ __forceinline__ v2h larger_of_row(v2h v) {
  const int o = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CONTROL, 0xF, 0xF, false);
  return __builtin_elementwise_max(v, __builtin_bit_cast(v2h, o));
}
__device__ __forceinline__ void exponents_of(const float (&m)[kEach], const float (&root)[kEach], int& first, int& second) {
  uint32_t most[2] = {0u, 0u};
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    const uint32_t a = __float_as_uint(m[e]) & 0x7FFFFFFFu, b = __float_as_uint(root[e]) & 0x7FFFFFFFu;
    most[0] = a > most[0] ? a : most[0];
    most[1] = b > most[1] ? b : most[1];
  }
  if (__any(most[0] >= 0x7F800000u || most[1] >= 0x7F800000u)) {
    most[0] = most[1] = 0u;
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      const uint32_t a = __float_as_uint(m[e]) & 0x7FFFFFFFu, b = __float_as_uint(root[e]) & 0x7FFFFFFFu;
      most[0] = a > most[0] && a < 0x7F800000u ? a : most[0];
      most[1] = b > most[1] && b < 0x7F800000u ? b : most[1];
    }
  }
  // the exponent of what comes after 1.75 times a power of two is the next
  v2h v = {(uint16_t)(most[0] + 0x1FFFFFu >> 23), (uint16_t)(most[1] + 0x1FFFFFu >> 23)};
  v = larger_of_row<0x128>(v);  // of the 16 lanes of a row, turned by 8, 4, 2 and 1
  v = larger_of_row<0x124>(v);
  v = larger_of_row<0x122>(v);
  v = larger_of_row<0x121>(v);
  const uint32_t u = __builtin_bit_cast(uint32_t, v);
  const auto rows = __builtin_amdgcn_permlane16_swap(u, u, false, false);
  v = __builtin_elementwise_max(__builtin_bit_cast(v2h, (uint32_t)rows[0]), __builtin_bit_cast(v2h, (uint32_t)rows[1]));
  const uint32_t w = __builtin_bit_cast(uint32_t, v);
  const auto halves = __builtin_amdgcn_permlane32_swap(w, w, false, false);
  v = __builtin_elementwise_max(__builtin_bit_cast(v2h, (uint32_t)halves[0]),
                                __builtin_bit_cast(v2h, (uint32_t)halves[1]));
  // the root of any float above 0 is 2^-75 or more: a 0 here is a block of zeros
  v = __builtin_elementwise_max(v, (v2h{37, (uint16_t)(v[1] ? 81 : 37)}));
  first = (int)v[0] - 135, second = (int)v[1] - 135;
}

__device__ __forceinline__ float power_of(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }

// Four elements from i on, of which `left` are there (WHOLE: all of the wave's are).
template <int BITS, bool WHOLE, typename P, typename G>
__device__ __forceinline__ void update(const Tensor& t, const Step& s, int64_t i, int some) {
  const int left = WHOLE ? kEach : some;
  const auto at = device<P>(t.parameter) + i;
  const auto first = device<uint8_t>(t.first) + i, second = device<uint8_t>(t.second) + i;
  float p[kEach], g[kEach], m[kEach], v[kEach], root[kEach];
  if (BITS == 32) {
    load_each(device<float>(t.first) + i, left, m);
    load_each(device<float>(t.second) + i, left, v);
    load_each(at, left, p);
    load_each(device<G>(t.gradient) + i, left, g);
  } else {
    uint8_t codes[2][kEach];
    load_raw(first, left, codes[0]);
    load_raw(second, left, codes[1]);
    float scale[2] = {0.0f, 0.0f};  // lanes past the end have a part in the wave's exponents
    if (left > 0) {
      scale[0] = device<float>(t.first_scales)[i / kBlock];
      scale[1] = device<float>(t.second_scales)[i / kBlock];
    }
    load_each(at, left, p);
    load_each(device<G>(t.gradient) + i, left, g);
    values_of(codes[0], m);
    values_of(codes[1], v);
#pragma unroll
    for (int e = 0; e < kEach; ++e) {
      m[e] *= scale[0];
      v[e] *= scale[1];
      v[e] *= v[e];
    }
  }
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    m[e] = s.beta1 * m[e] + s.rest1 * g[e];
    v[e] = s.beta2 * v[e] + s.rest2 * (g[e] * g[e]);
    if (BITS == 32) root[e] = sqrtf(v[e]);
  }
  if (BITS == 8) roots_of(v, root);
  P out[kEach];
  Chances chance[kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    if (BITS == 8 || sizeof(P) == 2) chance[e] = chances_of(t.place + i, e, s.key);
    // With f32 states the quotient is rounded once, which memory hides (21.1 M f32 parameters 126.8 us, with a
    // reciprocal 126.5).  With 8 bits, whose codes are 6% apart, it is a product with a reciprocal, two units in the last
    // place off at most (163.7 us for 62.1 M bfloat16 parameters, with the quotient 175.9).
    const float by = root[e] * s.cool + s.eps, most = s.rate * m[e];
    const float next = p[e] * s.keep - (BITS == 32 ? most / by : most * __builtin_amdgcn_rcpf(by));
    out[e] = stored(next, chance[e].parameter, P{});
  }
  store_each(at, left, out);
  if (BITS == 32) {
    store_each(device<float>(t.first) + i, left, m);
    store_each(device<float>(t.second) + i, left, v);
    return;
  }
  int e1, e2;
  exponents_of(m, root, e1, e2);
  const float by1 = power_of(-e1), by2 = power_of(-e2);
  uint8_t c[2][kEach];
#pragma unroll
  for (int e = 0; e < kEach; ++e) {
    c[0][e] = (uint8_t)first_code(m[e] * by1, chance[e].first);
    c[1][e] = (uint8_t)second_code(root[e] * by2, chance[e].second);
  }
  store_each(first, left, c[0]);
  store_each(second, left, c[1]);
  if (i % kBlock == 0 && left > 0) {
    device<float>(t.first_scales)[i / kBlock] = power_of(e1);
    device<float>(t.second_scales)[i / kBlock] = power_of(e2);
  }
}

template <int BITS, typename P, typename G>
__device__ __forceinline__ void update_chunk(const Tensor& t, const Step& s, int64_t first) {
  for (int64_t i = first + threadIdx.x * kEach; i < first + kChunk; i += kThreads * kEach) {
    // a wave goes on together: its lanes share a scale
    const int64_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave) * kBlock + (i - threadIdx.x * kEach);
    if (wave >= t.count) return;
    if (wave + kBlock <= t.count) {
      update<BITS, true, P, G>(t, s, i, kEach);
      continue;
    }
    const int64_t left = t.count - i;
    update<BITS, false, P, G>(t, s, i, left < 0 ? 0 : left > kEach ? kEach : (int)left);
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
