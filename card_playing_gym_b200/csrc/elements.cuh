// Element access shared by the training operators: one entry or a vector of four as floats, a float32 as bfloat16
// parts, and the activations.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "product.h"

namespace cg {

__device__ __forceinline__ float as_float(float v) { return v; }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ float2 pair_float(__half2 v) { return __half22float2(v); }
__device__ __forceinline__ float2 pair_float(__nv_bfloat162 v) { return __bfloat1622float2(v); }
__device__ __forceinline__ void pair_from(__half2& p, float x, float y) { p = __floats2half2_rn(x, y); }
__device__ __forceinline__ void pair_from(__nv_bfloat162& p, float x, float y) { p = __floats2bfloat162_rn(x, y); }

template <typename T>
struct PairOf;
template <>
struct PairOf<__half> {
  using type = __half2;
};
template <>
struct PairOf<__nv_bfloat16> {
  using type = __nv_bfloat162;
};

// Four entries at `p`, aligned to four.
__device__ __forceinline__ void load4(const float* p, float (&v)[4]) {
  const float4 f = *reinterpret_cast<const float4*>(p);
  v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
}
template <typename T>
__device__ __forceinline__ void load4(const T* p, float (&v)[4]) {
  const uint2 raw = *reinterpret_cast<const uint2*>(p);
  const auto* h = reinterpret_cast<const typename PairOf<T>::type*>(&raw);
  const float2 a = pair_float(h[0]), b = pair_float(h[1]);
  v[0] = a.x, v[1] = a.y, v[2] = b.x, v[3] = b.y;
}
__device__ __forceinline__ void store4(float* p, const float (&v)[4]) {
  *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
template <typename T>
__device__ __forceinline__ void store4(T* p, const float (&v)[4]) {
  uint2 raw;
  auto* h = reinterpret_cast<typename PairOf<T>::type*>(&raw);
  pair_from(h[0], v[0], v[1]);
  pair_from(h[1], v[2], v[3]);
  *reinterpret_cast<uint2*>(p) = raw;
}

// The first n (up to four) entries at `p`; `whole`: all four, aligned.
template <typename T>
__device__ __forceinline__ void load4(const T* p, int n, bool whole, float (&v)[4]) {
  if (whole) {
    load4(p, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) v[i] = i < n ? as_float(p[i]) : 0.f;
}
template <typename T>
__device__ __forceinline__ void store4(T* p, int n, bool whole, const float (&v)[4]) {
  if (whole) {
    store4(p, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (i < n) put(p + i, v[i]);
}

// Whether every row of a matrix is aligned to four entries.
template <typename T>
__host__ __device__ __forceinline__ bool aligned4(const void* base, int64_t stride) {
  return (reinterpret_cast<uintptr_t>(base) & (4 * sizeof(T) - 1)) == 0 && stride % 4 == 0;
}

// ---- float32 as tensor-core operands -----------------------------------------------------------------------------
// x = a + b + c exactly to 2^-24: a is x cut to eight bits (no rounding up, which could pass the largest finite
// value), b and c round what is left. An infinity or NaN is its own first part.
__device__ __forceinline__ void three_parts(float x, __nv_bfloat16 (&part)[3]) {
  part[0] = __float2bfloat16_rz(x);
  float rest = isfinite(x) ? x - __bfloat162float(part[0]) : 0.f;
  part[1] = __float2bfloat16_rn(rest);
  rest -= __bfloat162float(part[1]);
  part[2] = __float2bfloat16_rn(rest);
}

template <typename T>
struct OperandOf {
  using type = T;
};
template <>
struct OperandOf<float> {
  using type = __nv_bfloat16;
};

// ---- activations ---------------------------------------------------------------------------------------------------
__device__ __forceinline__ float reciprocal_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Phi(z) of the normal distribution and exp(-z^2 / 2), for 16-bit results: erfc by Abramowitz and Stegun 7.1.26,
// t p(t) exp(-u^2) with u = |z| / sqrt 2, t = 1 / (1 + 0.3275911 u), within 1.5e-7 of erfc, a thousandth
// of what the result's own rounding moves. One exponential serves the derivative too.
__device__ __forceinline__ float normal_cumulative(float z, float* bell) {
  const float t = reciprocal_fast(fmaf(0.3275911f * 0.70710678118654752f, fabsf(z), 1.f));
  const float e = __expf(-0.5f * z * z);
  float poly = fmaf(1.061405429f, t, -1.453152027f);
  poly = fmaf(poly, t, 1.421413741f);
  poly = fmaf(poly, t, -0.284496736f);
  poly = fmaf(poly, t, 0.254829592f);
  const float tail = 0.5f * poly * t * e;
  *bell = e;
  return z < 0.f ? tail : 1.f - tail;
}

template <typename T, int kActivation>
__device__ __forceinline__ float activate(float z) {
  if constexpr (kActivation == kActRelu) return z < 0.f ? 0.f : z;  // a NaN stays one
  if constexpr (kActivation == kActGelu) {
    if constexpr (sizeof(T) == 4) return gelu_erf(z);
    float bell;
    return z * normal_cumulative(z, &bell);
  }
  if constexpr (kActivation == kActSilu) return __fdividef(z, 1.f + __expf(-z));
  return z;
}

template <typename T, int kActivation>
__device__ __forceinline__ float activation_slope(float z) {
  if constexpr (kActivation == kActRelu) return z > 0.f ? 1.f : z == z ? 0.f : z;
  if constexpr (kActivation == kActGelu) {
    float bell, cumulative;
    if constexpr (sizeof(T) == 4) {
      cumulative = 0.5f * (1.f + erff(z * 0.70710678118654752f));
      bell = __expf(-0.5f * z * z);
    } else {
      cumulative = normal_cumulative(z, &bell);
    }
    return bell == 0.f ? cumulative : fmaf(z * 0.3989422804014327f, bell, cumulative);  // an infinity times zero
  }
  if constexpr (kActivation == kActSilu) {
    const float gate = __fdividef(1.f, 1.f + __expf(-z));
    return gate == 0.f ? 0.f : gate * fmaf(z, 1.f - gate, 1.f);
  }
  return 1.f;
}

// `body` with the activation as a constant.
template <typename F>
__device__ __forceinline__ void with_activation(int activation, F&& body) {
  if (activation == kActRelu)
    body(std::integral_constant<int, kActRelu>());
  else if (activation == kActGelu)
    body(std::integral_constant<int, kActGelu>());
  else if (activation == kActSilu)
    body(std::integral_constant<int, kActSilu>());
  else
    body(std::integral_constant<int, kActNone>());
}

}  // namespace cg
