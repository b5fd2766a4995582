// Element access shared by the training operators: one entry or a vector of four as floats, a float32 as bfloat16
// parts, and the activations.
#pragma once

#include <type_traits>

#include "common.cuh"
#include "product.h"

namespace cg {

// The larger value, a NaN if either is one (fmaxf would drop it).
__device__ __forceinline__ float max_nan(float x, float y) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(x), "f"(y));
  return m;
}

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

// Two fp32 values in one register pair, added, multiplied and combined in one instruction.
struct Two {
  uint64_t v;
};
__device__ __forceinline__ Two two(float lo, float hi) {
  Two t;
  asm("mov.b64 %0, {%1, %2};" : "=l"(t.v) : "f"(lo), "f"(hi));
  return t;
}
__device__ __forceinline__ float2 apart_of(Two t) {
  float2 f;
  asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(t.v));
  return f;
}
__device__ __forceinline__ Two operator+(Two a, Two b) {
  Two t;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(t.v) : "l"(a.v), "l"(b.v));
  return t;
}
__device__ __forceinline__ Two operator*(Two a, Two b) {
  Two t;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(t.v) : "l"(a.v), "l"(b.v));
  return t;
}
__device__ __forceinline__ Two fma(Two a, Two b, Two c) {
  Two t;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(t.v) : "l"(a.v), "l"(b.v), "l"(c.v));
  return t;
}
// ---- activations ---------------------------------------------------------------------------------------------------
__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ float reciprocal_fast(float x) {
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Phi(z) of the normal distribution and exp(-z^2 / 2) for two z's, for 16-bit results. The tail erfc(u) / 2, u = |z| / sqrt 2,
// is t P(t) exp(-u^2) with t = 1 / (1 + 0.376 u) and P of degree 6 fitted to erfc(u) exp(u^2) / 2 with the least largest
// relative error over u in [0, 12], 8.3e-7. In fp32 it is within 1.4e-6 of the tail to z = -4 and 9e-6 to z = -13, where
// float16's half step is 2.4e-4: GELU's small values left of zero are rounded as the others are. One exponential serves
// the derivative too; the packed arithmetic halves the rest.
__device__ __forceinline__ Two normal_cumulative(Two z, Two* bell) {
  const float2 f = apart_of(z);
  const Two u = fma(two(fabsf(f.x), fabsf(f.y)), two(0.26587215f, 0.26587215f), two(1.f, 1.f));  // 0.376 / sqrt 2
  const float2 fu = apart_of(u);
  const Two t = two(reciprocal_fast(fu.x), reciprocal_fast(fu.y));
  const float2 fe = apart_of(z * z * two(-0.72134752f, -0.72134752f));  // log2(e) / 2
  const Two e = two(exp2_fast(fe.x), exp2_fast(fe.y));
  Two poly = fma(two(-0.0661289045f, -0.0661289045f), t, two(0.187077036f, 0.187077036f));
  poly = fma(poly, t, two(-0.0563581805f, -0.0563581805f));
  poly = fma(poly, t, two(0.13621992f, 0.13621992f));
  poly = fma(poly, t, two(0.0854161346f, 0.0854161346f));
  poly = fma(poly, t, two(0.107799199f, 0.107799199f));
  poly = fma(poly, t, two(0.105974778f, 0.105974778f));
  const float2 tail = apart_of(poly * t * e);
  *bell = e;
  return two(f.x < 0.f ? tail.x : 1.f - tail.x, f.y < 0.f ? tail.y : 1.f - tail.y);
}

// 1 + exp(-z), the reciprocal of SiLU's gate: for 16-bit results by the fast exponential, whose error grows with |z| to
// 2^-18 at -58, far inside their rounding; in full precision for float32.
template <typename T>
__device__ __forceinline__ float silu_under(float z) {
  return 1.f + (sizeof(T) == 2 ? __expf(-z) : expf(-z));
}

template <typename T, int kActivation>
__device__ __forceinline__ float activate(float z) {
  if constexpr (kActivation == kActRelu) return z < 0.f ? 0.f : z;  // a NaN stays one
  if constexpr (kActivation == kActGelu && sizeof(T) == 2) {
    Two bell;
    return z * apart_of(normal_cumulative(two(z, z), &bell)).x;
  }
  if constexpr (kActivation == kActGelu && sizeof(T) == 4) return gelu_erf(z);
  if constexpr (kActivation == kActSilu && sizeof(T) == 2) return __fdividef(z, silu_under<T>(z));
  if constexpr (kActivation == kActSilu && sizeof(T) == 4) return z / silu_under<T>(z);
  return z;
}

// kCount (even) values at once.
template <typename T, int kActivation, int kCount>
__device__ __forceinline__ void activate4(float (&z)[kCount]) {
  if constexpr (kActivation == kActGelu && sizeof(T) == 2) {
#pragma unroll
    for (int k = 0; k < kCount; k += 2) {
      const Two v = two(z[k], z[k + 1]);
      Two bell;
      const float2 y = apart_of(v * normal_cumulative(v, &bell));
      z[k] = y.x, z[k + 1] = y.y;
    }
  } else {
#pragma unroll
    for (int k = 0; k < kCount; ++k) z[k] = activate<T, kActivation>(z[k]);
  }
}

template <typename T, int kActivation>
__device__ __forceinline__ float activation_slope(float z) {
  if constexpr (kActivation == kActRelu) return z > 0.f ? 1.f : z == z ? 0.f : z;
  if constexpr (kActivation == kActGelu) {
    // The fast exponential's error, 2^-24 z^2 / 2 of the bell, is an eighth of the 2^-25 that 1 + erff rounds by.
    const float cumulative = 0.5f * (1.f + erff(z * 0.70710678118654752f));
    const float bell = __expf(-0.5f * z * z);
    return bell == 0.f ? cumulative : fmaf(z * 0.3989422804014327f, bell, cumulative);  // an infinity times zero
  }
  if constexpr (kActivation == kActSilu) {
    const float gate = sizeof(T) == 2 ? __fdividef(1.f, silu_under<T>(z)) : 1.f / silu_under<T>(z);
    return gate == 0.f || gate == 1.f ? gate : gate * fmaf(z, 1.f - gate, 1.f);  // an infinity times zero
  }
  return 1.f;
}

// g *= act'(z) for kCount (even) values.
template <typename T, int kActivation, int kCount>
__device__ __forceinline__ void times_slope(float (&g)[kCount], const float (&z)[kCount]) {
  if constexpr (kActivation == kActGelu && sizeof(T) == 2) {
#pragma unroll
    for (int k = 0; k < kCount; k += 2) {
      // Past 14 the bell is zero, and an infinity times it is to be zero too.
      const Two v = two(z[k], z[k + 1]);
      const Two near = two(fminf(fmaxf(z[k], -14.f), 14.f), fminf(fmaxf(z[k + 1], -14.f), 14.f));
      Two bell;
      const Two cumulative = normal_cumulative(v, &bell);
      const float2 y = apart_of(two(g[k], g[k + 1]) * fma(near * two(0.3989422804f, 0.3989422804f), bell, cumulative));
      g[k] = y.x, g[k + 1] = y.y;
    }
  } else {
#pragma unroll
    for (int k = 0; k < kCount; ++k) g[k] *= activation_slope<T, kActivation>(z[k]);
  }
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
