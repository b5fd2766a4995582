// Element access shared by the training operators: one entry or a vector of four as floats, a float32 as bfloat16
// parts, and the activations.
#pragma once

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

__device__ __forceinline__ float activate(float z, int activation) {
  if (activation == kActRelu) return z < 0.f ? 0.f : z;  // a NaN stays one
  if (activation == kActGelu) return gelu_erf(z);
  if (activation == kActSilu) return z / (1.f + __expf(-z));
  return z;
}

__device__ __forceinline__ float activation_slope(float z, int activation) {
  if (activation == kActRelu) return z > 0.f ? 1.f : z == z ? 0.f : z;
  if (activation == kActGelu) {
    const float cumulative = 0.5f * (1.f + erff(z * 0.70710678118654752f));
    const float tail = z * z > 200.f ? 0.f : z * 0.3989422804014327f * __expf(-0.5f * z * z);
    return cumulative + tail;
  }
  if (activation == kActSilu) {
    const float gate = 1.f / (1.f + __expf(-z));
    const float rest = z < -80.f ? 0.f : z * (1.f - gate);  // z times zero where the gate has closed
    return gate * (1.f + rest);
  }
  return 1.f;
}

}  // namespace cg
