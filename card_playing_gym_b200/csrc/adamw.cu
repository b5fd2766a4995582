// One AdamW step over many tensors: the gradients' global norm, then every parameter and its moments.
//
//   g' = g min(1, max_norm / (|g| + 1e-6)),  m = b1 m + (1 - b1) g',  v = b2 v + (1 - b2) g'^2
//   p  = p (1 - lr wd) - lr / (1 - b1^t) * m / (sqrt(v) / sqrt(1 - b2^t) + eps)
//
// What bounds it is HBM: an fp32 weight moves 28 bytes with 32-bit moments and 16 with 8-bit ones, and the
// norm reads the gradient once more. So the step is two launches whatever the number of tensors: the table of
// tensors travels in the kernel's parameters (nothing is uploaded), a block takes one chunk of one tensor,
// and the norm kernel's last block turns the norm and the step count into the factors of every group on
// the device, so the host reads nothing back.
//
// 8-bit moments: m and sqrt(v) as e4m3, scaled by the largest magnitude of each block of 256 entries of a
// tensor (fp32). The root halves the exponent range that v needs; a root that is not zero keeps at least the
// smallest code, so that no entry with history divides by eps alone. A block's scale is held in fp32 (m's as the
// formula gives it, the root's within 2 units in the last place), so the block follows its largest entry through changes
// smaller than a code's step. The update itself uses the new fp32
// moments, before they are rounded. A block is one warp's eight entries a lane, so its maximum is one
// warp reduction.
#include <cuda_fp8.h>

#include <algorithm>

#include "elements.cuh"

namespace cg {
namespace {

constexpr int kBlockEntries = 256;  // entries of one scale; every tensor's state starts on a multiple
constexpr int kPerLane = 8;
constexpr int kThreads = 256;
constexpr int kChunk = 16384;  // entries of a thread block: eight 256-entry blocks a warp
constexpr int kGroupsAtOnce = 16;  // groups of a launch's parameters; more of them take launches of their own
constexpr int kNormBlocks = 1184;  // partial sums of the norm: one fixed order of addition
constexpr float kE4m3Max = 448.f;
constexpr float kE4m3Least = 0.001953125f;  // 2^-9
constexpr float kLeastPeak = 3.0e-36f;      // below it 448 / peak is not finite: the block is held as zero

struct Factors {
  float decay, step, root, eps, beta1, rest1, beta2, rest2;
};

// Zeroed before the first step; what the norm kernel leaves for the update. Every group's factors follow it.
struct Control {
  unsigned ticket;
  int skip;
  float clip;
  int reserved;
};
__device__ __forceinline__ Factors* factors_of(Control* control) { return reinterpret_cast<Factors*>(control + 1); }
__device__ __forceinline__ const Factors* factors_of(const Control* control) {
  return reinterpret_cast<const Factors*>(control + 1);
}

struct Groups {
  int first, count;
  cg_adamw_group g[kGroupsAtOnce];
};

struct Entry {
  void* param;
  const void* grad;
  int64_t numel;
  int64_t state;
  int32_t first_chunk;  // this tensor's first chunk in the launch
  int32_t group;
};

template <int kMax>
struct Table {
  int count, chunks;
  Entry e[kMax];
};

struct States {
  void* exp_avg;
  float* exp_avg_scale;
  void* exp_avg_sq;
  float* exp_avg_sq_scale;
  float* master;
};

template <int kMax>
__device__ __forceinline__ int find_tensor(const Table<kMax>& table, int chunk) {
  int lo = 0, hi = table.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (table.e[mid].first_chunk <= chunk)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
  asm volatile("ld.global.v8.f32 {%0,%1,%2,%3,%4,%5,%6,%7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "l"(p)
               : "memory");
}

__device__ __forceinline__ void store8(float* p, const float (&v)[8]) {
  asm volatile("st.global.v8.f32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(p), "f"(v[0]), "f"(v[1]), "f"(v[2]),
               "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7])
               : "memory");
}

__device__ __forceinline__ void load8(const __nv_bfloat16* p, float (&v)[8]) {
  const uint4 raw = *reinterpret_cast<const uint4*>(p);
  const __nv_bfloat162* h = reinterpret_cast<const __nv_bfloat162*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __bfloat1622float2(h[i]);
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}

__device__ __forceinline__ void load8(const __half* p, float (&v)[8]) {
  const uint4 raw = *reinterpret_cast<const uint4*>(p);
  const __half2* h = reinterpret_cast<const __half2*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(h[i]);
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}

__device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&v)[8]) {
  uint4 raw;
  __nv_bfloat162* h = reinterpret_cast<__nv_bfloat162*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = raw;
}

__device__ __forceinline__ void store8(__half* p, const float (&v)[8]) {
  uint4 raw;
  __half2* h = reinterpret_cast<__half2*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = raw;
}

// Eight entries of a tensor from `at`; those at or past `numel` read as zero. `whole`: all eight are inside
// and the address is aligned to eight entries.
template <typename T>
__device__ __forceinline__ void load_entries(const T* base, int64_t at, int64_t numel, bool whole, float (&v)[8]) {
  if (whole) {
    load8(base + at, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) v[i] = at + i < numel ? as_float(base[at + i]) : 0.f;
}

template <typename T>
__device__ __forceinline__ void store_entries(T* base, int64_t at, int64_t numel, bool whole, const float (&v)[8]) {
  if (whole) {
    store8(base + at, v);
    return;
  }
#pragma unroll
  for (int i = 0; i < kPerLane; ++i)
    if (at + i < numel) put(base + at + i, v[i]);
}

template <typename T>
__device__ __forceinline__ bool aligned8(const T* p) {
  return (reinterpret_cast<uintptr_t>(p) & (sizeof(T) * kPerLane - 1)) == 0;
}

// ---- 8-bit moments --------------------------------------------------------------------------------
__device__ __forceinline__ void decode8(const uint2& raw, float unit, float (&v)[8]) {
  const __nv_fp8x2_storage_t* pairs = reinterpret_cast<const __nv_fp8x2_storage_t*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2(pairs[i], __NV_E4M3)));
    v[2 * i] = f.x * unit, v[2 * i + 1] = f.y * unit;
  }
}

__device__ __forceinline__ void encode8(uint8_t* codes, const float (&v)[8]) {
  uint2 raw;
  __nv_fp8x2_storage_t* pairs = reinterpret_cast<__nv_fp8x2_storage_t*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i)
    pairs[i] = __nv_cvt_float2_to_fp8x2(make_float2(v[2 * i], v[2 * i + 1]), __NV_SATFINITE, __NV_E4M3);
  *reinterpret_cast<uint2*>(codes) = raw;
}

// Square root and reciprocal within 2 units in the last place: the update they make is the learning rate's fraction of a
// weight, and exact ones (some 30 instructions an entry) would cost more than the memory they hide behind.
__device__ __forceinline__ float root_fast(float v) {
  float r;  // of a subnormal v too, which is what a gradient of 1e-18 leaves
  asm("sqrt.approx.f32 %0, %1;" : "=f"(r) : "f"(v));
  return r;
}

// The reciprocal to its last bit, but for the rarest rounding cases: one step of Newton's method on the fast one.
__device__ __forceinline__ float reciprocal_near(float x) {
  const float r = reciprocal_fast(x);
  return fmaf(r, fmaf(-x, r, 1.f), r);
}

// Under the update's quotient at least, 2^-75: the root of any v above zero is larger, an entry without history does not
// divide zero by a zero eps, and one whose v has become zero below float32's range is updated as if it had the least one.
constexpr float kLeastUnder = 2.6469780e-23f;

// Largest of the warp's non-negative values; a NaN's bits compare above infinity's, so it is kept.
__device__ __forceinline__ float warp_peak(float v) {
  return __uint_as_float(__reduce_max_sync(0xffffffffu, __float_as_uint(v)));
}

// ---- the global norm and the step's factors ----------------------------------------------------------
// One thread per group, in double: 1 - b2^t loses half its digits in fp32. t: the step being made.
__device__ void make_factors(const Groups& groups, int64_t t, Control* control) {
  for (int k = threadIdx.x; k < groups.count; k += blockDim.x) {
    const cg_adamw_group g = groups.g[k];
    Factors f;
    f.decay = static_cast<float>(1.0 - g.lr * g.weight_decay);
    f.step = static_cast<float>(g.lr / (1.0 - pow(g.beta1, static_cast<double>(t))));
    f.root = static_cast<float>(1.0 / sqrt(1.0 - pow(g.beta2, static_cast<double>(t))));
    f.eps = static_cast<float>(g.eps);
    f.beta1 = static_cast<float>(g.beta1);
    f.rest1 = static_cast<float>(1.0 - g.beta1);
    f.beta2 = static_cast<float>(g.beta2);
    f.rest2 = static_cast<float>(1.0 - g.beta2);
    factors_of(control)[groups.first + k] = f;
  }
}

// The first groups' factors, the clip and the step's count.
__device__ void begin_step(const Groups& groups, int64_t* steps, bool finite, float clip, Control* control) {
  const int64_t t = *steps + 1;
  __syncthreads();
  if (threadIdx.x == 0) {
    control->clip = clip;
    control->skip = finite ? 0 : 1;
    if (finite) *steps = t;
  }
  make_factors(groups, t, control);
}

// Without a clip, or for the groups past the first ones: the step has been counted by then.
__global__ void __launch_bounds__(32) adamw_factors_kernel(const __grid_constant__ Groups groups, int64_t* steps,
                                                           Control* control) {
  pdl_trigger();
  if (groups.first == 0)
    begin_step(groups, steps, true, 1.f, control);
  else
    make_factors(groups, *steps, control);
}

// Squares are summed in fp32 over a thread's eight entries and in double from there on. Entries past 1.8e19, whose squares
// fp32 does not hold, are summed in double throughout: the norm of finite gradients is finite unless it passes fp32 itself.
__device__ __forceinline__ double sum_of_squares(const float (&g)[8]) {
  float sum = 0.f;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) sum = fmaf(g[i], g[i], sum);
  if (sum < INFINITY) return sum;
  double wide = 0;
#pragma unroll
  for (int i = 0; i < kPerLane; ++i) wide += static_cast<double>(g[i]) * g[i];
  return wide;
}

template <typename T, int kMax>
__global__ void __launch_bounds__(kThreads) adamw_norm_kernel(const __grid_constant__ Table<kMax> table,
                                                              const __grid_constant__ Groups groups, float max_norm,
                                                              int first_partial, int partials, double* partial,
                                                              int64_t* steps, float* norm_out, Control* control) {
  __shared__ double s[kThreads / 32];
  __shared__ bool last;
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  double total = 0;
  for (int chunk = blockIdx.x; chunk < table.chunks; chunk += gridDim.x) {
    const Entry& e = table.e[find_tensor(table, chunk)];
    const T* grad = static_cast<const T*>(e.grad);
    const bool aligned = aligned8(grad);
    const int64_t start = static_cast<int64_t>(chunk - e.first_chunk) * kChunk;
    constexpr int kSteps = kChunk / (kThreads * kPerLane), kAtOnce = sizeof(T) == 2 ? kSteps : kSteps / 2;
    if (aligned && start + kChunk <= e.numel) {
      // Loads of 128 bytes a lane are in flight at a time.
#pragma unroll
      for (int b = 0; b < kSteps; b += kAtOnce) {
        float g[kAtOnce][8];
#pragma unroll
        for (int c = 0; c < kAtOnce; ++c) load8(grad + start + ((b + c) * kThreads + threadIdx.x) * kPerLane, g[c]);
#pragma unroll
        for (int c = 0; c < kAtOnce; ++c) total += sum_of_squares(g[c]);
      }
      continue;
    }
    for (int b = 0; b < kSteps; ++b) {
      const int64_t at = start + (b * kThreads + threadIdx.x) * kPerLane;
      if (at >= e.numel) break;
      float g[8];
      load_entries(grad, at, e.numel, aligned && at + kPerLane <= e.numel, g);
      total += sum_of_squares(g);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) s[warp] = total;
  __syncthreads();
  if (threadIdx.x == 0) {
    for (int w = 1; w < kThreads / 32; ++w) total += s[w];
    partial[first_partial + blockIdx.x] = total;
    __threadfence();
    last = atomicInc(&control->ticket, partials - 1) == static_cast<unsigned>(partials - 1);
  }
  __syncthreads();
  if (!last) return;
  __threadfence();
  total = 0;
  for (int i = threadIdx.x; i < partials; i += kThreads) total += __ldcg(partial + i);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) s[warp] = total;
  __syncthreads();
  total = 0;
  for (int w = 0; w < kThreads / 32; ++w) total += s[w];
  const double norm = sqrt(total);
  if (threadIdx.x == 0) *norm_out = static_cast<float>(norm);
  begin_step(groups, steps, isfinite(static_cast<float>(norm)), static_cast<float>(fmin(1.0, max_norm / (norm + 1e-6))), control);
}

// ---- the update -----------------------------------------------------------------------------------------
// What a lane has in flight of one 256-entry block: its eight entries as they are in memory.
template <typename T, int kBits>
struct Loaded {
  float p[8], g[8], m[8], v[8];     // fp32 parts
  uint4 raw_g;                      // a 16-bit gradient
  uint2 codes_m, codes_v;           // 8-bit moments
  bool whole;
};

template <typename T, int kBits>
__device__ __forceinline__ void load_block(Loaded<T, kBits>& l, const Entry& e, const States& states, int64_t at, bool aligned) {
  const int64_t held = e.state + at;  // the state's arrays are padded: eight entries are always inside
  const T* param = static_cast<const T*>(e.param);
  const T* grad = static_cast<const T*>(e.grad);
  l.whole = aligned && at + kPerLane <= e.numel;
  if constexpr (sizeof(T) == 2) {
    if (l.whole)
      l.raw_g = *reinterpret_cast<const uint4*>(grad + at);
    else
      load_entries(grad, at, e.numel, false, l.g);
    load8(states.master + held, l.p);
  } else {
    load_entries(grad, at, e.numel, l.whole, l.g);
    load_entries(param, at, e.numel, l.whole, l.p);
  }
  if constexpr (kBits == 8) {
    l.codes_m = *reinterpret_cast<const uint2*>(static_cast<uint8_t*>(states.exp_avg) + held);
    l.codes_v = *reinterpret_cast<const uint2*>(static_cast<uint8_t*>(states.exp_avg_sq) + held);
  } else {
    load8(static_cast<float*>(states.exp_avg) + held, l.m);
    load8(static_cast<float*>(states.exp_avg_sq) + held, l.v);
  }
}

template <typename T, int kBits>
__device__ __forceinline__ void update_block(Loaded<T, kBits>& l, const Entry& e, const States& states, int64_t at,
                                             const Factors& f, float clip, float& scale_m, float& scale_r) {
  const int64_t held = e.state + at;
  if constexpr (sizeof(T) == 2) {
    if (l.whole) load8(reinterpret_cast<const T*>(&l.raw_g), l.g);
  }
  if constexpr (kBits == 8) {
    decode8(l.codes_m, scale_m * (1.f / kE4m3Max), l.m);
    decode8(l.codes_v, scale_r * (1.f / kE4m3Max), l.v);
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) l.v[i] *= l.v[i];
  }
  float peak_m = 0.f, peak_r = 0.f;
  const Two beta1 = two(f.beta1, f.beta1), rest1 = two(f.rest1, f.rest1), beta2 = two(f.beta2, f.beta2),
            rest2 = two(f.rest2, f.rest2), clips = two(clip, clip), decay = two(f.decay, f.decay),
            step = two(-f.step, -f.step), unbias = two(f.root, f.root), eps = two(f.eps, f.eps);
#pragma unroll
  for (int i = 0; i < kPerLane; i += 2) {
    const Two raw = two(l.g[i], l.g[i + 1]), g = raw * clips;
    // The products are rounded before their sum (packed ones are fused with a packed sum): an 8-bit code then is that of the
    // formula's own fp32 arithmetic, not of a neighbouring value at its edge.
    const float2 kept = apart_of(beta1 * two(l.m[i], l.m[i + 1])), added = apart_of(rest1 * g);
    const Two m = two(__fadd_rn(kept.x, added.x), __fadd_rn(kept.y, added.y));
    const Two v = fma(beta2, two(l.v[i], l.v[i + 1]), rest2 * (g * g));
    const float2 fv = apart_of(v), fm = apart_of(m);
    const float2 root = make_float2(root_fast(fv.x), root_fast(fv.y));
    const float2 under = apart_of(fma(two(root.x, root.y), unbias, eps));
    const Two update = m * two(reciprocal_fast(fmaxf(under.x, kLeastUnder)), reciprocal_fast(fmaxf(under.y, kLeastUnder)));
    const float2 p = apart_of(fma(step, update, two(l.p[i], l.p[i + 1]) * decay));
    l.p[i] = p.x, l.p[i + 1] = p.y;
    l.m[i] = fm.x, l.m[i + 1] = fm.y;
    if (kBits == 8) {
      l.v[i] = root.x, l.v[i + 1] = root.y;
      peak_m = max_nan(peak_m, max_nan(fabsf(fm.x), fabsf(fm.y)));
      peak_r = max_nan(peak_r, max_nan(root.x, root.y));
    } else {
      l.v[i] = fv.x, l.v[i + 1] = fv.y;
    }
  }
  if (sizeof(T) == 2) store8(states.master + held, l.p);
  store_entries(static_cast<T*>(e.param), at, e.numel, l.whole, l.p);
  if constexpr (kBits == 8) {
    peak_m = warp_peak(peak_m);
    peak_r = warp_peak(peak_r);
    const float to_m = peak_m < kLeastPeak ? 0.f : kE4m3Max * reciprocal_near(peak_m);
    const float to_r = peak_r < kLeastPeak ? 0.f : kE4m3Max * reciprocal_near(peak_r);
    float least = kE4m3Least;
#pragma unroll
    for (int i = 0; i < kPerLane; i += 2) {
      const float2 m = apart_of(two(l.m[i], l.m[i + 1]) * two(to_m, to_m));
      const float2 v = apart_of(two(l.v[i], l.v[i + 1]) * two(to_r, to_r));
      l.m[i] = m.x, l.m[i + 1] = m.y, l.v[i] = v.x, l.v[i + 1] = v.y;
      least = fminf(least, fminf(v.x, v.y));
    }
    if (least < kE4m3Least) {  // a root under the smallest code: it keeps that one unless it is zero
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) l.v[i] = l.v[i] > 0.f ? fmaxf(l.v[i], kE4m3Least) : l.v[i];
    }
    encode8(static_cast<uint8_t*>(states.exp_avg) + held, l.m);
    encode8(static_cast<uint8_t*>(states.exp_avg_sq) + held, l.v);
    scale_m = peak_m, scale_r = peak_r;
  } else {
    store8(static_cast<float*>(states.exp_avg) + held, l.m);
    store8(static_cast<float*>(states.exp_avg_sq) + held, l.v);
  }
}

// A warp takes eight neighbouring blocks, whose scales are one 32-byte sector: its lanes read and write them at once. (Read
// and written block by block, from sectors that eight warps were writing to, they were what the kernel waited for:
// 134 M float32 weights with 8-bit moments 510 us, with whole sectors 360.) Three thread blocks an SM, with the registers
// that leaves, do better than more (134 M bfloat16 weights, 8 bits: 376 us; four 400, five 472). The first loads go out
// before the wait for the factors: nothing the kernel before this one writes is among them. Without a clip,
// 134 M weights: 32-bit moments 571 us (float32, 6.6 TB/s) and 586 (bfloat16, 6.4), the copy bandwidth; 8-bit ones 338 (6.4)
// and 356 (6.0), short of it by their codes' arithmetic.
template <typename T, int kBits, int kMax>
__global__ void __launch_bounds__(kThreads, 3) adamw_update_kernel(const __grid_constant__ Table<kMax> table, const States states,
                                                                   const Control* control) {
  constexpr int kWarpBlocks = kChunk / kThreads * 32 / kBlockEntries;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const Entry& e = table.e[find_tensor(table, blockIdx.x)];
  const bool aligned = aligned8(static_cast<const T*>(e.param)) && aligned8(static_cast<const T*>(e.grad));
  const int64_t first = static_cast<int64_t>(blockIdx.x - e.first_chunk) * kChunk + warp * kWarpBlocks * kBlockEntries;
  if (first >= e.numel) return;
  const int blocks = static_cast<int>(min(static_cast<int64_t>(kWarpBlocks), (e.numel - first + kBlockEntries - 1) / kBlockEntries));
  Loaded<T, kBits> l;
  load_block(l, e, states, first + lane * kPerLane, aligned);
  const int64_t scale_at = (e.state + first) / kBlockEntries + lane;
  float scales_m = 0.f, scales_r = 0.f;  // of this lane's block
  if (kBits == 8 && lane < blocks) scales_m = states.exp_avg_scale[scale_at], scales_r = states.exp_avg_sq_scale[scale_at];
  pdl_wait();
  if (control->skip) return;  // a norm that is not finite: nothing moves
  const float clip = control->clip;
  const Factors f = factors_of(control)[e.group];
  for (int i = 0; i < blocks; ++i) {
    float scale_m = 0.f, scale_r = 0.f;
    if (kBits == 8) scale_m = __shfl_sync(0xffffffffu, scales_m, i), scale_r = __shfl_sync(0xffffffffu, scales_r, i);
    const int64_t at = first + i * kBlockEntries + lane * kPerLane;
    if (i > 0) load_block(l, e, states, at, aligned);
    update_block(l, e, states, at, f, clip, scale_m, scale_r);
    if (kBits == 8 && lane == i) scales_m = scale_m, scales_r = scale_r;
  }
  if (kBits == 8 && lane < blocks) states.exp_avg_scale[scale_at] = scales_m, states.exp_avg_sq_scale[scale_at] = scales_r;
}

constexpr int kFewTensors = 64, kManyTensors = 640;  // 2.6 and 25 KB of kernel parameters (32 KB is the limit)

// The tensors from `next` on that fit one launch; those without a gradient or without entries are left out.
struct Tensors {
  const cg_adamw_tensor* extents;
  void* const* params;
  const void* const* grads;
  int count;
  bool live(int i) const { return grads[i] && extents[i].numel > 0; }
};

template <int kMax>
void fill_table(const Tensors& tensors, int& next, Table<kMax>& table) {
  table.count = table.chunks = 0;
  while (next < tensors.count && table.count < kMax) {
    const cg_adamw_tensor& t = tensors.extents[next];
    if (tensors.live(next)) {
      const int64_t chunks = (t.numel + kChunk - 1) / kChunk;
      if (table.count && table.chunks + chunks > INT32_MAX) break;
      table.e[table.count++] = {tensors.params[next], tensors.grads[next], t.numel, t.state, table.chunks, t.group};
      table.chunks += static_cast<int>(chunks);
    }
    ++next;
  }
}

Groups groups_from(const cg_adamw_group* all, int count, int first) {
  Groups groups;
  groups.first = first;
  groups.count = std::min(count - first, kGroupsAtOnce);
  for (int k = 0; k < groups.count; ++k) groups.g[k] = all[first + k];
  return groups;
}

template <typename T, int kMax>
int run_step(const Tensors& tensors, const cg_adamw_group* all_groups, int group_count, int bits, const States& states,
             int64_t* steps, float max_norm, float* norm_out, Control* control, double* partial, cudaStream_t s) {
  Table<kMax> table;
  const Groups groups = groups_from(all_groups, group_count, 0);
  if (max_norm > 0) {
    int partials = 0;
    for (int next = 0; next < tensors.count;) {
      fill_table(tensors, next, table);
      partials += std::min(table.chunks, kNormBlocks);
    }
    int first = 0;
    for (int next = 0; next < tensors.count;) {
      fill_table(tensors, next, table);
      if (!table.chunks) continue;
      const int blocks = std::min(table.chunks, kNormBlocks);
      adamw_norm_kernel<T, kMax><<<blocks, kThreads, 0, s>>>(table, groups, max_norm, first, partials, partial, steps,
                                                             norm_out, control);
      if (int rc = check_launch("adamw_norm_kernel")) return rc;
      first += blocks;
    }
  } else {
    adamw_factors_kernel<<<1, 32, 0, s>>>(groups, steps, control);
    if (int rc = check_launch("adamw_factors_kernel")) return rc;
  }
  for (int more = kGroupsAtOnce; more < group_count; more += kGroupsAtOnce) {
    adamw_factors_kernel<<<1, 32, 0, s>>>(groups_from(all_groups, group_count, more), steps, control);
    if (int rc = check_launch("adamw_factors_kernel")) return rc;
  }
  for (int next = 0; next < tensors.count;) {
    fill_table(tensors, next, table);
    if (!table.chunks) continue;
    auto kernel = bits == 8 ? adamw_update_kernel<T, 8, kMax> : adamw_update_kernel<T, 32, kMax>;
    if (int rc = launch_pdl("adamw_update_kernel", kernel, dim3(table.chunks), dim3(kThreads), 0, s, table, states,
                            static_cast<const Control*>(control)))
      return rc;
  }
  return CG_OK;
}

}  // namespace
}  // namespace cg

extern "C" int64_t cg_adamw_control_bytes(int groups) {
  if (groups < 1) {
    cg::set_error(CG_ERR_ARGUMENT, "cg_adamw_control_bytes: no groups");
    return -1;
  }
  return static_cast<int64_t>(sizeof(cg::Control)) + groups * static_cast<int64_t>(sizeof(cg::Factors));
}

extern "C" int64_t cg_adamw_workspace_bytes(int count) {
  if (count < 0) {
    cg::set_error(CG_ERR_ARGUMENT, "cg_adamw_workspace_bytes: negative count");
    return -1;
  }
  return (static_cast<int64_t>(count) / cg::kFewTensors + 1) * cg::kNormBlocks * static_cast<int64_t>(sizeof(double));
}

extern "C" int cg_adamw_step(const cg_adamw_tensor* tensors, void* const* params, const void* const* grads, int count,
                             int dtype, const cg_adamw_group* groups, int group_count, int state_bits, void* exp_avg,
                             float* exp_avg_scale, void* exp_avg_sq, float* exp_avg_sq_scale, float* master, int64_t* steps,
                             float max_norm, float* norm_out, void* control, void* workspace, int64_t workspace_bytes,
                             void* stream) {
  using namespace cg;
  CG_REQUIRE(count >= 0 && (count == 0 || (tensors && params && grads)), "cg_adamw_step: bad tensor table");
  CG_REQUIRE(valid_dtype(dtype), "cg_adamw_step: dtype must be float32, float16 or bfloat16");
  CG_REQUIRE(state_bits == 8 || state_bits == 32, "cg_adamw_step: state_bits must be 8 or 32");
  CG_REQUIRE(groups && group_count > 0, "cg_adamw_step: no groups");
  CG_REQUIRE(exp_avg && exp_avg_sq && steps && control, "cg_adamw_step: NULL state");
  CG_REQUIRE(state_bits == 32 || (exp_avg_scale && exp_avg_sq_scale), "cg_adamw_step: 8-bit states need scales");
  CG_REQUIRE(dtype == CG_F32 || master, "cg_adamw_step: 16-bit parameters need fp32 master copies");
  CG_REQUIRE(!(max_norm > 0) || norm_out, "cg_adamw_step: max_norm needs norm_out");
  if (max_norm > 0 && (!workspace || workspace_bytes < cg_adamw_workspace_bytes(count)))
    return set_error(CG_ERR_WORKSPACE, "cg_adamw_step: workspace too small");
  for (int k = 0; k < group_count; ++k) {
    const cg_adamw_group& g = groups[k];
    CG_REQUIRE(g.beta1 >= 0 && g.beta1 < 1 && g.beta2 >= 0 && g.beta2 < 1, "cg_adamw_step: betas must lie in [0, 1)");
    CG_REQUIRE(g.eps >= 0, "cg_adamw_step: eps must not be negative");
  }
  const Tensors all{tensors, params, grads, count};
  int live = 0;
  for (int i = 0; i < count; ++i) {
    const cg_adamw_tensor& t = tensors[i];
    CG_REQUIRE(t.numel >= 0 && t.state >= 0 && t.state % kBlockEntries == 0, "cg_adamw_step: tensor %d: bad extent", i);
    CG_REQUIRE(t.numel <= static_cast<int64_t>(INT32_MAX) * kChunk, "cg_adamw_step: tensor %d is too large", i);
    CG_REQUIRE(t.group >= 0 && t.group < group_count, "cg_adamw_step: tensor %d: no such group", i);
    CG_REQUIRE(t.numel == 0 || !grads[i] || params[i], "cg_adamw_step: tensor %d: NULL parameter", i);
    live += all.live(i);
  }
  if (!live) return CG_OK;
  const States states{exp_avg, exp_avg_scale, exp_avg_sq, exp_avg_sq_scale, master};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  auto* c = static_cast<Control*>(control);
  auto* partial = static_cast<double*>(workspace);
  auto run = [&](auto sample) {
    using T = decltype(sample);
    return live <= kFewTensors
               ? run_step<T, kFewTensors>(all, groups, group_count, state_bits, states, steps, max_norm, norm_out, c, partial, s)
               : run_step<T, kManyTensors>(all, groups, group_count, state_bits, states, steps, max_norm, norm_out, c, partial, s);
  };
  if (dtype == CG_F32) return run(float{});
  if (dtype == CG_F16) return run(__half{});
  return run(__nv_bfloat16{});
}
