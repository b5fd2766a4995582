// The linear layer for a few tokens: y = act(x W^T + b) + residual with at most 32 rows of x (few_rows in product.h).
//
// W is read once and is all there is to read; it passes L1 by, which keeps the tokens.
//
// 16-bit operands: a block takes 16 or 32 outputs and all the tokens, and its eight warps split k. A lane loads W straight
// from memory into mma fragments. The products run on mma.sync m16n8k16 with W as the 16-row operand and eight tokens
// as its columns: at these sizes the tensor cores are idle either way, and what counts is that a token costs no
// instructions of its own. k's order inside a fragment does not matter as long as both operands agree, so a lane
// loads eight neighbouring k's in one access. The warps' sums join in shared memory in a fixed order.
//
// float32 operands: fused multiply-adds, which a few tokens leave time for beside the reading of W. A warp takes
// four outputs and all the tokens, its lanes split k.
//
// 4096 x 8192, floor 10.3 us for 16-bit W: bfloat16 17 us for one token and 20 for 24 (bound by the latency of W's loads
// and the launch). float32, floor 20.5: 33 us for one token, 41 for 8, 78 for 16, 172 for 32 (bound by the tokens' loads out
// of L1 and L2, a vector for 16 products; in tensor-core parts 60, 60, 105 and 188;
// such a layer goes to run_product from 25 tokens on).
#include "elements.cuh"

namespace cg {
namespace {

constexpr int kWarps = 8;

__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1, __nv_bfloat16) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                          uint32_t b1, __half) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// Eight neighbouring entries of a row as they are in memory; those at or past `n` are zero.
template <typename T>
struct Eight {
  T v[8];
};

// kAligned: rows are aligned to sixteen bytes and hold whole eights. kStream: they are used once and pass L1 by.
template <bool kAligned, bool kStream, typename T>
__device__ __forceinline__ Eight<T> load_eight(const T* p, int64_t n) {
  Eight<T> e;
  if constexpr (kAligned) {
    uint4* w = reinterpret_cast<uint4*>(&e);
#pragma unroll
    for (int i = 0; i < static_cast<int>(sizeof(T)) * 8 / 16; ++i) {
      w[i] = make_uint4(0, 0, 0, 0);
      if (n <= 0) continue;
      if (kStream)
        asm volatile("ld.global.nc.L1::no_allocate.v4.u32 {%0,%1,%2,%3}, [%4];"
                     : "=r"(w[i].x), "=r"(w[i].y), "=r"(w[i].z), "=r"(w[i].w)
                     : "l"(reinterpret_cast<const uint4*>(p) + i));
      else
        w[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      e.v[i] = T(0.f);
      if (i < n) e.v[i] = p[i];
    }
  }
  return e;
}

// Eight entries as the operand's four registers.
template <typename T>
struct Fragment {
  uint32_t w[4];
  __device__ __forceinline__ explicit Fragment(const Eight<T>& e) {
    const uint32_t* r = reinterpret_cast<const uint32_t*>(&e);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[i] = r[i];
  }
};
template <typename T, int kActivation>
__device__ __forceinline__ void finish_one(const ProductEpilogue& e, int token, int64_t j, int64_t outer, float z) {
  if (e.bias) z += as_float(static_cast<const T*>(e.bias)[j]);
  if (e.pre) put(static_cast<T*>(e.pre) + token * outer + j, z);
  z = activate<T, kActivation>(z);
  if (e.residual) z += as_float(static_cast<const T*>(e.residual)[token * e.residual_stride + j]);
  put(static_cast<T*>(e.out) + token * e.out_stride + j, z);
}

// kTokens: groups of eight tokens; kTiles: tiles of 16 outputs. A step is 64 k's. The next step's loads under this one's
// products would cost more in registers than they hide (24 tokens, 4096 x 8192: 23.2 us against 19.6).
template <typename T, int kTokens, int kTiles, bool kAligned>
__global__ void __launch_bounds__(kWarps * 32, 2) few_rows_kernel(
    const T* x, int64_t x_stride, const T* weight, int64_t weight_stride, int rows, int64_t inner, int64_t outer,
    const ProductEpilogue e) {
  constexpr int kOutputs = 16 * kTiles, kHalves = 2, kStep = 32 * kHalves;
  __shared__ float sums[kWarps][kTokens * 8][kOutputs + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int64_t j0 = static_cast<int64_t>(blockIdx.x) * kOutputs;
  const T* from_w = weight + (j0 + g) * weight_stride + t * 8;
  const T* from_x = x + g * x_stride + t * 8;
  float c[kTiles][kTokens][4] = {};
  for (int64_t k0 = warp * kStep; k0 < inner; k0 += kWarps * kStep) {
    Eight<T> a[kTiles][kHalves][2];
#pragma unroll
    for (int m = 0; m < kTiles; ++m)
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int64_t k = k0 + h * 32, row = m * 16 + r * 8;
          a[m][h][r] = load_eight<kAligned, true>(from_w + row * weight_stride + k, j0 + g + row < outer ? inner - k - t * 8 : 0);
        }
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      const int64_t k = k0 + h * 32;
#pragma unroll
      for (int n = 0; n < kTokens; ++n) {
        const Fragment<T> f(load_eight<kAligned, false>(from_x + n * 8 * x_stride + k, n * 8 + g < rows ? inner - k - t * 8 : 0));
#pragma unroll
        for (int m = 0; m < kTiles; ++m) {
          const Fragment<T> a0(a[m][h][0]), a1(a[m][h][1]);
          mma_16816(c[m][n], a0.w[0], a1.w[0], a0.w[1], a1.w[1], f.w[0], f.w[1], T());
          mma_16816(c[m][n], a0.w[2], a1.w[2], a0.w[3], a1.w[3], f.w[2], f.w[3], T());
        }
      }
    }
  }
#pragma unroll
  for (int m = 0; m < kTiles; ++m)
#pragma unroll
    for (int n = 0; n < kTokens; ++n)
#pragma unroll
      for (int k = 0; k < 4; ++k) sums[warp][n * 8 + 2 * t + (k & 1)][m * 16 + g + 8 * (k >> 1)] = c[m][n][k];
  __syncthreads();
  with_activation(e.activation, [&](auto activation) {
    for (int index = threadIdx.x; index < kTokens * 8 * kOutputs; index += kWarps * 32) {
      const int token = index / kOutputs, o = index % kOutputs;
      if (token >= rows || j0 + o >= outer) continue;
      float z = 0.f;
#pragma unroll
      for (int s = 0; s < kWarps; ++s) z += sums[s][token][o];
      finish_one<T, activation>(e, token, j0 + o, outer, z);
    }
  });
}

// ---- float32 ------------------------------------------------------------------------------------------------------------
constexpr int kOutputs32 = 4;  // a warp's

// Four of a row's entries for lane `lane` of a step of 128: neighbours where rows are aligned, else every 32nd.
template <bool kAligned, bool kStream>
__device__ __forceinline__ float4 load_four(const float* row, int64_t k0, int lane, int64_t inner) {
  float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
  if constexpr (kAligned) {
    const int64_t k = k0 + lane * 4;
    if (k >= inner) return f;
    if (kStream)
      asm volatile("ld.global.nc.L1::no_allocate.v4.f32 {%0,%1,%2,%3}, [%4];"
                   : "=f"(f.x), "=f"(f.y), "=f"(f.z), "=f"(f.w)
                   : "l"(row + k));
    else
      f = __ldg(reinterpret_cast<const float4*>(row + k));
  } else {
    float* v = reinterpret_cast<float*>(&f);
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (k0 + lane + 32 * i < inner) v[i] = row[k0 + lane + 32 * i];
  }
  return f;
}

// splits: of k, 1 to 8 (a power of two) of the block's warps to each four outputs.
template <int kTokens, bool kAligned>
__global__ void __launch_bounds__(kWarps * 32, kTokens > 16 ? 1 : 2) few_rows_f32_kernel(
    const float* x, int64_t x_stride, const float* weight, int64_t weight_stride, int rows, int64_t inner, int64_t outer,
    int splits, const ProductEpilogue e) {
  constexpr int kSums = kOutputs32 * kTokens;
  __shared__ float sums[kWarps][kSums];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, groups = kWarps / splits;
  const int64_t block_j = static_cast<int64_t>(blockIdx.x) * groups * kOutputs32, j0 = block_j + warp / splits * kOutputs32;
  float c[kSums] = {};
  float4 now[kOutputs32], next[kOutputs32];
  auto load = [&](float4 (&w)[kOutputs32], int64_t k0) {
#pragma unroll
    for (int o = 0; o < kOutputs32; ++o) {
      w[o] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (j0 + o < outer) w[o] = load_four<kAligned, true>(weight + (j0 + o) * weight_stride, k0, lane, inner);
    }
  };
  // A step's weights are loaded under the products of the one before.
  int64_t k0 = warp % splits * 128;
  load(now, k0);
  for (; k0 < inner; k0 += splits * 128) {
    if (k0 + splits * 128 < inner) load(next, k0 + splits * 128);
    // Some tokens at a time, so that their loads wait together: four (one by one 16 tokens take 153 us, not 78, on 4096 x
    // 8192), eight where one block an SM leaves the registers (32 tokens: 172 us against 220).
    constexpr int kTogether = kTokens > 16 ? 8 : kTokens < 4 ? kTokens : 4;
#pragma unroll
    for (int first = 0; first < kTokens; first += kTogether) {
      if (first >= rows) break;
      float4 f[kTogether];
#pragma unroll
      for (int t = 0; t < kTogether; ++t) {
        f[t] = make_float4(0.f, 0.f, 0.f, 0.f);
        if (first + t < rows) f[t] = load_four<kAligned, false>(x + (first + t) * x_stride, k0, lane, inner);
      }
#pragma unroll
      for (int t = 0; t < kTogether; ++t)
#pragma unroll
        for (int o = 0; o < kOutputs32; ++o) {
          float& sum = c[(first + t) * kOutputs32 + o];
          sum = fmaf(f[t].x, now[o].x, sum), sum = fmaf(f[t].y, now[o].y, sum);
          sum = fmaf(f[t].z, now[o].z, sum), sum = fmaf(f[t].w, now[o].w, sum);
        }
    }
#pragma unroll
    for (int o = 0; o < kOutputs32; ++o) now[o] = next[o];
  }
  // The lanes' sums: each exchange halves the sums a lane keeps, until it keeps one (or the rest of kSums / 32).
  int kept = 0;  // the first of this lane's
#pragma unroll
  for (int offset = 16, n = kSums / 2; offset > 0; offset >>= 1, n >>= 1) {
    if (n > 0) {
      const bool upper = lane & offset;
      kept += upper ? n : 0;
#pragma unroll
      for (int i = 0; i < n; ++i) {
        const float keep = upper ? c[i + n] : c[i], give = upper ? c[i] : c[i + n];
        c[i] = keep + __shfl_xor_sync(0xffffffffu, give, offset);
      }
    } else {
      c[0] += __shfl_xor_sync(0xffffffffu, c[0], offset);
    }
  }
  constexpr int kRest = kSums > 32 ? kSums / 32 : 1;
#pragma unroll
  for (int i = 0; i < kRest; ++i) sums[warp][kept + i] = c[i];
  __syncthreads();
  with_activation(e.activation, [&](auto activation) {
    for (int index = threadIdx.x; index < groups * kSums; index += kWarps * 32) {
      const int group = index / kSums, token = index % kSums / kOutputs32;
      const int64_t j = block_j + group * kOutputs32 + index % kOutputs32;
      if (token >= rows || j >= outer) continue;
      float z = 0.f;
      for (int s = 0; s < splits; ++s) z += sums[group * splits + s][index % kSums];
      finish_one<float, activation>(e, token, j, outer, z);
    }
  });
}

template <int kTokens>
int run_f32(const float* x, int64_t x_stride, const float* weight, int64_t weight_stride, int rows, int64_t inner, int64_t outer,
            bool whole, const ProductEpilogue& e, cudaStream_t s) {
  // As few warps to an output as give every SM a block.
  const int64_t fours = (outer + kOutputs32 - 1) / kOutputs32;
  int splits = 1;
  while (splits < kWarps && fours * splits < kWarps * 148) splits *= 2;
  const int64_t groups = kWarps / splits;
  auto kernel = whole ? few_rows_f32_kernel<kTokens, true> : few_rows_f32_kernel<kTokens, false>;
  kernel<<<static_cast<unsigned>((fours + groups - 1) / groups), kWarps * 32, 0, s>>>(x, x_stride, weight, weight_stride, rows,
                                                                                      inner, outer, splits, e);
  return check_launch("few_rows_f32_kernel");
}

template <typename T>
bool aligned_rows(const void* base, int64_t stride, int64_t count) {
  return (reinterpret_cast<uintptr_t>(base) & 15) == 0 && (count == 1 || stride * sizeof(T) % 16 == 0);
}

template <typename T, int kTokens, int kTiles>
int launch(const void* x, int64_t x_stride, const void* weight, int64_t weight_stride, int rows, int64_t inner, int64_t outer,
           const ProductEpilogue& e, cudaStream_t s) {
  constexpr int kOutputs = 16 * kTiles;
  const bool whole = aligned_rows<T>(x, x_stride, rows) && aligned_rows<T>(weight, weight_stride, outer) && inner % 8 == 0;
  auto kernel = whole ? few_rows_kernel<T, kTokens, kTiles, true> : few_rows_kernel<T, kTokens, kTiles, false>;
  kernel<<<static_cast<unsigned>((outer + kOutputs - 1) / kOutputs), kWarps * 32, 0, s>>>(
      static_cast<const T*>(x), x_stride, static_cast<const T*>(weight), weight_stride, rows, inner, outer, e);
  return check_launch("few_rows_kernel");
}

// Two tiles of outputs halve what the blocks read of the tokens (16 tokens, 4096 x 8192: 18 us against 23); one leaves more
// blocks, where two would leave SMs idle (4096 x 4096: 13 us against 15).
template <typename T, int kTokens>
int run_tokens(const void* x, int64_t x_stride, const void* weight, int64_t weight_stride, int rows, int64_t inner, int64_t outer,
               const ProductEpilogue& e, cudaStream_t s) {
  if (outer > 32 * 148) return launch<T, kTokens, 2>(x, x_stride, weight, weight_stride, rows, inner, outer, e, s);
  return launch<T, kTokens, 1>(x, x_stride, weight, weight_stride, rows, inner, outer, e, s);
}

template <typename T>
int run_typed(const void* x, int64_t x_stride, const void* weight, int64_t weight_stride, int rows, int64_t inner, int64_t outer,
              const ProductEpilogue& e, cudaStream_t s) {
  if (rows <= 8) return run_tokens<T, 1>(x, x_stride, weight, weight_stride, rows, inner, outer, e, s);
  if (rows <= 16) return run_tokens<T, 2>(x, x_stride, weight, weight_stride, rows, inner, outer, e, s);
  if (rows <= 24) return run_tokens<T, 3>(x, x_stride, weight, weight_stride, rows, inner, outer, e, s);
  return run_tokens<T, 4>(x, x_stride, weight, weight_stride, rows, inner, outer, e, s);
}

}  // namespace

int run_few_rows(const void* x, int64_t x_stride, const void* weight, int64_t weight_stride, int64_t rows, int64_t inner,
                 int64_t outer, int dtype, const ProductEpilogue& e, cudaStream_t s) {
  if (rows == 0 || outer == 0) return CG_OK;
  const int tokens = static_cast<int>(rows);
  if (dtype == CG_F32) {
    const auto* from = static_cast<const float*>(x);
    const auto* w = static_cast<const float*>(weight);
    const bool whole = aligned_rows<float>(x, x_stride, rows) && aligned_rows<float>(w, weight_stride, outer) && inner % 4 == 0;
    if (tokens <= 2) return run_f32<2>(from, x_stride, w, weight_stride, tokens, inner, outer, whole, e, s);
    if (tokens <= 8) return run_f32<8>(from, x_stride, w, weight_stride, tokens, inner, outer, whole, e, s);
    if (tokens <= 16) return run_f32<16>(from, x_stride, w, weight_stride, tokens, inner, outer, whole, e, s);
    return run_f32<32>(from, x_stride, w, weight_stride, tokens, inner, outer, whole, e, s);
  }
  if (dtype == CG_F16) return run_typed<__half>(x, x_stride, weight, weight_stride, tokens, inner, outer, e, s);
  return run_typed<__nv_bfloat16>(x, x_stride, weight, weight_stride, tokens, inner, outer, e, s);
}

}  // namespace cg
