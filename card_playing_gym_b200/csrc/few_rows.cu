// The linear layer for a few tokens: y = act(x W^T + b) + residual with at most 32 rows of x.
//
// W is read once and is all there is to read, so a block takes 16 or 32 outputs and all the tokens, and its eight warps
// split k. A lane loads W straight from memory into mma fragments, past L1, which keeps the tokens. The products run on mma.sync m16n8k16 with W as the 16-row operand and eight tokens as its
// columns: at these sizes the tensor cores are idle either way, and what counts is that a token costs no
// instructions of its own. k's order inside a fragment does not matter as long as both operands agree, so a lane
// loads eight neighbouring k's in one access. The warps' sums join in shared memory in a fixed order.
//
// float32 operands are cut into three bfloat16 parts in registers; six products of parts reach 2^-24.
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

// Eight entries as the operand's four registers (of each part).
template <typename T>
struct Fragment {
  static constexpr int kParts = 1;
  uint32_t w[1][4];
  __device__ __forceinline__ explicit Fragment(const Eight<T>& e) {
    const uint32_t* r = reinterpret_cast<const uint32_t*>(&e);
#pragma unroll
    for (int i = 0; i < 4; ++i) w[0][i] = r[i];
  }
};
template <>
struct Fragment<float> {
  static constexpr int kParts = 3;
  uint32_t w[3][4];
  __device__ __forceinline__ explicit Fragment(const Eight<float>& e) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      __nv_bfloat16 low[3], high[3];
      three_parts(e.v[2 * i], low);
      three_parts(e.v[2 * i + 1], high);
#pragma unroll
      for (int k = 0; k < 3; ++k) w[k][i] = __bfloat16_as_ushort(low[k]) | static_cast<uint32_t>(__bfloat16_as_ushort(high[k])) << 16;
    }
  }
};

// kTokens: groups of eight tokens; kTiles: tiles of 16 outputs. A step is 32 k's of float32 and 64 of 16-bit operands.
template <typename T, int kTokens, int kTiles, bool kAligned>
__global__ void __launch_bounds__(kWarps * 32, sizeof(T) == 2 ? 2 : 1) few_rows_kernel(
    const T* x, int64_t x_stride, const T* weight, int64_t weight_stride, int rows, int64_t inner, int64_t outer,
    const ProductEpilogue e) {
  using O = typename OperandOf<T>::type;
  constexpr int kOutputs = 16 * kTiles, kHalves = sizeof(T) == 2 ? 2 : 1, kStep = 32 * kHalves;
  __shared__ float sums[kWarps][kTokens * 8][kOutputs + 1];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int64_t j0 = static_cast<int64_t>(blockIdx.x) * kOutputs;
  const T* from_w = weight + (j0 + g) * weight_stride + t * 8;
  const T* from_x = x + g * x_stride + t * 8;
  float c[kTiles][kTokens][4] = {};
  struct Step {
    Eight<T> a[kTiles][kHalves][2];
  } now;
  // float32: the next step's loads run under this one's cutting into parts (8 tokens, 4096 x 8192: 59 against 64 us). 16-bit
  // operands have no such work to hide and do better with the registers (24 tokens: 19.6 us, with it 23.2).
  constexpr bool kAhead = sizeof(T) == 4;
  Step next;
  auto load = [&](Step& s, int64_t k0) {
#pragma unroll
    for (int m = 0; m < kTiles; ++m)
#pragma unroll
      for (int h = 0; h < kHalves; ++h)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int64_t k = k0 + h * 32, row = m * 16 + r * 8;
          s.a[m][h][r] = load_eight<kAligned, true>(from_w + row * weight_stride + k, j0 + g + row < outer ? inner - k - t * 8 : 0);
        }
  };
  int64_t k0 = warp * kStep;
  if (k0 < inner) load(now, k0);
  while (k0 < inner) {
    const int64_t after = k0 + kWarps * kStep;
    if (kAhead && after < inner) load(next, after);
#pragma unroll
    for (int h = 0; h < kHalves; ++h) {
      const int64_t k = k0 + h * 32;
#pragma unroll
      for (int n = 0; n < kTokens; ++n) {
        const Fragment<T> f(load_eight<kAligned, false>(from_x + n * 8 * x_stride + k, n * 8 + g < rows ? inner - k - t * 8 : 0));
#pragma unroll
        for (int m = 0; m < kTiles; ++m) {
          const Fragment<T> a0(now.a[m][h][0]), a1(now.a[m][h][1]);
          // Parts by falling total rank: the smallest products first.
#pragma unroll
          for (int rank = Fragment<T>::kParts - 1; rank >= 0; --rank)
#pragma unroll
            for (int pa = 0; pa <= rank; ++pa) {
              const int pb = rank - pa;
              mma_16816(c[m][n], a0.w[pa][0], a1.w[pa][0], a0.w[pa][1], a1.w[pa][1], f.w[pb][0], f.w[pb][1], O());
              mma_16816(c[m][n], a0.w[pa][2], a1.w[pa][2], a0.w[pa][3], a1.w[pa][3], f.w[pb][2], f.w[pb][3], O());
            }
        }
      }
    }
    if (kAhead)
      now = next;
    else if (after < inner)
      load(now, after);
    k0 = after;
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
      const int64_t j = j0 + o;
      if (token >= rows || j >= outer) continue;
      float z = 0.f;
#pragma unroll
      for (int s = 0; s < kWarps; ++s) z += sums[s][token][o];
      if (e.bias) z += as_float(static_cast<const T*>(e.bias)[j]);
      if (e.pre) put(static_cast<T*>(e.pre) + token * outer + j, z);
      z = activate<T, activation>(z);
      if (e.residual) z += as_float(static_cast<const T*>(e.residual)[token * e.residual_stride + j]);
      put(static_cast<T*>(e.out) + token * e.out_stride + j, z);
    }
  });
}

template <typename T, int kTokens, int kTiles>
int launch(const void* x, int64_t x_stride, const void* weight, int64_t weight_stride, int rows, int64_t inner, int64_t outer,
           const ProductEpilogue& e, cudaStream_t s) {
  constexpr int kOutputs = 16 * kTiles;
  auto aligned = [](const void* base, int64_t stride, int64_t count) {
    return (reinterpret_cast<uintptr_t>(base) & 15) == 0 && (count == 1 || stride * sizeof(T) % 16 == 0);
  };
  const bool whole = aligned(x, x_stride, rows) && aligned(weight, weight_stride, outer) && inner % 8 == 0;
  auto kernel = whole ? few_rows_kernel<T, kTokens, kTiles, true> : few_rows_kernel<T, kTokens, kTiles, false>;
  kernel<<<static_cast<unsigned>((outer + kOutputs - 1) / kOutputs), kWarps * 32, 0, s>>>(
      static_cast<const T*>(x), x_stride, static_cast<const T*>(weight), weight_stride, rows, inner, outer, e);
  return check_launch("few_rows_kernel");
}

// Two tiles of outputs halve what the blocks read of the tokens; one leaves more blocks, where two would leave SMs idle.
template <typename T, int kTokens>
int run_tokens(const void* x, int64_t x_stride, const void* weight, int64_t weight_stride, int rows, int64_t inner, int64_t outer,
               const ProductEpilogue& e, cudaStream_t s) {
  if constexpr (sizeof(T) == 2) {
    if (outer > 32 * 148) return launch<T, kTokens, 2>(x, x_stride, weight, weight_stride, rows, inner, outer, e, s);
  }
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
  if (dtype == CG_F32) return run_typed<float>(x, x_stride, weight, weight_stride, tokens, inner, outer, e, s);
  if (dtype == CG_F16) return run_typed<__half>(x, x_stride, weight, weight_stride, tokens, inner, outer, e, s);
  return run_typed<__nv_bfloat16>(x, x_stride, weight, weight_stride, tokens, inner, outer, e, s);
}

}  // namespace cg
