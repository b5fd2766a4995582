// A linear layer with its epilogue, and its backward pass:
//   y = act(x W^T + b) + residual          x [M, K], W [N, K], b [N], residual and y [M, N]
//   dpre = dy act'(pre), pre = x W^T + b;  dx = dpre W,  dW = dpre^T x,  db = sum over rows of dpre
// All three products are C[i, j] = sum_k A(i, k) B(j, k) over operands read in place through their strides.
// Sums are fp32 whatever the operands' type; results are rounded once to it.
#include <algorithm>

#include "common.cuh"

namespace cg {
namespace {

enum Activation { kNone = 0, kRelu = 1, kGelu = 2, kSilu = 3 };

template <typename T>
__device__ __forceinline__ float as_float(T v);
template <>
__device__ __forceinline__ float as_float(float v) { return v; }
template <>
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float as_float(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }

__device__ __forceinline__ float activate(float z, int activation) {
  if (activation == kRelu) return z < 0.f ? 0.f : z;  // a NaN stays one
  if (activation == kGelu) return gelu_erf(z);
  if (activation == kSilu) return z / (1.f + __expf(-z));
  return z;
}

__device__ __forceinline__ float activation_slope(float z, int activation) {
  if (activation == kRelu) return z > 0.f ? 1.f : z == z ? 0.f : z;
  if (activation == kGelu) {
    const float cumulative = 0.5f * (1.f + erff(z * 0.70710678118654752f));
    const float tail = z * z > 200.f ? 0.f : z * 0.3989422804014327f * __expf(-0.5f * z * z);
    return cumulative + tail;
  }
  if (activation == kSilu) {
    const float gate = 1.f / (1.f + __expf(-z));
    return gate * (1.f + z * (1.f - gate));
  }
  return 1.f;
}

struct Operand {
  const void* base;
  int64_t outer, inner;  // strides over i (or j) and over k
};

struct Epilogue {
  const void* bias;      // [J], or null
  const void* residual;  // [I, J], or null
  void* pre;             // [I, J] contiguous, or null: the sum before the activation, kept for the backward pass
  int64_t residual_stride, out_stride;
  int activation;
};

// ---- plain tiles: 64 x 64 outputs a block, 4 x 4 a thread, operands through shared memory -------------------
constexpr int kTile = 64, kDepth = 16;

template <typename T>
__global__ void __launch_bounds__(256) product_kernel(Operand a, Operand b, int64_t rows, int64_t cols, int64_t depth,
                                                      Epilogue e, T* out) {
  __shared__ float sa[kDepth][kTile + 1], sb[kDepth][kTile + 1];
  const int64_t i0 = static_cast<int64_t>(blockIdx.y) * kTile, j0 = static_cast<int64_t>(blockIdx.x) * kTile;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const T* pa = static_cast<const T*>(a.base);
  const T* pb = static_cast<const T*>(b.base);
  float acc[4][4] = {};
  for (int64_t k0 = 0; k0 < depth; k0 += kDepth) {
    for (int t = threadIdx.x; t < kTile * kDepth; t += 256) {
      const int i = a.inner == 1 ? t / kDepth : t % kTile, k = a.inner == 1 ? t % kDepth : t / kTile;
      sa[k][i] = i0 + i < rows && k0 + k < depth ? as_float(pa[(i0 + i) * a.outer + (k0 + k) * a.inner]) : 0.f;
    }
    for (int t = threadIdx.x; t < kTile * kDepth; t += 256) {
      const int j = b.inner == 1 ? t / kDepth : t % kTile, k = b.inner == 1 ? t % kDepth : t / kTile;
      sb[k][j] = j0 + j < cols && k0 + k < depth ? as_float(pb[(j0 + j) * b.outer + (k0 + k) * b.inner]) : 0.f;
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < kDepth; ++k)
#pragma unroll
      for (int u = 0; u < 4; ++u)
#pragma unroll
        for (int v = 0; v < 4; ++v) acc[u][v] = fmaf(sa[k][ty + 16 * u], sb[k][tx + 16 * v], acc[u][v]);
    __syncthreads();
  }
  for (int u = 0; u < 4; ++u)
    for (int v = 0; v < 4; ++v) {
      const int64_t i = i0 + ty + 16 * u, j = j0 + tx + 16 * v;
      if (i >= rows || j >= cols) continue;
      float z = acc[u][v];
      if (e.bias) z += as_float(static_cast<const T*>(e.bias)[j]);
      if (e.pre) put(static_cast<T*>(e.pre) + i * cols + j, z);
      z = activate(z, e.activation);
      if (e.residual) z += as_float(static_cast<const T*>(e.residual)[i * e.residual_stride + j]);
      put(out + i * e.out_stride + j, z);
    }
}

template <typename T>
int run_product(const Operand& a, const Operand& b, int64_t rows, int64_t cols, int64_t depth, const Epilogue& e, void* out,
                cudaStream_t s) {
  const dim3 grid(static_cast<unsigned>((cols + kTile - 1) / kTile), static_cast<unsigned>((rows + kTile - 1) / kTile));
  product_kernel<T><<<grid, 256, 0, s>>>(a, b, rows, cols, depth, e, static_cast<T*>(out));
  return check_launch("product_kernel");
}

// ---- dpre and the bias gradient -----------------------------------------------------------------------------------
// A block takes 32 columns of one slice of the rows; its warps' column sums join in shared memory, the slices' in
// order in the second kernel.
constexpr int kSlices = 64;

template <typename T>
__global__ void __launch_bounds__(256) slope_kernel(const T* dy, int64_t dy_stride, const T* pre, int64_t rows, int64_t cols,
                                                    int64_t slice, int activation, T* dpre, float* partial) {
  __shared__ float s[8][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t j = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  const int64_t lo = blockIdx.y * slice, hi = min(rows, lo + slice);
  float sum = 0.f;
  if (j < cols)
    for (int64_t i = lo + warp; i < hi; i += 8) {
      float g = as_float(dy[i * dy_stride + j]);
      if (pre) g *= activation_slope(as_float(pre[i * cols + j]), activation);
      if (dpre) put(dpre + i * cols + j, g);
      sum += g;
    }
  s[warp][lane] = sum;
  __syncthreads();
  if (partial && warp == 0 && j < cols) {
    for (int w = 1; w < 8; ++w) sum += s[w][lane];
    partial[blockIdx.y * cols + j] = sum;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) bias_sum_kernel(const float* partial, int slices, int64_t cols, T* db) {
  const int64_t j = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  pdl_wait();
  if (j >= cols) return;
  float sum = 0.f;
  for (int k = 0; k < slices; ++k) sum += partial[k * cols + j];
  put(db + j, sum);
}

bool valid_extent(int64_t rows, int64_t cols, int64_t depth) {
  constexpr int64_t most = int64_t{1} << 31;
  return rows >= 0 && cols >= 0 && depth >= 0 && rows < most && cols < most && depth < most;
}

template <typename T>
int forward(const void* x, int64_t x_stride, const void* weight, int64_t weight_stride, int64_t rows, int64_t inner,
            int64_t outer, const Epilogue& e, void* y, cudaStream_t s) {
  return run_product<T>({x, x_stride, 1}, {weight, weight_stride, 1}, rows, outer, inner, e, y, s);
}

template <typename T>
int backward(const void* dy, int64_t dy_stride, const void* pre, const void* x, int64_t x_stride, const void* weight,
             int64_t weight_stride, int64_t rows, int64_t inner, int64_t outer, int activation, void* dx, void* dweight,
             void* dbias, char* workspace, cudaStream_t s) {
  T* dpre = nullptr;
  float* partial = reinterpret_cast<float*>(workspace);
  if (activation != kNone) dpre = reinterpret_cast<T*>(workspace + kSlices * outer * sizeof(float));
  const int64_t slice = (rows + kSlices - 1) / kSlices;
  if ((dpre || dbias) && rows > 0 && outer > 0) {
    const dim3 grid(static_cast<unsigned>((outer + 31) / 32), static_cast<unsigned>((rows + slice - 1) / slice));
    slope_kernel<T><<<grid, 256, 0, s>>>(static_cast<const T*>(dy), dy_stride, static_cast<const T*>(pre), rows, outer, slice,
                                         activation, dpre, dbias ? partial : nullptr);
    if (int rc = check_launch("slope_kernel")) return rc;
  }
  if (dbias) {
    const int slices = rows > 0 ? static_cast<int>((rows + slice - 1) / slice) : 0;
    if (int rc = launch_pdl("bias_sum_kernel", bias_sum_kernel<T>, dim3(static_cast<unsigned>((outer + 255) / 256)), dim3(256),
                            0, s, static_cast<const float*>(partial), slices, outer, static_cast<T*>(dbias)))
      return rc;
  }
  const void* g = dpre ? dpre : dy;
  const int64_t g_stride = dpre ? outer : dy_stride;
  if (dx && rows > 0) {
    const Epilogue e = {nullptr, nullptr, nullptr, 0, inner, kNone};
    if (int rc = run_product<T>({g, g_stride, 1}, {weight, 1, weight_stride}, rows, inner, outer, e, dx, s)) return rc;
  }
  if (dweight) {
    const Epilogue e = {nullptr, nullptr, nullptr, 0, inner, kNone};
    if (int rc = run_product<T>({g, 1, g_stride}, {x, 1, x_stride}, outer, inner, rows, e, dweight, s)) return rc;
  }
  return CG_OK;
}

}  // namespace
}  // namespace cg

namespace cg {
namespace {
int64_t workspace_bytes_of(int dtype, int64_t rows, int64_t outer, bool backward) {
  return backward ? kSlices * outer * static_cast<int64_t>(sizeof(float)) + rows * outer * dtype_size(dtype) : 0;
}
}  // namespace
}  // namespace cg

extern "C" int64_t cg_linear_workspace_bytes(const void*, int64_t, const void*, int64_t, const void*, int64_t, int dtype,
                                             int64_t rows, int64_t inner, int64_t outer, int, int backward) {
  using namespace cg;
  if (!valid_extent(rows, outer, inner) || !valid_dtype(dtype)) {
    set_error(CG_ERR_ARGUMENT, "cg_linear_workspace_bytes: bad shape or dtype");
    return -1;
  }
  return workspace_bytes_of(dtype, rows, outer, backward);
}

extern "C" int cg_linear_forward(const void* x, int64_t x_stride, const void* weight, int64_t weight_stride, const void* bias,
                                 const void* residual, int64_t residual_stride, int dtype, int64_t rows, int64_t inner,
                                 int64_t outer, int activation, void* y, void* pre, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  using namespace cg;
  CG_REQUIRE(valid_dtype(dtype), "cg_linear_forward: dtype must be float32, float16 or bfloat16");
  CG_REQUIRE(valid_extent(rows, outer, inner), "cg_linear_forward: bad shape");
  CG_REQUIRE(activation >= kNone && activation <= kSilu, "cg_linear_forward: unknown activation");
  CG_REQUIRE(x_stride >= inner && weight_stride >= inner && (!residual || residual_stride >= outer),
             "cg_linear_forward: stride smaller than a row");
  if (rows == 0 || outer == 0) return CG_OK;
  CG_REQUIRE(y && (inner == 0 || (x && weight)), "cg_linear_forward: NULL pointer");
  (void)workspace;
  (void)workspace_bytes;
  const Epilogue e = {bias, residual, pre, residual_stride, outer, activation};
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == CG_F32) return forward<float>(x, x_stride, weight, weight_stride, rows, inner, outer, e, y, s);
  if (dtype == CG_F16) return forward<__half>(x, x_stride, weight, weight_stride, rows, inner, outer, e, y, s);
  return forward<__nv_bfloat16>(x, x_stride, weight, weight_stride, rows, inner, outer, e, y, s);
}

extern "C" int cg_linear_backward(const void* dy, int64_t dy_stride, const void* pre, const void* x, int64_t x_stride,
                                  const void* weight, int64_t weight_stride, int dtype, int64_t rows, int64_t inner,
                                  int64_t outer, int activation, void* dx, void* dweight, void* dbias, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  using namespace cg;
  CG_REQUIRE(valid_dtype(dtype), "cg_linear_backward: dtype must be float32, float16 or bfloat16");
  CG_REQUIRE(valid_extent(rows, outer, inner), "cg_linear_backward: bad shape");
  CG_REQUIRE(activation >= kNone && activation <= kSilu, "cg_linear_backward: unknown activation");
  CG_REQUIRE(dy_stride >= outer && x_stride >= inner && weight_stride >= inner,
             "cg_linear_backward: stride smaller than a row");
  CG_REQUIRE(rows == 0 || outer == 0 || (dy && (activation == kNone || pre)), "cg_linear_backward: NULL pointer");
  if (!workspace || workspace_bytes < workspace_bytes_of(dtype, rows, outer, true))
    return set_error(CG_ERR_WORKSPACE, "cg_linear_backward: workspace too small");
  char* w = static_cast<char*>(workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (inner == 0) dx = dweight = nullptr;
  if (outer == 0) dweight = dbias = nullptr;
  if (dtype == CG_F32)
    return backward<float>(dy, dy_stride, pre, x, x_stride, weight, weight_stride, rows, inner, outer, activation, dx, dweight,
                           dbias, w, s);
  if (dtype == CG_F16)
    return backward<__half>(dy, dy_stride, pre, x, x_stride, weight, weight_stride, rows, inner, outer, activation, dx, dweight,
                            dbias, w, s);
  return backward<__nv_bfloat16>(dy, dy_stride, pre, x, x_stride, weight, weight_stride, rows, inner, outer, activation, dx,
                                 dweight, dbias, w, s);
}
