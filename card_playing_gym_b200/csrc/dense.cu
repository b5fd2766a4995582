// A linear layer with its epilogue, and its backward pass:
//   y = act(x W^T + b) + residual          x [M, K], W [N, K], b [N], residual and y [M, N]
//   dpre = dy act'(pre), pre = x W^T + b;  dx = dpre W,  dW = dpre^T x,  db = sum over rows of dpre
// The products run on the tensor cores (product.cu), which reads 16-bit operands in place in either order; around them:
//
//   pack_kernel   float32 operands as three bfloat16 parts; 16-bit operands whose rows do not start on 16 bytes
//                 as a copy that does
//   slope_kernel  dpre, in the form the products read, and the column sums of db in the same pass over dy and pre
//
// Up to ten launches a pass: each is set up while the one before it drains.
//
// pre and dpre are kept in the operands' type: a 16-bit pre moves act' by its slope times 2^-8 |pre| (bfloat16) and a
// 16-bit dpre is what the tensor cores multiply; db sums dpre before that rounding.
#include <algorithm>

#include "elements.cuh"

namespace cg {
namespace {

// ---- operands in the products' form --------------------------------------------------------------------------------
// Four entries of a T matrix in operand form at `out`: T itself, or a float32's three parts, `part` entries apart.
template <typename T>
__device__ __forceinline__ void store_operand(typename OperandOf<T>::type* out, int64_t part, const float (&v)[4]) {
  if constexpr (sizeof(T) == 4) {
    __nv_bfloat16 p[4][3];
#pragma unroll
    for (int i = 0; i < 4; ++i) three_parts(v[i], p[i]);
#pragma unroll
    for (int k = 0; k < 3; ++k) {
      uint2 raw;
      auto* h = reinterpret_cast<__nv_bfloat16*>(&raw);
#pragma unroll
      for (int i = 0; i < 4; ++i) h[i] = p[i][k];
      *reinterpret_cast<uint2*>(out + k * part) = raw;
    }
  } else {
    store4(out, v);
  }
}

template <typename T>
__global__ void __launch_bounds__(256) pack_kernel(const T* in, int64_t stride, int64_t rows, int64_t cols,
                                                   typename OperandOf<T>::type* out, int64_t out_stride) {
  pdl_wait();
  pdl_trigger();
  const bool aligned = aligned4<T>(in, stride);
  const int64_t quads = (cols + 3) / 4, total = rows * quads;
  for (int64_t index = blockIdx.x * 256ll + threadIdx.x; index < total; index += gridDim.x * 256ll) {
    const int64_t i = index / quads, j = (index - i * quads) * 4;
    float v[4];
    load4(in + i * stride + j, static_cast<int>(min(int64_t{4}, cols - j)), aligned && j + 4 <= cols, v);
    store_operand<T>(out + i * out_stride + j, rows * out_stride, v);
  }
}

// ---- dpre and the bias gradient -----------------------------------------------------------------------------------
// A block takes 32 sixteen-byte vectors of columns of one slice of the rows, a vector a lane, a row a warp at a time. Its
// warps' column sums join in shared memory, the slices' in order in bias_sum_kernel. It is bound by memory once the
// activation's slope costs one exponential and rows are under way while others are computed: 8192 x 4096 bfloat16 with
// GELU 37 us for 201 MB, 83% of the copy bandwidth.
template <typename T>
constexpr int kSlopeVector = 16 / static_cast<int>(sizeof(T));

template <typename T>
__device__ __forceinline__ bool aligned_vector(const void* base, int64_t stride) {
  return (reinterpret_cast<uintptr_t>(base) & 15) == 0 && stride % kSlopeVector<T> == 0;
}

// The first n entries of a vector at `p`; `whole`: all of them, aligned to four.
template <typename T, int kVec>
__device__ __forceinline__ void load_vector(const T* __restrict__ p, int n, bool whole, float (&v)[kVec]) {
#pragma unroll
  for (int k = 0; k < kVec; k += 4) {
    float part[4];
    load4(p + k, n - k, whole, part);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[k + i] = part[i];
  }
}

template <typename T, int kActivation>
__global__ void __launch_bounds__(256, 3) slope_kernel(const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ pre,
                                                       int64_t rows, int64_t cols, int64_t slice,
                                                       typename OperandOf<T>::type* __restrict__ dpre, int64_t dpre_stride,
                                                       float* __restrict__ partial) {
  constexpr int kVec = kSlopeVector<T>, kRows = 2;
  __shared__ float s[8][32 * kVec];
  pdl_trigger();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t j = (static_cast<int64_t>(blockIdx.x) * 32 + lane) * kVec;
  const int64_t lo = blockIdx.y * slice, hi = min(rows, lo + slice);
  const int n = static_cast<int>(max(int64_t{0}, min(static_cast<int64_t>(kVec), cols - j)));
  const bool whole_dy = aligned_vector<T>(dy, dy_stride) && n == kVec, whole_pre = aligned_vector<T>(pre, cols) && n == kVec;
  float sum[kVec] = {};
  // One row's gradients, times the slopes, to their place and into the sums.
  auto take_row = [&](int64_t i, float (&g)[kVec], const float (&z)[kVec]) {
    if constexpr (kActivation != kActNone) times_slope<T, kActivation>(g, z);
#pragma unroll
    for (int k = 0; k < kVec; ++k) sum[k] += g[k];
    if (!dpre) return;
#pragma unroll
    for (int k = 0; k < kVec; k += 4) {
      const float part[4] = {g[k], g[k + 1], g[k + 2], g[k + 3]};
      if (k < n) store_operand<T>(dpre + i * dpre_stride + j + k, rows * dpre_stride, part);
    }
  };
  if (whole_dy && (kActivation == kActNone || whole_pre)) {
    // Two rows' vectors as they are in memory, the next two's under way while these are computed. Two sets of registers
    // are taken in turn: a copy would wait for its loads.
    struct Rows {
      uint4 g[kRows], z[kRows];
    } even, odd;
    auto load = [&](Rows& r, int64_t i0) {
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        const int64_t i = min(i0 + 8 * k, hi - 1);  // past the slice: a row that is not used
        r.g[k] = *reinterpret_cast<const uint4*>(dy + i * dy_stride + j);
        if (kActivation != kActNone) r.z[k] = *reinterpret_cast<const uint4*>(pre + i * cols + j);
      }
    };
    int64_t i0 = lo + warp;
    auto step = [&](Rows& now, Rows& next) {
      const int64_t after = i0 + 8 * kRows;
      if (after < hi) load(next, after);
#pragma unroll
      for (int k = 0; k < kRows; ++k) {
        if (i0 + 8 * k >= hi) continue;
        float g[kVec], z[kVec];
        load_vector<T, kVec>(reinterpret_cast<const T*>(&now.g[k]), kVec, true, g);
        if (kActivation != kActNone) load_vector<T, kVec>(reinterpret_cast<const T*>(&now.z[k]), kVec, true, z);
        take_row(i0 + 8 * k, g, z);
      }
      i0 = after;
      return after < hi;
    };
    if (i0 < hi) {
      load(even, i0);
      while (step(even, odd) && step(odd, even)) {
      }
    }
  } else if (n > 0) {
    for (int64_t i = lo + warp; i < hi; i += 8) {
      float g[kVec], z[kVec];
      load_vector<T, kVec>(dy + i * dy_stride + j, n, whole_dy, g);
      if (kActivation != kActNone) load_vector<T, kVec>(pre + i * cols + j, n, whole_pre, z);
      take_row(i, g, z);
    }
  }
  if (!partial) return;
#pragma unroll
  for (int k = 0; k < kVec; ++k) s[warp][k * 32 + lane] = sum[k];
  __syncthreads();
  for (int c = threadIdx.x; c < 32 * kVec; c += 256) {
    const int64_t column = static_cast<int64_t>(blockIdx.x) * 32 * kVec + (c & 31) * kVec + (c >> 5);
    if (column >= cols) continue;
    float total = s[0][c];
#pragma unroll
    for (int w = 1; w < 8; ++w) total += s[w][c];
    partial[blockIdx.y * cols + column] = total;
  }
}

template <typename T>
__global__ void __launch_bounds__(256) bias_sum_kernel(const float* partial, int slices, int64_t cols, T* db) {
  __shared__ float s[8][33];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t j = static_cast<int64_t>(blockIdx.x) * 32 + lane;
  pdl_wait();
  pdl_trigger();
  float sum = 0.f;
  if (j < cols)
    for (int k = warp; k < slices; k += 8) sum += partial[k * cols + j];
  s[warp][lane] = sum;
  __syncthreads();
  if (warp != 0 || j >= cols) return;
  for (int w = 1; w < 8; ++w) sum += s[w][lane];
  put(db + j, sum);
}

// ---- plans -----------------------------------------------------------------------------------------------------------
bool valid_extent(int64_t rows, int64_t cols, int64_t depth) {
  constexpr int64_t most = (int64_t{1} << 31) - 256;
  return rows >= 0 && cols >= 0 && depth >= 0 && rows < most && cols < most && depth < most;
}

int64_t padded(int64_t bytes) { return (bytes + 255) / 256 * 256; }
int64_t padded_row(int64_t entries) { return (entries + 7) / 8 * 8; }

// Whether an operand has to be packed: every float32 one, and a 16-bit one whose rows do not all start on 16 bytes.
bool needs_pack(const void* base, int64_t stride, int64_t rows, int dtype) {
  return dtype == CG_F32 || (reinterpret_cast<uintptr_t>(base) & 15) != 0 || (rows > 1 && stride % 8 != 0);
}

int64_t packed_bytes(int64_t rows, int64_t cols, int dtype) {
  return padded(rows * padded_row(cols) * 2 * (dtype == CG_F32 ? 3 : 1));
}

struct Layout {
  int64_t sums, dpre, x, weight, partial, bytes;  // byte offsets, -1 where a part is not needed
  int64_t slice;
  int slices;
};

Layout plan_layout(const void* x, int64_t x_stride, const void* weight, int64_t weight_stride, const void* dy, int64_t dy_stride,
                   int dtype, int64_t rows, int64_t inner, int64_t outer, int activation, bool backward) {
  Layout l = {-1, -1, -1, -1, -1, 0, 1, 0};
  auto take = [&](int64_t bytes) {
    const int64_t at = l.bytes;
    l.bytes += padded(bytes);
    return at;
  };
  if (backward) {
    // Blocks of 32 vectors of columns by slices of the rows: six blocks an SM, slices of at least 32 rows.
    const int64_t columns = 32 * (16 / (dtype == CG_F32 ? 4 : 2));
    const int64_t across = (outer + columns - 1) / columns;
    int64_t slices = std::max<int64_t>(1, 6 * 148 / std::max<int64_t>(across, 1));
    slices = std::max<int64_t>(1, std::min(slices, (rows + 31) / 32));
    l.slice = std::max<int64_t>(1, (rows + slices - 1) / slices);
    l.slices = static_cast<int>((rows + l.slice - 1) / l.slice);
    l.sums = take(l.slices * outer * static_cast<int64_t>(sizeof(float)));
    if (activation != kActNone || needs_pack(dy, dy_stride, rows, dtype)) l.dpre = take(packed_bytes(rows, outer, dtype));
  }
  if (!backward && few_rows(rows, inner, outer, dtype)) return l;
  if (needs_pack(x, x_stride, rows, dtype)) l.x = take(packed_bytes(rows, inner, dtype));
  if (needs_pack(weight, weight_stride, outer, dtype)) l.weight = take(packed_bytes(outer, inner, dtype));
  const int64_t partial = backward ? std::max(plan_product(rows, inner, outer, dtype).bytes(),
                                              plan_product(outer, inner, rows, dtype).bytes())
                                   : plan_product(rows, outer, inner, dtype).bytes();
  l.partial = take(partial);
  return l;
}

template <typename T>
int pack(const void* in, int64_t stride, int64_t rows, int64_t cols, void* out, cudaStream_t s) {
  const int64_t quads = rows * ((cols + 3) / 4);
  if (quads == 0) return CG_OK;
  const int blocks = static_cast<int>(std::min<int64_t>((quads + 255) / 256, 16 * sm_count()));
  return launch_pdl("pack_kernel", pack_kernel<T>, dim3(blocks), dim3(256), 0, s, static_cast<const T*>(in), stride, rows, cols,
                    static_cast<typename OperandOf<T>::type*>(out), padded_row(cols));
}

// An operand read in place. A single row has no stride to speak of.
ProductOperand in_place(const void* base, int64_t stride, int64_t rows, int64_t cols) {
  return {base, rows > 1 ? stride : padded_row(cols), 0, false};
}

// An operand stored [rows, cols], packed where its layout has a place for it.
template <typename T>
int operand(const void* base, int64_t stride, int64_t rows, int64_t cols, char* workspace, int64_t at, ProductOperand* o,
            cudaStream_t s) {
  *o = in_place(base, stride, rows, cols);
  if (at < 0) return CG_OK;
  *o = {workspace + at, padded_row(cols), rows * padded_row(cols), false};
  return pack<T>(base, stride, rows, cols, workspace + at, s);
}

ProductOperand across(ProductOperand o) {
  o.across = true;
  return o;
}

template <typename T>
int forward(const Layout& l, const void* x, int64_t x_stride, const void* weight, int64_t weight_stride, int dtype, int64_t rows,
            int64_t inner, int64_t outer, const ProductEpilogue& e, char* workspace, cudaStream_t s) {
  ProductOperand a, b;
  if (int rc = operand<T>(x, x_stride, rows, inner, workspace, l.x, &a, s)) return rc;
  if (int rc = operand<T>(weight, weight_stride, outer, inner, workspace, l.weight, &b, s)) return rc;
  return run_product(a, b, rows, outer, inner, dtype, e, workspace + l.partial, s);
}

template <typename T>
int backward(const Layout& l, const void* dy, int64_t dy_stride, const void* pre, const void* x, int64_t x_stride,
             const void* weight, int64_t weight_stride, int dtype, int64_t rows, int64_t inner, int64_t outer, int activation,
             void* dx, void* dweight, void* dbias, char* workspace, cudaStream_t s) {
  using O = typename OperandOf<T>::type;
  auto* sums = reinterpret_cast<float*>(workspace + l.sums);
  O* dpre = l.dpre < 0 || !(dx || dweight) ? nullptr : reinterpret_cast<O*>(workspace + l.dpre);
  if ((dpre || dbias) && rows > 0 && outer > 0) {
    constexpr int kColumns = 32 * kSlopeVector<T>;
    const dim3 grid(static_cast<unsigned>((outer + kColumns - 1) / kColumns), static_cast<unsigned>(l.slices));
    auto kernel = activation == kActRelu   ? slope_kernel<T, kActRelu>
                  : activation == kActGelu ? slope_kernel<T, kActGelu>
                  : activation == kActSilu ? slope_kernel<T, kActSilu>
                                           : slope_kernel<T, kActNone>;
    kernel<<<grid, 256, 0, s>>>(static_cast<const T*>(dy), dy_stride, static_cast<const T*>(pre), rows, outer, l.slice, dpre,
                                padded_row(outer), dbias ? sums : nullptr);
    if (int rc = check_launch("slope_kernel")) return rc;
  }
  if (dbias) {
    if (int rc = launch_pdl("bias_sum_kernel", bias_sum_kernel<T>, dim3(static_cast<unsigned>((outer + 31) / 32)), dim3(256), 0, s,
                            static_cast<const float*>(sums), rows > 0 ? l.slices : 0, outer, static_cast<T*>(dbias)))
      return rc;
  }
  const ProductOperand g = dpre ? ProductOperand{dpre, padded_row(outer), rows * padded_row(outer), false}
                                : in_place(dy, dy_stride, rows, outer);
  const ProductEpilogue into = {nullptr, nullptr, nullptr, nullptr, 0, inner, kActNone};
  ProductOperand o;
  if (dx) {
    if (int rc = operand<T>(weight, weight_stride, outer, inner, workspace, l.weight, &o, s)) return rc;
    ProductEpilogue e = into;
    e.out = dx;
    if (int rc = run_product(g, across(o), rows, inner, outer, dtype, e, workspace + l.partial, s)) return rc;
  }
  if (dweight) {
    if (int rc = operand<T>(x, x_stride, rows, inner, workspace, l.x, &o, s)) return rc;
    ProductEpilogue e = into;
    e.out = dweight;
    if (int rc = run_product(across(g), across(o), outer, inner, rows, dtype, e, workspace + l.partial, s)) return rc;
  }
  return CG_OK;
}

}  // namespace
}  // namespace cg

extern "C" int64_t cg_linear_workspace_bytes(const void* x, int64_t x_stride, const void* weight, int64_t weight_stride,
                                             const void* dy, int64_t dy_stride, int dtype, int64_t rows, int64_t inner,
                                             int64_t outer, int activation, int backward) {
  using namespace cg;
  if (!valid_extent(rows, outer, inner) || !valid_dtype(dtype)) {
    set_error(CG_ERR_ARGUMENT, "cg_linear_workspace_bytes: bad shape or dtype");
    return -1;
  }
  return plan_layout(x, x_stride, weight, weight_stride, dy, dy_stride, dtype, rows, inner, outer, activation, backward).bytes;
}

extern "C" int cg_linear_forward(const void* x, int64_t x_stride, const void* weight, int64_t weight_stride, const void* bias,
                                 const void* residual, int64_t residual_stride, int dtype, int64_t rows, int64_t inner,
                                 int64_t outer, int activation, void* y, void* pre, void* workspace,
                                 int64_t workspace_bytes, void* stream) {
  using namespace cg;
  CG_REQUIRE(valid_dtype(dtype), "cg_linear_forward: dtype must be float32, float16 or bfloat16");
  CG_REQUIRE(valid_extent(rows, outer, inner), "cg_linear_forward: bad shape");
  CG_REQUIRE(activation >= kActNone && activation <= kActSilu, "cg_linear_forward: unknown activation");
  CG_REQUIRE(x_stride >= inner && weight_stride >= inner && (!residual || residual_stride >= outer),
             "cg_linear_forward: stride smaller than a row");
  if (rows == 0 || outer == 0) return CG_OK;
  CG_REQUIRE(y && (inner == 0 || (x && weight)), "cg_linear_forward: NULL pointer");
  const Layout l = plan_layout(x, x_stride, weight, weight_stride, nullptr, 0, dtype, rows, inner, outer, activation, false);
  if (workspace_bytes < l.bytes || (l.bytes && !workspace))
    return set_error(CG_ERR_WORKSPACE, "cg_linear_forward: workspace too small");
  const ProductEpilogue e = {bias, residual, pre, y, residual_stride, outer, activation};
  char* w = static_cast<char*>(workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (few_rows(rows, inner, outer, dtype)) return run_few_rows(x, x_stride, weight, weight_stride, rows, inner, outer, dtype, e, s);
  if (dtype == CG_F32) return forward<float>(l, x, x_stride, weight, weight_stride, dtype, rows, inner, outer, e, w, s);
  if (dtype == CG_F16) return forward<__half>(l, x, x_stride, weight, weight_stride, dtype, rows, inner, outer, e, w, s);
  return forward<__nv_bfloat16>(l, x, x_stride, weight, weight_stride, dtype, rows, inner, outer, e, w, s);
}

extern "C" int cg_linear_backward(const void* dy, int64_t dy_stride, const void* pre, const void* x, int64_t x_stride,
                                  const void* weight, int64_t weight_stride, int dtype, int64_t rows, int64_t inner,
                                  int64_t outer, int activation, void* dx, void* dweight, void* dbias, void* workspace,
                                  int64_t workspace_bytes, void* stream) {
  using namespace cg;
  CG_REQUIRE(valid_dtype(dtype), "cg_linear_backward: dtype must be float32, float16 or bfloat16");
  CG_REQUIRE(valid_extent(rows, outer, inner), "cg_linear_backward: bad shape");
  CG_REQUIRE(activation >= kActNone && activation <= kActSilu, "cg_linear_backward: unknown activation");
  CG_REQUIRE(dy_stride >= outer && x_stride >= inner && weight_stride >= inner,
             "cg_linear_backward: stride smaller than a row");
  CG_REQUIRE(rows == 0 || outer == 0 || (dy && (activation == kActNone || pre)), "cg_linear_backward: NULL pointer");
  const Layout l = plan_layout(x, x_stride, weight, weight_stride, dy, dy_stride, dtype, rows, inner, outer, activation, true);
  if (workspace_bytes < l.bytes || (l.bytes && !workspace))
    return set_error(CG_ERR_WORKSPACE, "cg_linear_backward: workspace too small");
  char* w = static_cast<char*>(workspace);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (inner == 0) dx = dweight = nullptr;
  if (rows == 0) dx = nullptr;
  if (outer == 0) dweight = dbias = nullptr;
  CG_REQUIRE((!dx || weight || outer == 0) && (!dweight || x || rows == 0), "cg_linear_backward: NULL pointer");
  if (dtype == CG_F32)
    return backward<float>(l, dy, dy_stride, pre, x, x_stride, weight, weight_stride, dtype, rows, inner, outer, activation, dx,
                           dweight, dbias, w, s);
  if (dtype == CG_F16)
    return backward<__half>(l, dy, dy_stride, pre, x, x_stride, weight, weight_stride, dtype, rows, inner, outer, activation, dx,
                            dweight, dbias, w, s);
  return backward<__nv_bfloat16>(l, dy, dy_stride, pre, x, x_stride, weight, weight_stride, dtype, rows, inner, outer, activation,
                                 dx, dweight, dbias, w, s);
}
