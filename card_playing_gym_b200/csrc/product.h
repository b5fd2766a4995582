// The tensor-core product behind the linear layer: C[i, j] = sum_k A(i, k) B(j, k) with a fused epilogue.
#pragma once

#include "common.cuh"

namespace cg {

enum Activation { kActNone = 0, kActRelu = 1, kActGelu = 2, kActSilu = 3 };

// What becomes of a sum: + bias -> pre (kept, or null) -> activation -> + residual -> out, all in the output's type.
struct ProductEpilogue {
  const void* bias;      // [cols], or null
  const void* residual;  // [rows, cols], or null
  void* pre;             // [rows, cols] contiguous, or null
  void* out;
  int64_t residual_stride, out_stride;
  int activation;
};

// A 16-bit operand in memory: `across` false: rows i (or j) of k entries; true: rows k of i (or j) entries. float32
// operands come as three bfloat16 parts, `part` entries apart, that sum to them. base and stride are 16-byte multiples.
struct ProductOperand {
  const void* base;
  int64_t stride, part;
  bool across;
};

// The product's plan: a function of the sizes alone.
struct ProductPlan {
  int tile_n, tiles_i, tiles_j, blocks, whole, splits, per_split, chunk;
  int64_t partial_bytes;
};
ProductPlan plan_product(int64_t rows, int64_t cols, int64_t depth, int dtype);

// dtype is the output's; the operands are float16 for float16 outputs and bfloat16 otherwise.
int run_product(const ProductOperand& a, const ProductOperand& b, int64_t rows, int64_t cols, int64_t depth, int dtype,
                const ProductEpilogue& e, void* partial, cudaStream_t stream);

// The forward layer of at most kFewRows rows, its weights read once. (4096 x 8192, 24 tokens: bfloat16 20 us, by run_product
// 33; float32 139 against 165. 32 tokens: 22 against 32, and 172 against 166; 2048 x 512 float32 10 against 27.)
constexpr int kFewRows = 32;
int run_few_rows(const void* x, int64_t x_stride, const void* weight, int64_t weight_stride, int64_t rows, int64_t inner,
                 int64_t outer, int dtype, const ProductEpilogue& e, cudaStream_t stream);

}  // namespace cg
