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
  int64_t partial_bytes, running_bytes;  // of the workspace: split tiles' sums, then sums between chunks
  int64_t bytes() const { return partial_bytes + running_bytes; }
};
ProductPlan plan_product(int64_t rows, int64_t cols, int64_t depth, int dtype);

// dtype is the output's; the operands are float16 for float16 outputs and bfloat16 otherwise.
int run_product(const ProductOperand& a, const ProductOperand& b, int64_t rows, int64_t cols, int64_t depth, int dtype,
                const ProductEpilogue& e, void* partial, cudaStream_t stream);

// The forward layer of at most kFewRows rows, its weights read once: bfloat16 4096 x 8192 with 24 tokens 20 us, by run_product
// 33, with 32 tokens 22 against 32. float32 pays for each token, 4096 x 8192 with 16 tokens 117 us against 165, with 24 174
// against 165 and with 32 218 against 167, so more than 24 tokens of a large layer go to run_product: from 2^23 weights on
// (8000 x 1000 with 32 tokens 54 us against 52, 4096 x 512 20 against 28).
constexpr int kFewRows = 32, kFewRowsOfLarge32 = 24;
inline bool few_rows(int64_t rows, int64_t inner, int64_t outer, int dtype) {
  return rows <= (dtype == CG_F32 && inner * outer >= 1 << 23 ? kFewRowsOfLarge32 : kFewRows);
}
int run_few_rows(const void* x, int64_t x_stride, const void* weight, int64_t weight_stride, int64_t rows, int64_t inner,
                 int64_t outer, int dtype, const ProductEpilogue& e, cudaStream_t stream);

}  // namespace cg
