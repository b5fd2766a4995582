// The anchored policy objective: PPO's clipped surrogate with a KL term to a reference policy and an entropy
// bonus, over any vocabulary, with its gradient with respect to the logits in one call.
//
// Row i over its legal set S, logits z, reference logits r, lp = z - lse_S(z), lr = r - lse_S(r), p = exp(lp):
//   ratio = exp(lp_a - old), surr = -min(ratio A, clip(ratio) A), H = -sum p lp
//   KL = sum p (lp - lr)                       with the reference's logits, or
//   KL = exp(u) - u - 1, u = lr_a - lp_a       with the reference's log-probability of the action alone
//   L = sum_i w (surr + beta KL - alpha [|S| > 1] H / log |S|)
//   dL/dz_j = p_j (K0 + w beta ((z_j - r_j) - (max z - max r)) + w alpha' (z_j - max z)) + [j = a] w c
// with c = d surr / d ratio * ratio (+ beta (1 - exp(u))), alpha' = alpha / log |S| and
//   K0 = w (-c - beta (KL + log s - log t) + alpha' (H - log s)),
// s and t the sums of exp(z - max z) and exp(r - max r). The differences from the maxima are what keeps KL and H,
// sums of small terms, from cancelling against the large log-sum-exps. An illegal entry acts as a logit of minus
// infinity, whatever it holds.
//
// All row arithmetic is fp32; the nine totals are summed in double in a fixed order and rounded once.
#include <algorithm>

#include "common.cuh"

namespace cg {
namespace {

constexpr int kTotals = 9;
constexpr int kPartials = 1184;  // the grid's upper bound: a fixed order of addition for a given row count
constexpr float kLog2e = 1.4426950408889634f;

struct Args {
  const void* logits;
  const void* reference;           // logits, or null
  const float* reference_action;   // the action's log-probability, or null
  const uint8_t* legal;            // or null
  const int64_t* actions;
  const float* old_log_probs;
  const float* advantages;
  const float* weights;
  void* grad;                      // or null: the totals alone
  float* log_probs;                // or null: the actions' log-probabilities and nothing else
  double* partial;
  int64_t rows, stride, reference_stride, legal_stride, grad_stride;
  int width;
  float clip, beta, alpha;
};

__device__ __forceinline__ float exp2_fast(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// The larger value, a NaN if either is one (fmaxf would drop it, and a row of NaN would pass for an empty one).
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

// A row's sums over its legal entries.
struct RowSums {
  float peak, sum;              // max z, sum e with e = exp(z - max z)
  float spread;                 // sum e (z - max z)
  float apart;                  // sum e ((z - max z) - (r - max r))
  float reference_peak, reference_sum;
  float count;                  // legal entries
};

// What the gradient pass needs of a row.
struct RowGrad {
  float inv_sum, constant, beta, alpha, shift, action;
};

// The row's contribution to the totals (zeros unless it counts) and its gradient's coefficients.
// z_a: the action's logit, minus infinity where it is illegal.
__device__ __forceinline__ RowGrad finish_row(const Args& a, int64_t row, const RowSums& s, float z_a, bool counts,
                                              double (&acc)[kTotals]) {
  RowGrad g = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  if (!counts) return g;
  const float w = a.weights[row], advantage = a.advantages[row];
  const float log_sum = logf(s.sum);
  const float lp = (z_a - s.peak) - log_sum;
  const float log_ratio = lp - a.old_log_probs[row];
  const float ratio = expf(log_ratio);
  const float free = ratio * advantage;
  const float bounded = fminf(fmaxf(ratio, 1.f - a.clip), 1.f + a.clip) * advantage;
  const bool held = free > bounded;
  const float surrogate = -(held ? bounded : free);
  float slope = held ? 0.f : -advantage * ratio;
  const float entropy = log_sum - s.spread / s.sum;
  const bool eligible = s.count > 1.f;
  const float norm = eligible ? 1.f / logf(s.count) : 0.f;
  float kl = 0.f, log_apart = 0.f;
  g.inv_sum = 1.f / s.sum;
  if (a.reference) {
    log_apart = log_sum - logf(s.reference_sum);
    kl = s.apart * g.inv_sum - log_apart;
    g.beta = w * a.beta;
    g.shift = s.peak - s.reference_peak;
  } else if (a.reference_action) {
    const float u = a.reference_action[row] - lp;
    kl = expf(u) - u - 1.f;
    slope += a.beta * (1.f - expf(u));
  }
  g.alpha = w * a.alpha * norm;
  g.action = w * slope;
  g.constant = -g.action + g.alpha * (entropy - log_sum) - g.beta * (kl + log_apart);
  const float objective = surrogate + a.beta * kl - a.alpha * norm * entropy;
  const double wd = w;
  acc[0] += wd * surrogate;
  acc[1] += wd;
  acc[2] += wd * entropy;
  acc[3] += wd * (norm * entropy);
  acc[4] += eligible ? wd : 0.0;
  acc[5] += fabsf(ratio - 1.f) > a.clip ? wd : 0.0;
  acc[6] += wd * (ratio - 1.f - log_ratio);
  acc[7] += wd * kl;
  acc[8] += wd * objective;
  return g;
}

// Whether a row counts: it has an action inside the vocabulary and something legal, and for the objective its
// weight is not zero and its action is legal. Bad actions set the fault word.
__device__ __forceinline__ bool row_counts(const Args& a, int64_t row, int64_t action, const RowSums& s, float z_a,
                                           bool action_legal, bool report) {
  if (action < 0) return false;
  if (action >= a.width) {
    if (report) raise_fault(0x420);
    return false;
  }
  if (!(s.sum > 0.f) && !isnan(s.sum)) return false;  // nothing legal
  if (a.log_probs) return true;
  if (!action_legal) {
    if (report) raise_fault(0x421);
    return false;
  }
  return a.weights[row] != 0.f;
}

__device__ __forceinline__ float gradient_entry(const RowGrad& g, const RowSums& s, float z, float r, bool exact) {
  const float from_peak = z - s.peak;
  const float p = exp2_fast(from_peak * kLog2e) * g.inv_sum;
  float k = fmaf(g.alpha, from_peak, g.constant);
  if (exact) k = fmaf(g.beta, (z - r) - g.shift, k);
  return p == 0.f ? 0.f : p * k;  // a probability of zero times an infinite difference
}

// ---- any width: one block per row, the row read once for its maxima, once for its sums, once for its gradient ---
constexpr int kStreamThreads = 512;

template <int kOp>  // 0: sum, 1: max
__device__ __forceinline__ float block_reduce(float v, float* scratch) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float other = __shfl_xor_sync(0xffffffffu, v, o);
    v = kOp ? max_nan(v, other) : v + other;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) scratch[threadIdx.x >> 5] = v;
  __syncthreads();
  float out = scratch[0];
  for (int w = 1; w < static_cast<int>(blockDim.x >> 5); ++w) out = kOp ? max_nan(out, scratch[w]) : out + scratch[w];
  return out;
}

template <typename T>
__global__ void __launch_bounds__(kStreamThreads) anchored_stream_kernel(const Args a) {
  __shared__ float scratch[kStreamThreads / 32];
  double acc[kTotals] = {};
  const bool exact = a.reference != nullptr;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* z = static_cast<const T*>(a.logits) + row * a.stride;
    const T* r = exact ? static_cast<const T*>(a.reference) + row * a.reference_stride : nullptr;
    const uint8_t* legal = a.legal ? a.legal + row * a.legal_stride : nullptr;
    const int64_t action = a.actions[row];
    RowSums s = {};
    float peak = -INFINITY, reference_peak = -INFINITY, count = 0.f;
    for (int j = threadIdx.x; j < a.width; j += kStreamThreads) {
      if (legal && !legal[j]) continue;
      peak = max_nan(peak, as_float(z[j]));
      if (exact) reference_peak = max_nan(reference_peak, as_float(r[j]));
      count += 1.f;
    }
    s.peak = block_reduce<1>(peak, scratch);
    if (exact) s.reference_peak = block_reduce<1>(reference_peak, scratch);
    s.count = block_reduce<0>(count, scratch);
    // Nothing to exponentiate: every sum stays zero.
    const bool any = s.peak != -INFINITY;
    for (int j = threadIdx.x; any && j < a.width; j += kStreamThreads) {
      if (legal && !legal[j]) continue;
      const float from_peak = as_float(z[j]) - s.peak;
      const float e = exp2_fast(from_peak * kLog2e);
      s.sum += e;
      if (e != 0.f) s.spread = fmaf(e, from_peak, s.spread);
      if (exact) {
        const float reference_from_peak = as_float(r[j]) - s.reference_peak;
        s.reference_sum += exp2_fast(reference_from_peak * kLog2e);
        if (e != 0.f) s.apart = fmaf(e, from_peak - reference_from_peak, s.apart);
      }
    }
    s.sum = block_reduce<0>(s.sum, scratch);
    s.spread = block_reduce<0>(s.spread, scratch);
    if (exact) {
      s.reference_sum = block_reduce<0>(s.reference_sum, scratch);
      s.apart = block_reduce<0>(s.apart, scratch);
    }
    const bool inside = action >= 0 && action < a.width;
    const bool action_legal = inside && (!legal || legal[action]);
    const float z_a = action_legal ? as_float(z[action]) : -INFINITY;
    const bool counts = row_counts(a, row, action, s, z_a, action_legal, threadIdx.x == 0);
    if (a.log_probs) {
      if (threadIdx.x == 0) a.log_probs[row] = counts ? (z_a - s.peak) - logf(s.sum) : 0.f;
      continue;
    }
    double ignored[kTotals] = {};
    const RowGrad g = finish_row(a, row, s, z_a, counts, threadIdx.x == 0 ? acc : ignored);
    if (!a.grad) continue;
    T* out = static_cast<T*>(a.grad) + row * a.grad_stride;
    for (int j = threadIdx.x; j < a.width; j += kStreamThreads) {
      float v = 0.f;
      if (counts && !(legal && !legal[j])) {
        v = gradient_entry(g, s, as_float(z[j]), exact ? as_float(r[j]) : 0.f, exact);
        if (j == action) v += g.action;
      }
      put(out + j, v);
    }
  }
  if (!a.log_probs && threadIdx.x == 0)
    for (int k = 0; k < kTotals; ++k) a.partial[blockIdx.x * kTotals + k] = acc[k];
}

// Warp k sums total k over the blocks: lane l the partials l, l + 32, ..., then a butterfly.
__global__ void __launch_bounds__(kTotals * 32) anchored_totals_kernel(const double* partial, int count, float* totals) {
  const int lane = threadIdx.x & 31, k = threadIdx.x >> 5;
  pdl_wait();
  double total = 0;
  for (int b = lane; b < count; b += 32) total += partial[b * kTotals + k];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) totals[k] = static_cast<float>(total);
}

int run_rows(const Args& a, int dtype, int* blocks, cudaStream_t s) {
  *blocks = static_cast<int>(std::min<int64_t>(a.rows, kPartials));
  if (dtype == CG_F32)
    anchored_stream_kernel<float><<<*blocks, kStreamThreads, 0, s>>>(a);
  else if (dtype == CG_F16)
    anchored_stream_kernel<__half><<<*blocks, kStreamThreads, 0, s>>>(a);
  else
    anchored_stream_kernel<__nv_bfloat16><<<*blocks, kStreamThreads, 0, s>>>(a);
  return check_launch("anchored_stream_kernel");
}

}  // namespace
}  // namespace cg

extern "C" int64_t cg_anchored_objective_workspace_bytes(int64_t rows) {
  return std::min<int64_t>(std::max<int64_t>(rows, 1), cg::kPartials) * cg::kTotals * static_cast<int64_t>(sizeof(double));
}

extern "C" int cg_anchored_objective(const void* logits, int dtype, int64_t rows, int width, int64_t stride,
                                     const void* reference_logits, int64_t reference_stride,
                                     const float* reference_log_probs, const uint8_t* legal, int64_t legal_stride,
                                     const int64_t* actions, const float* old_log_probs, const float* advantages,
                                     const float* weights, float clip_ratio, float beta, float alpha, void* grad,
                                     int64_t grad_stride, float* totals, void* workspace, int64_t workspace_bytes,
                                     void* stream) {
  using namespace cg;
  CG_REQUIRE(valid_dtype(dtype), "cg_anchored_objective: dtype must be float32, float16 or bfloat16");
  CG_REQUIRE(rows >= 0 && width > 0, "cg_anchored_objective: bad shape");
  CG_REQUIRE(stride >= width && (!grad || grad_stride >= width) && (!reference_logits || reference_stride >= width) &&
                 (!legal || legal_stride >= width),
             "cg_anchored_objective: stride < width");
  CG_REQUIRE(!(reference_logits && reference_log_probs), "cg_anchored_objective: one reference at most");
  CG_REQUIRE(clip_ratio >= 0, "cg_anchored_objective: clip_ratio must not be negative");
  CG_REQUIRE(totals, "cg_anchored_objective: NULL totals");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int blocks = 0;
  auto* partial = static_cast<double*>(workspace);
  if (rows > 0) {
    CG_REQUIRE(logits && actions && old_log_probs && advantages && weights,
               "cg_anchored_objective: NULL pointer");
    if (!workspace || workspace_bytes < cg_anchored_objective_workspace_bytes(rows))
      return set_error(CG_ERR_WORKSPACE, "cg_anchored_objective: workspace too small");
    const Args a = {logits, reference_logits, reference_log_probs, legal, actions, old_log_probs, advantages, weights,
                    grad, nullptr, partial, rows, stride, reference_stride, legal_stride, grad_stride, width,
                    clip_ratio, beta, alpha};
    if (int rc = run_rows(a, dtype, &blocks, s)) return rc;
  }
  return launch_pdl("anchored_totals_kernel", anchored_totals_kernel, dim3(1), dim3(kTotals * 32), 0, s,
                    static_cast<const double*>(partial), blocks, totals);
}

extern "C" int cg_action_log_probs(const void* logits, int dtype, int64_t rows, int width, int64_t stride,
                                   const uint8_t* legal, int64_t legal_stride, const int64_t* actions,
                                   float* log_probs, void* stream) {
  using namespace cg;
  CG_REQUIRE(valid_dtype(dtype), "cg_action_log_probs: dtype must be float32, float16 or bfloat16");
  CG_REQUIRE(rows >= 0 && width > 0, "cg_action_log_probs: bad shape");
  CG_REQUIRE(stride >= width && (!legal || legal_stride >= width), "cg_action_log_probs: stride < width");
  if (rows == 0) return CG_OK;
  CG_REQUIRE(logits && actions && log_probs, "cg_action_log_probs: NULL pointer");
  Args a = {};
  a.logits = logits;
  a.legal = legal;
  a.actions = actions;
  a.log_probs = log_probs;
  a.rows = rows;
  a.stride = stride;
  a.legal_stride = legal_stride;
  a.width = width;
  int blocks = 0;
  return run_rows(a, dtype, &blocks, static_cast<cudaStream_t>(stream));
}
