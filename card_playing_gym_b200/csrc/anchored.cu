// The anchored policy objective: PPO's clipped surrogate with a KL term to a reference policy and an entropy
// bonus, over any vocabulary, with its gradient with respect to the logits in one call.
//
// Row i over its legal set S, logits z, reference logits r, lp = z - lse_S(z), lr = r - lse_S(r), p = exp(lp):
//   ratio = exp(lp_a - old), surr = -min(ratio A, clip(ratio) A), H = -sum p lp
//   KL = sum p (lp - lr)                       with the reference's logits, or
//   KL = exp(u) - u - 1, u = lr_a - lp_a       with the reference's log-probability of the action alone
//   L = sum_i w (surr + beta KL - alpha [|S| > 1] H / log |S|)
//   dL/dz_j = p_j (K0 + w beta (z_j - r_j) + w alpha' (z_j - max z)) + [j = a] w c
// with c = d surr / d ratio * ratio (+ beta (1 - exp(u))), alpha' = alpha / log |S| and
//   K0 = w (-c - beta (KL + log s - log t + max z - max r) + alpha' (H - log s)),
// s and t the sums of exp(z - max z) and exp(r - max r). The differences from the maxima are what keeps KL and H,
// sums of small terms, from cancelling against the large log-sum-exps. An illegal entry acts as a logit of minus
// infinity, whatever it holds.
//
// All row arithmetic is fp32. The totals are summed in fp32 over the rows of one thread (some tens) and in double
// from there on, in a fixed order.
#include <algorithm>

#include "elements.cuh"
#include "tcgen05.cuh"

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
  float inv_sum, constant, beta, alpha, action;
};

// The row's contribution to the totals (zeros unless it counts) and its gradient's coefficients.
// z_a: the action's logit, minus infinity where it is illegal.
__device__ __forceinline__ RowGrad finish_row(const Args& a, int64_t row, const RowSums& s, float z_a, bool counts,
                                              float (&acc)[kTotals]) {
  RowGrad g = {0.f, 0.f, 0.f, 0.f, 0.f};
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
  } else if (a.reference_action) {
    const float u = a.reference_action[row] - lp;
    kl = expf(u) - u - 1.f;
    slope += a.beta * (1.f - expf(u));
  }
  g.alpha = w * a.alpha * norm;
  g.action = w * slope;
  g.constant = -g.action + g.alpha * (entropy - log_sum) - g.beta * (kl + log_apart + (s.peak - s.reference_peak));
  const float objective = surrogate + a.beta * kl - a.alpha * norm * entropy;
  acc[0] += w * surrogate;
  acc[1] += w;
  acc[2] += w * entropy;
  acc[3] += w * (norm * entropy);
  acc[4] += eligible ? w : 0.f;
  acc[5] += fabsf(ratio - 1.f) > a.clip ? w : 0.f;
  acc[6] += w * (ratio - 1.f - log_ratio);
  acc[7] += w * kl;
  acc[8] += w * objective;
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

// dL/dz of an entry that is not the action. A probability of zero has a zero gradient whatever it is multiplied by.
__device__ __forceinline__ float gradient_entry(const RowGrad& g, float peak, float z, float r, bool exact) {
  const float from_peak = z - peak;
  const float p = exp2_fast(from_peak * kLog2e) * g.inv_sum;
  float k = fmaf(g.alpha, from_peak, g.constant);
  if (exact) k = fmaf(g.beta, z - r, k);
  return p == 0.f ? 0.f : p * k;
}

// One entry's part of a row's sums.
__device__ __forceinline__ void add_entry(RowSums& s, float z, float r, bool exact) {
  const float from_peak = z - s.peak;
  const float e = exp2_fast(from_peak * kLog2e);
  s.sum += e;
  if (exact) {
    const float reference_from_peak = r - s.reference_peak;
    s.reference_sum += exp2_fast(reference_from_peak * kLog2e);
    if (e != 0.f) s.apart = fmaf(e, from_peak - reference_from_peak, s.apart);
  }
  if (e != 0.f) s.spread = fmaf(e, from_peak, s.spread);
}

// Sixteen bytes of a row as floats and back.
template <typename T>
constexpr int kVector = 16 / static_cast<int>(sizeof(T));

__device__ __forceinline__ void unpack(const uint4& raw, float (&v)[4]) {
  v[0] = __uint_as_float(raw.x), v[1] = __uint_as_float(raw.y), v[2] = __uint_as_float(raw.z), v[3] = __uint_as_float(raw.w);
}
__device__ __forceinline__ void unpack(const uint4& raw, float (&v)[8], __half) {
  const __half2* h = reinterpret_cast<const __half2*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 f = __half22float2(h[i]);
    v[2 * i] = f.x, v[2 * i + 1] = f.y;
  }
}
__device__ __forceinline__ void unpack(const uint4& raw, float (&v)[8], __nv_bfloat16) {
  const uint32_t w[4] = {raw.x, raw.y, raw.z, raw.w};
#pragma unroll
  for (int i = 0; i < 4; ++i) v[2 * i] = __uint_as_float(w[i] << 16), v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u);
}
__device__ __forceinline__ void unpack(const uint4& raw, float (&v)[4], float) { unpack(raw, v); }
__device__ __forceinline__ uint4 repack(const float (&v)[4], float) {
  return make_uint4(__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3]));
}
template <typename T>
__device__ __forceinline__ uint4 repack(const float (&v)[8], T) {
  uint4 raw;
  auto* h = reinterpret_cast<typename PairOf<T>::type*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) pair_from(h[i], v[2 * i], v[2 * i + 1]);
  return raw;
}

// The largest entry of sixteen-byte units, a NaN if there is one. 16-bit entries are compared in pairs.
template <typename T>
struct UnitMax {
  typename PairOf<T>::type top;
  __device__ __forceinline__ UnitMax() { pair_from(top, -INFINITY, -INFINITY); }
  __device__ __forceinline__ void take(const uint4& raw) {
    const auto* h = reinterpret_cast<const typename PairOf<T>::type*>(&raw);
    top = __hmax2_nan(top, __hmax2_nan(__hmax2_nan(h[0], h[1]), __hmax2_nan(h[2], h[3])));
  }
  __device__ __forceinline__ float value() const {
    const float2 f = pair_float(top);
    return max_nan(f.x, f.y);
  }
};
template <>
struct UnitMax<float> {
  float top = -INFINITY;
  __device__ __forceinline__ void take(const uint4& raw) {
    top = max_nan(top, max_nan(max_nan(__uint_as_float(raw.x), __uint_as_float(raw.y)),
                               max_nan(__uint_as_float(raw.z), __uint_as_float(raw.w))));
  }
  __device__ __forceinline__ float value() const { return top; }
};

// Whether every row of a plane starts on sixteen bytes.
template <typename T>
__device__ __forceinline__ bool aligned_rows(const void* base, int64_t stride, int64_t rows) {
  return (reinterpret_cast<uintptr_t>(base) & 15) == 0 && (rows == 1 || stride * static_cast<int64_t>(sizeof(T)) % 16 == 0);
}

// ---- up to 1024 entries: a row in the registers of four lanes or of a warp --------------------------------------------
// A row has some 300 instructions of its own (reductions, logarithms, the ratio) beside 30 an entry, so rows of up to 64
// entries take four lanes, eight rows a warp. The row is read once and written once,
// and the grid is one resident wave of warps. Aligned rows move in vectors of sixteen bytes, a lane holding every
// kLanes-th vector; others entry by entry, a lane holding every kLanes-th entry, so that both are coalesced.
template <typename T, int kLanes, int kVectors>
__global__ void __launch_bounds__(256, 2) anchored_narrow_kernel(const Args a) {
  constexpr int kVec = kVector<T>, kPer = kVec * kVectors, kGroups = 32 / kLanes;
  __shared__ double scratch[8][kTotals];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = lane / kLanes, l = lane % kLanes;
  const uint32_t group_mask = kLanes == 32 ? 0xffffffffu : ((1u << (kLanes & 31)) - 1u) << (group * kLanes);
  const bool exact = a.reference != nullptr;
  const bool vectors = aligned_rows<T>(a.logits, a.stride, a.rows) &&
                       (!exact || aligned_rows<T>(a.reference, a.reference_stride, a.rows)) &&
                       (!a.grad || aligned_rows<T>(a.grad, a.grad_stride, a.rows)) &&
                       (!a.legal || ((reinterpret_cast<uintptr_t>(a.legal) & (kVec - 1)) == 0 &&
                                     (a.rows == 1 || a.legal_stride % kVec == 0)));
  float acc[kTotals] = {};
  // The entry of slot (v, e).
  auto entry = [&](int v, int e) { return vectors ? (l + kLanes * v) * kVec + e : l + kLanes * (v * kVec + e); };
  auto reduce = [&](float v, bool largest) {
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) {
      const float other = __shfl_xor_sync(0xffffffffu, v, o);
      v = largest ? max_nan(v, other) : v + other;
    }
    return v;
  };
  const int64_t step = static_cast<int64_t>(gridDim.x) * 8 * kGroups;
  const int64_t warp_first = (static_cast<int64_t>(blockIdx.x) * 8 + warp) * kGroups;
  // Every group of a warp runs the same iterations, so that the shuffles stay converged.
  for (int64_t base = warp_first; base < a.rows; base += step) {
    const int64_t row = base + group;
    const bool live = row < a.rows;
    const T* gz = static_cast<const T*>(a.logits) + row * a.stride;
    const T* gr = exact ? static_cast<const T*>(a.reference) + row * a.reference_stride : nullptr;
    const uint8_t* gl = a.legal ? a.legal + row * a.legal_stride : nullptr;
    const int64_t action = live ? a.actions[row] : -1;
    // Illegal entries, and those past the row, are minus infinity.
    float z[kPer], r[kPer], z_a = 0.f, count = 0.f;
    bool mine = false;
    if (vectors) {
      uint4 raw_z[kVectors], raw_r[kVectors];
      uint2 raw_l[kVectors];
#pragma unroll
      for (int v = 0; v < kVectors; ++v) {
        const int j = (l + kLanes * v) * kVec;
        raw_z[v] = raw_r[v] = make_uint4(0, 0, 0, 0);
        raw_l[v] = make_uint2(0x01010101u, 0x01010101u);
        if (!live || j + kVec > a.width) continue;
        raw_z[v] = *reinterpret_cast<const uint4*>(gz + j);
        if (exact) raw_r[v] = *reinterpret_cast<const uint4*>(gr + j);
        if (gl) {
          if constexpr (kVec == 4)
            raw_l[v].x = *reinterpret_cast<const uint32_t*>(gl + j);
          else
            raw_l[v] = *reinterpret_cast<const uint2*>(gl + j);
        }
      }
#pragma unroll
      for (int v = 0; v < kVectors; ++v) {
        const int j = (l + kLanes * v) * kVec;
        float t[kVec], u[kVec];
        uint32_t in[kVec];
        if (live && j < a.width && j + kVec > a.width) {  // the row's last entries, fewer than a vector
#pragma unroll
          for (int e = 0; e < kVec; ++e) {
            const bool inside = j + e < a.width;
            t[e] = inside ? as_float(gz[j + e]) : 0.f;
            u[e] = inside && exact ? as_float(gr[j + e]) : 0.f;
            in[e] = inside ? (gl ? gl[j + e] : 1u) : 0u;
          }
        } else {
          unpack(raw_z[v], t, T());
          unpack(raw_r[v], u, T());
#pragma unroll
          for (int e = 0; e < kVec; ++e)
            in[e] = live && j < a.width ? (e < 4 ? raw_l[v].x : raw_l[v].y) >> (8 * (e & 3)) & 255u : 0u;
        }
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const int k = v * kVec + e;
          z[k] = in[e] ? t[e] : -INFINITY;
          r[k] = in[e] ? u[e] : -INFINITY;
          count += in[e] ? 1.f : 0.f;
          if (in[e] && j + e == action) z_a = z[k], mine = true;
        }
      }
    } else {
#pragma unroll
      for (int k = 0; k < kPer; ++k) {
        const int j = l + kLanes * k;
        const bool in = live && j < a.width && (!gl || gl[j]);
        z[k] = in ? as_float(gz[j]) : -INFINITY;
        r[k] = in && exact ? as_float(gr[j]) : -INFINITY;
        count += in ? 1.f : 0.f;
        if (in && j == action) z_a = z[k], mine = true;
      }
    }
    RowSums s = {};
    float peak = -INFINITY, reference_peak = -INFINITY;
#pragma unroll
    for (int k = 0; k < kPer; ++k) {
      peak = max_nan(peak, z[k]);
      if (exact) reference_peak = max_nan(reference_peak, r[k]);
    }
    s.peak = reduce(peak, true);
    if (exact) s.reference_peak = reduce(reference_peak, true);
    s.count = reduce(count, false);
    const bool action_legal = (__ballot_sync(0xffffffffu, mine) & group_mask) != 0;
    z_a = reduce(z_a, false);  // one lane holds it
    if (!action_legal) z_a = -INFINITY;
    if (s.peak != -INFINITY) {
#pragma unroll
      for (int k = 0; k < kPer; ++k) add_entry(s, z[k], exact ? r[k] : 0.f, exact);
    }
    s.sum = reduce(s.sum, false);
    if (!a.log_probs) s.spread = reduce(s.spread, false);
    if (exact) {
      s.reference_sum = reduce(s.reference_sum, false);
      s.apart = reduce(s.apart, false);
    }
    const bool counts = row_counts(a, row, action, s, z_a, action_legal, l == 0);
    if (a.log_probs) {
      if (live && l == 0) a.log_probs[row] = counts ? (z_a - s.peak) - logf(s.sum) : 0.f;
      continue;
    }
    const RowGrad g = finish_row(a, row, s, z_a, counts, acc);  // every lane of the group keeps the same totals
    if (!a.grad || !live) continue;
    T* out = static_cast<T*>(a.grad) + row * a.grad_stride;
#pragma unroll
    for (int v = 0; v < kVectors; ++v) {
      float t[kVec];
#pragma unroll
      for (int e = 0; e < kVec; ++e) {
        const int k = v * kVec + e;
        t[e] = counts ? gradient_entry(g, s.peak, z[k], exact ? r[k] : 0.f, exact) : 0.f;
        if (counts && entry(v, e) == action) t[e] += g.action;
      }
      const int j = (l + kLanes * v) * kVec;
      if (vectors && j + kVec <= a.width) {
        *reinterpret_cast<uint4*>(out + j) = repack(t, T());
      } else {
#pragma unroll
        for (int e = 0; e < kVec; ++e)
          if (entry(v, e) < a.width) put(out + entry(v, e), t[e]);
      }
    }
  }
  if (a.log_probs) return;
  // The groups' leaders in order, then the warps.
#pragma unroll
  for (int k = 0; k < kTotals; ++k) {
    double total = acc[k];
#pragma unroll
    for (int other = 1; other < kGroups; ++other) {
      total += __shfl_sync(0xffffffffu, acc[k], other * kLanes);
    }
    if (lane == 0) scratch[warp][k] = total;
  }
  __syncthreads();
  if (threadIdx.x < kTotals) {
    double total = 0;
    for (int w = 0; w < 8; ++w) total += scratch[w][threadIdx.x];
    a.partial[blockIdx.x * kTotals + threadIdx.x] = total;
  }
}

// ---- wider rows: a row in the shared memory of a cluster --------------------------------------------------------------
// The row is read once, by bulk copies, and stays in shared memory for its maxima, its sums and its gradient. A cluster
// of C blocks holds it, C the least that leaves room for three blocks an SM, so that one block's copies and barriers
// run under another's arithmetic; narrow slices have two buffers, the next row's copies running under this one's arithmetic.
// Every thread sums its own entries relative to its own maxima, and the maxima and sums are joined once, over the
// block and then over the cluster through each other's shared memory: one cluster barrier a row.
//
// What bounds it is instruction issue beside HBM: three exponentials an entry and, in pairs of packed fp32
// arithmetic, some 20 instructions. Entries at minus infinity, which the packed sums turn into NaN, are found by
// that and summed again with tests.
//
// Slices are copied with the alignment they have in memory: the sixteen-byte units inside by the copy engine, the few
// bytes at the ends by threads. The arithmetic runs over the same units; planes whose rows are aligned differently
// from the logits' are read entry by entry from shared memory.
constexpr int kWideThreads = 256;
constexpr int kMaxCluster = 16;

// Partial results over some entries, each relative to their own maxima.
struct Part {
  float peak, reference_peak, sum, spread, reference_sum, apart, count;
};
constexpr int kSlots = sizeof(Part) / sizeof(float);

// The parts of 2^steps neighbouring lanes (or of the whole warp) joined; every lane gets the result.
template <bool kExact>
__device__ __forceinline__ void join_lanes(Part& p, int lanes) {
  float peak = p.peak, reference_peak = p.reference_peak;
  for (int o = lanes / 2; o > 0; o >>= 1) {
    peak = max_nan(peak, __shfl_xor_sync(0xffffffffu, peak, o));
    if (kExact) reference_peak = max_nan(reference_peak, __shfl_xor_sync(0xffffffffu, reference_peak, o));
  }
  const float up = p.peak == -INFINITY ? 0.f : p.peak - peak;
  const float scale = p.peak == -INFINITY ? 0.f : exp2_fast(up * kLog2e);
  if (kExact) {
    const float reference_up = p.reference_peak == -INFINITY ? 0.f : p.reference_peak - reference_peak;
    p.reference_sum *= p.reference_peak == -INFINITY ? 0.f : exp2_fast(reference_up * kLog2e);
    // Without a reference entry above minus infinity the part's differences are infinite already.
    p.apart = scale == 0.f ? 0.f : scale * fmaf(up - reference_up, p.sum, p.apart);
  }
  p.spread = scale == 0.f ? 0.f : scale * fmaf(up, p.sum, p.spread);
  p.sum = scale == 0.f ? 0.f : scale * p.sum;
  p.peak = peak, p.reference_peak = reference_peak;
  for (int o = lanes / 2; o > 0; o >>= 1) {
    p.sum += __shfl_xor_sync(0xffffffffu, p.sum, o);
    p.spread += __shfl_xor_sync(0xffffffffu, p.spread, o);
    p.count += __shfl_xor_sync(0xffffffffu, p.count, o);
    if (kExact) {
      p.reference_sum += __shfl_xor_sync(0xffffffffu, p.reference_sum, o);
      p.apart += __shfl_xor_sync(0xffffffffu, p.apart, o);
    }
  }
}

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
__device__ __forceinline__ Two exp2_two(Two x) {
  const float2 f = apart_of(x);
  return two(exp2_fast(f.x), exp2_fast(f.y));
}

// The bytes before the first sixteen-byte boundary of `bytes` bytes at `src`, and those in whole units after it.
__device__ __forceinline__ uint32_t aligned_part(const void* src, int bytes, int* head) {
  const int lead = static_cast<int>((16 - (reinterpret_cast<uintptr_t>(src) & 15)) & 15);
  *head = min(lead, bytes);
  return static_cast<uint32_t>((bytes - *head) & ~15);
}

__device__ __forceinline__ void store_remote(uint32_t address, float v) {
  asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(address), "f"(v) : "memory");
}

// One plane of a row's slice: where it is in memory and where in shared memory, at the same misalignment.
struct Plane {
  const unsigned char* from;
  unsigned char* to;  // entry 0
  int bytes, head;
  uint32_t inner;
  __device__ __forceinline__ Plane(const void* src, unsigned char* base, int size) {
    from = static_cast<const unsigned char*>(src);
    to = base + (reinterpret_cast<uintptr_t>(src) & 15);
    bytes = src ? size : 0;
    inner = aligned_part(src, bytes, &head);
  }
  __device__ __forceinline__ int tail() const { return bytes - head - static_cast<int>(inner); }
  __device__ __forceinline__ void copy_units(uint64_t* barrier) const {
    if (inner) tc::bulk_g2s(to + head, from + head, inner, barrier);
  }
  __device__ __forceinline__ void copy_ends(int tid) const {
    if (tid < head) to[tid] = from[tid];
    if (tid >= 32 && tid < 32 + tail()) to[head + inner + tid - 32] = from[head + inner + tid - 32];
  }
};

template <typename T, bool kExact>
__global__ void __launch_bounds__(kWideThreads, 3) anchored_wide_kernel(const Args a, int slice, int clusters, int buffer_bytes,
                                                                        int buffers) {
  constexpr int kVec = kVector<T>;
  extern __shared__ __align__(16) unsigned char smem[];
  __shared__ __align__(8) uint64_t arrived[2];
  __shared__ float warp_parts[kWideThreads / 32][kSlots], cluster_parts[2][kMaxCluster][kSlots];
  __shared__ RowGrad row_grad;
  __shared__ float row_peak;
  __shared__ bool row_live;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  uint32_t rank = 0, size = 1;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
  asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(size));
  const int plane = slice * static_cast<int>(sizeof(T)) + 32;  // a slice and its misalignment
  const int lo = static_cast<int>(rank) * slice;
  const int n = max(0, min(slice, a.width - lo));
  if (tid == 0) {
    tc::bar_init(&arrived[0], 1);
    tc::bar_init(&arrived[1], 1);
    tc::bar_fence_init();
  }
  __syncthreads();
  if (size > 1) tc::cluster_sync();

  auto plane_z = [&](int64_t row, int buffer) {
    return Plane(static_cast<const T*>(a.logits) + row * a.stride + lo, smem + buffer * buffer_bytes,
                 n * static_cast<int>(sizeof(T)));
  };
  auto plane_r = [&](int64_t row, int buffer) {
    return Plane(kExact ? static_cast<const T*>(a.reference) + row * a.reference_stride + lo : nullptr,
                 smem + buffer * buffer_bytes + plane, n * static_cast<int>(sizeof(T)));
  };
  auto plane_l = [&](int64_t row, int buffer) {
    return Plane(a.legal ? a.legal + row * a.legal_stride + lo : nullptr,
                 smem + buffer * buffer_bytes + (kExact ? 2 : 1) * plane, n);
  };
  // Thread 0 starts a row's copies. Whatever the block read from and wrote to the buffer is done.
  auto issue = [&](int64_t row, int buffer) {
    if (tid != 0 || row >= a.rows) return;
    const Plane pz = plane_z(row, buffer), pr = plane_r(row, buffer), pl = plane_l(row, buffer);
    tc::fence_async_smem();
    tc::bar_expect_tx(&arrived[buffer], pz.inner + pr.inner + pl.inner);
    pz.copy_units(&arrived[buffer]);
    if (kExact) pr.copy_units(&arrived[buffer]);
    pl.copy_units(&arrived[buffer]);
  };

  float acc[kTotals] = {};
  uint32_t turn = 0;  // rows done: the buffer and its barrier's phase
  const int64_t first = blockIdx.x / size;
  issue(first, 0);
  for (int64_t row = first; row < a.rows; row += clusters, ++turn) {
    const int buffer = buffers == 2 ? turn & 1 : 0;
    if (buffers == 2) issue(row + clusters, buffer ^ 1);
    const Plane pz = plane_z(row, buffer), pr = plane_r(row, buffer), pl = plane_l(row, buffer);
    const bool masked = a.legal != nullptr;
    const int64_t action = a.actions[row];
    if (pz.head | pz.tail() | pr.head | pr.tail() | pl.head | pl.tail()) {
      pz.copy_ends(tid);
      if (kExact) pr.copy_ends(tid);
      pl.copy_ends(tid);
      __syncthreads();
    }
    tc::bar_wait(&arrived[buffer], (buffers == 2 ? turn >> 1 : turn) & 1u, 0x422);

    T* z = reinterpret_cast<T*>(pz.to);
    T* r = reinterpret_cast<T*>(pr.to);
    const uint8_t* legal = pl.to;
    const int head = pz.head / static_cast<int>(sizeof(T));  // entries before the first unit
    const int units = static_cast<int>(pz.inner) / 16;
    const int ends = n - units * kVec;  // entries outside the units, head first
    const bool alike = !kExact || ((reinterpret_cast<uintptr_t>(pz.from) ^ reinterpret_cast<uintptr_t>(pr.from)) & 15) == 0;
    auto end_entry = [&](int k) { return k < head ? k : k + units * kVec; };
    auto load_unit = [&](const T* base, int j, bool whole, float (&v)[kVec]) {
      if (whole) {
        unpack(*reinterpret_cast<const uint4*>(base + j), v, T());
      } else {
#pragma unroll
        for (int e = 0; e < kVec; ++e) v[e] = as_float(base[j + e]);
      }
    };

    // This thread's maxima. An illegal entry becomes a logit of minus infinity, here and in the reference.
    RowSums s = {};
    float count = 0.f;
    s.peak = s.reference_peak = -INFINITY;
    if (!masked && alike) {
      UnitMax<T> top_z, top_r;
#pragma unroll 4
      for (int u = tid; u < units; u += kWideThreads) {
        top_z.take(*reinterpret_cast<const uint4*>(z + head + u * kVec));
        if (kExact) top_r.take(*reinterpret_cast<const uint4*>(r + head + u * kVec));
      }
      s.peak = top_z.value();
      if (kExact) s.reference_peak = top_r.value();
    } else {
      for (int u = tid; u < units; u += kWideThreads) {
        const int j = head + u * kVec;
        float vz[kVec], vr[kVec];
        load_unit(z, j, true, vz);
        if (kExact) load_unit(r, j, alike, vr);
#pragma unroll
        for (int e = 0; e < kVec; ++e) {
          const bool in = !masked || legal[j + e];
          if (!in) {
            put(z + j + e, -INFINITY);
            if (kExact) put(r + j + e, -INFINITY);
          } else {
            count += 1.f;
            s.peak = max_nan(s.peak, vz[e]);
            if (kExact) s.reference_peak = max_nan(s.reference_peak, vr[e]);
          }
        }
      }
    }
    if (tid < ends) {
      const int j = end_entry(tid);
      if (masked && !legal[j]) {
        put(z + j, -INFINITY);
        if (kExact) put(r + j, -INFINITY);
      } else {
        count += 1.f;
        s.peak = max_nan(s.peak, as_float(z[j]));
        if (kExact) s.reference_peak = max_nan(s.reference_peak, as_float(r[j]));
      }
    }

    // This thread's sums.
    const float reference_base = s.reference_peak == -INFINITY ? 0.f : s.reference_peak;
    auto sum_tested = [&] {
      RowSums t = s;
      t.sum = t.spread = t.apart = t.reference_sum = 0.f;
      t.peak = s.peak == -INFINITY ? 0.f : s.peak;
      t.reference_peak = reference_base;
      for (int u = tid; u < units; u += kWideThreads) {
        const int j = head + u * kVec;
        float vz[kVec], vr[kVec];
        load_unit(z, j, true, vz);
        if (kExact) load_unit(r, j, alike, vr);
#pragma unroll
        for (int e = 0; e < kVec; ++e) add_entry(t, vz[e], kExact ? vr[e] : 0.f, kExact);
      }
      if (tid < ends) {
        const int j = end_entry(tid);
        add_entry(t, as_float(z[j]), kExact ? as_float(r[j]) : 0.f, kExact);
      }
      s.sum = t.sum, s.spread = t.spread, s.apart = t.apart, s.reference_sum = t.reference_sum;
    };
    bool tested = masked || !alike;  // whether this thread's entries need tests for minus infinity
    if (s.peak != -INFINITY) {
      if (!tested) {
        const Two from = two(-s.peak, -s.peak), reference_from = two(-reference_base, -reference_base);
        const Two scale = two(kLog2e, kLog2e), minus = two(-1.f, -1.f);
        Two sum = two(0.f, 0.f), spread = sum, apart = sum, reference_sum = sum;
#pragma unroll 2
        for (int u = tid; u < units; u += kWideThreads) {
          const int j = head + u * kVec;
          float vz[kVec], vr[kVec];
          load_unit(z, j, true, vz);
          if (kExact) load_unit(r, j, true, vr);
#pragma unroll
          for (int e = 0; e < kVec; e += 2) {
            const Two x = two(vz[e], vz[e + 1]) + from;
            const Two p = exp2_two(x * scale);
            sum = sum + p;
            spread = fma(p, x, spread);
            if (kExact) {
              const Two y = two(vr[e], vr[e + 1]) + reference_from;
              reference_sum = reference_sum + exp2_two(y * scale);
              apart = fma(p, fma(y, minus, x), apart);
            }
          }
        }
        const float2 fs = apart_of(sum), fd = apart_of(spread), fa = apart_of(apart), fr = apart_of(reference_sum);
        s.sum = fs.x + fs.y, s.spread = fd.x + fd.y, s.apart = fa.x + fa.y, s.reference_sum = fr.x + fr.y;
        if (tid < ends) {
          const int j = end_entry(tid);
          add_entry(s, as_float(z[j]), kExact ? as_float(r[j]) : 0.f, kExact);
        }
        tested = isnan(s.spread) || isnan(s.apart);
      }
      if (tested) sum_tested();
    } else {
      tested = true;
      if (kExact) sum_tested();  // the reference's sum counts where this thread has no logit above minus infinity
    }

    Part part = {s.peak, s.reference_peak, s.sum, s.spread, s.reference_sum, s.apart, count};
    join_lanes<kExact>(part, 32);
    if (lane == 0) *reinterpret_cast<Part*>(warp_parts[warp]) = part;
    __syncthreads();
    if (warp == 0) {
      part = *reinterpret_cast<const Part*>(warp_parts[lane & (kWideThreads / 32 - 1)]);
      join_lanes<kExact>(part, kWideThreads / 32);
      if (size > 1 && lane < static_cast<int>(size)) {
        const float* value = reinterpret_cast<const float*>(&part);
        const uint32_t to = tc::map_shared(tc::smem_u32(cluster_parts[turn & 1][rank]), lane);
#pragma unroll
        for (int k = 0; k < kSlots; ++k) store_remote(to + 4 * k, value[k]);
      }
      __syncwarp();
    }
    if (size > 1) tc::cluster_sync();
    if (warp == 0) {
      if (size > 1) {
        part = *reinterpret_cast<const Part*>(cluster_parts[turn & 1][lane & (size - 1)]);
        join_lanes<kExact>(part, static_cast<int>(size));
      }
      const RowSums t = {part.peak, part.sum, part.spread, part.apart, kExact ? part.reference_peak : 0.f, part.reference_sum,
                         masked ? part.count : static_cast<float>(a.width)};
      const bool inside = action >= 0 && action < a.width;
      const bool action_legal = inside && (!masked || a.legal[row * a.legal_stride + action]);
      const float z_a = action_legal ? as_float(static_cast<const T*>(a.logits)[row * a.stride + action]) : -INFINITY;
      const bool live = row_counts(a, row, action, t, z_a, action_legal, rank == 0 && lane == 0);
      if (a.log_probs) {
        if (rank == 0 && lane == 0) a.log_probs[row] = live ? (z_a - t.peak) - logf(t.sum) : 0.f;
      } else {
        const RowGrad grad = finish_row(a, row, t, z_a, live, acc);
        if (lane == 0) row_grad = grad, row_live = live, row_peak = t.peak;
      }
    }
    if (a.grad) {
      __syncthreads();
      const RowGrad g = row_grad;
      const float peak = row_peak;
      const bool counts = row_live;
      // Large coefficients could take a finite difference past the largest float: then a probability of zero is tested.
      tested |= g.alpha > 0.5f || g.beta > 0.5f;
      T* out = static_cast<T*>(a.grad) + row * a.grad_stride + lo;
      const bool alike_out = ((reinterpret_cast<uintptr_t>(pz.from) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
      const int64_t at = action - lo;  // the action inside this slice
      const Two from = two(-peak, -peak), scale = two(kLog2e, kLog2e), minus = two(-1.f, -1.f);
      const Two inv_sum = two(g.inv_sum, g.inv_sum), alpha = two(g.alpha, g.alpha), beta = two(g.beta, g.beta),
                constant = two(g.constant, g.constant);
#pragma unroll 2
      for (int u = tid; u < units; u += kWideThreads) {
        const int j = head + u * kVec;
        float vz[kVec], vr[kVec], v[kVec];
        load_unit(z, j, true, vz);
        if (kExact) load_unit(r, j, alike, vr);
        if (!counts) {
#pragma unroll
          for (int e = 0; e < kVec; ++e) v[e] = 0.f;
        } else if (tested) {
#pragma unroll
          for (int e = 0; e < kVec; ++e) v[e] = gradient_entry(g, peak, vz[e], kExact ? vr[e] : 0.f, kExact);
        } else {
#pragma unroll
          for (int e = 0; e < kVec; e += 2) {
            const Two zz = two(vz[e], vz[e + 1]);
            const Two x = zz + from;
            Two k = fma(alpha, x, constant);
            if (kExact) k = fma(beta, fma(two(vr[e], vr[e + 1]), minus, zz), k);
            const float2 f = apart_of(exp2_two(x * scale) * inv_sum * k);
            v[e] = f.x, v[e + 1] = f.y;
          }
        }
        if (counts && at >= j && at < j + kVec) {
#pragma unroll
          for (int e = 0; e < kVec; ++e)
            if (at == j + e) v[e] += g.action;
        }
        if (alike_out) {
          *reinterpret_cast<uint4*>(out + j) = repack(v, T());
        } else {
#pragma unroll
          for (int e = 0; e < kVec; ++e) put(out + j + e, v[e]);
        }
      }
      if (tid < ends) {
        const int j = end_entry(tid);
        float v = counts ? gradient_entry(g, peak, as_float(z[j]), kExact ? as_float(r[j]) : 0.f, kExact) : 0.f;
        if (counts && at == j) v += g.action;
        put(out + j, v);
      }
    }
    __syncthreads();  // the buffer may be overwritten
    if (buffers == 1) issue(row + clusters, 0);
  }
  if (!a.log_probs && rank == 0 && tid == 0)
    for (int k = 0; k < kTotals; ++k) a.partial[blockIdx.x / size * kTotals + k] = acc[k];
  __syncwarp();
  if (size > 1) tc::cluster_sync();  // no block leaves while another may still write to its shared memory
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
  float acc[kTotals] = {};
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
      add_entry(s, as_float(z[j]), exact ? as_float(r[j]) : 0.f, exact);
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
    const RowGrad g = finish_row(a, row, s, z_a, counts, acc);
    if (!a.grad) continue;
    T* out = static_cast<T*>(a.grad) + row * a.grad_stride;
    for (int j = threadIdx.x; j < a.width; j += kStreamThreads) {
      float v = 0.f;
      if (counts && !(legal && !legal[j])) {
        v = gradient_entry(g, s.peak, as_float(z[j]), exact ? as_float(r[j]) : 0.f, exact);
        if (j == action) v += g.action;
      }
      put(out + j, v);
    }
  }
  if (!a.log_probs && threadIdx.x == 0)
    for (int k = 0; k < kTotals; ++k) a.partial[blockIdx.x * kTotals + k] = acc[k];
}

// Warp k sums total k over the blocks: lane l the partials l, l + 32, ..., then a butterfly. The last total, the
// objective, is written once more after them.
__global__ void __launch_bounds__(kTotals * 32) anchored_totals_kernel(const double* partial, int count, float* totals) {
  const int lane = threadIdx.x & 31, k = threadIdx.x >> 5;
  pdl_wait();
  double total = 0;
#pragma unroll 8
  for (int b = lane; b < count; b += 32) total += partial[b * kTotals + k];
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) total += __shfl_xor_sync(0xffffffffu, total, o);
  if (lane == 0) totals[k] = static_cast<float>(total);
  if (lane == 0 && k == kTotals - 1) totals[kTotals] = static_cast<float>(total);
}

// A gradient times the gradient of the objective. The usual one is 1, and then there is nothing to do.
template <typename T>
__global__ void __launch_bounds__(256) anchored_scale_kernel(T* grad, int64_t rows, int64_t width, int64_t stride,
                                                             const float* scale) {
  const float by = *scale;
  if (by == 1.f) return;
  for (int64_t row = blockIdx.x; row < rows; row += gridDim.x)
    for (int64_t j = threadIdx.x; j < width; j += 256) {
      T* at = grad + row * stride + j;
      put(at, as_float(*at) * by);
    }
}

// The blocks of a kernel that are resident at once.
template <typename K>
int resident_blocks(K kernel, int threads) {
  int per_sm = 0;
  if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, 0) != cudaSuccess || per_sm < 1) per_sm = 1;
  return std::min(per_sm * sm_count(), kPartials);
}

template <typename T, int kLanes, int kVectors>
int run_narrow(const Args& a, int* blocks, cudaStream_t s) {
  static const int resident = resident_blocks(anchored_narrow_kernel<T, kLanes, kVectors>, 256);
  constexpr int kRows = 8 * (32 / kLanes);
  *blocks = static_cast<int>(std::min<int64_t>((a.rows + kRows - 1) / kRows, resident));
  anchored_narrow_kernel<T, kLanes, kVectors><<<*blocks, 256, 0, s>>>(a);
  return check_launch("anchored_narrow_kernel");
}

constexpr int kSharedPerSm = 227 * 1024;
constexpr int kSharedPerBlock = 224 * 1024;           // beside the static part
constexpr int kSliceBytes = kSharedPerSm / 3 - 2048;  // three blocks an SM

template <typename T, bool kExact>
int run_wide(const Args& a, int* blocks, cudaStream_t s, bool* fits) {
  auto kernel = anchored_wide_kernel<T, kExact>;
  static const cudaError_t configured = [&] {
    const cudaError_t rc = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kSharedPerBlock);
    return rc != cudaSuccess ? rc : cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
  }();
  if (configured != cudaSuccess) return set_error(CG_ERR_CUDA, "anchored_wide_kernel: %s", cudaGetErrorString(configured));
  constexpr int kPlanes = kExact ? 2 : 1;
  auto shared_of = [&](int slice) {  // a multiple of 16: slices are
    return kPlanes * (slice * static_cast<int>(sizeof(T)) + 32) + (a.legal ? slice + 32 : 0);
  };
  int size = 1, slice = 0, shared = 0;
  for (;; size *= 2) {
    // Slices of whole units, so that every block's slice is aligned as the row is.
    const int64_t each = (static_cast<int64_t>(a.width) + size - 1) / size;
    if (each < (1 << 20)) {
      slice = static_cast<int>((each + 15) / 16 * 16);
      shared = shared_of(slice);
      if (shared <= kSliceBytes) break;
      if (size == kMaxCluster) break;
    } else if (size == kMaxCluster) {
      shared = kSharedPerBlock + 1;
      break;
    }
  }
  *fits = shared <= kSharedPerBlock;
  if (!*fits) return CG_OK;
  // Two buffers where three blocks an SM still fit.
  const int buffers = 2 * shared <= kSliceBytes ? 2 : 1;
  const int per_sm = std::max(1, std::min(3, kSharedPerSm / (buffers * shared + 2048)));
  const int clusters = static_cast<int>(std::min<int64_t>(a.rows, std::max(1, per_sm * sm_count() / size)));
  *blocks = clusters;  // one partial sum a cluster
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(static_cast<unsigned>(clusters * size));
  config.blockDim = dim3(kWideThreads);
  config.dynamicSmemBytes = buffers * shared;
  config.stream = s;
  cudaLaunchAttribute attribute[1];
  attribute[0].id = cudaLaunchAttributeClusterDimension;
  attribute[0].val.clusterDim.x = size;
  attribute[0].val.clusterDim.y = attribute[0].val.clusterDim.z = 1;
  config.attrs = attribute;
  config.numAttrs = 1;
  const cudaError_t err = cudaLaunchKernelEx(&config, kernel, a, slice, clusters, shared, buffers);
  if (err != cudaSuccess) return set_error(CG_ERR_CUDA, "anchored_wide_kernel launch: %s", cudaGetErrorString(err));
  return check_launch("anchored_wide_kernel");
}

// A row goes where it fits: registers of four lanes (64 entries) or of a warp (1024), a cluster's shared memory, or nowhere
// (it is streamed three times).
template <typename T>
int run_typed(const Args& a, int* blocks, cudaStream_t s) {
  constexpr int kUnit = 8 / kVector<T>;  // vectors of eight entries
  if (a.width <= 64) return run_narrow<T, 4, 2 * kUnit>(a, blocks, s);
  if (a.width <= 256) return run_narrow<T, 32, kUnit>(a, blocks, s);
  if (a.width <= 512) return run_narrow<T, 32, 2 * kUnit>(a, blocks, s);
  if (a.width <= 1024) return run_narrow<T, 32, 4 * kUnit>(a, blocks, s);
  bool fits = false;
  if (int rc = a.reference ? run_wide<T, true>(a, blocks, s, &fits) : run_wide<T, false>(a, blocks, s, &fits)) return rc;
  if (fits) return CG_OK;
  *blocks = static_cast<int>(std::min<int64_t>(a.rows, kPartials));
  anchored_stream_kernel<T><<<*blocks, kStreamThreads, 0, s>>>(a);
  return check_launch("anchored_stream_kernel");
}

int run_rows(const Args& a, int dtype, int* blocks, cudaStream_t s) {
  if (dtype == CG_F32) return run_typed<float>(a, blocks, s);
  if (dtype == CG_F16) return run_typed<__half>(a, blocks, s);
  return run_typed<__nv_bfloat16>(a, blocks, s);
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

extern "C" int cg_anchored_scale(void* grad, int dtype, int64_t rows, int width, int64_t stride, const float* scale,
                                 void* stream) {
  using namespace cg;
  CG_REQUIRE(valid_dtype(dtype), "cg_anchored_scale: dtype must be float32, float16 or bfloat16");
  CG_REQUIRE(rows >= 0 && width > 0 && stride >= width, "cg_anchored_scale: bad shape");
  if (rows == 0) return CG_OK;
  CG_REQUIRE(grad && scale, "cg_anchored_scale: NULL pointer");
  const int blocks = static_cast<int>(std::min<int64_t>(rows, 8 * sm_count()));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == CG_F32)
    anchored_scale_kernel<<<blocks, 256, 0, s>>>(static_cast<float*>(grad), rows, width, stride, scale);
  else if (dtype == CG_F16)
    anchored_scale_kernel<<<blocks, 256, 0, s>>>(static_cast<__half*>(grad), rows, width, stride, scale);
  else
    anchored_scale_kernel<<<blocks, 256, 0, s>>>(static_cast<__nv_bfloat16*>(grad), rows, width, stride, scale);
  return check_launch("anchored_scale_kernel");
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
