// The anchored policy objective: PPO's clipped surrogate with a KL term to a reference policy and an entropy
// bonus, over any vocabulary, with its gradient with respect to the logits in one call.
//
// Row i over its legal set S, logits z, reference logits r, lp = z - lse_S(z), lr = r - lse_S(r), p = exp(lp):
//   ratio = exp(lp_a - old), surr = -min(ratio A, clip(ratio) A), H = -sum p lp
//   KL = sum p (lp - lr)                       with the reference's logits, or
//   KL = exp(u) - u - 1, u = lr_a - lp_a       with the reference's log-probability of the action alone (excess())
//   L = sum_i w (surr + beta KL - alpha [|S| > 1] H / log |S|)
//   dL/dz_j = p_j (K0 + w beta (z_j - r_j) + w alpha' (z_j - max z)) + [j = a] w c
// with c = d surr / d ratio * ratio (+ beta (1 - exp(u))), alpha' = alpha / log |S| and
//   K0 = w (-c - beta (KL + log s - log t + max z - max r) + alpha' (H - log s)),
// s and t the sums of exp(z - max z) and exp(r - max r). The differences from the maxima are what keeps KL and H,
// sums of small terms, from cancelling against the large log-sum-exps. An illegal entry acts as a logit of minus
// infinity, whatever it holds.
//
// All row arithmetic is fp32. The totals are summed in fp32 over the rows of one thread (rows over the resident groups of
// lanes, or over the resident blocks for wide rows: 14 of 262,144 rows of 52, 150 to 600 of as many wide ones) and in double
// from there on, in a fixed order. The entries' exponentials are ex2.approx, off by 2^-22 and by 2^-24 of
// the exponent's size, since kernels that wait for issue would pay for every instruction of a full-precision one: against 64
// bits the float32 gradient of 262,144 rows of 52 is 6.1e-7 off, by plain fp32 operations 1.1e-6.
#include <algorithm>

#include "elements.cuh"

namespace cg {
namespace {

constexpr int kTotals = 9;
constexpr int kPartials = 4736;  // the grid's upper bound: a fixed order of addition for a given row count
constexpr int kMostEntries = 1 << 30;  // of a row, counted in 32 bits with room for a batch past its end
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
  double* partial;                 // or null: no totals
  int64_t rows, stride, reference_stride, legal_stride, grad_stride;
  int width;
  float clip, beta, alpha;
  const float* scale;              // of the gradient, or null for 1
  bool given;                      // grad holds the gradient for a scale of 1 already

  // Nothing to do: the gradient of the usual scale is there. (Every thread reads the same word.)
  __device__ __forceinline__ bool done() const { return given && *scale == 1.f; }
};

// A row's sums over its legal entries, relative to a base near the largest logit (every formula is the same for any
// base; one within kLazy of the maximum keeps the exponentials in range).
struct RowSums {
  float peak, sum;              // the base m, sum e with e = exp(z - m)
  float spread;                 // sum e (z - m)
  float apart;                  // sum e ((z - m) - (r - m_r))
  float reference_peak, reference_sum;  // m_r, sum exp(r - m_r)
  float count;                  // legal entries
};
constexpr float kLazy = 8.f;

// What the gradient pass needs of a row.
struct RowGrad {
  float inv_sum, constant, beta, alpha, action;
};

// What a row brings beside its planes, loaded before the planes are waited for.
struct RowIn {
  int64_t action;
  float weight, advantage, old_log_prob, reference_log_prob;
};

__device__ __forceinline__ RowIn load_row(const Args& a, int64_t row) {
  RowIn in = {a.actions[row], 1.f, 0.f, 0.f, 0.f};
  if (!a.log_probs) {
    in.weight = a.weights[row];
    in.advantage = a.advantages[row];
    in.old_log_prob = a.old_log_probs[row];
    if (a.reference_action) in.reference_log_prob = a.reference_action[row];
  }
  return in;
}

// exp(u) - u - 1, given exp(u), as exactly for small u, where the terms cancel (at u = 1e-3 to a tenth of the result), as for
// large: below a half by its series, whose first term left out is 2^-24 of it.
__device__ __forceinline__ float excess(float u, float grown) {
  float series = fmaf(u, 1.f / 362880.f, 1.f / 40320.f);
  series = fmaf(u, series, 1.f / 5040.f);
  series = fmaf(u, series, 1.f / 720.f);
  series = fmaf(u, series, 1.f / 120.f);
  series = fmaf(u, series, 1.f / 24.f);
  series = fmaf(u, series, 1.f / 6.f);
  series = fmaf(u, series, 0.5f);
  return fabsf(u) < 0.5f ? u * u * series : grown - u - 1.f;
}

// The row's contribution to the totals (zeros unless it counts) and its gradient's coefficients.
// z_a: the action's logit, minus infinity where it is illegal.
__device__ __forceinline__ RowGrad finish_row(const Args& a, const RowIn& in, const RowSums& s, float z_a, bool counts,
                                              float (&acc)[kTotals]) {
  RowGrad g = {0.f, 0.f, 0.f, 0.f, 0.f};
  if (!counts) return g;
  const float w = in.weight, advantage = in.advantage;
  const float grad_w = a.scale ? w * *a.scale : w;  // scaled before the gradient is rounded to its type
  const float log_sum = logf(s.sum);
  const float lp = (z_a - s.peak) - log_sum;
  const float log_ratio = lp - in.old_log_prob;
  const float ratio = expf(log_ratio);
  const float free = ratio * advantage;
  const float bounded = fminf(fmaxf(ratio, 1.f - a.clip), 1.f + a.clip) * advantage;
  const bool held = free > bounded;
  const float surrogate = -(held ? bounded : free);
  float slope = held ? 0.f : -advantage * ratio;
  g.inv_sum = 1.f / s.sum;
  const float entropy = log_sum - s.spread * g.inv_sum;
  const bool eligible = s.count > 1.f;
  const float norm = eligible ? 1.f / logf(s.count) : 0.f;
  float kl = 0.f, log_apart = 0.f;
  if (a.reference) {
    log_apart = log_sum - logf(s.reference_sum);
    kl = s.apart * g.inv_sum - log_apart;
    g.beta = grad_w * a.beta;
  } else if (a.reference_action) {
    const float u = in.reference_log_prob - lp;
    kl = excess(u, expf(u));
    slope -= a.beta * (u + kl);  // 1 - exp(u)
  }
  g.alpha = grad_w * a.alpha * norm;
  g.action = grad_w * slope;
  g.constant = -g.action + g.alpha * (entropy - log_sum) - g.beta * (kl + log_apart);
  const float objective = surrogate + a.beta * kl - a.alpha * norm * entropy;
  acc[0] += w * surrogate;
  acc[1] += w;
  acc[2] += w * entropy;
  acc[3] += w * (norm * entropy);
  acc[4] += eligible ? w : 0.f;
  acc[5] += fabsf(ratio - 1.f) > a.clip ? w : 0.f;
  acc[6] += w * excess(log_ratio, ratio);
  acc[7] += w * kl;
  acc[8] += w * objective;
  return g;
}

// Whether a row counts: it has an action inside the vocabulary and something legal, and for the objective its
// weight is not zero and its action is legal. Bad actions set the fault word (once: not again for the gradient alone).
__device__ __forceinline__ bool row_counts(const Args& a, const RowIn& in, const RowSums& s, bool action_legal, bool report) {
  if (in.action < 0) return false;
  if (in.action >= a.width) {
    if (report) raise_fault(0x420);
    return false;
  }
  if (!(s.sum > 0.f) && !isnan(s.sum)) return false;  // nothing legal
  if (a.log_probs) return true;
  if (!action_legal) {
    if (report) raise_fault(0x421);
    return false;
  }
  return in.weight != 0.f;
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

__device__ __forceinline__ Two exp2_two(Two x) {
  const float2 f = apart_of(x);
  return two(exp2_fast(f.x), exp2_fast(f.y));
}

// Minus infinity in the entries of a unit whose byte of `keep` is zero; the others are 255.
template <typename T>
__device__ __forceinline__ void hide(uint4& unit, uint2 keep) {
  uint32_t* w = reinterpret_cast<uint32_t*>(&unit);
  constexpr uint32_t kInf = sizeof(T) == 4 ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
#pragma unroll
  for (int e = 0; e < 4; ++e) {
    const uint32_t mask = sizeof(T) == 4 ? __byte_perm(keep.x, 0, 0x1111 * e)
                                         : __byte_perm(e < 2 ? keep.x : keep.y, 0, e & 1 ? 0x3322 : 0x1100);
    w[e] = (w[e] & mask) | (kInf & ~mask);
  }
}

// A row's planes, and where its units and the entries outside them are.
template <typename T>
struct Row {
  const T* z;
  const T* r;
  const uint8_t* legal;
  int width, lead, head, units, ends;  // lead: entries from the aligned address at or before the row to it
  bool alike;
  __device__ __forceinline__ Row(const Args& a, int64_t row) {
    z = static_cast<const T*>(a.logits) + row * a.stride;
    r = a.reference ? static_cast<const T*>(a.reference) + row * a.reference_stride : nullptr;
    legal = a.legal ? a.legal + row * a.legal_stride : nullptr;
    width = a.width;
    lead = static_cast<int>((reinterpret_cast<uintptr_t>(z) & 15) / sizeof(T));
    head = min((kVector<T> - lead) % kVector<T>, width);
    units = (width - head) / kVector<T>;
    ends = width - units * kVector<T>;
    alike = !r || ((reinterpret_cast<uintptr_t>(z) ^ reinterpret_cast<uintptr_t>(r)) & 15) == 0;
  }
  __device__ __forceinline__ int unit_entry(int unit) const { return head + unit * kVector<T>; }
  __device__ __forceinline__ int end_entry(int k) const { return k < head ? k : k + units * kVector<T>; }
  __device__ __forceinline__ bool in(int j) const { return !legal || legal[j]; }
};

// The mask bytes of a unit: one or two aligned words where they lie inside the row, else byte by byte.
template <typename T>
__device__ __forceinline__ uint2 mask_bytes(const Row<T>& row, int j) {
  constexpr int kVec = kVector<T>;
  const uint8_t* p = row.legal + j;
  const int off = static_cast<int>(reinterpret_cast<uintptr_t>(p) & (kVec - 1));
  uint2 m = make_uint2(0, 0);
  if (off == 0 || (j - off >= 0 && j - off + 2 * kVec <= row.width)) {
    if constexpr (kVec == 8) {
      const uint64_t* w = reinterpret_cast<const uint64_t*>(p - off);
      uint64_t v = w[0];
      if (off) v = v >> (8 * off) | w[1] << (64 - 8 * off);
      m = make_uint2(static_cast<uint32_t>(v), static_cast<uint32_t>(v >> 32));
    } else {
      const uint32_t* w = reinterpret_cast<const uint32_t*>(p - off);
      m.x = off ? __funnelshift_r(w[0], w[1], 8 * off) : w[0];
    }
    return m;
  }
#pragma unroll
  for (int e = 0; e < kVec; ++e) {
    const uint32_t b = p[e];
    if (e < 4)
      m.x |= b << (8 * e);
    else
      m.y |= b << (8 * (e - 4));
  }
  return m;
}

template <typename T>
__device__ __forceinline__ uint4 gather_unit(const T* p) {
  T v[kVector<T>];
#pragma unroll
  for (int e = 0; e < kVector<T>; ++e) v[e] = p[e];
  return *reinterpret_cast<const uint4*>(v);
}

// ---- up to 1024 entries: a row in the registers of a few lanes ----------------------------------------------------------
// A row has some 350 instructions of its own (reductions, logarithms, the ratio) beside 25 an entry, so as few lanes as hold
// it, sixteen entries each, take a row, and a warp takes up to sixteen rows at a time (100,000 x 100: 50 us; with eight
// entries a lane 62). The row is read once and written once, and the grid is one resident wave of warps, two blocks an SM
// (with three the registers spill: 262,144 x 52 73 us instead of 61). A lane holds every kLanes-th unit of sixteen bytes from
// the aligned address at or before the row's start; the units that the row only partly fills, and planes aligned
// differently from the logits', go entry by entry.
//
// What bounds it is the issue of those instructions: 262,144 masked float32 rows of 52 with a reference take 61 us (164 MB, 41%
// of the copy bandwidth), 40,000 rows of 1000 113 us (65%).
//
// An entry whose exponential is zero counts for nothing. So that no test is needed, its distance from the maximum is
// held to kFar, where the exponential is zero too, and its distance from the reference is set to zero.
constexpr float kFar = -1e4f;

template <typename T, bool kExact, int kLanes, int kPer>
__global__ void __launch_bounds__(256, 2) anchored_narrow_kernel(const Args a) {
  constexpr int kVec = kVector<T>, kVectors = kPer / kVec, kGroups = 32 / kLanes;
  __shared__ double scratch[8][kTotals];
  if (a.done()) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int group = lane / kLanes, l = lane % kLanes;
  auto whole = [&](const void* base, int64_t stride, int size) {
    return ((reinterpret_cast<uintptr_t>(base) | (a.rows > 1 ? stride * size : 0)) & (size * kVec - 1)) == 0;
  };
  const bool plain_planes = whole(a.logits, a.stride, sizeof(T)) &&
                            (!kExact || whole(a.reference, a.reference_stride, sizeof(T))) &&
                            (!a.legal || whole(a.legal, a.legal_stride, 1));
  const Two scale = two(kLog2e, kLog2e), minus = two(-1.f, -1.f);
  float acc[kTotals] = {};
  auto total = [&](float v) {
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
  };
  auto largest = [&](float v) {
#pragma unroll
    for (int o = kLanes / 2; o > 0; o >>= 1) v = max_nan(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
  };
  const int64_t step = static_cast<int64_t>(gridDim.x) * 8 * kGroups;
  const int64_t warp_first = (static_cast<int64_t>(blockIdx.x) * 8 + warp) * kGroups;
  // Every group of a warp runs the same iterations, so that the shuffles stay converged.
  for (int64_t first = warp_first; first < a.rows; first += step) {
    const int64_t row = first + group;
    const bool live = row < a.rows;
    const Row<T> planes(a, row);
    const int lead = planes.lead;
    RowIn in = {-1, 0.f, 0.f, 0.f, 0.f};
    if (live) in = load_row(a, row);
    // Illegal entries, and those outside the row, are minus infinity.
    float z[kPer], r[kPer];
    uint4 raw_z[kVectors], raw_r[kVectors];
    uint2 keep[kVectors];
    // The planes alike, the mask's words whole: no branch between the loads, which wait together.
    auto fetch = [&](auto which) {
      constexpr bool plain = decltype(which)::value;
#pragma unroll
      for (int v = 0; v < kVectors; ++v) {
        const int j = (l + kLanes * v) * kVec - (plain ? 0 : lead);
        raw_z[v] = raw_r[v] = make_uint4(0, 0, 0, 0);
        keep[v] = make_uint2(0, 0);
        if (!live || j >= a.width) continue;
        if ((plain || j >= 0) && j + kVec <= a.width) {
          raw_z[v] = *reinterpret_cast<const uint4*>(planes.z + j);
          if (kExact)
            raw_r[v] = plain || planes.alike ? *reinterpret_cast<const uint4*>(planes.r + j) : gather_unit(planes.r + j);
          keep[v] = make_uint2(~0u, ~0u);
          if (planes.legal) {
            if constexpr (!plain)
              keep[v] = mask_bytes(planes, j);
            else if constexpr (kVec == 4)
              keep[v].x = *reinterpret_cast<const uint32_t*>(planes.legal + j);
            else
              keep[v] = *reinterpret_cast<const uint2*>(planes.legal + j);
          }
        } else {  // a unit that the row fills in part
          T tz[kVec], tr[kVec];
#pragma unroll
          for (int e = 0; e < kVec; ++e) {
            const bool inside = j + e >= 0 && j + e < a.width;
            put(&tz[e], 0.f), put(&tr[e], 0.f);
            if (inside) tz[e] = planes.z[j + e];
            if (inside && kExact) tr[e] = planes.r[j + e];
            const uint32_t byte = !inside ? 0u : planes.legal ? planes.legal[j + e] : 1u;
            (e < 4 ? keep[v].x : keep[v].y) |= byte << (8 * (e & 3));
          }
          raw_z[v] = *reinterpret_cast<const uint4*>(tz), raw_r[v] = *reinterpret_cast<const uint4*>(tr);
        }
      }
    };
    if (plain_planes)
      fetch(std::true_type());
    else
      fetch(std::false_type());
    int bits = 0;
#pragma unroll
    for (int v = 0; v < kVectors; ++v) {
      uint2 k = make_uint2(__vcmpne4(keep[v].x, 0), 0u);
      if constexpr (kVec == 8) k.y = __vcmpne4(keep[v].y, 0);
      bits += __popc(k.x) + __popc(k.y);
      hide<T>(raw_z[v], k);
      float t[kVec];
      unpack(raw_z[v], t, T());
#pragma unroll
      for (int e = 0; e < kVec; ++e) z[v * kVec + e] = t[e];
      if (kExact) {
        hide<T>(raw_r[v], k);
        unpack(raw_r[v], t, T());
#pragma unroll
        for (int e = 0; e < kVec; ++e) r[v * kVec + e] = t[e];
      }
    }
    const float count = static_cast<float>(bits >> 3);
    const bool action_legal = in.action >= 0 && in.action < a.width && planes.in(static_cast<int>(in.action));
    const float z_a = action_legal ? as_float(planes.z[in.action]) : -INFINITY;
    const float r_a = kExact && action_legal ? as_float(planes.r[in.action]) : -INFINITY;
    RowSums s = {};
    float peak = z[0], reference_peak = kExact ? r[0] : 0.f;
#pragma unroll
    for (int k = 1; k < kPer; ++k) {
      peak = max_nan(peak, z[k]);
      if (kExact) reference_peak = max_nan(reference_peak, r[k]);
    }
    s.peak = largest(peak);
    if (kExact) s.reference_peak = largest(reference_peak);
    s.count = total(count);
    const float base = s.peak == -INFINITY ? 0.f : s.peak;
    Two x[kPer / 2], e[kPer / 2], d[kPer / 2], sum = two(0.f, 0.f), spread = sum, apart = sum, reference_sum = sum;
    // An entry's distance from the maximum, its exponential, and its distance from the reference's.
    auto measure = [&](Two zz, Two rr, Two* xx, Two* ee, Two* dd, Two* reference_e) {
      const float2 far = apart_of(zz + two(-base, -base));
      *xx = two(max_nan(far.x, kFar), max_nan(far.y, kFar));
      *ee = exp2_two(*xx * scale);
      if (kExact) {
        const Two y = rr + two(-s.reference_peak, -s.reference_peak);
        *reference_e = exp2_two(y * scale);
        const float2 g = apart_of(fma(y, minus, *xx)), f = apart_of(*ee);
        *dd = two(f.x == 0.f ? 0.f : g.x, f.y == 0.f ? 0.f : g.y);
      }
    };
#pragma unroll
    for (int k = 0; k < kPer / 2; ++k) {
      Two reference_e;
      measure(two(z[2 * k], z[2 * k + 1]), kExact ? two(r[2 * k], r[2 * k + 1]) : sum, &x[k], &e[k], &d[k], &reference_e);
      sum = sum + e[k];
      spread = fma(e[k], x[k], spread);
      if (kExact) {
        reference_sum = reference_sum + reference_e;
        apart = fma(e[k], d[k], apart);
      }
    }
    const float2 fs = apart_of(sum), fd = apart_of(spread), fa = apart_of(apart), fr = apart_of(reference_sum);
    s.sum = total(fs.x + fs.y);
    if (!a.log_probs) s.spread = total(fd.x + fd.y);
    if (kExact) {
      s.reference_sum = total(fr.x + fr.y);
      s.apart = total(fa.x + fa.y);
    }
    const bool counts = row_counts(a, in, s, action_legal, l == 0 && !a.scale);
    if (a.log_probs) {
      if (live && l == 0) a.log_probs[row] = counts ? (z_a - s.peak) - logf(s.sum) : 0.f;
      continue;
    }
    const RowGrad g = finish_row(a, in, s, z_a, counts, acc);  // every lane of the group keeps the same totals
    if (!a.grad || !live) continue;
    T* out = static_cast<T*>(a.grad) + row * a.grad_stride;
    const bool alike_out = ((reinterpret_cast<uintptr_t>(planes.z) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
    const Two inv_sum = two(g.inv_sum, g.inv_sum), alpha = two(g.alpha, g.alpha), beta = two(g.beta, g.beta),
              constant = two(g.constant, g.constant);
    const bool plain = counts && isfinite(g.constant);
    auto gradient = [&](Two xx, Two ee, Two dd) {
      const Two p = ee * inv_sum;
      Two k = fma(alpha, xx, constant);
      if (kExact) k = fma(beta, dd, k);
      const float2 v = apart_of(p * k), f = apart_of(ee);
      if (plain) return v;
      // No gradient where the row does not count or the probability is zero, whatever it is multiplied by.
      return make_float2(counts && f.x != 0.f ? v.x : 0.f, counts && f.y != 0.f ? v.y : 0.f);
    };
#pragma unroll
    for (int v = 0; v < kVectors; ++v) {
      float t[kVec];
#pragma unroll
      for (int k = 0; k < kVec; k += 2) {
        const int at = (v * kVec + k) / 2;
        const float2 f = gradient(x[at], e[at], d[at]);
        t[k] = f.x, t[k + 1] = f.y;
      }
      const int j = (l + kLanes * v) * kVec - lead;
      if (alike_out && j >= 0 && j + kVec <= a.width) {
        *reinterpret_cast<uint4*>(out + j) = repack(t, T());
      } else {
#pragma unroll
        for (int k = 0; k < kVec; ++k)
          if (j + k >= 0 && j + k < a.width) put(out + j + k, t[k]);
      }
    }
    // The action's entry, once more by the lane that has just written it.
    if (counts && l == (static_cast<int>(in.action) + lead) / kVec % kLanes) {
      Two xx, ee, dd, reference_e;
      measure(two(z_a, z_a), two(r_a, r_a), &xx, &ee, &dd, &reference_e);
      put(out + in.action, gradient(xx, ee, dd).x + g.action);
    }
  }
  if (!a.partial) return;
  // The groups' leaders in order, then the warps.
#pragma unroll
  for (int k = 0; k < kTotals; ++k) {
    double sum = acc[k];
#pragma unroll
    for (int other = 1; other < kGroups; ++other) {
      sum += __shfl_sync(0xffffffffu, acc[k], other * kLanes);
    }
    if (lane == 0) scratch[warp][k] = sum;
  }
  __syncthreads();
  if (threadIdx.x < kTotals) {
    double sum = 0;
    for (int w = 0; w < 8; ++w) sum += scratch[w][threadIdx.x];
    a.partial[blockIdx.x * kTotals + threadIdx.x] = sum;
  }
}

// ---- wider rows: a block a row ------------------------------------------------------------------------------------------
// A thread holds its share of the row, or of a batch of it, in registers as it is in memory: up to four units of sixteen
// bytes of each plane in flight at a time. It sums a batch relative to the batch's own maxima and merges the result into
// its running sums, so the row's maxima are never waited for; the block joins its threads once a row.
// A row of one batch (kHeld) is read once and its gradient computed from the registers (16,384 x 4096 bfloat16: 124 us, read
// twice 230). A longer one is read again for the gradient, out of L2 where the rows in work at one time fit (see run_wide).
//
// What bounds it is instruction issue beside memory: three exponentials an entry and, in packed fp32 pairs, some 25
// instructions at 2.2 a cycle and SM. 4096 x 131072 bfloat16 with a reference: 860 us for 3.2 GB, 57% of the copy bandwidth;
// 4000 x 32000 float32 361 us, 65%; log-probabilities of 1500 x 50,021 float16 42 us, 55%.
//
// Entries at minus infinity, which the packed sums turn into NaN, are found by that and summed again with tests. Units
// start where the logits' row is aligned; the few entries before and after them go one a thread, and planes aligned
// differently from the logits' are read entry by entry.

// Partial results over some entries, each relative to their own maxima. `tested`: minus infinity was among them.
struct Part {
  float peak, reference_peak, sum, spread, reference_sum, apart, count, tested;
};
__device__ __forceinline__ Part no_part() { return {-INFINITY, -INFINITY, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f}; }

// The part relative to larger maxima.
template <bool kExact>
__device__ __forceinline__ void rebase(Part& p, float peak, float reference_peak) {
  const float up = p.peak == -INFINITY ? 0.f : p.peak - peak;
  const float scale = p.peak == -INFINITY ? 0.f : exp2_fast(up * kLog2e);
  if (kExact) {
    const float reference_up = p.reference_peak == -INFINITY ? 0.f : p.reference_peak - reference_peak;
    p.reference_sum *= p.reference_peak == -INFINITY ? 0.f : exp2_fast(reference_up * kLog2e);
    // Without a reference entry above minus infinity the part's differences are infinite already.
    p.apart = scale == 0.f ? 0.f : scale * fmaf(up - reference_up, p.sum, p.apart);
    p.reference_peak = reference_peak;
  }
  p.spread = scale == 0.f ? 0.f : scale * fmaf(up, p.sum, p.spread);
  p.sum = scale == 0.f ? 0.f : scale * p.sum;
  p.peak = peak;
}

// Bases for more entries whose maxima are top and reference_top: the part keeps its own, so that its sums need no scaling,
// unless an exponential would pass exp(kLazy).
template <bool kExact>
__device__ __forceinline__ void lift(Part& p, float top, float reference_top) {
  if (top <= p.peak + kLazy && (!kExact || reference_top <= p.reference_peak + kLazy) && p.peak != -INFINITY) return;
  const float peak = top <= p.peak + kLazy ? p.peak : top;
  const float reference_peak = reference_top <= p.reference_peak + kLazy ? p.reference_peak : reference_top;
  rebase<kExact>(p, max_nan(p.peak, peak), max_nan(p.reference_peak, reference_peak));
}

__device__ __forceinline__ float warp_max_nan(float v) {
  float m;
  asm("redux.sync.max.NaN.f32 %0, %1, 0xffffffff;" : "=f"(m) : "f"(v));
  return m;
}

// The parts of the first `lanes` lanes of a warp joined (the others hold no_part()); lane 0 gets the result.
template <bool kExact>
__device__ __forceinline__ void join_lanes(Part& p, int lanes, bool masked) {
  rebase<kExact>(p, warp_max_nan(p.peak), kExact ? warp_max_nan(p.reference_peak) : 0.f);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    if (o >= lanes) continue;
    p.sum += __shfl_xor_sync(0xffffffffu, p.sum, o);
    p.spread += __shfl_xor_sync(0xffffffffu, p.spread, o);
    if (kExact) {
      p.reference_sum += __shfl_xor_sync(0xffffffffu, p.reference_sum, o);
      p.apart += __shfl_xor_sync(0xffffffffu, p.apart, o);
    }
    if (masked) p.count += __shfl_xor_sync(0xffffffffu, p.count, o);
  }
  p.tested = __any_sync(0xffffffffu, p.tested != 0.f) ? 1.f : 0.f;
}

// One unit of a row, what the mask hides at minus infinity; the number of legal entries is added to `count`.
template <typename T, bool kExact>
__device__ __forceinline__ void load_unit(const Row<T>& row, int j, uint4& z, uint4& r, float& count) {
  z = *reinterpret_cast<const uint4*>(row.z + j);
  if (kExact) r = row.alike ? *reinterpret_cast<const uint4*>(row.r + j) : gather_unit(row.r + j);
  if (!row.legal) return;
  uint2 m = mask_bytes(row, j);
  m = make_uint2(__vcmpne4(m.x, 0), __vcmpne4(m.y, 0));
  count += static_cast<float>((__popc(m.x) + __popc(m.y)) >> 3);
  hide<T>(z, m);
  if (kExact) hide<T>(r, m);
}

// A batch's units, the first `n` of which exist, added to a part.
template <typename T, bool kExact, int kUnits>
__device__ __forceinline__ void add_units(Part& p, const uint4 (&z)[kUnits], const uint4 (&r)[kUnits], int n) {
  constexpr int kVec = kVector<T>;
  UnitMax<T> top_z, top_r;
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    if (i >= n) continue;
    top_z.take(z[i]);
    if (kExact) top_r.take(r[i]);
  }
  lift<kExact>(p, top_z.value(), kExact ? top_r.value() : 0.f);
  const float base = p.peak == -INFINITY ? 0.f : p.peak;
  const float reference_base = p.reference_peak == -INFINITY ? 0.f : p.reference_peak;
  const Two from = two(-base, -base), reference_from = two(-reference_base, -reference_base);
  const Two scale = two(kLog2e, kLog2e), minus = two(-1.f, -1.f);
  Two sum = two(0.f, 0.f), spread = sum, apart = sum, reference_sum = sum;
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    if (i >= n) continue;
    float vz[kVec], vr[kVec];
    unpack(z[i], vz, T());
    if (kExact) unpack(r[i], vr, T());
#pragma unroll
    for (int e = 0; e < kVec; e += 2) {
      const Two x = two(vz[e], vz[e + 1]) + from;
      const Two e2 = exp2_two(x * scale);
      sum = sum + e2;
      spread = fma(e2, x, spread);
      if (kExact) {
        const Two y = two(vr[e], vr[e + 1]) + reference_from;
        reference_sum = reference_sum + exp2_two(y * scale);
        apart = fma(e2, fma(y, minus, x), apart);
      }
    }
  }
  float2 fs = apart_of(sum), fd = apart_of(spread), fa = apart_of(apart), fr = apart_of(reference_sum);
  const float odd = (fd.x + fd.y) + (fa.x + fa.y);
  if (isnan(odd)) {
    p.tested = 1.f;
    RowSums t = {};
    t.peak = base, t.reference_peak = reference_base;
#pragma unroll
    for (int i = 0; i < kUnits; ++i) {
      if (i >= n) continue;
      float vz[kVec], vr[kVec];
      unpack(z[i], vz, T());
      if (kExact) unpack(r[i], vr, T());
#pragma unroll
      for (int e = 0; e < kVec; ++e) add_entry(t, vz[e], kExact ? vr[e] : 0.f, kExact);
    }
    fs = make_float2(t.sum, 0.f), fd = make_float2(t.spread, 0.f), fa = make_float2(t.apart, 0.f);
    fr = make_float2(t.reference_sum, 0.f);
  }
  p.sum += fs.x + fs.y, p.spread += fd.x + fd.y;
  if (kExact) p.apart += fa.x + fa.y, p.reference_sum += fr.x + fr.y;
}

// An entry outside the units added to a part.
template <typename T, bool kExact>
__device__ __forceinline__ void add_end(Part& p, const Row<T>& row, int j) {
  if (!row.in(j)) return;
  const float z = as_float(row.z[j]), r = kExact ? as_float(row.r[j]) : 0.f;
  lift<kExact>(p, z, r);
  RowSums t = {};
  t.peak = p.peak == -INFINITY ? 0.f : p.peak, t.reference_peak = p.reference_peak == -INFINITY ? 0.f : p.reference_peak;
  add_entry(t, z, r, kExact);
  p.sum += t.sum, p.spread += t.spread, p.count += 1.f;
  if (kExact) p.apart += t.apart, p.reference_sum += t.reference_sum;
}

// The gradient of a unit.
template <typename T, bool kExact>
__device__ __forceinline__ uint4 gradient_unit(const RowGrad& g, float peak, bool tested, const uint4& z, const uint4& r,
                                               int at) {
  constexpr int kVec = kVector<T>;
  float vz[kVec], vr[kVec], v[kVec];
  unpack(z, vz, T());
  if (kExact) unpack(r, vr, T());
  if (tested) {
#pragma unroll
    for (int e = 0; e < kVec; ++e) v[e] = gradient_entry(g, peak, vz[e], kExact ? vr[e] : 0.f, kExact);
  } else {
    const Two from = two(-peak, -peak), scale = two(kLog2e, kLog2e), minus = two(-1.f, -1.f);
    const Two inv_sum = two(g.inv_sum, g.inv_sum), alpha = two(g.alpha, g.alpha), beta = two(g.beta, g.beta),
              constant = two(g.constant, g.constant);
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
  if (at >= 0) {  // the action's place in the unit
#pragma unroll
    for (int e = 0; e < kVec; ++e)
      if (at == e) v[e] += g.action;
  }
  return repack(v, T());
}

// What a row's gradient needs, from the warp that finishes the row to the others.
struct RowOut {
  RowGrad grad;
  float peak;
  int live, tested;
};

template <typename T, bool kExact, int kThreads, bool kHeld>
__global__ void __launch_bounds__(kThreads, (kThreads >= 512 ? 1024 : 768) / kThreads) anchored_row_kernel(const Args a) {
  constexpr int kUnits = kThreads >= 512 ? 2 : 4, kWarps = kThreads / 32, kVec = kVector<T>;
  __shared__ Part warp_parts[2][kWarps];
  __shared__ RowOut row_out[2];
  if (a.done()) return;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  float acc[kTotals] = {};
  int turn = 0;  // rows done: what the warps exchange alternates, so that two barriers a row are enough
  for (int64_t index = blockIdx.x; index < a.rows; index += gridDim.x, turn ^= 1) {
    const Row<T> row(a, index);
    const bool masked = row.legal != nullptr;
    const RowIn in = load_row(a, index);
    bool action_legal = in.action >= 0 && in.action < a.width;
    float z_a = -INFINITY;
    uint4 z[kUnits], r[kUnits];
    Part part = no_part();
    constexpr int kBatch = kUnits * kThreads;  // units of a batch
    // A batch's units, all in flight; returns how many this thread has.
    auto load_batch = [&](int first) {
      int n = 0;
      if (!masked && row.alike && first + kBatch <= row.units) {
        const T* from_z = row.z + row.unit_entry(first + tid);
        const T* from_r = row.r + row.unit_entry(first + tid);
#pragma unroll
        for (int i = 0; i < kUnits; ++i) {
          z[i] = *reinterpret_cast<const uint4*>(from_z + i * kThreads * kVec);
          if (kExact) r[i] = *reinterpret_cast<const uint4*>(from_r + i * kThreads * kVec);
        }
        return kUnits;
      }
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int u = first + tid + i * kThreads;
        if (u >= row.units) continue;
        load_unit<T, kExact>(row, row.unit_entry(u), z[i], r[i], part.count);
        n = i + 1;
      }
      return n;
    };
    const int held = load_batch(0);
    if (warp == 0 && action_legal) {
      action_legal = row.in(static_cast<int>(in.action));
      if (action_legal) z_a = as_float(row.z[in.action]);
    }
    add_units<T, kExact, kUnits>(part, z, r, held);
    if (!kHeld) {
      for (int first = kBatch; first < row.units; first += kBatch) {
        const int n = load_batch(first);
        add_units<T, kExact, kUnits>(part, z, r, n);
      }
    }
    if (tid < row.ends) add_end<T, kExact>(part, row, row.end_entry(tid));
    join_lanes<kExact>(part, 32, masked);
    if (lane == 0) warp_parts[turn][warp] = part;
    __syncthreads();
    if (warp == 0) {
      part = lane < kWarps ? warp_parts[turn][lane] : no_part();
      join_lanes<kExact>(part, kWarps, masked);
      const RowSums s = {part.peak, part.sum, part.spread, part.apart, kExact ? part.reference_peak : 0.f, part.reference_sum,
                         masked ? part.count : static_cast<float>(a.width)};
      const bool live = row_counts(a, in, s, action_legal, lane == 0 && !a.scale);
      if (a.log_probs) {
        if (lane == 0) a.log_probs[index] = live ? (z_a - s.peak) - logf(s.sum) : 0.f;
      } else {
        RowGrad g = finish_row(a, in, s, z_a, live, acc);
        if (kExact) g.constant -= g.beta * (s.peak - s.reference_peak);  // the entries' own differences are z - r here
        // Large coefficients, of either sign, could take a finite difference past the largest float: then a probability of
        // zero is tested.
        if (lane == 0) row_out[turn] = {g, s.peak, live, part.tested != 0.f || fabsf(g.alpha) > 0.5f || fabsf(g.beta) > 0.5f};
      }
    }
    if (!a.grad) continue;
    __syncthreads();
    const RowOut o = row_out[turn];
    T* out = static_cast<T*>(a.grad) + index * a.grad_stride;
    const bool alike_out = ((reinterpret_cast<uintptr_t>(row.z) ^ reinterpret_cast<uintptr_t>(out)) & 15) == 0;
    const int action_unit = in.action >= row.head ? (static_cast<int>(in.action) - row.head) / kVec : -1;
    const int action_entry = (static_cast<int>(in.action) - row.head) % kVec;
    auto store_batch = [&](int first) {
      T* to = out + row.unit_entry(first + tid);
      const bool whole = first + kBatch <= row.units;
#pragma unroll
      for (int i = 0; i < kUnits; ++i) {
        const int u = first + tid + i * kThreads;
        if (!whole && u >= row.units) continue;
        const uint4 v = o.live ? gradient_unit<T, kExact>(o.grad, o.peak, o.tested, z[i], r[i], u == action_unit ? action_entry : -1)
                               : make_uint4(0, 0, 0, 0);
        if (alike_out) {
          __stcs(reinterpret_cast<uint4*>(to + i * kThreads * kVec), v);
        } else {
          const T* e = reinterpret_cast<const T*>(&v);
#pragma unroll
          for (int k = 0; k < kVec; ++k) to[i * kThreads * kVec + k] = e[k];
        }
      }
    };
    if (kHeld) {
      store_batch(0);
    } else {
      for (int first = 0; first < row.units; first += kBatch) {
        load_batch(first);
        store_batch(first);
      }
    }
    if (tid < row.ends) {
      const int j = row.end_entry(tid);
      float v = 0.f;
      if (o.live && row.in(j)) {
        v = gradient_entry(o.grad, o.peak, as_float(row.z[j]), kExact ? as_float(row.r[j]) : 0.f, kExact);
        if (j == in.action) v += o.grad.action;
      }
      put(out + j, v);
    }
  }
  if (a.partial && tid == 0)
    for (int k = 0; k < kTotals; ++k) a.partial[blockIdx.x * kTotals + k] = acc[k];
}

// Every total over the blocks: thread (g, k) takes total k of the blocks g, g + 112, ... in order, then one thread a total
// the 112 sums in order. The last total, the objective, is written once more after them.
constexpr int kTotalGroups = 112;

__global__ void __launch_bounds__(1024) anchored_totals_kernel(const double* partial, int count, float* totals) {
  __shared__ double sums[kTotalGroups][kTotals];
  const int g = threadIdx.x / kTotals, k = threadIdx.x % kTotals;
  pdl_wait();
  if (g < kTotalGroups) {
    double total = 0;
#pragma unroll 8
    for (int b = g; b < count; b += kTotalGroups) total += partial[b * kTotals + k];
    sums[g][k] = total;
  }
  __syncthreads();
  if (threadIdx.x >= kTotals) return;
  double total = 0;
#pragma unroll 16
  for (int i = 0; i < kTotalGroups; ++i) total += sums[i][k];
  totals[k] = static_cast<float>(total);
  if (k == kTotals - 1) totals[kTotals] = static_cast<float>(total);
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

template <typename T, bool kExact, int kLanes, int kPer>
int run_narrow(const Args& a, int* blocks, cudaStream_t s) {
  static const int resident = resident_blocks(anchored_narrow_kernel<T, kExact, kLanes, kPer>, 256);
  constexpr int kRows = 8 * (32 / kLanes);
  *blocks = static_cast<int>(std::min<int64_t>((a.rows + kRows - 1) / kRows, resident));
  anchored_narrow_kernel<T, kExact, kLanes, kPer><<<*blocks, 256, 0, s>>>(a);
  return check_launch("anchored_narrow_kernel");
}

template <typename T, bool kExact, int kThreads, bool kHeld>
int run_row(const Args& a, int* blocks, cudaStream_t s) {
  static const int resident = resident_blocks(anchored_row_kernel<T, kExact, kThreads, kHeld>, kThreads);
  *blocks = static_cast<int>(std::min<int64_t>(a.rows, resident));
  anchored_row_kernel<T, kExact, kThreads, kHeld><<<*blocks, kThreads, 0, s>>>(a);
  return check_launch("anchored_row_kernel");
}

// The smallest block that holds the row in its registers. Longer rows: 16-bit ones take 256 threads, whether or not the
// rows in work fit L2 (131,072 entries, which do not: 859 us, with 1024 threads 878; 32,000: 220 against 264). So do float32 ones whose resident
// blocks' rows stay in L2 between their two readings (80 of its 126 MB, the rest for the gradient passing through:
// 10,000 entries 123 us against 185), else 1024 threads, which have fewer rows in work (32,000: 361 against 411).
template <typename T, bool kExact>
int run_wide(const Args& a, int* blocks, cudaStream_t s) {
  constexpr int kHeldEntries = 4 * kVector<T>;  // a thread's
  if (a.width <= 64 * kHeldEntries) return run_row<T, kExact, 64, true>(a, blocks, s);
  if (a.width <= 128 * kHeldEntries) return run_row<T, kExact, 128, true>(a, blocks, s);
  if (a.width <= 256 * kHeldEntries) return run_row<T, kExact, 256, true>(a, blocks, s);
  if constexpr (sizeof(T) == 4) {
    const int64_t row_bytes = static_cast<int64_t>(a.width) * sizeof(T) * (kExact ? 2 : 1);
    if (a.grad && 3 * sm_count() * row_bytes > int64_t{80} << 20) return run_row<T, kExact, 1024, false>(a, blocks, s);
  }
  return run_row<T, kExact, 256, false>(a, blocks, s);
}

// A row goes where it fits: registers of two lanes (32 entries) to a warp (1024; 40,000 x 1000 float32: 113 us, by the next
// rule's blocks 170) or of a block, or a block that reads it twice. An unaligned row takes up to a unit more.
template <typename T, bool kExact>
int run_typed(const Args& a, int* blocks, cudaStream_t s) {
  const bool aligned = (reinterpret_cast<uintptr_t>(a.logits) & 15) == 0 && (a.rows == 1 || a.stride % kVector<T> == 0);
  const int64_t span = static_cast<int64_t>(a.width) + (aligned ? 0 : kVector<T> - 1);
  if (span <= 32) return run_narrow<T, kExact, 2, 16>(a, blocks, s);
  if (span <= 64) return run_narrow<T, kExact, 4, 16>(a, blocks, s);
  if (span <= 128) return run_narrow<T, kExact, 8, 16>(a, blocks, s);
  if (span <= 256) return run_narrow<T, kExact, 16, 16>(a, blocks, s);
  if (span <= 512) return run_narrow<T, kExact, 32, 16>(a, blocks, s);
  if (span <= 1024) return run_narrow<T, kExact, 32, 32>(a, blocks, s);
  return run_wide<T, kExact>(a, blocks, s);
}

template <typename T>
int run_typed(const Args& a, int* blocks, cudaStream_t s) {
  return a.reference ? run_typed<T, true>(a, blocks, s) : run_typed<T, false>(a, blocks, s);
}

int run_rows(const Args& a, int dtype, int* blocks, cudaStream_t s) {
  if (dtype == CG_F32) return run_typed<float>(a, blocks, s);
  if (dtype == CG_F16) return run_typed<__half>(a, blocks, s);
  return run_typed<__nv_bfloat16>(a, blocks, s);
}

}  // namespace
}  // namespace cg

namespace cg {
namespace {

// The checks that the objective and its gradient share.
int check_rows(const char* name, const Args& a, int dtype) {
  CG_REQUIRE(valid_dtype(dtype), "%s: dtype must be float32, float16 or bfloat16", name);
  CG_REQUIRE(a.rows >= 0 && a.width > 0 && a.width <= kMostEntries, "%s: bad shape", name);
  CG_REQUIRE(a.stride >= a.width && (!a.grad || a.grad_stride >= a.width) &&
                 (!a.reference || a.reference_stride >= a.width) && (!a.legal || a.legal_stride >= a.width),
             "%s: stride < width", name);
  CG_REQUIRE(!(a.reference && a.reference_action), "%s: one reference at most", name);
  CG_REQUIRE(a.clip >= 0, "%s: clip_ratio must not be negative", name);
  CG_REQUIRE(a.rows == 0 || (a.logits && a.actions && a.old_log_probs && a.advantages && a.weights), "%s: NULL pointer",
             name);
  return CG_OK;
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
  auto* partial = static_cast<double*>(workspace);
  const Args a = {logits, reference_logits, reference_log_probs, legal, actions, old_log_probs, advantages, weights,
                  grad, nullptr, partial, rows, stride, reference_stride, legal_stride, grad_stride, width,
                  clip_ratio, beta, alpha, nullptr, false};
  if (int rc = check_rows("cg_anchored_objective", a, dtype)) return rc;
  CG_REQUIRE(totals, "cg_anchored_objective: NULL totals");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  int blocks = 0;
  if (rows > 0) {
    if (!workspace || workspace_bytes < cg_anchored_objective_workspace_bytes(rows))
      return set_error(CG_ERR_WORKSPACE, "cg_anchored_objective: workspace too small");
    if (int rc = run_rows(a, dtype, &blocks, s)) return rc;
  }
  return launch_pdl("anchored_totals_kernel", anchored_totals_kernel, dim3(1), dim3(1024), 0, s,
                    static_cast<const double*>(partial), blocks, totals);
}

extern "C" int cg_anchored_gradient(const void* logits, int dtype, int64_t rows, int width, int64_t stride,
                                    const void* reference_logits, int64_t reference_stride,
                                    const float* reference_log_probs, const uint8_t* legal, int64_t legal_stride,
                                    const int64_t* actions, const float* old_log_probs, const float* advantages,
                                    const float* weights, float clip_ratio, float beta, float alpha, const float* scale,
                                    int given, void* grad, int64_t grad_stride, void* stream) {
  using namespace cg;
  const Args a = {logits, reference_logits, reference_log_probs, legal, actions, old_log_probs, advantages, weights,
                  grad, nullptr, nullptr, rows, stride, reference_stride, legal_stride, grad_stride, width,
                  clip_ratio, beta, alpha, scale, given != 0};
  if (int rc = check_rows("cg_anchored_gradient", a, dtype)) return rc;
  if (rows == 0) return CG_OK;
  CG_REQUIRE(grad && scale, "cg_anchored_gradient: NULL pointer");
  int blocks = 0;
  return run_rows(a, dtype, &blocks, static_cast<cudaStream_t>(stream));
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
  CG_REQUIRE(rows >= 0 && width > 0 && width <= kMostEntries, "cg_action_log_probs: bad shape");
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
