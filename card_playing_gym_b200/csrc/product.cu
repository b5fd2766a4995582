// C[i, j] = sum_k A(i, k) B(j, k) on the tensor cores, with the linear layer's epilogue.
//
// Pairs of CTAs on two SMs compute 256 x tile_n outputs: one tcgen05.mma.cta_group::2 (M = 256, K = 16) reads each
// CTA's own 128 rows of A and its half of B's tile_n rows from its own shared memory, so a stage of 64 k's is 32 KB per
// SM for 2 x 256 x 256 x 64 FMAs, and each CTA's tensor memory receives its own 128 rows. The kernel is persistent: tensor
// memory holds two accumulators, and the epilogue of one tile runs while the next is multiplied.
//   warps 0-7  epilogue: 32 columns of a row a lane from tensor memory to registers and, where rows are aligned, from there to
//              their place in whole sectors; else through a 4 KB shared-memory square per warp, four columns a lane
//   warp 8     lane 0 fills the ring of six stages by TMA (128-byte swizzle; both operand orders, so neither product of
//              the backward pass transposes anything in memory)
//   warp 9     allocates tensor memory; in the even CTA lane 0 issues the MMAs
// Loads of both CTAs complete on the even CTA's barriers; MMA completions are committed to both CTAs'.
//
// float32 operands are three bfloat16 parts each (8 bits of mantissa apiece): the six products of parts that reach
// 2^-24 of the result run from one stage that holds all three parts of both operands, at six times the bfloat16 work
// and three times its traffic. The tensor cores cut their running sum at each step (measured on terms of one sign: by
// 1.7e-7 of it every 16 k's, always toward zero; of random signs a tenth of that), which a long float32 sum would show:
// the five small products have an accumulator of their own, and after kChunkBlocks blocks of k the epilogue takes both
// sums into registers, where they are added with rounding, and the next chunk starts from zero in the other pair of
// accumulators. An infinity or NaN is its own first part, so the product of first parts is the float32 one; what it
// makes of the small products (an infinity times parts of either sign, or of zero) is left out. tile_n is 128 for
// float32, so that two pairs fit tensor memory.
//
// 16-bit results keep one running sum as far as its cuts stay well inside their own rounding: 16,384 k's of float16
// (9e-5 of the sum at most, against 4.9e-4) and 65,536 of bfloat16 (3.9e-4 against 3.9e-3). Deeper products, the weight
// gradients of long batches, add such sums with rounding, in a place of each lane's own that stays in L2 (262,144 rows
// of float16 in one sum: 1.5e-3 short).
//
// Where the last round of tiles leaves half the pairs idle, k is split for the tiles of that round: every split writes
// fp32 partial sums and product_join_kernel adds them in order and applies the epilogue (8192 k's of 4096 x 4096: 256
// tiles are three rounds of 74 and 34 tiles in two halves, 232 us with the join and 254 unsplit; 256 rows x 8192 x 1024:
// 21 us against 56).
//
// What bounds it is the tensor cores' feed: 8192 x 4096 x 4096 bfloat16 with its epilogue takes 207 us, 1330 TFLOP/s, 79%
// of what the library reaches on its best shape, and 16,384 x 720 x 240 float32 52 us, 650 TFLOP/s of bfloat16
// parts. A single round of tiles costs 10 to 15 us beside its products, in launch, first loads and last epilogue.
#include "product.h"

#include <cuda.h>

#include <algorithm>

#include "elements.cuh"
#include "tcgen05.cuh"

namespace cg {
namespace {

constexpr int kPairs = 74;  // of the B200's 148 SMs
constexpr int kTileM = 256, kTileK = 64;  // a pair's rows; k's of a stage (128 bytes of 16-bit entries)
constexpr int kHalfBytes = 128 * kTileK * 2;  // one CTA's rows of A (or of B at tile_n 256) of a stage
constexpr int kEpilogueWarps = 8;
constexpr int kLoadWarp = 8, kMmaWarp = 9;
constexpr int kThreads = 10 * 32;
constexpr int kSquareBytes = 32 * 32 * 4;
constexpr int kAccumulatorColumns = 256;  // of one of the two accumulators (float32: the main products' and the small ones')
constexpr int kBoxRows = 64;              // rows of a box of an operand stored across
constexpr int kLeastSplitBlocks = 4;      // k blocks a split is worth (100 x 1024 x 1024: 16 us, with 8 or 16 19)
constexpr int kLongestHalfSum = 256;      // k blocks (16,384 k's) of one running sum of a float16 product
constexpr int kLongestBfloatSum = 1024;   // and of a bfloat16 one (65,536 k's)
constexpr int kRunningFloats = kEpilogueWarps * 4 * 32 * 32;  // of one CTA: 128 rows by 256 columns
constexpr int kChunkBlocks = 4;           // k blocks (256 k's) of one running sum of a float32 product: 16 steps

// What a stage holds: one part of each operand, or a float32's three.
template <typename T>
struct Shape {
  static constexpr bool kPromote = sizeof(T) == 4;
  static constexpr int kParts = kPromote ? 3 : 1;
  static constexpr int kTileN = kPromote ? 128 : 256;
  static constexpr int kPartB = kTileN / 2 * kTileK * 2;  // bytes of one CTA's part of B at the widest tile
  static constexpr int kStageBytes = kParts * (kHalfBytes + kPartB);
  static constexpr int kStages = kPromote ? 2 : 6;
  static constexpr int kSmemBytes = kStages * kStageBytes + kEpilogueWarps * kSquareBytes + 1024;
};

struct Params {
  int64_t rows, cols;
  int tile_n, tiles_i, tiles_j, blocks, whole, splits, per_split;  // tiles from `whole` on are split
  int chunk;  // blocks of one running sum; for float32 its k blocks times the parts
  uint32_t instruction;
  int across_a, across_b;
  float* partial;  // [split tile][split][256][tile_n]
  float* running;  // sums of 16-bit products between chunks: [CTA][warp][chunk of columns][column][lane]
  ProductEpilogue e;
};

struct Item {
  int i, j, slot, first, last;  // slot: of its partial sums, or -1
};

// Tiles go in groups of eight columns, down the rows inside a group, so that the pairs working at one time share
// their operands in L2.
__device__ __forceinline__ void place_tile(int tile, int tiles_i, int tiles_j, int* i, int* j) {
  const int group = tile / (8 * tiles_i);
  const int width = min(8, tiles_j - group * 8);
  const int inside = tile - group * 8 * tiles_i;
  *i = inside / width;
  *j = group * 8 + inside % width;
}

__device__ __forceinline__ Item item_of(const Params& p, int index) {
  Item t = {0, 0, -1, 0, p.blocks};
  int tile = index;
  if (index >= p.whole) {
    t.slot = index - p.whole;
    tile = p.whole + t.slot / p.splits;
    t.first = t.slot % p.splits * p.per_split;
    t.last = min(t.first + p.per_split, p.blocks);
  }
  place_tile(tile, p.tiles_i, p.tiles_j, &t.i, &t.j);
  return t;
}

// K-major, 128-byte swizzle: eight-row atoms of 1024 bytes; a K = 16 step is 32 bytes along the row.
// Across (MN-major): 64 i's by 8 k's per atom, k groups 1024 bytes apart, the next 64 i's a box (64 k's) further.
__device__ __forceinline__ uint64_t operand_desc(uint32_t address, bool across) {
  uint64_t d = (address >> 4) & 0x3FFFu;
  d |= static_cast<uint64_t>(across ? (kBoxRows * 128) >> 4 : 1) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, int x, int y, int z, uint32_t barrier) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%2, %3, %4}], "
      "[%5];" ::"r"(dst),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(barrier)
      : "memory");
}

template <typename T>
__device__ __forceinline__ void load_bias(const ProductEpilogue& e, int64_t j, int64_t cols, float (&bias)[4]) {
#pragma unroll
  for (int k = 0; k < 4; ++k) bias[k] = e.bias && j + k < cols ? as_float(static_cast<const T*>(e.bias)[j + k]) : 0.f;
}

// Four columns of one row: the fp32 sums to their place.
template <typename T, int kActivation>
__device__ __forceinline__ void finish4(const ProductEpilogue& e, int64_t i, int64_t j, int64_t cols, const float (&bias)[4],
                                        bool aligned, float (&z)[4]) {
  const int n = static_cast<int>(min(static_cast<int64_t>(4), cols - j));
  const bool whole = aligned && n == 4;
#pragma unroll
  for (int k = 0; k < 4; ++k) z[k] += bias[k];
  if (e.pre) store4(static_cast<T*>(e.pre) + i * cols + j, n, whole, z);
  activate4<T, kActivation>(z);
  if (e.residual) {
    float r[4];
    load4(static_cast<const T*>(e.residual) + i * e.residual_stride + j, n, whole, r);
#pragma unroll
    for (int k = 0; k < 4; ++k) z[k] += r[k];
  }
  store4(static_cast<T*>(e.out) + i * e.out_stride + j, n, whole, z);
}

// Thirty-two entries of a row in memory, as they are: 16-byte aligned, `sectors`: to 32 bytes too, which then move whole.
template <typename T>
struct RowOf32 {
  static constexpr int kWords = static_cast<int>(sizeof(T)) * 8;
  uint32_t w[kWords];
  __device__ __forceinline__ void load(const T* p, bool sectors) {
    const char* from = reinterpret_cast<const char*>(p);
    if (sectors) {
#pragma unroll
      for (int k = 0; k < kWords; k += 8)
        asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(w[k]), "=r"(w[k + 1]), "=r"(w[k + 2]), "=r"(w[k + 3]), "=r"(w[k + 4]), "=r"(w[k + 5]),
                       "=r"(w[k + 6]), "=r"(w[k + 7])
                     : "l"(from + 4 * k));
    } else {
#pragma unroll
      for (int k = 0; k < kWords; k += 4) *reinterpret_cast<uint4*>(w + k) = *reinterpret_cast<const uint4*>(from + 4 * k);
    }
  }
  __device__ __forceinline__ void store(T* p, bool sectors) const {
    char* to = reinterpret_cast<char*>(p);
    if (sectors) {
#pragma unroll
      for (int k = 0; k < kWords; k += 8)
        asm volatile("st.global.v8.b32 [%8], {%0, %1, %2, %3, %4, %5, %6, %7};" ::"r"(w[k]), "r"(w[k + 1]), "r"(w[k + 2]),
                     "r"(w[k + 3]), "r"(w[k + 4]), "r"(w[k + 5]), "r"(w[k + 6]), "r"(w[k + 7]), "l"(to + 4 * k)
                     : "memory");
    } else {
#pragma unroll
      for (int k = 0; k < kWords; k += 4)
        *reinterpret_cast<uint4*>(to + 4 * k) = make_uint4(w[k], w[k + 1], w[k + 2], w[k + 3]);
    }
  }
  __device__ __forceinline__ void set(const float (&z)[32]) {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int k = 0; k < 32; ++k) w[k] = __float_as_uint(z[k]);
    } else {
#pragma unroll
      for (int k = 0; k < 16; ++k) pair_from(*reinterpret_cast<typename PairOf<T>::type*>(&w[k]), z[2 * k], z[2 * k + 1]);
    }
  }
  __device__ __forceinline__ void add_to(float (&z)[32]) const {
    if constexpr (sizeof(T) == 4) {
#pragma unroll
      for (int k = 0; k < 32; ++k) z[k] += __uint_as_float(w[k]);
    } else {
#pragma unroll
      for (int k = 0; k < 16; ++k) {
        const float2 f = pair_float(*reinterpret_cast<const typename PairOf<T>::type*>(&w[k]));
        z[2 * k] += f.x, z[2 * k + 1] += f.y;
      }
    }
  }
};

// Row i's 32 sums from column j on, all inside the matrix, to their place. A lane a row, without a detour through shared
// memory: every 32-byte sector moves whole all the same (8192 x 1024 x 4096 bfloat16 with GELU 70 us, through squares 82).
template <typename T, int kActivation>
__device__ __forceinline__ void finish_row32(const ProductEpilogue& e, const RowOf32<T>& residual, int64_t i, int64_t j,
                                             int64_t cols, bool inside, bool sectors, float (&z)[32]) {
  RowOf32<T> row;
  if (e.bias) {
    row.load(static_cast<const T*>(e.bias) + j, false);
    row.add_to(z);
  }
  if (e.pre) {
    row.set(z);
    if (inside) row.store(static_cast<T*>(e.pre) + i * cols + j, sectors);
  }
  activate4<T, kActivation>(z);
  if (e.residual) residual.add_to(z);
  row.set(z);
  if (inside) row.store(static_cast<T*>(e.out) + i * e.out_stride + j, sectors);
}

// The same for a square of 32 x 32 sums in shared memory (a row of eight four-column vectors, vector q of row r at
// q ^ (r & 7)) that the matrix's edge cuts or whose rows are not aligned: four rows at a time, four columns a lane.
template <typename T, int kActivation>
__device__ __forceinline__ void finish_square(const ProductEpilogue& e, const float4* square, int lane, int64_t i0, int64_t rows,
                                              int64_t j, int64_t cols, bool aligned) {
  const int q = lane & 7, first = lane >> 3;
  if (j >= cols) return;
  float bias[4];
  load_bias<T>(e, j, cols, bias);
  for (int r = 0; r < 8; ++r) {
    const int row = r * 4 + first;
    if (i0 + row >= rows) return;
    const float4 f = square[row * 8 + (q ^ (row & 7))];
    float z[4] = {f.x, f.y, f.z, f.w};
    finish4<T, kActivation>(e, i0 + row, j, cols, bias, aligned, z);
  }
}

template <typename T>
__device__ __forceinline__ bool epilogue_aligned(const ProductEpilogue& e, int64_t cols) {
  return aligned4<T>(e.out, e.out_stride) && (!e.residual || aligned4<T>(e.residual, e.residual_stride)) &&
         (!e.pre || aligned4<T>(e.pre, cols));
}

// kDeep: a 16-bit product of more than one running sum (a kernel of its own: the others' epilogues are 5% slower with it).
template <typename T, bool kDeep>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(kThreads, 1)
    product_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                   const __grid_constant__ Params p) {
  using S = Shape<T>;
  constexpr bool kPromote = S::kPromote;
  constexpr int kStages = S::kStages;
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t full[kStages], empty[kStages], acc_full[2], acc_empty[2];
  __shared__ uint32_t tmem_slot;
  unsigned char* smem = reinterpret_cast<unsigned char*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t{1023});
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const uint32_t rank = tc::cluster_ctarank();
  if (threadIdx.x == 0) {
    for (int s = 0; s < kStages; ++s) {
      tc::bar_init(&full[s], 1);
      tc::bar_init(&empty[s], 1);
    }
    for (int s = 0; s < 2; ++s) {
      tc::bar_init(&acc_full[s], 1);
      tc::bar_init(&acc_empty[s], 2 * kEpilogueWarps);
    }
    tc::bar_fence_init();
  }
  if (warp == kMmaWarp) {
    tc::tmem_alloc_pair(&tmem_slot, 512);
    tc::tmem_relinquish_pair();
  }
  tc::fence_before_sync();
  __syncthreads();
  tc::cluster_sync();  // barriers and tensor memory are ready in both CTAs
  tc::fence_after_sync();
  pdl_wait();
  pdl_trigger();
  const uint32_t tmem = tmem_slot;
  const int items = p.whole + (p.tiles_i * p.tiles_j - p.whole) * p.splits;
  const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int half_n = p.tile_n / 2;
  bool ok = true;

  if (warp == kLoadWarp) {
    if (lane == 0) {
      const uint32_t bytes = S::kParts * (kHalfBytes + half_n * kTileK * 2);
      int stage = 0;
      uint32_t lap = 0;
      for (int index = pair; index < items && ok; index += pairs) {
        const Item t = item_of(p, index);
        const int i0 = t.i * kTileM + static_cast<int>(rank) * 128;
        const int j0 = t.j * p.tile_n + static_cast<int>(rank) * half_n;
        for (int b = t.first; b < t.last; ++b) {
          if (lap > 0 && !(ok = tc::bar_wait(&empty[stage], (lap - 1) & 1u, 0x500))) break;
          const int k0 = b * kTileK;
          const uint32_t at = tc::smem_u32(smem + stage * S::kStageBytes);
          const uint32_t barrier = tc::map_shared(tc::smem_u32(&full[stage]), 0);
          if (rank == 0) tc::bar_expect_tx(&full[stage], 2 * bytes);
#pragma unroll
          for (int part = 0; part < S::kParts; ++part) {
            const uint32_t to_a = at + part * kHalfBytes, to_b = at + S::kParts * kHalfBytes + part * S::kPartB;
            if (p.across_a) {
              for (int c = 0; c < 2; ++c) load_box(to_a + c * kBoxRows * 128, &map_a, i0 + c * 64, k0, part, barrier);
            } else {
              load_box(to_a, &map_a, k0, i0, part, barrier);
            }
            if (p.across_b) {
              for (int c = 0; c < half_n / 64; ++c) load_box(to_b + c * kBoxRows * 128, &map_b, j0 + c * 64, k0, part, barrier);
            } else {
              load_box(to_b, &map_b, k0, j0, part, barrier);
            }
          }
          if (++stage == kStages) {
            stage = 0;
            ++lap;
          }
        }
      }
      // Every stage that was filled has been read before this CTA leaves.
      for (int s = 0; s < kStages && ok; ++s) {
        const uint32_t fills = lap + (s < stage ? 1 : 0);
        if (fills > 0) ok = tc::bar_wait(&empty[s], (fills - 1) & 1u, 0x501);
      }
    }
  } else if (warp == kMmaWarp) {
    if (lane == 0 && rank == 0) {
      const uint32_t step_a = p.across_a ? (16 * 128) >> 4 : 32 >> 4, step_b = p.across_b ? (16 * 128) >> 4 : 32 >> 4;
      int stage = 0, done = 0;  // running sums so far: they alternate between the accumulators
      uint32_t lap = 0;
      for (int index = pair; index < items && ok; index += pairs) {
        const Item t = item_of(p, index);
        for (int first = t.first; first < t.last && ok; first += p.chunk, ++done) {
          const int s = done & 1, last = min(first + p.chunk, t.last);
          if (done >= 2 && !(ok = tc::bar_wait_cluster(&acc_empty[s], ((done >> 1) - 1) & 1u, 0x502))) break;
          tc::fence_after_sync();
          const uint32_t accumulator = tmem + s * kAccumulatorColumns;
          for (int b = first; b < last; ++b) {
            if (!(ok = tc::bar_wait_cluster(&full[stage], lap & 1u, 0x503))) break;
            tc::fence_after_sync();
            const uint32_t at = tc::smem_u32(smem + stage * S::kStageBytes);
            // The product of part pa of A and part pb of B.
            auto multiply = [&](int pa, int pb, uint32_t into, bool fresh) {
              uint64_t da = operand_desc(at + pa * kHalfBytes, p.across_a);
              uint64_t db = operand_desc(at + S::kParts * kHalfBytes + pb * S::kPartB, p.across_b);
#pragma unroll
              for (int k = 0; k < kTileK / 16; ++k) {
                tc::mma_bf16_pair(into, da, db, p.instruction, !fresh || k > 0);
                da += step_a;
                db += step_b;
              }
            };
            if constexpr (kPromote) {
              const uint32_t small = accumulator + S::kTileN;
              multiply(2, 0, small, b == first);
              multiply(0, 2, small, false);
              multiply(1, 1, small, false);
              multiply(1, 0, small, false);
              multiply(0, 1, small, false);
            }
            multiply(0, 0, accumulator, b == first);
            tc::mma_commit_pair(&empty[stage]);
            if (++stage == kStages) {
              stage = 0;
              ++lap;
            }
          }
          if (ok) tc::mma_commit_pair(&acc_full[s]);
        }
      }
    }
  } else {
    float4* square = reinterpret_cast<float4*>(smem + kStages * S::kStageBytes + warp * kSquareBytes);
    const int quarter = warp & 3, half = warp >> 2;
    const bool aligned = epilogue_aligned<T>(p.e, p.cols);
    const int chunks = half_n / 32;  // 32-column chunks of this warp's half of the columns
    int done = 0;
    // The next running sum is complete; false where the wait ran out.
    auto wait_sum = [&] {
      ok = tc::bar_wait(&acc_full[done & 1], (done >> 1) & 1u, 0x504);
      ok = __all_sync(0xffffffffu, ok);
      tc::fence_after_sync();
      return ok;
    };
    auto read_sum = [&](int c, int column, float (&v)[32]) {
      tc::tmem_ld32(tmem + (static_cast<uint32_t>(quarter * 32) << 16) + (done & 1) * kAccumulatorColumns + column +
                        (half * chunks + c) * 32,
                    v);
    };
    // This warp has read all it needs of the running sum: its accumulator may be written again.
    auto release_sum = [&] {
      tc::fence_before_sync();
      __syncwarp();
      if (lane == 0) tc::bar_arrive_cluster(tc::map_shared(tc::smem_u32(&acc_empty[done & 1]), 0));
      ++done;
    };
    // Every plane's rows start on a multiple of `bytes`.
    auto rows_start_on = [&](int bytes) {
      auto on = [&](const void* base, int64_t stride) {
        return !base || ((reinterpret_cast<uintptr_t>(base) | (stride * sizeof(T))) & (bytes - 1)) == 0;
      };
      return on(p.e.out, p.e.out_stride) && on(p.e.residual, p.e.residual_stride) && on(p.e.pre, p.cols) && on(p.e.bias, 0);
    };
    const bool direct = rows_start_on(16), sectors = rows_start_on(32);
    for (int index = pair; index < items && ok; index += pairs) {
      const Item t = item_of(p, index);
      const int64_t i0 = static_cast<int64_t>(t.i) * kTileM + rank * 128 + quarter * 32, i = i0 + lane;
      auto first_column = [&](int c) { return static_cast<int64_t>(t.j) * p.tile_n + (half * chunks + c) * 32; };
      auto row_at_once = [&](int c) { return direct && t.slot < 0 && first_column(c) + 32 <= p.cols; };
      // A row's residual, under way before its sums are.
      auto residual_of = [&](int c) {
        RowOf32<T> r;
        if (p.e.residual && i < p.rows && row_at_once(c))
          r.load(static_cast<const T*>(p.e.residual) + i * p.e.residual_stride + first_column(c), sectors);
        return r;
      };
      // 32 rows by 32 columns of sums, a row a lane, to their place.
      auto store_sums = [&](int c, float (&v)[32], const RowOf32<T>& residual) {
        const int64_t j0 = first_column(c);
        if (i0 >= p.rows || j0 >= p.cols) return;
        if (row_at_once(c)) {
          with_activation(p.e.activation, [&](auto activation) {
            finish_row32<T, activation>(p.e, residual, i, j0, p.cols, i < p.rows, sectors, v);
          });
          return;
        }
#pragma unroll
        for (int q = 0; q < 8; ++q)
          square[lane * 8 + (q ^ (lane & 7))] = make_float4(v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]);
        __syncwarp();
        if (t.slot >= 0) {
          const int64_t row0 = static_cast<int64_t>(t.slot) * kTileM + rank * 128 + quarter * 32 + (lane >> 3);
          float* to = p.partial + row0 * p.tile_n + (half * chunks + c) * 32 + (lane & 7) * 4;
#pragma unroll
          for (int r = 0; r < 8; ++r) {
            const int row = r * 4 + (lane >> 3);
            *reinterpret_cast<float4*>(to + r * 4 * p.tile_n) = square[row * 8 + ((lane & 7) ^ (row & 7))];
          }
        } else {
          with_activation(p.e.activation, [&](auto activation) {
            finish_square<T, activation>(p.e, square, lane, i0, p.rows, j0 + (lane & 7) * 4, p.cols, aligned);
          });
        }
        __syncwarp();
      };
      if constexpr (kPromote) {
        float sums[2][32];
        for (int first = t.first; first < t.last && ok; first += p.chunk) {
          if (!wait_sum()) break;
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            float v[32];
            read_sum(c, S::kTileN, v);
#pragma unroll
            for (int k = 0; k < 32; ++k) {
              const float small = fabsf(v[k]) < INFINITY ? v[k] : 0.f;
              sums[c][k] = first == t.first ? small : sums[c][k] + small;
            }
            read_sum(c, 0, v);
#pragma unroll
            for (int k = 0; k < 32; ++k) sums[c][k] += v[k];
          }
          release_sum();
        }
        if (!ok) break;
#pragma unroll
        for (int c = 0; c < 2; ++c) store_sums(c, sums[c], residual_of(c));
      } else {
        // Between the chunks of a deep product its sums wait in a place of this lane's own.
        auto running = [&](int c) { return p.running + (((blockIdx.x * kEpilogueWarps + warp) * 4 + c) * 32) * 32 + lane; };
        auto add_running = [&](int c, float (&v)[32]) {
#pragma unroll
          for (int k = 0; k < 32; ++k) v[k] += __ldcg(running(c) + k * 32);
        };
        int first = t.first;
        if constexpr (kDeep) {
          for (; first + p.chunk < t.last && wait_sum(); first += p.chunk) {
            for (int c = 0; c < chunks; ++c) {
              float v[32];
              read_sum(c, 0, v);
              if (c == chunks - 1) release_sum();
              if (first > t.first) add_running(c, v);
#pragma unroll
              for (int k = 0; k < 32; ++k) __stcg(running(c) + k * 32, v[k]);
            }
          }
          if (!ok) break;
        }
        RowOf32<T> residual = residual_of(0);
        if (!wait_sum()) break;
        for (int c = 0; c < chunks; ++c) {
          float v[32];
          read_sum(c, 0, v);
          if (c == chunks - 1) release_sum();
          if (kDeep && first > t.first) add_running(c, v);
          store_sums(c, v, residual);
          if (c + 1 < chunks) residual = residual_of(c + 1);
        }
      }
    }
  }
  if (!ok) {
    // A wait ran out: give copies in flight time to land before the shared memory goes.
    const uint64_t start = tc::now_ns();
    while (tc::now_ns() - start < 10000000ull) {
    }
  }
  __syncwarp();
  tc::fence_before_sync();
  __syncthreads();
  tc::cluster_sync();
  tc::fence_after_sync();
  if (warp == kMmaWarp) tc::tmem_dealloc_pair(tmem, 512);
}

// The split tiles' sums, from `whole` on, to their place. splits is zero for a product of no depth.
template <typename T>
__global__ void __launch_bounds__(256) product_join_kernel(const float* partial, int whole, int splits, int tile_n, int tiles_i,
                                                           int tiles_j, int64_t rows, int64_t cols, const ProductEpilogue e) {
  pdl_wait();
  pdl_trigger();
  const bool aligned = epilogue_aligned<T>(e, cols);
  const int shift = tile_n == 256 ? 6 : 5;  // vectors of four columns in a tile's row
  // At most 37 split tiles, but every tile of a product of no depth.
  const int64_t total = static_cast<int64_t>(tiles_i * tiles_j - whole) * kTileM << shift;
  for (int64_t index = blockIdx.x * 256 + threadIdx.x; index < total; index += gridDim.x * 256) {
    const int tile = static_cast<int>((index >> shift) / kTileM), row = static_cast<int>((index >> shift) % kTileM);
    const int q = static_cast<int>(index) & ((1 << shift) - 1);
    int ti, tj;
    place_tile(whole + tile, tiles_i, tiles_j, &ti, &tj);
    const int64_t i = static_cast<int64_t>(ti) * kTileM + row, j = static_cast<int64_t>(tj) * tile_n + q * 4;
    if (i >= rows || j >= cols) continue;
    float z[4] = {0.f, 0.f, 0.f, 0.f};
    const float* from = partial + (static_cast<int64_t>(tile) * splits * kTileM + row) * tile_n + q * 4;
#pragma unroll 4
    for (int s = 0; s < splits; ++s) {
      const float4 f = *reinterpret_cast<const float4*>(from + static_cast<int64_t>(s) * kTileM * tile_n);
      z[0] += f.x, z[1] += f.y, z[2] += f.z, z[3] += f.w;
    }
    float bias[4];
    load_bias<T>(e, j, cols, bias);
    with_activation(e.activation, [&](auto activation) { finish4<T, activation>(e, i, j, cols, bias, aligned, z); });
  }
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
  static EncodeTiled found = [] {
    void* entry = nullptr;
    cudaDriverEntryPointQueryResult result;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &entry, 12000, cudaEnableDefault, &result) != cudaSuccess ||
        result != cudaDriverEntryPointSuccess)
      entry = nullptr;
    return reinterpret_cast<EncodeTiled>(entry);
  }();
  return found;
}

// The map of an operand: [parts][outer][inner] with boxes of 64 inner entries by `box` rows.
int make_map(CUtensorMap* map, const ProductOperand& o, int64_t inner, int64_t outer, int parts, int box, bool half) {
  EncodeTiled encode = encode_tiled();
  if (!encode) return set_error(CG_ERR_CUDA, "cuTensorMapEncodeTiled is not available");
  CG_REQUIRE((reinterpret_cast<uintptr_t>(o.base) & 15) == 0 && o.stride % 8 == 0 && o.part % 8 == 0,
             "run_product: operands must be aligned to 16 bytes");
  const cuuint64_t dims[3] = {static_cast<cuuint64_t>(inner), static_cast<cuuint64_t>(outer), static_cast<cuuint64_t>(parts)};
  const cuuint64_t row_bytes = static_cast<cuuint64_t>(std::max(o.stride, inner)) * 2;
  const cuuint64_t strides[2] = {(row_bytes + 15) & ~cuuint64_t{15},
                                 parts > 1 ? static_cast<cuuint64_t>(o.part) * 2 : (row_bytes + 15) & ~cuuint64_t{15}};
  const cuuint32_t boxes[3] = {64, static_cast<cuuint32_t>(box), 1}, steps[3] = {1, 1, 1};
  auto make = [&] {
    return encode(map, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 3, const_cast<void*>(o.base),
                  dims, strides, boxes, steps, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult rc = make();
  if (rc == CUDA_ERROR_INVALID_CONTEXT) {
    // The thread's first CUDA call (an autograd worker's, whose memory came from torch's cache): the driver call needs a
    // current context, which the runtime sets at its own calls only.
    int device = 0;
    if (cudaGetDevice(&device) == cudaSuccess && cudaSetDevice(device) == cudaSuccess) rc = make();
  }
  if (rc != CUDA_SUCCESS) return set_error(CG_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", static_cast<int>(rc));
  return CG_OK;
}

template <typename T>
int run_typed(const ProductOperand& a, const ProductOperand& b, int64_t rows, int64_t cols, int64_t depth, int dtype,
              const ProductEpilogue& e, float* partial, cudaStream_t stream) {
  const ProductPlan plan = plan_product(rows, cols, depth, dtype);
  if (plan.blocks > 0) {
    const bool half = dtype == CG_F16;
    const int parts = dtype == CG_F32 ? 3 : 1;
    CUtensorMap map_a, map_b;
    if (int rc = make_map(&map_a, a, a.across ? rows : depth, a.across ? depth : rows, parts, a.across ? kBoxRows : 128, half))
      return rc;
    if (int rc = make_map(&map_b, b, b.across ? cols : depth, b.across ? depth : cols, parts,
                          b.across ? kBoxRows : plan.tile_n / 2, half))
      return rc;
    Params p;
    p.rows = rows, p.cols = cols;
    p.tile_n = plan.tile_n, p.tiles_i = plan.tiles_i, p.tiles_j = plan.tiles_j;
    p.blocks = plan.blocks, p.whole = plan.whole, p.splits = plan.splits, p.per_split = plan.per_split, p.chunk = plan.chunk;
    p.across_a = a.across, p.across_b = b.across;
    // fp32 accumulator; A and B both float16 or both bfloat16; the transpose bits say "across".
    p.instruction = (1u << 4) | (half ? 0u : (1u << 7) | (1u << 10)) | (a.across ? 1u << 15 : 0u) | (b.across ? 1u << 16 : 0u) |
                    (static_cast<uint32_t>(plan.tile_n >> 3) << 17) | (static_cast<uint32_t>(kTileM >> 4) << 24);
    p.partial = partial;
    p.running = partial + plan.partial_bytes / 4;
    p.e = e;
    auto kernel = sizeof(T) == 2 && plan.blocks > plan.chunk ? product_kernel<T, sizeof(T) == 2> : product_kernel<T, false>;
    static bool configured[64] = {false};
    int device = 0;
    cudaGetDevice(&device);
    if (!configured[device & 63]) {
      for (auto each : {product_kernel<T, sizeof(T) == 2>, product_kernel<T, false>}) {
        cudaError_t err = cudaFuncSetAttribute(each, cudaFuncAttributeMaxDynamicSharedMemorySize, Shape<T>::kSmemBytes);
        if (err != cudaSuccess) return set_error(CG_ERR_CUDA, "product_kernel smem: %s", cudaGetErrorString(err));
      }
      configured[device & 63] = true;
    }
    const int items = plan.whole + (plan.tiles_i * plan.tiles_j - plan.whole) * plan.splits;
    const int pairs = std::min({items, sm_count() / 2, kPairs});
    if (int rc = launch_pdl("product_kernel", kernel, dim3(2 * pairs), dim3(kThreads), Shape<T>::kSmemBytes, stream,
                            map_a, map_b, p))
      return rc;
    if (plan.whole == plan.tiles_i * plan.tiles_j) return CG_OK;
  }
  const int64_t quads = static_cast<int64_t>(plan.tiles_i * plan.tiles_j - plan.whole) * kTileM * (plan.tile_n / 4);
  const int blocks = static_cast<int>(std::min<int64_t>((quads + 255) / 256, 16 * sm_count()));
  return launch_pdl("product_join_kernel", product_join_kernel<T>, dim3(blocks), dim3(256), 0, stream, partial, plan.whole,
                    plan.splits, plan.tile_n, plan.tiles_i, plan.tiles_j, rows, cols, e);
}

}  // namespace

ProductPlan plan_product(int64_t rows, int64_t cols, int64_t depth, int dtype) {
  ProductPlan plan = {};
  const int64_t pairs = kPairs;
  auto tiles_of = [&](int tile_n) { return (rows + kTileM - 1) / kTileM * ((cols + tile_n - 1) / tile_n); };
  // 16-bit operands: half tiles where they fill more than half the pairs in one round and whole ones would be split
  // (2048 x 1024 x 1024: 18 us against 25; 512 x 4096 x 4096: equal).
  plan.tile_n = dtype == CG_F32 || cols <= 128 || (tiles_of(128) <= pairs && 2 * tiles_of(128) > pairs) ? 128 : 256;
  plan.tiles_i = static_cast<int>((rows + kTileM - 1) / kTileM);
  plan.tiles_j = static_cast<int>((cols + plan.tile_n - 1) / plan.tile_n);
  const int64_t k_blocks = (depth + kTileK - 1) / kTileK, tiles = static_cast<int64_t>(plan.tiles_i) * plan.tiles_j;
  // A split is a whole number of units: kLeastSplitBlocks k blocks, or a float32 chunk.
  const int64_t unit = dtype == CG_F32 ? kChunkBlocks : kLeastSplitBlocks, units = (k_blocks + unit - 1) / unit;
  const int64_t last_round = tiles % pairs;  // tiles that would not fill a round of pairs
  int64_t splits = 1;
  if (last_round > 0 && 2 * last_round <= pairs) splits = std::max<int64_t>(1, std::min(pairs / last_round, units));
  const int64_t units_each = units > 0 ? (units + splits - 1) / splits : 1;
  splits = units > 0 ? (units + units_each - 1) / units_each : 0;
  plan.blocks = static_cast<int>(k_blocks);
  plan.per_split = static_cast<int>(units_each * unit);
  plan.splits = static_cast<int>(splits);
  plan.whole = static_cast<int>(splits == 1 ? tiles : splits == 0 ? 0 : tiles - last_round);
  plan.chunk = dtype == CG_F32 ? kChunkBlocks : dtype == CG_F16 ? kLongestHalfSum : kLongestBfloatSum;
  plan.partial_bytes = (tiles - plan.whole) * splits * kTileM * plan.tile_n * 4;
  plan.running_bytes = dtype != CG_F32 && plan.blocks > plan.chunk ? 2 * pairs * kRunningFloats * 4 : 0;
  return plan;
}

int run_product(const ProductOperand& a, const ProductOperand& b, int64_t rows, int64_t cols, int64_t depth, int dtype,
                const ProductEpilogue& e, void* partial, cudaStream_t stream) {
  if (rows == 0 || cols == 0) return CG_OK;
  auto* sums = static_cast<float*>(partial);
  if (dtype == CG_F32) return run_typed<float>(a, b, rows, cols, depth, dtype, e, sums, stream);
  if (dtype == CG_F16) return run_typed<__half>(a, b, rows, cols, depth, dtype, e, sums, stream);
  return run_typed<__nv_bfloat16>(a, b, rows, cols, depth, dtype, e, sums, stream);
}

}  // namespace cg
