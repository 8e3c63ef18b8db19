// Products of MXFP4 rows (mxfp4.cuh) with MXFP4 matrices:
//   llmopt_mxfp4_linear_{f16,bf16,f32}    [x codes, x scales, w codes, w scales, bias or any, out], {m, n, k, has bias}
//   llmopt_mxfp4_expert_rows_{f16,bf16}   [x codes, x scales, w codes, w scales, plan, score of every slot, out],
//                                         {slots, n, k, experts, paired}: rows sorted by expert (llmopt_route_plan)
//
// y[m, n] = sum over blocks b of 2^(sx + sw - 254) (x block . w block): the tensor cores take both operands as they are held, 64 elements
// of k at a time with two powers of two per row (tcgen05.mma kind::mxf4), so no weight is ever converted.  The weights are the M side
// (128 rows of a tile are the lanes of tensor memory, one output column each), the rows of x the N side: one token costs an N of 16,
// and a ragged tile of an expert costs its rows rounded up to 16.
//
// A CTA: warp 0 brings the codes of 256 elements of k of 128 weight rows and of the tile's rows of x by TMA (128-byte swizzle); warps 2 to 5
// bring their exponents, a word (128 elements) per thread and row, requested four stages ahead and laid down in the order that tcgen05.cp
// spreads over tensor memory; one thread of warp 1 issues copies and products; the other warps read the sums out.
//
// Every wait on an mbarrier is bounded; a wait that runs out raises the context's device error word, and the CTA lets its copies land,
// frees its tensor memory and returns.
#include <cuda.h>

#include "mxfp4.cuh"
#include "w4a16_tc_device.cuh"

namespace llmopt {
using namespace tc;

uint32_t* context_device_error(Context* ctx);

namespace {
using namespace mxfp4;

constexpr uint32_t kColumns = 128, kDepth = 256, kRowBytes = kDepth / 2;  // weight rows of a tile, elements of k of a stage
constexpr uint32_t kStageWords = kDepth / kWordValues, kAtom = 512;       // an atom: the words of 128 rows
constexpr uint32_t kScaleWarps = 4, kAhead = 4;

template <uint32_t NT>
struct Shape {
  static constexpr uint32_t kAtoms = (NT + 127) / 128;  // of x, per word
  static constexpr uint32_t kWeightBytes = kColumns * kRowBytes, kInputBytes = NT * kRowBytes;
  static constexpr uint32_t kScalesAt = kWeightBytes + kInputBytes;
  static constexpr uint32_t kStageBytes = kScalesAt + kStageWords * (1 + kAtoms) * kAtom;
  static constexpr uint32_t kStages = NT == 256 ? 4 : NT == 128 ? 6 : NT == 64 ? 4 : 5;
  static constexpr uint32_t kSums = NT == 256 ? 1 : 2;  // accumulators
  static constexpr uint32_t kScaleColumns = kStageWords * 4 * (1 + kAtoms);
  static constexpr uint32_t kUsedColumns = kSums * NT + 2 * kScaleColumns;
  static constexpr uint32_t kTmemColumns = kUsedColumns <= 64 ? 64 : kUsedColumns <= 128 ? 128 : kUsedColumns <= 256 ? 256 : 512;
  static constexpr uint32_t kBarriers = kStages * kStageBytes;
  static constexpr uint32_t kHolder = kBarriers + (3 * kStages + 4) * 8;
  static constexpr uint32_t kAbort = kHolder + 4;
  static constexpr uint32_t kSharedBytes = kAbort + 4 + 1024;  // slack: 1024-byte alignment of the tiles
  static constexpr uint32_t kEpilogueWarps = NT >= 128 ? 8 : 4;
  static constexpr uint32_t kThreads = (2 + kScaleWarps + kEpilogueWarps) * 32;
  static constexpr uint32_t kResident = NT >= 128 ? 1 : 2;
};

// kind::mxf4, e2m1 A and B (format 1), e8m0 scales, both K-major; `pair` picks the half of a scale word.
__device__ __forceinline__ uint32_t mxf4_instruction(uint32_t n, uint32_t pair) {
  return (pair << 5) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | (1u << 23) | ((kColumns >> 4) << 24) | (pair << 30);
}
__device__ __forceinline__ void mma_mxf4(uint32_t sums, uint64_t a, uint64_t b, uint32_t instruction, uint32_t a_scales, uint32_t b_scales,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
      ::"r"(sums), "l"(a), "l"(b), "r"(instruction), "r"(accumulate), "r"(a_scales), "r"(b_scales)
      : "memory");
}
// An atom (32 rows of 16 bytes, unswizzled, eight rows every 128 bytes) to four columns, the same in all four quarters of the lanes.
__device__ __forceinline__ void copy_atom(uint32_t columns, uint32_t shared_address) {
  const uint64_t descriptor = (uint64_t)((shared_address & 0x3ffffu) >> 4) | (uint64_t)(128 >> 4) << 16 | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(columns), "l"(descriptor) : "memory");
}

enum Store : uint32_t { kStoreHalf, kStoreBf16, kStoreFloat, kStorePairHalf, kStorePairBf16 };
template <Store S> struct Element { typedef float Type; };
template <> struct Element<kStoreHalf> { typedef __half Type; };
template <> struct Element<kStorePairHalf> { typedef __half Type; };
template <> struct Element<kStoreBf16> { typedef bf16 Type; };
template <> struct Element<kStorePairBf16> { typedef bf16 Type; };

__device__ __forceinline__ uint32_t packed(__half a, __half b) { return (uint32_t)__half_as_ushort(a) | (uint32_t)__half_as_ushort(b) << 16; }
__device__ __forceinline__ uint32_t packed(bf16 a, bf16 b) { return (uint32_t)__bfloat16_as_ushort(a) | (uint32_t)__bfloat16_as_ushort(b) << 16; }

// Sums of COUNT rows from `row` on, of the output column that is this lane's, on their way out; the whole warp takes part.  Sixteen-bit
// results go two columns at a time: neighbouring lanes exchange the sums of every other row.
template <Store S, int COUNT>
__device__ __forceinline__ void store_rows(const Problem& p, uint32_t row, uint32_t end, uint32_t column, const uint32_t (&raw)[COUNT]) {
  typedef typename Element<S>::Type T;
  const bool odd = threadIdx.x & 1u;
  if constexpr (S == kStoreFloat) {
    if (column >= p.n) return;
    const float bias = p.bias ? reinterpret_cast<const float*>(p.bias)[column] : 0.0f;
    float* out = reinterpret_cast<float*>(p.out) + (size_t)row * p.n + column;
#pragma unroll
    for (int i = 0; i < COUNT; ++i, out += p.n)
      if (row + i < end) *out = __uint_as_float(raw[i]) + bias;
  } else {
    const uint32_t even_column = column & ~1u;
    constexpr bool kPair = S == kStorePairHalf || S == kStorePairBf16;
    float bias[2] = {};
    if (!kPair && p.bias) {
      if (even_column < p.n) bias[0] = as_float(reinterpret_cast<const T*>(p.bias)[even_column]);
      if (even_column + 1u < p.n) bias[1] = as_float(reinterpret_cast<const T*>(p.bias)[even_column + 1u]);
    }
    const bool words = p.n % 2u == 0 && ((uintptr_t)p.out & 3u) == 0;
#pragma unroll
    for (int i = 0; i < COUNT; i += 2) {
      const uint32_t away = __shfl_xor_sync(0xffffffffu, odd ? raw[i] : raw[i + 1], 1);
      const float first = __uint_as_float(odd ? away : raw[i]), second = __uint_as_float(odd ? raw[i + 1] : away);
      const uint32_t at = row + i + (odd ? 1 : 0);
      if (at >= end || even_column >= p.n) continue;
      if constexpr (kPair) {
        const float scale = p.row_scale[at];
        reinterpret_cast<T*>(p.out)[(size_t)at * (p.n / 2u) + even_column / 2u] = from_float<T>(silu_f32(first * scale) * (second * scale));
      } else {
        T* out = reinterpret_cast<T*>(p.out) + (size_t)at * p.n + even_column;
        const T low = from_float<T>(first + bias[0]), high = from_float<T>(second + bias[1]);
        if (words) {
          *reinterpret_cast<uint32_t*>(out) = packed(low, high);
        } else {
          out[0] = low;
          if (even_column + 1u < p.n) out[1] = high;
        }
      }
    }
  }
}

// What a launch is shared out by.  splits > 1: a cluster of so many CTAs shares a tile's k, one tile per cluster.
struct Work {
  uint32_t row_tiles, column_tiles, splits, box_rows;
};

template <uint32_t NT, Store S>
__global__ void __launch_bounds__(Shape<NT>::kThreads, Shape<NT>::kResident)
product_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ Problem p,
               const Work work, uint32_t* error_word) {
  using Z = Shape<NT>;
  extern __shared__ unsigned char shared_raw[];
  grid_chain_prologue();
  const uint32_t base = (smem_u32(shared_raw) + 1023u) & ~1023u;
  unsigned char* base_pointer = shared_raw + (base - smem_u32(shared_raw));
  const uint32_t full = base + Z::kBarriers, scales_full = full + Z::kStages * 8, empty = scales_full + Z::kStages * 8;
  const uint32_t sums_full = empty + Z::kStages * 8, sums_empty = sums_full + 16;
  volatile uint32_t* holder = reinterpret_cast<volatile uint32_t*>(base_pointer + Z::kHolder);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(base_pointer + Z::kAbort);
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const uint32_t row_tiles = p.plan.tiles ? min(p.plan.tiles[0], work.row_tiles) : work.row_tiles;
  const uint32_t splits = work.splits, rank = blockIdx.x % splits, tiles = row_tiles * work.column_tiles;
  const uint32_t first_tile = blockIdx.x / splits, tile_step = gridDim.x / splits;
  // rows of x and first weight row of a tile; the column of its first weight row
  struct Place {
    uint32_t row, end, w_row, column;
  };
  auto place = [&](uint32_t tile) -> Place {
    const uint32_t row_tile = tile % row_tiles, column = tile / row_tiles * kColumns;
    if (!p.plan.tiles) return {row_tile * NT, min(p.m, (row_tile + 1u) * NT), column, column};
    const DenseTile rows = dense_tile(p.plan, row_tile);
    const uint32_t row = min(rows.first, p.m), end = max(row, min(min(rows.end, p.m), row + kExpertTile));  // whatever the plan says
    return {row, min(end, row + NT), min(rows.expert, p.plan.experts - 1u) * p.n + column, column};
  };
  const uint32_t k_stages = (p.k + kDepth - 1u) / kDepth;
  const uint32_t stage0 = k_stages * rank / splits, stage1 = k_stages * (rank + 1u) / splits;

  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < Z::kStages; ++s) {
      barrier_init(full + s * 8, 1);  // the copies' expect_tx arrival; completes by byte count
      barrier_init(scales_full + s * 8, kScaleWarps);
      barrier_init(empty + s * 8, 1);  // one tcgen05.commit
    }
    for (uint32_t s = 0; s < 2; ++s) {
      barrier_init(sums_full + s * 8, 1);  // one tcgen05.commit
      barrier_init(sums_empty + s * 8, Z::kEpilogueWarps);
    }
    *abort_flag = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + Z::kHolder), "r"(Z::kTmemColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = *holder;
  auto give_up = [&]() {
    *abort_flag = 1u;
    if (error_word) atomicExch(error_word, 1u);
  };

  if (warp == 0) {
    if (lane == 0) {
      uint32_t issued = 0;  // stages over all tiles of this CTA
      bool ok = true;
      for (uint32_t tile = first_tile; tile < tiles && ok; tile += tile_step) {
        const Place at = place(tile);
        const uint32_t boxes = (at.end - at.row + work.box_rows - 1u) / work.box_rows;
        for (uint32_t ks = stage0; ks < stage1; ++ks, ++issued) {
          const uint32_t s = issued % Z::kStages, stage = base + s * Z::kStageBytes;
          ok = !*abort_flag && barrier_wait(empty + s * 8, ((issued / Z::kStages) & 1u) ^ 1u);
          if (!ok) {
            give_up();
            break;
          }
          barrier_expect_tx(full + s * 8, Z::kWeightBytes + boxes * work.box_rows * kRowBytes);
          tma_load_2d(stage, &map_w, (int32_t)(ks * kRowBytes), (int32_t)at.w_row, full + s * 8);
          for (uint32_t box = 0; box < boxes; ++box)
            tma_load_2d(stage + Z::kWeightBytes + box * work.box_rows * kRowBytes, &map_x, (int32_t)(ks * kRowBytes),
                        (int32_t)(at.row + box * work.box_rows), full + s * 8);
        }
      }
      // on the way out after a failure the copies already started must land first
      if (!ok || *abort_flag)
        for (uint32_t i = issued > Z::kStages ? issued - Z::kStages : 0u; i < issued; ++i)
          barrier_wait(full + (i % Z::kStages) * 8, (i / Z::kStages) & 1u);
    }
  } else if (warp == 1) {
    if (lane == 0) {
      uint32_t consumed = 0, turn = 0;
      bool ok = true;
      for (uint32_t tile = first_tile; tile < tiles && ok; tile += tile_step, ++turn) {
        const Place at = place(tile);
        const uint32_t rows = p.plan.tiles ? max((at.end - at.row + 15u) / 16u * 16u, 16u) : NT;
        const uint32_t which = turn % Z::kSums, sums = tmem_base + which * NT;
        ok = !*abort_flag && barrier_wait(sums_empty + which * 8, ((turn / Z::kSums) & 1u) ^ 1u);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        for (uint32_t ks = stage0; ks < stage1 && ok; ++ks, ++consumed) {
          const uint32_t s = consumed % Z::kStages, stage = base + s * Z::kStageBytes;
          ok = !*abort_flag && barrier_wait(full + s * 8, (consumed / Z::kStages) & 1u) &&
               barrier_wait(scales_full + s * 8, (consumed / Z::kStages) & 1u);
          if (!ok) break;
          asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
          const uint32_t scales = tmem_base + Z::kSums * NT + (consumed & 1u) * Z::kScaleColumns, left = p.k - ks * kDepth;
#pragma unroll
          for (uint32_t g = 0; g < kStageWords; ++g) {
            if (g * kWordValues >= left) break;
            const uint32_t columns = scales + g * 4u * (1u + Z::kAtoms), atoms = stage + Z::kScalesAt + g * (1u + Z::kAtoms) * kAtom;
#pragma unroll
            for (uint32_t a = 0; a <= Z::kAtoms; ++a) copy_atom(columns + a * 4u, atoms + a * kAtom);
          }
#pragma unroll
          for (uint32_t j = 0; j < kDepth / 64; ++j) {
            if (j * 64u >= left) break;
            const uint32_t columns = scales + j / 2u * 4u * (1u + Z::kAtoms);
            mma_mxf4(sums, operand_descriptor(stage + j * 32u), operand_descriptor(stage + Z::kWeightBytes + j * 32u), mxf4_instruction(rows, j & 1u),
                     columns, columns + 4u, (ks > stage0 || j > 0) ? 1u : 0u);
          }
          mma_commit(empty + s * 8);
        }
        if (ok) mma_commit(sums_full + which * 8);
      }
      if (!ok) give_up();
    }
  } else if (warp < 2u + kScaleWarps) {
    // a thread per row: its words of a stage, of the weights and of x
    constexpr uint32_t kWords = kStageWords * (1 + Z::kAtoms);
    const uint32_t t = (warp - 2u) * 32u + lane, words = words_of(p.k), target = (t & 31u) * 16u + (t >> 5) * 4u;
    const uint32_t last_mask = p.k % kWordValues ? (1u << (p.k % kWordValues / kBlock * 8u)) - 1u : 0xffffffffu;  // bytes behind k: no exponents
    uint32_t held[kAhead][kWords];
    uint32_t ahead_tile = first_tile, ahead_stage = stage0, mine = 0, left_tiles = 0;
    for (uint32_t tile = first_tile; tile < tiles; tile += tile_step) ++left_tiles;
    const uint32_t all = left_tiles * (stage1 - stage0);
    Place ahead = {};
    if (all > 0) ahead = place(first_tile);
    auto fetch = [&](uint32_t (&into)[kWords]) {
      if (mine >= all) return;
      ++mine;
#pragma unroll
      for (uint32_t g = 0; g < kStageWords; ++g) {
        const uint32_t group = ahead_stage * kStageWords + g, mask = group + 1u == words ? last_mask : 0xffffffffu;
        const uint32_t w_row = ahead.w_row + t;
        into[g * (1 + Z::kAtoms)] = group < words && w_row < p.w_rows ? p.w_scales[(size_t)group * p.w_rows + w_row] & mask : 0u;
#pragma unroll
        for (uint32_t a = 0; a < Z::kAtoms; ++a) {
          const uint32_t row = ahead.row + a * 128u + t;
          into[g * (1 + Z::kAtoms) + 1 + a] = group < words && row < ahead.end ? p.x_scales[(size_t)group * p.m + row] & mask : 0u;
        }
      }
      if (++ahead_stage == stage1) {
        ahead_stage = stage0;
        ahead_tile += tile_step;
        if (mine < all) ahead = place(ahead_tile);
      }
    };
#pragma unroll
    for (uint32_t a = 0; a < kAhead; ++a) fetch(held[a]);
    bool ok = true;
    for (uint32_t first = 0; first < all && ok; first += kAhead) {
#pragma unroll
      for (uint32_t a = 0; a < kAhead; ++a) {
        const uint32_t i = first + a, s = i % Z::kStages;
        if (i >= all || !ok) break;
        ok = !*abort_flag && barrier_wait(empty + s * 8, ((i / Z::kStages) & 1u) ^ 1u);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        unsigned char* atoms = base_pointer + s * Z::kStageBytes + Z::kScalesAt + target;
#pragma unroll
        for (uint32_t w = 0; w < kWords; ++w) *reinterpret_cast<uint32_t*>(atoms + w * kAtom) = held[a][w];
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) barrier_arrive(scales_full + s * 8);
        fetch(held[a]);
      }
    }
    if (!ok) give_up();
  } else {
    const uint32_t worker = warp - 2u - kScaleWarps, quarter = warp & 3u, side = worker >> 2;  // lanes of tensor memory; share of the columns
    constexpr uint32_t kPiece = NT == 16 ? 16 : 32, kSides = Z::kEpilogueWarps / 4;
    uint32_t turn = 0;
    bool ok = true;
    for (uint32_t tile = first_tile; tile < tiles && ok; tile += tile_step, ++turn) {
      const uint32_t which = turn % Z::kSums;
      const Place at = place(tile);
      ok = !*abort_flag && barrier_wait(sums_full + which * 8, (turn / Z::kSums) & 1u);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {
        give_up();
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t address = tmem_base + which * NT + ((quarter * 32u) << 16);
#pragma unroll 1
      for (uint32_t piece = side; piece < NT / kPiece; piece += kSides) {
        const uint32_t row = at.row + piece * kPiece;
        if (row >= at.end) break;
        uint32_t raw[kPiece];
        if constexpr (kPiece == 16) tmem_load_16(address + piece * kPiece, raw);
        else tmem_load_32(address + piece * kPiece, raw);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        if (splits == 1u) {
          store_rows<S>(p, row, at.end, at.column + quarter * 32u + lane, raw);
        } else {
          // [row][column] of the partial sums, over the ring: every stage of it has been read
          float* partial = reinterpret_cast<float*>(base_pointer) + piece * kPiece * kColumns + quarter * 32u + lane;
#pragma unroll
          for (uint32_t i = 0; i < kPiece; ++i) partial[i * kColumns] = __uint_as_float(raw[i]);
        }
        __syncwarp();  // tcgen05.ld needs the whole warp
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) barrier_arrive(sums_empty + which * 8);
    }
  }

  __syncthreads();
  // before CTAs of a cluster wait for one another: a CTA that another grid's columns keep from its own must not be waited for with these held
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(Z::kTmemColumns) : "memory");
  }
  if (splits == 1u) return;
  cluster_sync();
  if (first_tile < tiles) {
    // each CTA joins a share of the rows, always the partial sums of rank 0 first; a warp has 32 columns of two rows at a time
    const Place at = place(first_tile);
    const float* partial = reinterpret_cast<const float*>(base_pointer);
    const uint32_t pairs = (at.end - at.row + 1u) / 2u;
    for (uint32_t item = rank * (Z::kThreads / 32u) + warp; item < pairs * 4u; item += splits * (Z::kThreads / 32u)) {
      const uint32_t row = item / 4u * 2u, column = item % 4u * 32u + lane;
      float sum[2] = {};
      for (uint32_t from = 0; from < splits; ++from)
        for (int i = 0; i < 2; ++i) sum[i] += cluster_load(partial + (row + i) * kColumns + column, from);
      const uint32_t raw[2] = {__float_as_uint(sum[0]), __float_as_uint(sum[1])};
      store_rows<S>(p, at.row + row, at.end, at.column + column, raw);
    }
  }
  cluster_sync();  // nobody leaves while its sums are read
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Codes [rows, k / 2] read in boxes of 128 bytes x `box_rows` with the 128-byte swizzle; absent bytes read zero.
bool make_map(CUtensorMap* map, const void* codes, uint64_t k, uint64_t rows, uint32_t box_rows) {
  static EncodeTiled encode = []() -> EncodeTiled {
    void* pointer = nullptr;
    cudaDriverEntryPointQueryResult result;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &pointer, cudaEnableDefault, &result) != cudaSuccess ||
        result != cudaDriverEntryPointSuccess)
      return nullptr;
    return reinterpret_cast<EncodeTiled>(pointer);
  }();
  if (encode == nullptr) return false;
  const cuuint64_t dims[2] = {k / 2, rows}, strides[1] = {k / 2};
  const cuuint32_t box[2] = {kRowBytes, box_rows}, element_strides[2] = {1, 1};
  return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), dims, strides, box, element_strides, CU_TENSOR_MAP_INTERLEAVE_NONE,
                CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

uint32_t most_plan_tiles(uint32_t slots, uint32_t experts) { return slots / kExpertTile + (slots < experts ? slots : experts); }

// What both products ask of their operands.
int check_operands(const KernelArgs& args, const Problem& p) {
  LLMOPT_REQUIRE(p.n > 0 && p.k > 0 && p.k % kBlock == 0, "needs n > 0 and k a positive multiple of 32");
  LLMOPT_REQUIRE(p.k <= (1u << 23) && p.m < (1u << 30), "too many rows, or k is too large");
  LLMOPT_REQUIRE(args.lengths[0] >= (size_t)p.m * (p.k / 2u) && args.lengths[1] >= (size_t)p.m * words_of(p.k) * 4 &&
                     args.lengths[2] >= (size_t)p.w_rows * (p.k / 2u) && args.lengths[3] >= (size_t)p.w_rows * words_of(p.k) * 4,
                 "buffer is too short");
  LLMOPT_REQUIRE((((uintptr_t)p.x | (uintptr_t)p.w) & 15u) == 0 && (((uintptr_t)p.x_scales | (uintptr_t)p.w_scales) & 3u) == 0,
                 "codes must be 16-byte aligned, scales 4-byte");
  return 0;
}

template <uint32_t NT, Store S>
int run(const KernelArgs& args, const Problem& p, uint32_t row_tiles) {
  using Z = Shape<NT>;
  const uint32_t sms = (uint32_t)context_sm_count(args.ctx), k_stages = (p.k + kDepth - 1u) / kDepth;
  Work work = {row_tiles, (p.n + kColumns - 1u) / kColumns, 1u, p.plan.tiles && NT > 32 ? 32u : NT};
  const size_t tiles = (size_t)work.row_tiles * work.column_tiles;
  LLMOPT_REQUIRE(tiles < (1u << 28), "too many tiles");
  // CTAs that share a tile's k while the tiles leave SMs without work
  if (NT <= 64)
    while (work.splits < 8u && tiles * work.splits * 2u <= (size_t)Z::kResident * sms && k_stages >= work.splits * 4u) work.splits *= 2u;
  CUtensorMap map_w, map_x;
  LLMOPT_REQUIRE(make_map(&map_w, p.w, p.k, p.w_rows, kColumns) && make_map(&map_x, p.x, p.k, p.m, work.box_rows), "tensor map was refused");
  auto kernel = product_kernel<NT, S>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Z::kSharedBytes) != cudaSuccess) {
    cudaGetLastError();
    return fail(args, "shared memory request was refused");
  }
  const uint32_t slots = Z::kResident * sms;
  if (work.splits == 1u)
    launch_kernel(args, kernel, dim3(tiles < slots ? (uint32_t)tiles : slots), dim3(Z::kThreads), Z::kSharedBytes, map_w, map_x, p, work,
                  context_device_error(args.ctx));
  else
    launch_cluster_kernel(args, kernel, dim3((uint32_t)tiles * work.splits), dim3(Z::kThreads), Z::kSharedBytes, work.splits, map_w, map_x, p, work,
                          context_device_error(args.ctx));
  return check_launch(args);
}

template <Store S>
int run_product(const KernelArgs& args, const Problem& p, uint32_t plan_tiles) {
  LLMOPT_REQUIRE(args.ctx != nullptr, "needs a context");
  auto tiles = [&](uint32_t rows) { return p.plan.tiles ? plan_tiles : (p.m + rows - 1u) / rows; };
  if (p.m <= 16u) return run<16, S>(args, p, tiles(16));
  if (p.m <= 32u) return run<32, S>(args, p, tiles(32));
  if (p.m <= 64u) return run<64, S>(args, p, tiles(64));
  if (p.m <= 128u || p.plan.tiles) return run<128, S>(args, p, tiles(128));
  return run<256, S>(args, p, tiles(256));
}

Problem operands(const KernelArgs& args) {
  Problem p = {};
  p.x = (const uint8_t*)args.buffers[0], p.x_scales = (const uint32_t*)args.buffers[1];
  p.w = (const uint8_t*)args.buffers[2], p.w_scales = (const uint32_t*)args.buffers[3];
  p.m = param_u32(args, 0), p.n = param_u32(args, 1), p.k = param_u32(args, 2);
  return p;
}

}  // namespace

template <typename T> constexpr Store kPlain = kStoreFloat;
template <> constexpr Store kPlain<__half> = kStoreHalf;
template <> constexpr Store kPlain<bf16> = kStoreBf16;
template <typename T> constexpr Store kPairs = kStorePairHalf;
template <> constexpr Store kPairs<bf16> = kStorePairBf16;

template <typename T>
int launch_mxfp4_linear(const KernelArgs& args) {
  LLMOPT_REQUIRE(args.buffer_count == 6 && args.param_bytes == 16, "expects 6 buffers and 16 parameter bytes");
  Problem p = operands(args);
  const bool has_bias = param_u32(args, 3) != 0;
  p.w_rows = p.n, p.bias = has_bias ? args.buffers[4] : nullptr, p.out = args.buffers[5];
  LLMOPT_REQUIRE(p.n < (1u << 31), "too many columns");
  if (const int status = check_operands(args, p)) return status;
  LLMOPT_REQUIRE((!has_bias || args.lengths[4] >= (size_t)p.n * sizeof(T)) && args.lengths[5] / sizeof(T) >= (size_t)p.m * p.n, "buffer is too short");
  LLMOPT_REQUIRE((((uintptr_t)p.bias | (uintptr_t)p.out) & (sizeof(T) - 1)) == 0, "bias and out must lie at multiples of their element");
  if (p.m == 0) return 0;
  return run_product<kPlain<T>>(args, p, 0);
}

template <typename T>
int launch_mxfp4_expert_rows(const KernelArgs& args) {
  LLMOPT_REQUIRE(args.buffer_count == 7 && args.param_bytes == 20, "expects 7 buffers and 20 parameter bytes");
  Problem p = operands(args);
  p.plan.tiles = (const uint32_t*)args.buffers[4], p.plan.experts = param_u32(args, 3);
  const bool paired = param_u32(args, 4) != 0;
  p.row_scale = (const float*)args.buffers[5], p.out = args.buffers[6];
  LLMOPT_REQUIRE(p.plan.experts > 0 && p.plan.experts <= 8192u && (!paired || p.n % 2u == 0), "needs experts, at most 8192, and whole pairs");
  LLMOPT_REQUIRE((size_t)p.plan.experts * p.n < (1u << 31), "too many rows");
  p.w_rows = p.plan.experts * p.n;
  if (const int status = check_operands(args, p)) return status;
  const uint32_t most = most_plan_tiles(p.m, p.plan.experts);
  LLMOPT_REQUIRE(args.lengths[4] >= 16 * (1 + (size_t)most) && (!paired || args.lengths[5] >= (size_t)p.m * 4) &&
                     args.lengths[6] / (paired ? sizeof(T) : 4) >= (size_t)p.m * (paired ? p.n / 2u : p.n),
                 "buffer is too short");
  LLMOPT_REQUIRE(((uintptr_t)args.buffers[4] & 15u) == 0 && (!paired || ((uintptr_t)p.row_scale & 3u) == 0) &&
                     ((uintptr_t)p.out & (paired ? sizeof(T) - 1 : 3u)) == 0,
                 "the plan must be 16-byte aligned, scores and out lie at multiples of their element");
  if (p.m == 0) return 0;
  if (!paired) return run_product<kStoreFloat>(args, p, most);
  return run_product<kPairs<T>>(args, p, most);
}

template int launch_mxfp4_linear<__half>(const KernelArgs&);
template int launch_mxfp4_linear<bf16>(const KernelArgs&);
template int launch_mxfp4_linear<float>(const KernelArgs&);
template int launch_mxfp4_expert_rows<__half>(const KernelArgs&);
template int launch_mxfp4_expert_rows<bf16>(const KernelArgs&);

}  // namespace llmopt
