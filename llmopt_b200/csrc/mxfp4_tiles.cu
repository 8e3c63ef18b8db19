// Products of many MXFP4 rows: persistent CTAs walk over tiles of 128 weight rows by 128 or 256 rows of x.
//
// A CTA: warp 0 brings the codes of 256 elements of k of 128 weight rows and of the tile's rows of x by TMA (128-byte swizzle); warps 2 to 5
// bring their exponents, a word (128 elements) per thread and row, requested four stages ahead and laid down in the order that tcgen05.cp
// spreads over tensor memory; one thread of warp 1 issues copies and products; the other warps read the sums out.
//
// Every wait on an mbarrier is bounded; a wait that runs out raises the context's device error word, and the CTA lets its copies land,
// frees its tensor memory and returns.
#include "mxfp4_tc.cuh"

namespace llmopt {
namespace {
using namespace mxfp4;

constexpr uint32_t kAhead = 4, kDepth = kBoxDepth, kStageWords = kDepth / kWordValues;  // of a stage

template <uint32_t NT>
struct Shape {
  static constexpr uint32_t kAtoms = (NT + 127) / 128;  // of x, per word
  static constexpr uint32_t kWeightBytes = kColumns * kRowBytes, kInputBytes = NT * kRowBytes;
  static constexpr uint32_t kScalesAt = kWeightBytes + kInputBytes;
  static constexpr uint32_t kStageBytes = kScalesAt + kStageWords * (1 + kAtoms) * kAtom;
  static constexpr uint32_t kStages = NT == 256 ? 4 : 6;
  static constexpr uint32_t kSums = NT == 256 ? 1 : 2;  // accumulators
  static constexpr uint32_t kScaleColumns = kStageWords * 4 * (1 + kAtoms);
  static constexpr uint32_t kUsedColumns = kSums * NT + 2 * kScaleColumns;
  static constexpr uint32_t kTmemColumns = 512;
  static_assert(kUsedColumns <= kTmemColumns, "tensor memory");
  static constexpr uint32_t kBarriers = kStages * kStageBytes;
  static constexpr uint32_t kHolder = kBarriers + (3 * kStages + 4) * 8;
  static constexpr uint32_t kAbort = kHolder + 4;
  static constexpr uint32_t kSharedBytes = kAbort + 4 + 1024;  // slack: 1024-byte alignment of the tiles
  static constexpr uint32_t kEpilogueWarps = 8;
  static constexpr uint32_t kThreads = (2 + kScaleWarps + kEpilogueWarps) * 32;
};

struct Work {
  uint32_t row_tiles, column_tiles, box_rows;
};

template <uint32_t NT, Store S>
__global__ void __launch_bounds__(Shape<NT>::kThreads, 1)
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
  const uint32_t warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31u;
  const uint32_t row_tiles = p.plan.tiles ? min(p.plan.tiles[0], work.row_tiles) : work.row_tiles;
  const uint32_t tiles = row_tiles * work.column_tiles, k_stages = (p.k + kDepth - 1u) / kDepth;
  auto place = [&](uint32_t tile) { return place_of<NT>(p, tile % row_tiles, 1u, tile / row_tiles * kColumns); };

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
  const uint32_t tmem_base = uniform(*holder);
  auto give_up = [&]() {
    *abort_flag = 1u;
    if (error_word) atomicExch(error_word, 1u);
  };

  if (warp == 0) {
    uint32_t issued = 0, s = 0, phase = 1;  // stages over all tiles of this CTA
    bool ok = true;
    for (uint32_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x) {
      const Place at = place(tile);
      const uint32_t boxes = (at.end - at.row + work.box_rows - 1u) / work.box_rows;
      for (uint32_t ks = 0; ks < k_stages; ++ks, ++issued) {
        const uint32_t stage = base + s * Z::kStageBytes;
        ok = !*abort_flag && warp_wait(empty + s * 8, phase);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) {
          give_up();
          break;
        }
        if (elect_one()) {
          barrier_expect_tx(full + s * 8, Z::kWeightBytes + boxes * work.box_rows * kRowBytes);
          tma_load_2d(stage, &map_w, (int32_t)(ks * kRowBytes), (int32_t)at.w_row, full + s * 8);
          for (uint32_t box = 0; box < boxes; ++box)
            tma_load_2d(stage + Z::kWeightBytes + box * work.box_rows * kRowBytes, &map_x, (int32_t)(ks * kRowBytes),
                        (int32_t)(at.row + box * work.box_rows), full + s * 8);
        }
        __syncwarp();
        if (++s == Z::kStages) s = 0, phase ^= 1u;
      }
    }
    // on the way out after a failure the copies already started must land first
    if (!ok || *abort_flag)
      for (uint32_t i = issued > Z::kStages ? issued - Z::kStages : 0u; i < issued; ++i)
        barrier_wait(full + (i % Z::kStages) * 8, (i / Z::kStages) & 1u);
    __syncwarp();
  } else if (warp == 1) {
    uint32_t s = 0, phase = 0, half = 0, turn = 0;
    bool ok = true;
    for (uint32_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x, ++turn) {
      uint32_t rows = NT;
      if (p.plan.tiles) {
        const Place at = place(tile);
        rows = uniform(max((at.end - at.row + 15u) / 16u * 16u, 16u));
      }
      const uint32_t low = mxf4_instruction(rows, 0u), high = mxf4_instruction(rows, 1u);
      const uint32_t which = turn % Z::kSums, sums = tmem_base + which * NT;
      ok = !*abort_flag && warp_wait(sums_empty + which * 8, ((turn / Z::kSums) & 1u) ^ 1u);
      ok = __all_sync(0xffffffffu, ok);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      for (uint32_t ks = 0; ks < k_stages && ok; ++ks) {
        const uint32_t stage = base + s * Z::kStageBytes;
        ok = !*abort_flag && warp_wait(full + s * 8, phase) && warp_wait(scales_full + s * 8, phase);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t scales = tmem_base + Z::kSums * NT + half * Z::kScaleColumns, left = p.k - ks * kDepth;
        const uint64_t a = operand_descriptor(stage), b = operand_descriptor(stage + Z::kWeightBytes);
        if (elect_one()) {
#pragma unroll
          for (uint32_t g = 0; g < kStageWords; ++g) {
            if (g * kWordValues >= left) break;
            const uint32_t columns = scales + g * 4u * (1u + Z::kAtoms), atoms = stage + Z::kScalesAt + g * (1u + Z::kAtoms) * kAtom;
#pragma unroll
            for (uint32_t atom = 0; atom <= Z::kAtoms; ++atom) copy_atom(columns + atom * 4u, atoms + atom * kAtom);
          }
#pragma unroll
          for (uint32_t j = 0; j < kDepth / 64; ++j) {
            if (j * 64u >= left) break;
            const uint32_t columns = scales + j / 2u * 4u * (1u + Z::kAtoms);
            mma_mxf4(sums, a + j * 2u, b + j * 2u, j & 1u ? high : low, columns, columns + 4u, (ks > 0 || j > 0) ? 1u : 0u);
          }
          mma_commit(empty + s * 8);
          if (ks + 1u == k_stages) mma_commit(sums_full + which * 8);
        }
        __syncwarp();
        half ^= 1u;
        if (++s == Z::kStages) s = 0, phase ^= 1u;
      }
    }
    if (!ok) give_up();
  } else if (warp < 2u + kScaleWarps) {
    // a thread per row: its words of a stage, of the weights and of x
    constexpr uint32_t kWords = kStageWords * (1 + Z::kAtoms);
    const uint32_t t = (warp - 2u) * 32u + lane, words = words_of(p.k), target = (t & 31u) * 16u + (t >> 5) * 4u, last_mask = last_word_mask(p.k);
      uint32_t held[kAhead][kWords];
    uint32_t ahead_tile = blockIdx.x, ahead_stage = 0, mine = 0, left_tiles = 0;
    for (uint32_t tile = blockIdx.x; tile < tiles; tile += gridDim.x) ++left_tiles;
    const uint32_t all = left_tiles * k_stages;
    Place ahead = {};
    if (all > 0) ahead = place(blockIdx.x);
    auto fetch = [&](uint32_t (&into)[kWords]) {
      if (mine >= all) return;
      ++mine;
#pragma unroll
      for (uint32_t g = 0; g < kStageWords; ++g) {
        const uint32_t group = ahead_stage * kStageWords + g, w_row = ahead.w_row + t;
        uint32_t& of_w = into[g * (1 + Z::kAtoms)];
        of_w = 0u;
        if (group < words && w_row < p.w_rows) of_w = p.w_scales[(size_t)group * p.w_rows + w_row];
#pragma unroll
        for (uint32_t a = 0; a < Z::kAtoms; ++a) {
          const uint32_t row = ahead.row + a * 128u + t;
          uint32_t& of_x = into[g * (1 + Z::kAtoms) + 1 + a];
          of_x = 0u;
          if (group < words && row < ahead.end) of_x = p.x_scales[(size_t)group * p.m + row];
        }
      }
      if (++ahead_stage == k_stages) {
        ahead_stage = 0;
        ahead_tile += gridDim.x;
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
        for (uint32_t w = 0; w < kWords; ++w)
          *reinterpret_cast<uint32_t*>(atoms + w * kAtom) =
              held[a][w] & (i % k_stages * kStageWords + w / (1 + Z::kAtoms) + 1u == words ? last_mask : 0xffffffffu);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) barrier_arrive(scales_full + s * 8);
        fetch(held[a]);
      }
    }
    if (!ok) give_up();
  } else {
    const uint32_t worker = warp - 2u - kScaleWarps, quarter = warp & 3u, side = worker >> 2;  // lanes of tensor memory; share of the columns
    constexpr uint32_t kPiece = 32, kSides = Z::kEpilogueWarps / 4;
    uint32_t turn = 0;
    bool ok = true;
    for (uint32_t tile = blockIdx.x; tile < tiles && ok; tile += gridDim.x, ++turn) {
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
        tmem_load_32(address + piece * kPiece, raw);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        store_rows<S>(p, row, at.end, at.column + quarter * 32u + lane, raw);
        __syncwarp();  // tcgen05.ld needs the whole warp
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) barrier_arrive(sums_empty + which * 8);
    }
  }

  __syncthreads();
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(Z::kTmemColumns) : "memory");
  }
}

template <uint32_t NT, Store S>
int run(const KernelArgs& args, const Problem& p, uint32_t row_tiles) {
  using Z = Shape<NT>;
  const uint32_t sms = (uint32_t)context_sm_count(args.ctx);
  const Work work = {row_tiles, (p.n + kColumns - 1u) / kColumns, p.plan.tiles ? 32u : NT};
  const size_t tiles = (size_t)work.row_tiles * work.column_tiles;
  LLMOPT_REQUIRE(tiles < (1u << 28), "too many tiles");
  CUtensorMap map_w, map_x;
  LLMOPT_REQUIRE(make_map(&map_w, p.w, p.k, p.w_rows, kColumns) && make_map(&map_x, p.x, p.k, p.m, work.box_rows), "tensor map was refused");
  auto kernel = product_kernel<NT, S>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Z::kSharedBytes) != cudaSuccess) {
    cudaGetLastError();
    return fail(args, "shared memory request was refused");
  }
  launch_kernel(args, kernel, dim3(tiles < sms ? (uint32_t)tiles : sms), dim3(Z::kThreads), Z::kSharedBytes, map_w, map_x, p, work,
                context_device_error(args.ctx));
  return check_launch(args);
}

}  // namespace

namespace mxfp4 {

template <Store S>
int run_tiles(const KernelArgs& args, const Problem& p, uint32_t plan_tiles) {
  auto tiles = [&](uint32_t rows) { return p.plan.tiles ? plan_tiles : (p.m + rows - 1u) / rows; };
  if (p.m <= 128u || p.plan.tiles) return run<128, S>(args, p, tiles(128));
  return run<256, S>(args, p, tiles(256));
}

template int run_tiles<kStoreHalf>(const KernelArgs&, const Problem&, uint32_t);
template int run_tiles<kStoreBf16>(const KernelArgs&, const Problem&, uint32_t);
template int run_tiles<kStoreFloat>(const KernelArgs&, const Problem&, uint32_t);
template int run_tiles<kStorePairHalf>(const KernelArgs&, const Problem&, uint32_t);
template int run_tiles<kStorePairBf16>(const KernelArgs&, const Problem&, uint32_t);

}  // namespace mxfp4
}  // namespace llmopt
