// Products of many MXFP4 rows: pairs of CTAs walk over tiles of 256 weight rows by up to 224 rows of x (256 where no pair has a second tile).
//
// Why pairs: a tile's operands come from L2, and tcgen05.mma with cta_group::2 multiplies 256 weight rows, half of them in either
// CTA's shared memory, with rows of x of which either CTA holds half as well: per 256 elements of k 30 KB a CTA where one by itself needs
// 44 KB.  In each CTA warp 0 brings the codes of 512 elements of k of its halves by TMA (128-byte swizzle); warps 2 to 5 bring
// exponents, a warp per word of a stage, those of the CTA's 128 weight rows and of all rows of x, requested three stages ahead and laid
// down in the order that tcgen05.cp spreads over tensor memory.  One lane of warp 1 of the first CTA issues copies and products
// for both, and its barriers count both CTAs' copies and exponents (the second one's when its warp 1 says so).  Eight more warps read a
// tile's sums out, each a quarter of the lanes (output columns), while the next tile's are formed in other columns of tensor memory; results
// of 16 bits change places in shared memory and leave as boxes of 32 rows by TMA, ragged ones by vector stores.
//
// What bounds it: a stage costs the tensor cores 4 cycles per row of x and 200 to 500 for copies of exponents (12 of them, in the same
// pipe) and the handover of the ring.  Stages of 512 rather than 256 elements halve the handovers: 4096 x 4096 x 14336 108 -> 99 us, 2048 x
// 4096 x 4096 24.9 -> 21.3, 512 x 14336 x 4096 25.7 -> 20.9.  (These three are 92 to 96, 19.7 and 19.8 now.)  The large
// product runs at up to 5.2 PFLOP/s (k 8192: 5.8) and takes 82 to 87 us where all codes are zero: what is left between the two is power,
// 1000 W, and repeated for a second it takes 110 at 1.6 to 1.7 GHz.  Rows sorted by expert have tiles of 128, which spend up to half a
// stage outside the products; many are joined to tiles of up to 224: 4096 of 16 experts through 4096 x 7168 85 -> 73 us, 3.3 PFLOP/s and
// 3.1 TB/s, down through 3584 x 4096 with fp32 sums 46.  Small products are bound by their ends: 128 rows through 4096 x 14336 11.4 us, 777 x
// 2048 x 7168 10.5; copies and exponents start without waiting for tensor memory (0.5 us).
//
// Every wait on an mbarrier is bounded; a wait that runs out raises the launch's error word, and the CTA lets its copies and
// products end, frees its tensor memory and returns; a pair gives up together.
#include "mxfp4_tc.cuh"

namespace llmopt {
namespace {
using namespace mxfp4;

constexpr uint32_t kDepth = 512, kBoxes = kDepth / kBoxDepth, kStageWords = kDepth / kWordValues;  // of a stage
constexpr uint32_t kAhead = 3;  // stages of exponents that are under way in registers
static_assert(kStageWords == kScaleWarps, "a warp per word of a stage");
constexpr uint32_t kMostRows = 224, kLoneRows = 256, kInputAtoms = 2;  // of a tile; of the only one of every pair
constexpr uint32_t kEpilogueWarps = 8, kThreads = (2 + kScaleWarps + kEpilogueWarps) * 32;
constexpr uint32_t kBoxBytes = kColumns * kRowBytes;  // of weights
// A stage: codes of weights, exponents of weights and of x, codes of x, of as many rows as the launch's tiles have, which says how many
// stages there are.
constexpr uint32_t kScalesAt = kBoxes * kBoxBytes, kInputScalesAt = kScalesAt + kStageWords * kAtom;
constexpr uint32_t kInputAt = kInputScalesAt + kStageWords * kInputAtoms * kAtom;
constexpr uint32_t kMostStages = 4, kSums = 2;  // sums of two tiles in tensor memory
constexpr uint32_t kWordColumns = 4 * (1 + kInputAtoms), kScaleColumns = kStageWords * kWordColumns, kTmemColumns = 512;
static_assert(kSums * kMostRows + kScaleColumns <= kTmemColumns && kInputAt % 1024 == 0, "tensor memory, alignment of tiles");
// In front of the ring: barriers, tensor memory's address, abort flag, and the staging of the warps that store, which lies over the ring where
// no pair has a second tile that would be on its way into it.
constexpr uint32_t kHolder = (5 * kMostStages + 2 * kSums + 1) * 8, kAbort = kHolder + 4, kFront = 1024, kMostShared = 227 * 1024;
constexpr uint32_t kStaging = kEpilogueWarps * kStagingBytes;
// Joined tiles of a plan: their number, then first row and expert << 16 | rows of each, in front of the staging.
constexpr uint32_t kCount = kAbort + 4, kMostJoined = 512, kList = kMostJoined * 8;
constexpr uint32_t kIssued = kCount + 4;  // stages that either CTA has asked for, where somebody gave up
static_assert(kIssued + 8 <= kFront && kStaging % 1024 == 0 && kList % 1024 == 0, "alignment of tiles");
static_assert(kStagingBytes >= 32 * 64, "a box of results");

struct Work {
  uint32_t row_tiles, column_tiles;    // of x, of pairs of weight tiles
  uint32_t rows;                       // most of a tile; either CTA copies half of them, whatever there are
  uint32_t stages, stage_bytes, ring;  // of shared memory; where the ring begins
  uint32_t boxes;                      // results leave in boxes
  uint32_t list;                       // bytes of the list of joined tiles; 0: the plan's
  uint32_t wait_limit;                 // how often a wait looks; 0: all give up at once
};

// A word or barrier of either CTA, from either; the first one's barriers.
__device__ __forceinline__ uint32_t pair_address(uint32_t local, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
  return remote;
}
__device__ __forceinline__ uint32_t first_address(uint32_t local) { return pair_address(local, 0u); }
__device__ __forceinline__ void pair_store(uint32_t local, uint32_t rank, uint32_t value) {
  asm volatile("st.relaxed.cluster.shared::cluster.b32 [%0], %1;" ::"r"(pair_address(local, rank)), "r"(value) : "memory");
}
// The two CTAs hand each other shared memory (exponents laid down, stages read) and tensor memory (sums read out) by barriers whose arrivals and
// waits have to be of the cluster's scope: one that names none is the CTA's, and orders nothing between threads of two CTAs.  They are relaxed,
// with fences restricted to shared memory where that changes hands and tcgen05.fence for tensor memory: release and acquire of
// everything wait for global memory too.  The warps that bring exponents take part in none of it: even a restricted fence waits for the loads that
// they have under way, so warp 0 tells them when a stage is theirs, and the second CTA's warp 1 tells the first what they have laid down.
// us, cold, of 777 x 2048 x 7168, 4096 x 4096 x 14336 and 32 x 4096 x 128256 (fp32): 10.5, 92 to 96, 48 to 51; with fences in those warps 10.8, 98, 55; with
// release and acquire of everything 15.4, 156, 87.
__device__ __forceinline__ void shared_release() { asm volatile("fence.release.sync_restrict::shared::cta.cluster;" ::: "memory"); }
__device__ __forceinline__ void first_arrive(uint32_t first) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(first) : "memory");
}
__device__ __forceinline__ bool pair_wait(uint32_t bar, uint32_t parity, uint32_t limit = kWaitLimit) {
  uint32_t done = 0, looks = 0;
  do {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.relaxed.cluster.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
  } while (!done && ++looks < limit);
  asm volatile("fence.acquire.sync_restrict::shared::cluster.cluster;" ::: "memory");
  return __all_sync(0xffffffffu, done != 0u);
}
// Bytes that the barrier waits for and nobody will send.
__device__ __forceinline__ void barrier_forgo(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.complete_tx.relaxed.cta.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// A tile to this CTA's shared memory whose bytes the barrier of the first one counts.
__device__ __forceinline__ void pair_load(uint32_t destination, const CUtensorMap* map, int32_t x, int32_t y, uint32_t first) {
  asm volatile(
      "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
      ::"r"(destination), "l"(map), "r"(first), "r"(x), "r"(y)
      : "memory");
}
__device__ __forceinline__ void pair_mma(uint32_t sums, uint64_t a, uint64_t b, uint32_t instruction, uint32_t a_scales, uint32_t b_scales,
                                         uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}"
      ::"r"(sums), "l"(a), "l"(b), "r"(instruction), "r"(accumulate), "r"(a_scales), "r"(b_scales)
      : "memory");
}
__device__ __forceinline__ void pair_copy_atom(uint32_t columns, uint32_t shared_address) {
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(columns), "l"(atom_descriptor(shared_address)) : "memory");
}
// arrives on both CTAs' barriers
__device__ __forceinline__ void pair_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3)
               : "memory");
}

// A box of shared memory to the rows and columns of the results it belongs to.
__device__ __forceinline__ void store_box(const CUtensorMap* map, int32_t x, int32_t y, uint32_t source) {
  asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%1, %2}], [%3];" ::"l"(map), "r"(x), "r"(y), "r"(source) : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
// Until this thread's boxes have been read.
__device__ __forceinline__ void await_box() { asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory"); }

// The plan's tiles of an expert lie behind one another and have up to 128 rows: 32 of the plan's at a time, runs of one expert's are divided
// evenly into as few as have no more than `rows`.  A warp's; no more tiles come out than went in.
__device__ __forceinline__ void join_tiles(const Problem& p, uint32_t plan_tiles, uint32_t rows, volatile uint32_t* number, uint2* list) {
  const uint32_t lane = threadIdx.x & 31u;
  uint32_t made = 0, count = plan_tiles;
  for (uint32_t base = 0; base < count; base += 32u) {
    Place at = {};
    if (base + lane < plan_tiles) at = place_of(p, base + lane, kExpertTile, 0u);
    count = min(p.plan.tiles[0], plan_tiles);
    const bool present = base + lane < count;
    const uint32_t of_before = __shfl_up_sync(0xffffffffu, at.w_row, 1), end_before = __shfl_up_sync(0xffffffffu, at.end, 1);
    const bool begins = lane == 0 || of_before != at.w_row || end_before != at.row;
    // runs end ahead of the next one, or of what is not there
    const uint32_t ends = __ballot_sync(0xffffffffu, begins || !present) & (0xfffffffeu << lane);
    const uint32_t end = __shfl_sync(0xffffffffu, at.end, ends ? __ffs(ends) - 2 : 31);
    const uint32_t tiles = present && begins ? (end - at.row + rows - 1u) / rows : 0u;
    uint32_t before = tiles;
#pragma unroll
    for (uint32_t offset = 1; offset < 32u; offset <<= 1) {
      const uint32_t other = __shfl_up_sync(0xffffffffu, before, offset);
      if (lane >= offset) before += other;
    }
    uint2* const target = list + made + before - tiles;
    made += __shfl_sync(0xffffffffu, before, 31);
    if (tiles > 0) {
      const uint32_t each = ((end - at.row + tiles - 1u) / tiles + 31u) / 32u * 32u, expert = at.w_row / p.n;
      for (uint32_t t = 0, row = at.row; t < tiles; ++t, row += each) target[t] = make_uint2(row, expert << 16 | min(each, end - row));
    }
  }
  if (lane == 0) *number = made;
}

template <Store S>
__global__ void __launch_bounds__(kThreads, 1)
tiles_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ CUtensorMap map_out,
             const __grid_constant__ Problem p, const Work work, uint32_t* error_word) {
  extern __shared__ unsigned char shared_raw[];
  grid_launch_dependents();
  const uint32_t base = (smem_u32(shared_raw) + 1023u) & ~1023u;
  unsigned char* base_pointer = shared_raw + (base - smem_u32(shared_raw));
  const uint32_t full = base, scales_full = full + kMostStages * 8, empty = scales_full + kMostStages * 8;
  const uint32_t sums_full = empty + kMostStages * 8, sums_empty = sums_full + kSums * 8, drained = sums_empty + kSums * 8;
  const uint32_t laid = drained + 8, vacant = laid + kMostStages * 8;
  volatile uint32_t* holder = reinterpret_cast<volatile uint32_t*>(base_pointer + kHolder);
  volatile uint32_t* abort_flag = reinterpret_cast<volatile uint32_t*>(base_pointer + kAbort);
  const uint32_t warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31u, rank = blockIdx.x & 1u, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < work.stages; ++s) {
      barrier_init(full + s * 8, 1);  // of the first CTA, for both: its expect_tx arrival; completes by byte count
      barrier_init(scales_full + s * 8, kScaleWarps + 1);  // the same: its own warps, and warp 1 of the second CTA for that one's
      barrier_init(laid + s * 8, kScaleWarps);  // of the second CTA
      barrier_init(vacant + s * 8, 1);          // warp 0's word to the warps that bring exponents: the stage is empty
      barrier_init(empty + s * 8, 1);  // one tcgen05.commit
    }
    for (uint32_t s = 0; s < kSums; ++s) {
      barrier_init(sums_full + s * 8, 1);  // one tcgen05.commit
      barrier_init(sums_empty + s * 8, 2 * kEpilogueWarps);
    }
    barrier_init(drained, 1);
    *abort_flag = work.wait_limit == 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  __syncwarp();
  cluster_arrive();
  grid_dependency_wait();  // ahead of tensor memory, which CTAs of the kernel before may still have to ask for
  // Copies and exponents start without tensor memory, which warp 1 and the warps that store wait for.
  uint32_t tmem_base = 0;
  if (warp == 1u || warp >= 2u + kScaleWarps) {
    if (warp == 1u) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + kHolder), "r"(kTmemColumns) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    asm volatile("bar.sync 1, %0;" ::"n"((1 + kEpilogueWarps) * 32) : "memory");
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    tmem_base = uniform(*holder);
  }
  cluster_wait();  // either CTA's barriers are there for the other
  uint2* const list = reinterpret_cast<uint2*>(base_pointer + kFront);
  uint32_t row_tiles = work.row_tiles;
  if (work.list > 0) {
    volatile uint32_t* joined = reinterpret_cast<volatile uint32_t*>(base_pointer + kCount);
    if (warp == 2u) join_tiles(p, work.row_tiles, work.rows, joined, list);
    __syncthreads();
    row_tiles = *joined;
  } else if (p.plan.tiles) {
    row_tiles = min(p.plan.tiles[0], work.row_tiles);
  }
  const uint32_t tiles = row_tiles * work.column_tiles, k_stages = (p.k + kDepth - 1u) / kDepth;
  // tiles of the same weights follow one another
  auto place = [&](uint32_t tile) -> Place {
    const uint32_t column = tile / row_tiles * 2u * kColumns;
    if (work.list == 0) return place_of(p, tile % row_tiles, work.rows, column);
    const uint2 at = list[tile % row_tiles];
    return {at.x, at.x + (at.y & 0xffffu), (at.y >> 16) * p.n + column, column};
  };
  const uint32_t half_bytes = work.rows / 2u * kRowBytes;
  auto boxes_of = [&](uint32_t ks) { return min(kBoxes, (p.k - ks * kDepth + kBoxDepth - 1u) / kBoxDepth); };
  // rows that a product takes, half of them from either CTA
  auto width = [&](const Place& at) { return max((at.end - at.row + 31u) / 32u * 32u, 32u); };
  auto give_up = [&]() {  // for both CTAs
    pair_store(base + kAbort, 0u, 1u);
    pair_store(base + kAbort, 1u, 1u);
    if (error_word) atomicExch(error_word, 1u);
  };

  uint32_t issued = 0;      // stages over all tiles of this pair, by warp 0
  bool multiplied = false;  // by warp 1 of the first CTA
  if (warp == 0) {
    uint32_t s = 0, phase = 1;
    bool ok = true;
    for (uint32_t tile = pair; tile < tiles && ok; tile += pairs) {
      const Place at = place(tile);
      const uint32_t x_row = uniform(at.row + rank * (width(at) / 2u)), w_row = uniform(at.w_row) + rank * kColumns;
      for (uint32_t ks = 0; ks < k_stages; ++ks, ++issued) {
        const uint32_t stage = base + work.ring + s * work.stage_bytes, boxes = boxes_of(ks);
        ok = !*abort_flag && pair_wait(empty + s * 8, phase, work.wait_limit);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) {
          give_up();
          break;
        }
        if (elect_one()) {
          barrier_arrive(vacant + s * 8);
          const uint32_t first = first_address(full + s * 8);
          if (rank == 0u) barrier_expect_tx(full + s * 8, 2u * boxes * (kBoxBytes + half_bytes));
          for (uint32_t box = 0; box < boxes; ++box) {
            const int32_t x = (int32_t)((ks * kBoxes + box) * kRowBytes);
            pair_load(stage + box * kBoxBytes, &map_w, x, (int32_t)w_row, first);
            pair_load(stage + kInputAt + box * half_bytes, &map_x, x, (int32_t)x_row, first);
          }
        }
        __syncwarp();
        if (++s == work.stages) s = 0, phase ^= 1u;
      }
    }
  } else if (warp == 1 && rank == 1u) {
    // the first CTA issues for both, and hears from here that exponents lie in the second one's memory
    uint32_t s = 0, phase = 0;
    bool ok = true;
    for (uint32_t tile = pair; tile < tiles && ok; tile += pairs)
      for (uint32_t ks = 0; ks < k_stages; ++ks) {
        ok = !*abort_flag && warp_wait(laid + s * 8, phase, work.wait_limit);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (lane == 0) {
          shared_release();
          first_arrive(first_address(scales_full + s * 8));
        }
        __syncwarp();
        if (++s == work.stages) s = 0, phase ^= 1u;
      }
    if (!ok) give_up();
  } else if (warp == 1) {
    uint32_t s = 0, phase = 0, turn = 0;
    bool ok = true;
    for (uint32_t tile = pair; tile < tiles && ok; tile += pairs, ++turn) {
      const uint32_t rows = uniform(width(place(tile)));
      const uint32_t low = mxf4_instruction(2u * kColumns, rows, 0u), high = mxf4_instruction(2u * kColumns, rows, 1u);
      const uint32_t which = turn % kSums, sums = tmem_base + which * kMostRows, scales = tmem_base + kSums * kMostRows;
      ok = !*abort_flag && pair_wait(sums_empty + which * 8, ((turn / kSums) & 1u) ^ 1u, work.wait_limit);
      ok = __all_sync(0xffffffffu, ok);
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      for (uint32_t ks = 0; ks < k_stages && ok; ++ks) {
        const uint32_t stage = base + work.ring + s * work.stage_bytes;
        ok = !*abort_flag && pair_wait(full + s * 8, phase, work.wait_limit) && pair_wait(scales_full + s * 8, phase, work.wait_limit);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        multiplied = true;
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        const uint32_t left = p.k - ks * kDepth;
        const uint64_t a = operand_descriptor(stage), b = operand_descriptor(stage + kInputAt);
        if (elect_one()) {
#pragma unroll
          for (uint32_t g = 0; g < kStageWords; ++g) {
            if (g * kWordValues >= left) break;
            const uint32_t columns = scales + g * kWordColumns, atoms = stage + kInputScalesAt + g * kInputAtoms * kAtom;
            pair_copy_atom(columns, stage + kScalesAt + g * kAtom);
            pair_copy_atom(columns + 4u, atoms);
            if (rows > 128u) pair_copy_atom(columns + 8u, atoms + kAtom);
#pragma unroll
            for (uint32_t j = 0; j < 2; ++j) {
              if (g * kWordValues + j * 64u >= left) break;
              const uint32_t box = g / 2u, at_box = (g % 2u * 2u + j) * 2u;  // 32 bytes of the box's rows, in the descriptor's 16
              pair_mma(sums, a + box * (kBoxBytes / 16u) + at_box, b + box * (half_bytes / 16u) + at_box, j ? high : low, columns, columns + 4u,
                       (ks > 0 || g > 0 || j > 0) ? 1u : 0u);
            }
          }
          pair_commit(empty + s * 8);
          if (ks + 1u == k_stages) pair_commit(sums_full + which * 8);
        }
        __syncwarp();
        if (++s == work.stages) s = 0, phase ^= 1u;
      }
    }
    if (!ok) give_up();
  } else if (warp < 2u + kScaleWarps) {
    // the words of group warp - 2 of a stage, of the CTA's weight rows and of the tile's rows of x: lane, lane + 32, ...
    const uint32_t group = warp - 2u, words = words_of(p.k), last_mask = last_word_mask(p.k);
    uint32_t held[kAhead][kWordColumns];
    uint32_t all = 0, mine = 0, ahead_tile = pair, ahead_stage = 0;
    for (uint32_t tile = pair; tile < tiles; tile += pairs) all += k_stages;
    Place ahead = {};
    if (all > 0) ahead = place(pair);
    // Nothing looks at them before they are laid down, so that nothing waits for them here.
    auto fetch = [&](uint32_t (&into)[kWordColumns]) {
      if (mine >= all) return;
      ++mine;
      const uint32_t at = ahead_stage * kStageWords + group, w_row = ahead.w_row + rank * kColumns + lane, x_row = ahead.row + lane;
      const uint32_t w_end = at < words ? p.w_rows : 0u, x_end = at < words ? ahead.end : 0u;
      const uint32_t *const of_w = p.w_scales + (size_t)at * p.w_rows, *const of_x = p.x_scales + (size_t)at * p.m;
#pragma unroll
      for (uint32_t i = 0; i < 4; ++i) {
        into[i] = 0u;
        if (w_row + i * 32u < w_end) into[i] = of_w[w_row + i * 32u];
      }
#pragma unroll
      for (uint32_t i = 0; i < 4 * kInputAtoms; ++i) {
        into[4 + i] = 0u;
        if (x_row + i * 32u < x_end) into[4 + i] = of_x[x_row + i * 32u];
      }
      if (++ahead_stage == k_stages) {
        ahead_stage = 0;
        ahead_tile += pairs;
        if (mine < all) ahead = place(ahead_tile);
      }
    };
#pragma unroll
    for (uint32_t a = 0; a < kAhead; ++a) fetch(held[a]);
    uint32_t s = 0, phase = 0, ks = 0;
    bool ok = true;
    for (uint32_t first = 0; first < all && ok; first += kAhead) {
#pragma unroll
      for (uint32_t a = 0; a < kAhead; ++a) {
        if (first + a >= all || !ok) break;
        ok = !*abort_flag && warp_wait(vacant + s * 8, phase, work.wait_limit);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint32_t mask = ks * kStageWords + group + 1u == words ? last_mask : 0xffffffffu;
        const uint32_t(&v)[kWordColumns] = held[a];
        unsigned char* const stage = base_pointer + work.ring + s * work.stage_bytes;
        auto line = [&](uint32_t atom, uint32_t first) {  // a lane's four rows are a line of an atom
          *reinterpret_cast<uint4*>(stage + atom + lane * 16u) = make_uint4(v[first] & mask, v[first + 1] & mask, v[first + 2] & mask, v[first + 3] & mask);
        };
        line(kScalesAt + group * kAtom, 0u);
        line(kInputScalesAt + group * kInputAtoms * kAtom, 4u);
        line(kInputScalesAt + (group * kInputAtoms + 1u) * kAtom, 8u);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) barrier_arrive((rank == 0u ? scales_full : laid) + s * 8);
        fetch(held[a]);
        if (++ks == k_stages) ks = 0;
        if (++s == work.stages) s = 0, phase ^= 1u;
      }
    }
    if (!ok) give_up();
  } else {
    const uint32_t worker = warp - 2u - kScaleWarps, quarter = warp & 3u, side = worker >> 2;  // lanes of tensor memory; every other piece
    unsigned char* const staging = base_pointer + kFront + work.list + worker * kStagingBytes;
    uint32_t turn = 0;
    bool ok = true;
    for (uint32_t tile = pair; tile < tiles && ok; tile += pairs, ++turn) {
      const uint32_t which = turn % kSums;
      const Place at = place(tile);
      const uint32_t column = at.column + rank * kColumns + quarter * 32u;
      float own = piece_operand<S>(p, at.row + side * 32u, at.end, column);
      ok = !*abort_flag && pair_wait(sums_full + which * 8, (turn / kSums) & 1u, work.wait_limit);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {
        give_up();
        break;
      }
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t address = tmem_base + which * kMostRows + ((quarter * 32u) << 16);
#pragma unroll 1
      for (uint32_t piece = side; piece < kLoneRows / 32u; piece += kEpilogueWarps / 4u) {
        const uint32_t row = at.row + piece * 32u;
        if (row >= at.end) break;
        uint32_t raw[32];
        tmem_load_32(address + piece * 32u, raw);
        const float mine = own;
        if (kPaired<S>) own = piece_operand<S>(p, row + kEpilogueWarps / 4u * 32u, at.end, column);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        constexpr uint32_t kWidth = kPaired<S> ? 16 : 32;  // columns of results
        const uint32_t out_column = kPaired<S> ? column / 2u : column, columns = kPaired<S> ? p.n / 2u : p.n;
        if (lane == 0) await_box();
        __syncwarp();
        if (S != kStoreFloat && work.boxes && row + 32u <= at.end && out_column + kWidth <= columns) {
          if constexpr (S != kStoreFloat) stage_piece<S, kWidth * 2>(32u, raw, mine, staging);
          asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
          __syncwarp();
          if (lane == 0) store_box(&map_out, (int32_t)out_column, (int32_t)row, smem_u32(staging));
        } else {
          store_piece<S>(p, row, at.end, column, raw, mine, staging);
        }
        __syncwarp();  // tcgen05.ld needs the whole warp
      }
      asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
      __syncwarp();
      if (lane == 0) first_arrive(first_address(sums_empty + which * 8));
    }
    if (lane == 0) await_box();
    __syncwarp();
  }

  __syncthreads();
  cluster_sync();  // neither CTA leaves, or gives its tensor memory back, while the other's products or arrivals reach it
  // Whoever gave up has said so to both by now.  What was started then must end before the pair leaves: products, and the copies of both, which
  // the first one's barriers count and of which those that nobody waited for are among the ring's last.  Of a stage that one CTA alone
  // came to ask for they would wait for the other's share too.
  if (*abort_flag) {
    if (threadIdx.x == 0) pair_store(base + kIssued + rank * 4u, 0u, issued);
    __syncwarp();
    cluster_sync();
    if (rank == 0u && warp == 0) {
      const volatile uint32_t* const of = reinterpret_cast<const volatile uint32_t*>(base_pointer + kIssued);
      const uint32_t first = of[0], second = of[1], last = max(first, second);
      for (uint32_t i = last > work.stages ? last - work.stages : 0u; i < last; ++i) {
        const uint32_t bar = full + (i % work.stages) * 8, bytes = boxes_of(i % k_stages) * (kBoxBytes + half_bytes);
        if (lane == 0 && i >= first) barrier_expect_tx(bar, bytes);
        if (lane == 0 && i >= second) barrier_forgo(bar, bytes);
        __syncwarp();
        barrier_wait(bar, (i / work.stages) & 1u);
      }
    } else if (multiplied) {
      if (elect_one())
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(drained) : "memory");
      __syncwarp();
      pair_wait(drained, 0u);
    }
    __syncwarp();
    cluster_sync();
  }
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(kTmemColumns) : "memory");
  }
}

}  // namespace

namespace mxfp4 {

template <Store S>
int run_tiles(const KernelArgs& args, const Problem& p, uint32_t plan_tiles) {
  const uint32_t pairs = (uint32_t)context_sm_count(args.ctx) / 2u, k_stages = (p.k + kDepth - 1u) / kDepth;
  Work work = {plan_tiles, (p.n + 2u * kColumns - 1u) / (2u * kColumns), kExpertTile, 0u, 0u, 0u, 0u, 0u, context_mxfp4_wait_limit(args.ctx)};
  if (!p.plan.tiles) {
    // the height with the shortest estimate: rounds of tiles times the cycles of one, of which a stage takes about 500 and four per row
    uint64_t least = ~0ull;
    for (uint32_t rows = kLoneRows; rows >= 32u; rows -= 32u) {
      const uint32_t row_tiles = (p.m + rows - 1u) / rows;
      if (rows > kMostRows && (uint64_t)row_tiles * work.column_tiles > pairs) continue;  // its sums lie over those of the next
      const uint64_t rounds = ((uint64_t)row_tiles * work.column_tiles + pairs - 1u) / pairs, cost = rounds * ((uint64_t)k_stages * (500u + 4u * rows) + 1000u);
      if (cost < least) least = cost, work.rows = rows, work.row_tiles = row_tiles;
    }
  } else if (p.m >= p.plan.experts * kExpertTile && p.k >= 4u * kDepth && plan_tiles <= kMostJoined) {
    // The plan's tiles joined where experts have as many rows as one on average, and products enough to make up for taller boxes and one stage
    // less.  us, the plan's and joined, through 4096 x 7168: 16384 rows of 16 experts 276, 228, 8192 of 8 137, 111, 4096 of 16 85, 73, 1024 of 8
    // 36.0, 32.3; 16384 of 64 through 2048 x 2816 75.7, 70.3.  Fewer rows: 1024 of 16 45.7, 45.0 (through 3584 x 4096 21.3, 23.1), 4096 of 64 through
    // 2048 x 2048 28.4, 29.9; smaller k: 16384 of 64 through 1408 x 2048 52.5, 54.4, 1200 of 8 10.4, 12.4.
    work.rows = kMostRows, work.list = kList;
  }
  const uint64_t tiles = (uint64_t)work.row_tiles * work.column_tiles;
  LLMOPT_REQUIRE(tiles < (1u << 28), "too many tiles");
  work.stage_bytes = kInputAt + kBoxes * (work.rows / 2u * kRowBytes);
  work.ring = kFront + work.list + (tiles > pairs ? kStaging : 0u);
  work.stages = (kMostShared - 1024u - work.ring) / work.stage_bytes;
  if (work.stages > kMostStages) work.stages = kMostStages;
  if (!allow_shared<tiles_kernel<S>, kMostShared>()) return fail_launch(args, "shared memory request was refused");
  CUtensorMap map_w, map_x;
  if (!make_map(&map_w, p.w, p.k, p.w_rows, kColumns) || !make_map(&map_x, p.x, p.k, p.m, work.rows / 2u)) return fail_launch(args, "tensor map was refused");
  CUtensorMap map_out = map_x;  // not read without boxes
  const uint32_t columns = kPaired<S> ? p.n / 2u : p.n;
  if (S != kStoreFloat && columns % 8u == 0 && ((uintptr_t)p.out & 15u) == 0) {
    const bool half = sizeof(typename Element<S>::Type) == 2 && (S == kStoreHalf || S == kStorePairHalf);
    work.boxes = make_map(&map_out, half ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2u, p.out, columns, p.m,
                          kPaired<S> ? 16u : 32u, 32u, CU_TENSOR_MAP_SWIZZLE_NONE);
  }
  const uint32_t shared = 1024u + work.ring + work.stages * work.stage_bytes;  // 1024 for the alignment of the ring
  launch_cluster_kernel(args, tiles_kernel<S>, dim3(2u * (tiles < pairs ? (uint32_t)tiles : pairs)), dim3(kThreads), shared, 2u, map_w, map_x,
                        map_out, p, work, error_word_of(args));
  return check_launch(args);
}

template int run_tiles<kStoreHalf>(const KernelArgs&, const Problem&, uint32_t);
template int run_tiles<kStoreBf16>(const KernelArgs&, const Problem&, uint32_t);
template int run_tiles<kStoreFloat>(const KernelArgs&, const Problem&, uint32_t);
template int run_tiles<kStorePairHalf>(const KernelArgs&, const Problem&, uint32_t);
template int run_tiles<kStorePairBf16>(const KernelArgs&, const Problem&, uint32_t);

}  // namespace mxfp4
}  // namespace llmopt
