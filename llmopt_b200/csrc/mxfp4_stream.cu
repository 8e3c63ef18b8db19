// Products of few MXFP4 rows with MXFP4 matrices: the stream of the weights is what they cost, n k 17 / 32 bytes.
//
// A CTA has one tile of 128 weight rows and all of k or, as one of a cluster, a share of it, in stages of 512 elements of k.  Warp 0 brings
// the codes by TMA (128-byte swizzle); warps 2 to 5 bring the exponents, a warp per word (128 elements) of the stage, requested ahead in
// registers and laid down in the order that tcgen05.cp spreads over tensor memory; one lane of warp 1 issues copies and products; then
// warps 2 to 5 read the sums out.  CTAs of a cluster hand each row's sums to the one that joins them, in the order of k.
//
// The copies start before the block's other warps: the barriers are warp 0's own until it says that they are there.  Weights cold, calls of a
// kind behind one another (k x columns, as everywhere here): 14336 x 57344 1 row 68 to 75 us (6.4 to 5.8 TB/s, by GPU); 4096 x 128256 46 to 50;
// 4096 x 14336 7.8, 64 rows 8.8, where the launch, the first copies' latency and the way out are half of it; 14336 x 4096 8.3, 4096 x 4096 4.7.
// Stages of 256 had the same bytes in flight and twice the handovers, 485 cycles each, more than the copies of a stage take.  Asking for the
// weights while the previous kernel ends made both slower.
//
// Every wait on an mbarrier is bounded; a wait that runs out raises the launch's error word, and the CTA lets its copies and
// products end, frees its tensor memory and returns.
#include "mxfp4_tc.cuh"

namespace llmopt {
namespace {
using namespace mxfp4;

constexpr uint32_t kThreads = (2 + kScaleWarps) * 32, kMostSplits = 8, kMostShared = 227 * 1024;
constexpr uint32_t kAhead = 4;               // stages of exponents that are under way in registers
constexpr uint32_t kDepth = 512, kBoxes = kDepth / kBoxDepth, kStageWords = kDepth / kWordValues;
static_assert(kStageWords == kScaleWarps, "a warp per word of a stage");

template <uint32_t NT>
struct Shape {
  static constexpr uint32_t kWeightBytes = kBoxes * kColumns * kRowBytes, kInputBytes = kBoxes * NT * kRowBytes;
  static constexpr uint32_t kScalesAt = kWeightBytes + kInputBytes, kInputScalesAt = kScalesAt + kStageWords * kAtom;
  static constexpr uint32_t kStageBytes = kInputScalesAt + kStageWords * kAtom;
  static constexpr uint32_t kStages = 4;  // at most
  static constexpr uint32_t kScaleColumns = kStageWords * 8;
  static constexpr uint32_t kTmemColumns = 128;
  static_assert(NT + 2 * kScaleColumns <= kTmemColumns, "tensor memory");
  static constexpr uint32_t kHolder = (3 * kStages + 2) * 8;  // behind the ring: barriers, tensor memory's address, abort flag
  static constexpr uint32_t kBehind = kHolder + 8;
  static constexpr uint32_t kPiece = NT == 16 ? 16 : 32;
};

struct Work {
  uint32_t row_tiles, column_tiles, splits, stages, box_rows;
  uint32_t share;  // rows that a CTA of a cluster joins
  uint32_t wait_limit;  // how often a wait looks; 0: all give up at once
};
// Shared memory, 1024 of it for the alignment of the ring; behind the barriers the sums of a cluster's CTAs, [from][row of the share][column],
// and a row that may be read but not used.
template <uint32_t NT>
uint32_t shared_bytes(const Work& work) {
  using Z = Shape<NT>;
  return 1024u + work.stages * Z::kStageBytes + Z::kBehind + (work.splits > 1u ? (work.splits * work.share + 1u) * kColumns * 4u : 0u);
}

__device__ __forceinline__ void cluster_store(uint32_t local, uint32_t rank, uint32_t value) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(local), "r"(rank));
  asm volatile("st.shared::cluster.b32 [%0], %1;" ::"r"(remote), "r"(value) : "memory");
}

template <uint32_t NT, Store S>
__global__ void __launch_bounds__(kThreads, 2)
stream_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ Problem p, const Work work,
              uint32_t* error_word) {
  using Z = Shape<NT>;
  extern __shared__ unsigned char shared_raw[];
  grid_launch_dependents();
  const uint32_t base = (smem_u32(shared_raw) + 1023u) & ~1023u;
  unsigned char* base_pointer = shared_raw + (base - smem_u32(shared_raw));
  const uint32_t behind = work.stages * Z::kStageBytes;
  const uint32_t full = base + behind, scales_full = full + Z::kStages * 8, empty = scales_full + Z::kStages * 8, sums_full = empty + Z::kStages * 8;
  const uint32_t drained = sums_full + 8;
  const uint32_t joined = base + behind + Z::kBehind;
  volatile uint32_t* holder = reinterpret_cast<volatile uint32_t*>(base_pointer + behind + Z::kHolder);
  volatile uint32_t* abort_flag = holder + 1;
  const uint32_t warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31u;
  const uint32_t splits = work.splits, rank = blockIdx.x % splits, tile = blockIdx.x / splits;
  // tiles that the plan does not have come last
  const uint32_t row_tile = tile / work.column_tiles, column = tile % work.column_tiles * kColumns, k_stages = (p.k + kDepth - 1u) / kDepth;
  const uint32_t stage0 = k_stages * rank / splits, stage1 = k_stages * (rank + 1u) / splits, words = words_of(p.k);

  if (warp == 0) {
    if (lane == 0) {
      for (uint32_t s = 0; s < work.stages; ++s) {
        barrier_init(full + s * 8, 1);  // the copies' expect_tx arrival; completes by byte count
        barrier_init(scales_full + s * 8, kScaleWarps);
        barrier_init(empty + s * 8, 1);  // one tcgen05.commit
      }
      barrier_init(sums_full, 1);  // one tcgen05.commit
      barrier_init(drained, 1);    // the same, where somebody gave up
      *abort_flag = work.wait_limit == 0u;
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    asm volatile("bar.arrive 1, %0;" ::"n"(kThreads) : "memory");
  }
  if (splits > 1u) cluster_arrive();  // this CTA runs: others may write into its shared memory
  grid_dependency_wait();
  if (p.plan.tiles && row_tile >= min(p.plan.tiles[0], work.row_tiles)) return;  // the whole cluster
  const Place at = place_of(p, row_tile, NT, column);

  auto give_up = [&]() {
    *abort_flag = 1u;
    if (error_word) atomicExch(error_word, 1u);
  };
  const uint32_t x_boxes = uniform((at.end - at.row + work.box_rows - 1u) / work.box_rows), w_row = uniform(at.w_row), x_row = uniform(at.row);
  auto load = [&](uint32_t ks, uint32_t s) {
    const uint32_t stage = base + s * Z::kStageBytes, boxes = min(kBoxes, (p.k - ks * kDepth + kBoxDepth - 1u) / kBoxDepth);
    if (elect_one()) {
      barrier_expect_tx(full + s * 8, boxes * (kColumns + x_boxes * work.box_rows) * kRowBytes);
      for (uint32_t box = 0; box < boxes; ++box) {
        const int32_t x = (int32_t)((ks * kBoxes + box) * kRowBytes);
        tma_load_2d(stage + box * kColumns * kRowBytes, &map_w, x, (int32_t)w_row, full + s * 8);
        for (uint32_t i = 0; i < x_boxes; ++i)
          tma_load_2d(stage + Z::kWeightBytes + (box * NT + i * work.box_rows) * kRowBytes, &map_x, x, (int32_t)(x_row + i * work.box_rows), full + s * 8);
      }
    }
    __syncwarp();
  };
  // The words of group warp - 2 of a stage: of the weight rows lane, lane + 32, ..., and of as many rows of x.  Nothing looks at them before
  // they are laid down, so that nothing waits for them here.
  constexpr uint32_t kInputWords = NT <= 32 ? 1 : NT / 32;
  uint32_t held[kAhead][4 + kInputWords];
  auto fetch = [&](uint32_t ks, uint32_t (&into)[4 + kInputWords]) {
    const uint32_t group = ks * kStageWords + warp - 2u;
    const bool present = ks < stage1 && group < words;
#pragma unroll
    for (uint32_t i = 0; i < 4; ++i) {
      into[i] = 0u;
      if (present && at.w_row + i * 32u + lane < p.w_rows) into[i] = p.w_scales[(size_t)group * p.w_rows + at.w_row + i * 32u + lane];
    }
#pragma unroll
    for (uint32_t i = 0; i < kInputWords; ++i) {
      into[4 + i] = 0u;
      if (present && at.row + i * 32u + lane < at.end) into[4 + i] = p.x_scales[(size_t)group * p.m + at.row + i * 32u + lane];
    }
  };
  // ahead of the block's first synchronisation: the barriers are this warp's own, the words lie in registers
  if (warp == 0) {
    for (uint32_t s = 0; s < work.stages && stage0 + s < stage1; ++s) load(stage0 + s, s);
  } else if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + behind + Z::kHolder), "r"(Z::kTmemColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else {
#pragma unroll
    for (uint32_t a = 0; a < kAhead; ++a) fetch(stage0 + a, held[a]);
  }
  // warp 0 has said that its barriers are there, and goes on to copy
  if (warp > 0) {
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    asm volatile("bar.sync 1, %0;" ::"n"(kThreads) : "memory");
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  }
  const uint32_t tmem_base = warp > 0 ? uniform(*holder) : 0u;

  uint32_t issued = min(work.stages, stage1 - stage0);  // stages, by warp 0
  bool multiplied = false;                              // by warp 1
  if (warp == 0) {
    bool ok = true;
    uint32_t s = 0, phase = 0;
    for (uint32_t ks = stage0 + issued; ks < stage1; ++ks, ++issued) {
      ok = !*abort_flag && warp_wait(empty + s * 8, phase, work.wait_limit);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {
        give_up();
        break;
      }
      load(ks, s);
      if (++s == work.stages) s = 0, phase ^= 1u;
    }
  } else if (warp == 1) {
    const uint32_t rows = p.plan.tiles ? uniform(max((at.end - at.row + 15u) / 16u * 16u, 16u)) : NT;
    const uint32_t low = mxf4_instruction(kColumns, rows, 0u), high = mxf4_instruction(kColumns, rows, 1u);
    bool ok = true;
    uint32_t s = 0, phase = 0;
    for (uint32_t ks = stage0; ks < stage1; ++ks) {
      const uint32_t stage = base + s * Z::kStageBytes;
      ok = !*abort_flag && warp_wait(full + s * 8, phase, work.wait_limit) && warp_wait(scales_full + s * 8, phase, work.wait_limit);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      multiplied = true;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t scales = tmem_base + NT + (ks & 1u) * Z::kScaleColumns, x_scales = scales + kStageWords * 4u, left = p.k - ks * kDepth;
      const uint64_t a = operand_descriptor(stage), b = operand_descriptor(stage + Z::kWeightBytes);
      if (elect_one()) {
#pragma unroll
        for (uint32_t g = 0; g < kStageWords; ++g) {
          if (g * kWordValues >= left) break;
          copy_atom(scales + g * 4u, stage + Z::kScalesAt + g * kAtom);
          copy_atom(x_scales + g * 4u, stage + Z::kInputScalesAt + g * kAtom);
#pragma unroll
          for (uint32_t j = 0; j < 2; ++j) {
            if (g * kWordValues + j * 64u >= left) break;
            const uint32_t box = g / 2u, at_box = (g % 2u * 2u + j) * 2u;  // 32 bytes of the box's rows, in the descriptor's 16
            mma_mxf4(tmem_base, a + box * (kColumns * kRowBytes / 16u) + at_box, b + box * (NT * kRowBytes / 16u) + at_box, j ? high : low,
                     scales + g * 4u, x_scales + g * 4u, (ks > stage0 || g > 0 || j > 0) ? 1u : 0u);
          }
        }
        mma_commit(empty + s * 8);
        if (ks + 1u == stage1) mma_commit(sums_full);
      }
      __syncwarp();
      if (++s == work.stages) s = 0, phase ^= 1u;
    }
    if (!ok) give_up();
  } else {
    const uint32_t group = warp - 2u, last_mask = last_word_mask(p.k);
    bool ok = true;
    uint32_t s = 0, phase = 1;
    for (uint32_t first = stage0; first < stage1 && ok; first += kAhead) {
#pragma unroll
      for (uint32_t a = 0; a < kAhead; ++a) {
        const uint32_t ks = first + a;
        if (ks >= stage1 || !ok) break;
        ok = !*abort_flag && warp_wait(empty + s * 8, phase, work.wait_limit);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        const uint32_t mask = ks * kStageWords + group + 1u == words ? last_mask : 0xffffffffu;
        unsigned char* const stage = base_pointer + s * Z::kStageBytes;
        // a lane's four rows are a line of the atom
        *reinterpret_cast<uint4*>(stage + Z::kScalesAt + group * kAtom + lane * 16u) =
            make_uint4(held[a][0] & mask, held[a][1] & mask, held[a][2] & mask, held[a][3] & mask);
#pragma unroll
        for (uint32_t i = 0; i < kInputWords; ++i)
          *reinterpret_cast<uint32_t*>(stage + Z::kInputScalesAt + group * kAtom + lane * 16u + i * 4u) = held[a][4 + i] & mask;
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) barrier_arrive(scales_full + s * 8);
        fetch(ks + kAhead, held[a]);
        if (++s == work.stages) s = 0, phase ^= 1u;
      }
    }
    const uint32_t quarter = warp & 3u;
    float own = splits == 1u ? piece_operand<S>(p, at.row, at.end, at.column + quarter * 32u) : 0.0f;
    if (ok) {
      ok = !*abort_flag && warp_wait(sums_full, 0u, work.wait_limit);
      ok = __all_sync(0xffffffffu, ok);
    }
    if (splits > 1u) cluster_wait();
    if (!ok) {
      give_up();
    } else {
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t address = tmem_base + ((quarter * 32u) << 16), place = quarter * 32u + lane;
      uint32_t owner = 0, share_row = 0;
#pragma unroll 1
      for (uint32_t piece = 0; piece < NT / Z::kPiece; ++piece) {
        const uint32_t row = at.row + piece * Z::kPiece;
        if (row >= at.end) break;
        uint32_t raw[Z::kPiece];
        if constexpr (Z::kPiece == 16) tmem_load_16(address + piece * Z::kPiece, raw);
        else tmem_load_32(address + piece * Z::kPiece, raw);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        if (splits == 1u) {
          // through the ring: every stage of it has been read
          if (kPaired<S> && piece > 0) own = piece_operand<S>(p, row, at.end, at.column + quarter * 32u);
          store_piece<S>(p, row, at.end, at.column + quarter * 32u, raw, own, base_pointer + quarter * kStagingBytes);
        } else {
#pragma unroll
          for (uint32_t i = 0; i < Z::kPiece; ++i) {
            if (row + i >= at.end) break;
            cluster_store(joined + ((rank * work.share + share_row) * kColumns + place) * 4u, owner, raw[i]);
            if (++share_row == work.share) share_row = 0, ++owner;
          }
        }
        __syncwarp();  // tcgen05.ld needs the whole warp
      }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  }
  if (warp < 2u && splits > 1u) cluster_wait();

  __syncthreads();
  // Whoever gave up has said so by now.  What was started then must end before the CTA leaves its shared and tensor memory to others: copies, of
  // which those that nobody waited for are among the ring's last, and products.
  if (*abort_flag) {
    if (warp == 0) {
      for (uint32_t i = issued > work.stages ? issued - work.stages : 0u; i < issued; ++i)
        barrier_wait(full + (i % work.stages) * 8, (i / work.stages) & 1u);
    } else if (multiplied) {
      if (elect_one()) mma_commit(drained);
      __syncwarp();
      warp_wait(drained, 0u);
    }
    __syncwarp();
  }
  // Before CTAs of a cluster wait for one another's sums: one that waits for columns which another grid holds must not be waited for with
  // these held.
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(Z::kTmemColumns) : "memory");
  }
  if (splits == 1u) return;
  cluster_arrive();
  cluster_wait();
  // this CTA's share of the rows, always the sums of rank 0 first; a warp has 32 columns of two rows at a time
  const float* sums = reinterpret_cast<const float*>(base_pointer + behind + Z::kBehind);
  const uint32_t first_row = rank * work.share, all = at.end - at.row, mine = first_row < all ? min(work.share, all - first_row) : 0u;
  for (uint32_t item = warp; item < (mine + 1u) / 2u * 4u; item += kThreads / 32u) {
    const uint32_t row = item / 4u * 2u, place = item % 4u * 32u + lane;
    uint32_t raw[2];
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
      float sum = sums[(row + i) * kColumns + place];
      for (uint32_t from = 1; from < splits; ++from) sum += sums[(from * work.share + row + i) * kColumns + place];
      raw[i] = __float_as_uint(sum);
    }
    store_rows<S>(p, at.row + first_row + row, at.row + first_row + mine, at.column + place, raw);
  }
}

template <uint32_t NT, Store S>
int run(const KernelArgs& args, const Problem& p, uint32_t row_tiles) {
  using Z = Shape<NT>;
  const uint32_t sms = (uint32_t)context_sm_count(args.ctx), k_stages = (p.k + kDepth - 1u) / kDepth;
  Work work = {row_tiles, (p.n + kColumns - 1u) / kColumns, 1u, 0u, p.plan.tiles ? 16u : NT, 0u, context_mxfp4_wait_limit(args.ctx)};
  const size_t tiles = (size_t)work.row_tiles * work.column_tiles;
  LLMOPT_REQUIRE(tiles < (1u << 28), "too many tiles");
  // CTAs that share a tile's k while tiles leave SMs without work; powers of two, which leave the fewest SMs of a GPC over.  us with 1, 2, 4, 8
  // of them: 4096 x 4096 6.1, 5.3, 4.7, 6.0; 14336 x 4096 15.0, 9.9, 8.3, 10.0; 4096 x 14336 (112 tiles) 7.9, 9.4.
  while (work.splits < kMostSplits && tiles * work.splits * 2u <= sms && p.k / kDepth >= work.splits * 2u) work.splits *= 2u;
  const uint32_t mine = (k_stages + work.splits - 1u) / work.splits;
  // a CTA per SM: a deep ring; more: two of them per SM, which start and end beside one another (4 and 2 stages: 4096 x 14336 7.8, 9.1 us,
  // 14336 x 4096 8.3, 9.5; 4096 x 128256 56.3, 49.7)
  const uint32_t most = tiles * work.splits <= sms ? Z::kStages : 2u;
  work.stages = mine < most ? mine : most;
  const uint32_t rows = p.m < NT ? p.m : NT;
  work.share = (rows + work.splits - 1u) / work.splits;
  while (shared_bytes<NT>(work) > kMostShared) --work.stages;
  auto kernel = stream_kernel<NT, S>;
  if (!allow_shared<stream_kernel<NT, S>, kMostShared>()) return fail_launch(args, "shared memory request was refused");
  CUtensorMap map_w, map_x;
  if (!make_map(&map_w, p.w, p.k, p.w_rows, kColumns) || !make_map(&map_x, p.x, p.k, p.m, work.box_rows)) return fail_launch(args, "tensor map was refused");
  const dim3 grid((uint32_t)tiles * work.splits);
  if (work.splits == 1u)
    launch_kernel(args, kernel, grid, dim3(kThreads), shared_bytes<NT>(work), map_w, map_x, p, work, error_word_of(args));
  else
    launch_cluster_kernel(args, kernel, grid, dim3(kThreads), shared_bytes<NT>(work), work.splits, map_w, map_x, p, work,
                          error_word_of(args));
  return check_launch(args);
}

}  // namespace

namespace mxfp4 {

template <Store S>
int run_stream(const KernelArgs& args, const Problem& p, uint32_t plan_tiles) {
  const uint32_t row_tiles = p.plan.tiles ? plan_tiles : 1u;
  if (p.m <= 16u) return run<16, S>(args, p, row_tiles);
  if (p.m <= 32u) return run<32, S>(args, p, row_tiles);
  return run<64, S>(args, p, row_tiles);
}

template int run_stream<kStoreHalf>(const KernelArgs&, const Problem&, uint32_t);
template int run_stream<kStoreBf16>(const KernelArgs&, const Problem&, uint32_t);
template int run_stream<kStoreFloat>(const KernelArgs&, const Problem&, uint32_t);
template int run_stream<kStorePairHalf>(const KernelArgs&, const Problem&, uint32_t);
template int run_stream<kStorePairBf16>(const KernelArgs&, const Problem&, uint32_t);

}  // namespace mxfp4
}  // namespace llmopt
