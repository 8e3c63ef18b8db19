// Products of few MXFP4 rows with MXFP4 matrices: the stream of the weights is what they cost, n k 17 / 32 bytes.
//
// A CTA has one tile of 128 weight rows and all of k or, as one of a cluster, a share of it: four thread blocks of 192 threads live on an SM,
// so that while one starts or stores the others stream.  Warp 0 brings the codes of 256 elements of k at a time by TMA
// (128-byte swizzle); warps 2 to 5 bring the exponents, a word (128 elements) per thread and row, requested ahead in registers and laid
// down in the order that tcgen05.cp spreads over tensor memory; one thread of warp 1 issues copies and products; then warps 2 to
// 5 read the sums out.  CTAs of a cluster leave their sums in shared memory and each joins a share of the rows, in the order of k.
//
// While the kernel before still runs, the tile's weights are asked into L2: that changes nothing that anybody reads, whoever writes them.
//
// Every wait on an mbarrier is bounded; a wait that runs out raises the context's device error word, and the CTA lets its copies land,
// frees its tensor memory and returns.
#include "mxfp4_tc.cuh"

namespace llmopt {
namespace {
using namespace mxfp4;

constexpr uint32_t kThreads = (2 + kScaleWarps) * 32, kAhead = 4, kMostSplits = 8;

template <uint32_t NT>
struct Shape {
  static constexpr uint32_t kWeightBytes = kColumns * kRowBytes, kInputBytes = NT * kRowBytes;
  static constexpr uint32_t kScalesAt = kWeightBytes + kInputBytes;
  static constexpr uint32_t kStageBytes = kScalesAt + kStageWords * 2 * kAtom;
  static constexpr uint32_t kStages = 3;
  static constexpr uint32_t kScaleColumns = kStageWords * 4 * 2;
  static constexpr uint32_t kUsedColumns = NT + 2 * kScaleColumns;
  static constexpr uint32_t kTmemColumns = kUsedColumns <= 64 ? 64 : kUsedColumns <= 128 ? 128 : 256;
  static constexpr uint32_t kHolder = (3 * kStages + 1) * 8;  // behind the ring: barriers, tensor memory's address, abort flag
  static constexpr uint32_t kBehind = kHolder + 8;
  static constexpr uint32_t kPiece = NT == 16 ? 16 : 32;
  // slack: 1024-byte alignment of the tiles; the ring holds the sums of a cluster's CTA afterwards
  static constexpr __host__ __device__ uint32_t bytes(uint32_t stages) {
    const uint32_t ring = stages * kStageBytes, sums = NT * kColumns * 4;
    return (ring > sums ? ring : sums) + kBehind + 1024;
  }
};

struct Work {
  uint32_t row_tiles, column_tiles, splits, stages, box_rows;
};

template <uint32_t NT, Store S>
__global__ void __launch_bounds__(kThreads, NT <= 32 ? 3 : 2)
stream_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const __grid_constant__ Problem p, const Work work,
              uint32_t* error_word) {
  using Z = Shape<NT>;
  extern __shared__ unsigned char shared_raw[];
  grid_launch_dependents();
  const uint32_t base = (smem_u32(shared_raw) + 1023u) & ~1023u;
  unsigned char* base_pointer = shared_raw + (base - smem_u32(shared_raw));
  const uint32_t behind = Z::bytes(work.stages) - Z::kBehind - 1024u;
  const uint32_t full = base + behind, scales_full = full + Z::kStages * 8, empty = scales_full + Z::kStages * 8, sums_full = empty + Z::kStages * 8;
  volatile uint32_t* holder = reinterpret_cast<volatile uint32_t*>(base_pointer + behind + Z::kHolder);
  volatile uint32_t* abort_flag = holder + 1;
  const uint32_t warp = uniform(threadIdx.x >> 5), lane = threadIdx.x & 31u, t = threadIdx.x - 64u;  // t: row of the exponents' threads
  const uint32_t splits = work.splits, rank = blockIdx.x % splits, tile = blockIdx.x / splits;
  const uint32_t column = tile / work.row_tiles * kColumns, k_stages = (p.k + kDepth - 1u) / kDepth;
  const uint32_t stage0 = k_stages * rank / splits, stage1 = k_stages * (rank + 1u) / splits, words = words_of(p.k);

  if (threadIdx.x == 0) {
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_w) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&map_x) : "memory");
    for (uint32_t s = 0; s < work.stages; ++s) {
      barrier_init(full + s * 8, 1);  // the copies' expect_tx arrival; completes by byte count
      barrier_init(scales_full + s * 8, kScaleWarps);
      barrier_init(empty + s * 8, 1);  // one tcgen05.commit
    }
    barrier_init(sums_full, 1);  // one tcgen05.commit
    *abort_flag = 0u;
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    if (!p.plan.tiles)
      for (uint32_t ks = stage0; ks < stage1; ++ks)
        asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];" ::"l"(&map_w), "r"((int32_t)(ks * kRowBytes)), "r"((int32_t)column)
                     : "memory");
  }
  grid_dependency_wait();
  if (p.plan.tiles && tile % work.row_tiles >= min(p.plan.tiles[0], work.row_tiles)) return;  // the whole cluster
  const Place at = place_of<NT>(p, tile % work.row_tiles, column);

  auto give_up = [&]() {
    *abort_flag = 1u;
    if (error_word) atomicExch(error_word, 1u);
  };
  const uint32_t boxes = (at.end - at.row + work.box_rows - 1u) / work.box_rows;
  auto load = [&](uint32_t ks, uint32_t s) {
    const uint32_t stage = base + s * Z::kStageBytes;
    barrier_expect_tx(full + s * 8, Z::kWeightBytes + boxes * work.box_rows * kRowBytes);
    tma_load_2d(stage, &map_w, (int32_t)(ks * kRowBytes), (int32_t)at.w_row, full + s * 8);
    for (uint32_t box = 0; box < boxes; ++box)
      tma_load_2d(stage + Z::kWeightBytes + box * work.box_rows * kRowBytes, &map_x, (int32_t)(ks * kRowBytes), (int32_t)(at.row + box * work.box_rows),
                  full + s * 8);
  };
  // words of the weights and of x, a stage each; nothing looks at them before they are laid down, so that nothing waits for them here
  uint32_t held[kAhead][kStageWords * 2];
  auto fetch = [&](uint32_t ks, uint32_t (&into)[kStageWords * 2]) {
#pragma unroll
    for (uint32_t g = 0; g < kStageWords; ++g) {
      const uint32_t group = ks * kStageWords + g;
      const bool present = ks < stage1 && group < words;
      into[2 * g] = into[2 * g + 1] = 0u;
      if (present && at.w_row + t < p.w_rows) into[2 * g] = p.w_scales[(size_t)group * p.w_rows + at.w_row + t];
      if (present && t < NT && at.row + t < at.end) into[2 * g + 1] = p.x_scales[(size_t)group * p.m + at.row + t];
    }
  };
  // ahead of the block's first synchronisation: the barriers are this thread's own, the words lie in registers
  if (threadIdx.x == 0) {
    for (uint32_t s = 0; s < work.stages && stage0 + s < stage1; ++s) load(stage0 + s, s);
  } else if (warp == 1) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(base + behind + Z::kHolder), "r"(Z::kTmemColumns) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
  } else if (warp >= 2) {
#pragma unroll
    for (uint32_t a = 0; a < kAhead; ++a) fetch(stage0 + a, held[a]);
  }
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  __syncthreads();
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
  const uint32_t tmem_base = uniform(*holder);

  if (warp == 0) {
    bool ok = true;
    uint32_t s = 0, phase = 0, issued = min(work.stages, stage1 - stage0);
    for (uint32_t ks = stage0 + issued; ks < stage1; ++ks, ++issued) {
      ok = !*abort_flag && warp_wait(empty + s * 8, phase);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) {
        give_up();
        break;
      }
      if (elect_one()) load(ks, s);
      __syncwarp();
      if (++s == work.stages) s = 0, phase ^= 1u;
    }
    // on the way out after a failure the copies already started must land first
    if (!ok || *abort_flag)
      for (uint32_t i = issued > work.stages ? issued - work.stages : 0u; i < issued; ++i)
        barrier_wait(full + (i % work.stages) * 8, (i / work.stages) & 1u);
    __syncwarp();
  } else if (warp == 1) {
    const uint32_t rows = p.plan.tiles ? uniform(max((at.end - at.row + 15u) / 16u * 16u, 16u)) : NT;
    const uint32_t low = mxf4_instruction(rows, 0u), high = mxf4_instruction(rows, 1u);
    bool ok = true;
    uint32_t s = 0, phase = 0;
    for (uint32_t ks = stage0; ks < stage1; ++ks) {
      const uint32_t stage = base + s * Z::kStageBytes;
      ok = !*abort_flag && warp_wait(full + s * 8, phase) && warp_wait(scales_full + s * 8, phase);
      ok = __all_sync(0xffffffffu, ok);
      if (!ok) break;
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t scales = tmem_base + NT + (ks & 1u) * Z::kScaleColumns, left = p.k - ks * kDepth;
      const uint64_t a = operand_descriptor(stage), b = operand_descriptor(stage + Z::kWeightBytes);
      if (elect_one()) {
#pragma unroll
        for (uint32_t g = 0; g < kStageWords; ++g) {
          if (g * kWordValues >= left) break;
          copy_atom(scales + g * 8u, stage + Z::kScalesAt + 2u * g * kAtom);
          copy_atom(scales + g * 8u + 4u, stage + Z::kScalesAt + (2u * g + 1u) * kAtom);
        }
#pragma unroll
        for (uint32_t j = 0; j < kDepth / 64; ++j) {
          if (j * 64u >= left) break;
          const uint32_t columns = scales + j / 2u * 8u;
          mma_mxf4(tmem_base, a + j * 2u, b + j * 2u, j & 1u ? high : low, columns, columns + 4u, (ks > stage0 || j > 0) ? 1u : 0u);
        }
        mma_commit(empty + s * 8);
        if (ks + 1u == stage1) mma_commit(sums_full);
      }
      __syncwarp();
      if (++s == work.stages) s = 0, phase ^= 1u;
    }
    if (!ok) give_up();
  } else {
    const uint32_t target = (t & 31u) * 16u + (t >> 5) * 4u, last_mask = last_word_mask(p.k);  // a row's place in an atom
    bool ok = true;
    uint32_t s = 0, phase = 1;
    for (uint32_t first = stage0; first < stage1 && ok; first += kAhead) {
#pragma unroll
      for (uint32_t a = 0; a < kAhead; ++a) {
        const uint32_t ks = first + a;
        if (ks >= stage1 || !ok) break;
        ok = !*abort_flag && barrier_wait(empty + s * 8, phase);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        unsigned char* atoms = base_pointer + s * Z::kStageBytes + Z::kScalesAt + target;
#pragma unroll
        for (uint32_t w = 0; w < kStageWords * 2; ++w)
          *reinterpret_cast<uint32_t*>(atoms + w * kAtom) = held[a][w] & (ks * kStageWords + w / 2 + 1u == words ? last_mask : 0xffffffffu);
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
        __syncwarp();
        if (lane == 0) barrier_arrive(scales_full + s * 8);
        fetch(ks + kAhead, held[a]);
        if (++s == work.stages) s = 0, phase ^= 1u;
      }
    }
    if (ok) {
      ok = !*abort_flag && barrier_wait(sums_full, 0u);
      ok = __all_sync(0xffffffffu, ok);
    }
    if (!ok) {
      give_up();
    } else {
      asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
      const uint32_t quarter = warp & 3u, address = tmem_base + ((quarter * 32u) << 16);
#pragma unroll 1
      for (uint32_t piece = 0; piece < NT / Z::kPiece; ++piece) {
        const uint32_t row = at.row + piece * Z::kPiece;
        if (row >= at.end) break;
        uint32_t raw[Z::kPiece];
        if constexpr (Z::kPiece == 16) tmem_load_16(address + piece * Z::kPiece, raw);
        else tmem_load_32(address + piece * Z::kPiece, raw);
        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
        if (splits == 1u) {
          store_rows<S>(p, row, at.end, at.column + quarter * 32u + lane, raw);
        } else {
          // [row][column] of the partial sums, over the ring: every stage of it has been read
          float* partial = reinterpret_cast<float*>(base_pointer) + piece * Z::kPiece * kColumns + quarter * 32u + lane;
#pragma unroll
          for (uint32_t i = 0; i < Z::kPiece; ++i) partial[i * kColumns] = __uint_as_float(raw[i]);
        }
        __syncwarp();  // tcgen05.ld needs the whole warp
      }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
  }

  __syncthreads();
  // Before CTAs of a cluster wait for one another: one that waits for columns which another grid holds must not be waited for with these held.
  if (warp == 1) {
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(Z::kTmemColumns) : "memory");
  }
  if (splits == 1u) return;
  cluster_sync();
  // each CTA joins a share of the rows, always the partial sums of rank 0 first; a warp has 32 columns of two rows at a time
  const float* partial = reinterpret_cast<const float*>(base_pointer);
  const uint32_t pairs = (at.end - at.row + 1u) / 2u;
  for (uint32_t item = rank * (kThreads / 32u) + warp; item < pairs * 4u; item += splits * (kThreads / 32u)) {
    const uint32_t row = item / 4u * 2u, place = item % 4u * 32u + lane;
    float part[2][kMostSplits];
#pragma unroll
    for (uint32_t from = 0; from < kMostSplits; ++from)
#pragma unroll
      for (uint32_t i = 0; i < 2; ++i) part[i][from] = from < splits ? cluster_load(partial + (row + i) * kColumns + place, from) : 0.0f;
    uint32_t raw[2];
#pragma unroll
    for (uint32_t i = 0; i < 2; ++i) {
      float sum = part[i][0];
#pragma unroll
      for (uint32_t from = 1; from < kMostSplits; ++from)
        if (from < splits) sum += part[i][from];
      raw[i] = __float_as_uint(sum);
    }
    store_rows<S>(p, at.row + row, at.end, at.column + place, raw);
  }
  cluster_sync();  // nobody leaves while its sums are read
}

template <uint32_t NT, Store S>
int run(const KernelArgs& args, const Problem& p, uint32_t row_tiles) {
  using Z = Shape<NT>;
  const uint32_t sms = (uint32_t)context_sm_count(args.ctx), k_stages = (p.k + kDepth - 1u) / kDepth;
  Work work = {row_tiles, (p.n + kColumns - 1u) / kColumns, 1u, 0u, p.plan.tiles ? 16u : NT};
  const size_t tiles = (size_t)work.row_tiles * work.column_tiles;
  LLMOPT_REQUIRE(tiles < (1u << 28), "too many tiles");
  // CTAs that share a tile's k while the tiles leave SMs without work
  while (work.splits < kMostSplits && tiles * work.splits < 2u * (size_t)sms && k_stages >= work.splits * 4u) work.splits *= 2u;
  const uint32_t mine = (k_stages + work.splits - 1u) / work.splits;
  work.stages = mine < Z::kStages ? mine : Z::kStages;
  CUtensorMap map_w, map_x;
  LLMOPT_REQUIRE(make_map(&map_w, p.w, p.k, p.w_rows, kColumns) && make_map(&map_x, p.x, p.k, p.m, work.box_rows), "tensor map was refused");
  auto kernel = stream_kernel<NT, S>;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, Z::bytes(Z::kStages)) != cudaSuccess) {
    cudaGetLastError();
    return fail(args, "shared memory request was refused");
  }
  const dim3 grid((uint32_t)tiles * work.splits);
  if (work.splits == 1u)
    launch_kernel(args, kernel, grid, dim3(kThreads), Z::bytes(work.stages), map_w, map_x, p, work, context_device_error(args.ctx));
  else
    launch_cluster_kernel(args, kernel, grid, dim3(kThreads), Z::bytes(work.stages), work.splits, map_w, map_x, p, work,
                          context_device_error(args.ctx));
  return check_launch(args);
}

}  // namespace

namespace mxfp4 {

template <Store S>
int run_stream(const KernelArgs& args, const Problem& p, uint32_t plan_tiles) {
  const uint32_t row_tiles = p.plan.tiles ? plan_tiles : 1u;
  if (p.m <= 16u) return run<16, S>(args, p, row_tiles);
  if (p.m <= 32u) return run<32, S>(args, p, row_tiles);
  if (p.m <= 64u) return run<64, S>(args, p, row_tiles);
  return run<128, S>(args, p, row_tiles);
}

template int run_stream<kStoreHalf>(const KernelArgs&, const Problem&, uint32_t);
template int run_stream<kStoreBf16>(const KernelArgs&, const Problem&, uint32_t);
template int run_stream<kStoreFloat>(const KernelArgs&, const Problem&, uint32_t);
template int run_stream<kStorePairHalf>(const KernelArgs&, const Problem&, uint32_t);
template int run_stream<kStorePairBf16>(const KernelArgs&, const Problem&, uint32_t);

}  // namespace mxfp4
}  // namespace llmopt
