// Products of MXFP4 rows (mxfp4.cuh) with MXFP4 matrices:
//   llmopt_mxfp4_linear_{f16,bf16,f32}    [x codes, x scales, w codes, w scales, bias or any, out], {m, n, k, has bias}
//   llmopt_mxfp4_expert_rows_{f16,bf16}   [x codes, x scales, w codes, w scales, plan, score of every slot, out],
//                                         {slots, n, k, experts, paired}: rows sorted by expert (llmopt_route_plan)
#include "mxfp4_tc.cuh"

namespace llmopt {
namespace {
using namespace mxfp4;

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

template <Store S>
int run_product(const KernelArgs& args, const Problem& p, uint32_t plan_tiles) {
  LLMOPT_REQUIRE(args.ctx != nullptr, "needs a context");
  // Up to 64 rows the stream, us beside the tiles': 64 rows through 4096 x 14336 10.4, 12.2, k 14336 x 4096 12.7, 18.4; 32 sorted rows of 16 experts
  // through 4096 x 7168 25.7, 28.2.  Tiles that would be more than 13 CTAs for every two SMs go to the kernel whose CTAs stay for the next
  // (stream, tiles: 448 tiles, 32 rows through 4096 x 57344 26.7, 28.7; 896, 64 sorted rows through 4096 x 7168 37.2, 36.7; 1002, 4096 x 128256
  // 32 rows 53.6, 51.8, 64 rows 58.3, 54.4; 1024, 64 sorted rows of 64 experts 15.6, 14.8; 7168, 64 of 128 experts 110, 80), unless all read the
  // same rows and those are few (1 row through 4096 x 128256 48.8, 50.0, 16 rows 51.6, 51.1).  Between, by how the tiles fill the last round
  // of the stream's two CTAs per SM (32 and 64 rows, in another series): 512 tiles 28.0, 29.1 and 29.0, 29.6; 640 36.1, 35.4 and 37.8, 36.1; 768
  // 40.1, 41.1 and 41.9, 42.3; 896 47.2, 46.7 and 49.5, 48.2.  With small k the line would lie lower: k 1024, 64 rows, 448 10.9, 10.4, 896
  // 17.9, 15.8.
  const uint64_t tiles = (uint64_t)(p.plan.tiles ? plan_tiles : 1u) * ((p.n + kColumns - 1u) / kColumns);
  const bool few = tiles * 2u <= (uint64_t)context_sm_count(args.ctx) * 13u || (!p.plan.tiles && p.m <= 16u);
  return p.m <= 64u && few ? run_stream<S>(args, p, plan_tiles) : run_tiles<S>(args, p, plan_tiles);
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
