// Products of MXFP4 rows (mxfp4.cuh) with MXFP4 matrices:
//   llmopt_mxfp4_linear_{f16,bf16,f32}    [x codes, x scales, w codes, w scales, bias or any, out], {m, n, k, has bias}
//   llmopt_mxfp4_expert_rows_{f16,bf16}   [x codes, x scales, w codes, w scales, plan, score of every slot, out],
//                                         {slots, n, k, experts, paired}: rows sorted by expert (llmopt_route_plan)
#include "mxfp4.cuh"

namespace llmopt {
namespace {
using namespace mxfp4;

constexpr uint32_t kTileM = 32, kTileN = 64, kDepth = 64;

// Sums in fp32 of values in fp32, a 32 x 64 tile per CTA.
template <typename T>
__global__ void __launch_bounds__(256) product_kernel(const Problem p, uint32_t most_tiles) {
  grid_chain_prologue();
  __shared__ float xs[kTileM][kDepth + 1], ws[kTileN][kDepth + 1];
  DenseTile rows = {0u, blockIdx.y * kTileM, p.m};
  if (p.plan.tiles) {
    const uint32_t parts = kExpertTile / kTileM, tile = blockIdx.y / parts;
    if (tile >= min(p.plan.tiles[0], most_tiles)) return;
    rows = dense_tile(p.plan, tile);
    rows.expert = min(rows.expert, p.plan.experts - 1u);
    rows.first += blockIdx.y % parts * kTileM;
    rows.end = min(rows.end, p.m);
    if (rows.first >= rows.end) return;
  }
  const uint32_t n0 = blockIdx.x * kTileN, w0 = rows.expert * p.n;
  const uint32_t r = threadIdx.x / 16u, c = threadIdx.x % 16u;  // rows r, r + 16; columns 4 c ..
  float sum[2][4] = {};
  for (uint32_t k0 = 0; k0 < p.k; k0 += kDepth) {
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < (kTileM + kTileN) * (kDepth / 8u); i += 256u) {
      const uint32_t at = i / (kDepth / 8u), k = k0 + i % (kDepth / 8u) * 8u;
      const bool of_x = at < kTileM;
      const uint32_t row = of_x ? rows.first + at : n0 + at - kTileM;
      float v[8] = {};
      if (k < p.k && row < (of_x ? rows.end : p.n)) {
        const size_t held = of_x ? row : w0 + row;
        elements(*reinterpret_cast<const uint32_t*>((of_x ? p.x : p.w) + held * (p.k / 2u) + k / 2u), v);
        const uint32_t word = of_x ? p.x_scales[(size_t)(k / kWordValues) * p.m + held] : p.w_scales[(size_t)(k / kWordValues) * p.w_rows + held];
        const float scale = scale_value(word >> (8u * (k / kBlock % 4u)) & 255u);
        for (int j = 0; j < 8; ++j) v[j] *= scale;
      }
      float* target = of_x ? &xs[at][k - k0] : &ws[at - kTileM][k - k0];
      for (int j = 0; j < 8; ++j) target[j] = v[j];
    }
    __syncthreads();
    for (uint32_t k = 0; k < kDepth; ++k)
      for (int i = 0; i < 2; ++i)
        for (int j = 0; j < 4; ++j) sum[i][j] = fmaf(xs[r + 16 * i][k], ws[4 * c + j][k], sum[i][j]);
  }
  for (int i = 0; i < 2; ++i) {
    const uint32_t row = rows.first + r + 16 * i;
    if (row >= rows.end) continue;
    for (int j = 0; j < 4; ++j) {
      const uint32_t column = n0 + 4 * c + j;
      if (column >= p.n) continue;
      if (p.paired) {
        if (j % 2) continue;
        const float scale = p.row_scale[row], gate = sum[i][j] * scale, up = sum[i][j + 1] * scale;
        reinterpret_cast<T*>(p.out)[(size_t)row * (p.n / 2u) + column / 2u] = from_float<T>(silu_f32(gate) * up);
      } else if (p.plan.tiles) {
        reinterpret_cast<float*>(p.out)[(size_t)row * p.n + column] = sum[i][j];
      } else {
        const float bias = p.bias ? as_float(reinterpret_cast<const T*>(p.bias)[column]) : 0.0f;
        reinterpret_cast<T*>(p.out)[(size_t)row * p.n + column] = from_float<T>(sum[i][j] + bias);
      }
    }
  }
}

uint32_t most_plan_tiles(uint32_t slots, uint32_t experts) { return slots / kExpertTile + (slots < experts ? slots : experts); }

// What both products ask of their operands.
int check_operands(const KernelArgs& args, const Problem& p) {
  LLMOPT_REQUIRE(p.n > 0 && p.k > 0 && p.k % kBlock == 0, "needs n > 0 and k a positive multiple of 32");
  LLMOPT_REQUIRE(p.k <= (1u << 23) && p.m < (1u << 31), "too many rows, or k is too large");
  LLMOPT_REQUIRE(args.lengths[0] >= (size_t)p.m * (p.k / 2u) && args.lengths[1] >= (size_t)p.m * words_of(p.k) * 4 &&
                     args.lengths[2] >= (size_t)p.w_rows * (p.k / 2u) && args.lengths[3] >= (size_t)p.w_rows * words_of(p.k) * 4,
                 "buffer is too short");
  LLMOPT_REQUIRE((((uintptr_t)p.x | (uintptr_t)p.w) & 15u) == 0 && (((uintptr_t)p.x_scales | (uintptr_t)p.w_scales) & 3u) == 0,
                 "codes must be 16-byte aligned, scales 4-byte");
  return 0;
}

template <typename T>
int run_product(const KernelArgs& args, const Problem& p, uint32_t most) {
  const uint32_t row_tiles = p.plan.tiles ? most * (kExpertTile / kTileM) : (p.m + kTileM - 1u) / kTileM;
  launch_kernel(args, product_kernel<T>, dim3((p.n + kTileN - 1u) / kTileN, row_tiles), dim3(256), 0, p, most);
  return check_launch(args);
}

Problem operands(const KernelArgs& args) {
  Problem p = {};
  p.x = (const uint8_t*)args.buffers[0], p.x_scales = (const uint32_t*)args.buffers[1];
  p.w = (const uint8_t*)args.buffers[2], p.w_scales = (const uint32_t*)args.buffers[3];
  p.m = param_u32(args, 0), p.n = param_u32(args, 1), p.k = param_u32(args, 2);
  return p;
}

}  // namespace

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
  return run_product<T>(args, p, 0);
}

template <typename T>
int launch_mxfp4_expert_rows(const KernelArgs& args) {
  LLMOPT_REQUIRE(args.buffer_count == 7 && args.param_bytes == 20, "expects 7 buffers and 20 parameter bytes");
  Problem p = operands(args);
  p.plan.tiles = (const uint32_t*)args.buffers[4], p.plan.experts = param_u32(args, 3), p.paired = param_u32(args, 4) != 0;
  p.row_scale = (const float*)args.buffers[5], p.out = args.buffers[6];
  LLMOPT_REQUIRE(p.plan.experts > 0 && p.plan.experts <= 8192u && (!p.paired || p.n % 2u == 0), "needs experts, at most 8192, and whole pairs");
  LLMOPT_REQUIRE((size_t)p.plan.experts * p.n < (1u << 31) && p.m < (1u << 30), "too many rows");
  p.w_rows = p.plan.experts * p.n;
  if (const int status = check_operands(args, p)) return status;
  const uint32_t most = most_plan_tiles(p.m, p.plan.experts);
  LLMOPT_REQUIRE(args.lengths[4] >= 16 * (1 + (size_t)most) && (!p.paired || args.lengths[5] >= (size_t)p.m * 4) &&
                     args.lengths[6] / (p.paired ? sizeof(T) : 4) >= (size_t)p.m * (p.paired ? p.n / 2u : p.n),
                 "buffer is too short");
  LLMOPT_REQUIRE(((uintptr_t)args.buffers[4] & 15u) == 0 && (!p.paired || ((uintptr_t)p.row_scale & 3u) == 0) &&
                     ((uintptr_t)p.out & (p.paired ? sizeof(T) - 1 : 3u)) == 0,
                 "the plan must be 16-byte aligned, scores and out lie at multiples of their element");
  if (p.m == 0) return 0;
  return run_product<T>(args, p, most);
}

template int launch_mxfp4_linear<__half>(const KernelArgs&);
template int launch_mxfp4_linear<bf16>(const KernelArgs&);
template int launch_mxfp4_linear<float>(const KernelArgs&);
template int launch_mxfp4_expert_rows<__half>(const KernelArgs&);
template int launch_mxfp4_expert_rows<bf16>(const KernelArgs&);

}  // namespace llmopt
