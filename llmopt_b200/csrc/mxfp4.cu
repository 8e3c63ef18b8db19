// MXFP4 (mxfp4.cuh) on the device: rows into codes and exponents, and back.
//   llmopt_mxfp4_quantize_{f16,bf16,f32}       [x, codes, scales], {rows, k, stride of x}
//   llmopt_mxfp4_quantize_rows_{f16,bf16,f32}  [x, row of every slot, codes, scales], {slots, k, stride, rows of x}: the rows that
//                                              routed experts read, in the order of llmopt_route_plan
//   llmopt_mxfp4_dequantize_{f16,bf16,f32}     [codes, scales, out], {rows, k}
//
// s - 127 = floor(log2 of the block's largest size) - 2, which puts that one at 4 to 8 units of it: beyond 6 it saturates, as the
// specification has it.  The quotient is exact (a power of two), its rounding to e2m1 is to nearest, ties to even.  A block with an
// infinity or a NaN becomes one of NaNs.
#include "mxfp4.cuh"

namespace llmopt {
namespace {
using namespace mxfp4;

constexpr uint32_t kTileRows = 32, kTileColumns = 256, kWarps = 8, kRowsPerWarp = kTileRows / kWarps;

// Eight values of a row as floats.
template <typename T>
__device__ __forceinline__ void load_eight(const T* source, bool vectors, float (&v)[8]) {
  if (vectors) {
    constexpr int kLoads = sizeof(T) / 2;
    uint4 raw[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) raw[i] = reinterpret_cast<const uint4*>(source)[i];
    const T* values = reinterpret_cast<const T*>(raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = as_float(values[i]);
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) v[i] = as_float(source[i]);
}

// A CTA takes 32 rows x 256 columns, a warp four of the rows, a lane eight neighbouring values.  Four lanes share a block, sixteen a
// word of exponents; the words of the 32 rows leave together.
template <typename T, bool GATHER>
__global__ void __launch_bounds__(kWarps * 32) quantize_kernel(const T* x, const uint32_t* index, uint8_t* codes, uint32_t* scales, uint32_t rows,
                                                               uint32_t source_rows, uint32_t k, size_t stride, bool vectors) {
  grid_chain_prologue();
  __shared__ uint32_t words[2][kTileRows];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const uint32_t row0 = blockIdx.x * kTileRows, column = blockIdx.y * kTileColumns + lane * 8u;
  float v[kRowsPerWarp][8];
#pragma unroll
  for (uint32_t i = 0; i < kRowsPerWarp; ++i) {
    const uint32_t row = row0 + warp + i * kWarps;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[i][j] = 0.0f;
    if (row < rows && column < k) {
      const uint32_t source = GATHER ? min(index[row], source_rows - 1u) : row;  // whatever the index says
      load_eight(x + source * stride + column, vectors, v[i]);
    }
  }
#pragma unroll
  for (uint32_t i = 0; i < kRowsPerWarp; ++i) {
    const uint32_t at = warp + i * kWarps, row = row0 + at;
    uint32_t most = 0;  // sizes compare as integers, NaN above infinity
#pragma unroll
    for (int j = 0; j < 8; ++j) most = max(most, __float_as_uint(v[i][j]) & 0x7fffffffu);
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
    const bool number = most < 0x7f800000u;
    const uint32_t s = number ? max(most >> 23, 2u) - 2u : 255u;
    const float inverse = __uint_as_float((254u - min(s, 253u)) << 23);
    uint32_t packed = 0;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      uint32_t pair;
      asm("{\n\t.reg .b8 b, z;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %2, %1;\n\tmov.b32 %0, {b, z, z, z};\n\t}"
          : "=r"(pair)
          : "f"(v[i][2 * j] * inverse), "f"(v[i][2 * j + 1] * inverse));
      packed |= (pair & 255u) << (8 * j);
    }
    if (row < rows && column < k) *reinterpret_cast<uint32_t*>(codes + (size_t)row * (k / 2u) + column / 2u) = number ? packed : 0u;
    uint32_t word = column < k ? s << (8u * (lane >> 2 & 3u)) : 0u;
    word |= __shfl_xor_sync(0xffffffffu, word, 4);
    word |= __shfl_xor_sync(0xffffffffu, word, 8);
    if ((lane & 15u) == 0u) words[lane >> 4][at] = word;
  }
  __syncthreads();
  const uint32_t group = blockIdx.y * 2u + (threadIdx.x >> 5), row = row0 + lane;
  if (threadIdx.x < 64u && group < words_of(k) && row < rows) scales[(size_t)group * rows + row] = words[threadIdx.x >> 5][lane];
}

template <typename T>
__device__ __forceinline__ void store_eight(T* target, const float (&v)[8], bool vectors) {
  constexpr int kStores = sizeof(T) / 2;
  uint4 raw[kStores];
  T* values = reinterpret_cast<T*>(raw);
#pragma unroll
  for (int i = 0; i < 8; ++i) values[i] = from_float<T>(v[i]);
  if (vectors) {
#pragma unroll
    for (int i = 0; i < kStores; ++i) reinterpret_cast<uint4*>(target)[i] = raw[i];
    return;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) target[i] = values[i];
}

// The same tiles the other way.  A value has two significant bits, so its product with the power of two is exact in fp32 and leaves
// with the one rounding of its type.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32) dequantize_kernel(const uint8_t* codes, const uint32_t* scales, T* out, uint32_t rows, uint32_t k,
                                                                 bool vectors) {
  grid_chain_prologue();
  __shared__ uint32_t words[2][kTileRows];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const uint32_t row0 = blockIdx.x * kTileRows, column = blockIdx.y * kTileColumns + lane * 8u;
  uint32_t packed[kRowsPerWarp];
#pragma unroll
  for (uint32_t i = 0; i < kRowsPerWarp; ++i) {
    const uint32_t row = row0 + warp + i * kWarps;
    packed[i] = row < rows && column < k ? *reinterpret_cast<const uint32_t*>(codes + (size_t)row * (k / 2u) + column / 2u) : 0u;
  }
  const uint32_t group = blockIdx.y * 2u + warp;
  if (warp < 2u) words[warp][lane] = group < words_of(k) && row0 + lane < rows ? scales[(size_t)group * rows + row0 + lane] : 0u;
  __syncthreads();
#pragma unroll
  for (uint32_t i = 0; i < kRowsPerWarp; ++i) {
    const uint32_t at = warp + i * kWarps, row = row0 + at;
    if (row >= rows || column >= k) continue;
    const float scale = scale_value(words[lane >> 4][at] >> (8u * (lane >> 2 & 3u)) & 255u);
    float v[8];
    elements(packed[i], v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] *= scale;
    store_eight(out + (size_t)row * k + column, v, vectors);
  }
}

bool aligned(const void* pointer) { return ((uintptr_t)pointer & 15u) == 0; }

// Rows and k that every launch here takes: whole blocks, grids that fit.
int check_rows(const KernelArgs& args, uint32_t rows, uint32_t k) {
  LLMOPT_REQUIRE(k > 0 && k % kBlock == 0, "k must be a positive multiple of 32");
  LLMOPT_REQUIRE(k <= (1u << 23), "k is too large");
  LLMOPT_REQUIRE(rows < (1u << 31), "too many rows");
  return 0;
}
dim3 tiles_of(uint32_t rows, uint32_t k) { return dim3((rows + kTileRows - 1u) / kTileRows, (k + kTileColumns - 1u) / kTileColumns); }

template <typename T, bool GATHER>
int launch_quantize(const KernelArgs& args) {
  LLMOPT_REQUIRE(args.buffer_count == (GATHER ? 4 : 3) && args.param_bytes == (GATHER ? 16 : 12),
                 GATHER ? "expects 4 buffers and 16 parameter bytes" : "expects 3 buffers and 12 parameter bytes");
  const uint32_t rows = param_u32(args, 0), k = param_u32(args, 1), stride = param_u32(args, 2), source_rows = GATHER ? param_u32(args, 3) : rows;
  const int codes = GATHER ? 2 : 1;
  if (const int status = check_rows(args, rows, k)) return status;
  LLMOPT_REQUIRE(stride >= k, "the rows of x overlap");
  LLMOPT_REQUIRE(rows == 0 || source_rows > 0, "no rows to gather from");
  if (rows == 0) return 0;
  LLMOPT_REQUIRE(args.lengths[0] / sizeof(T) >= (size_t)(source_rows - 1u) * stride + k && (!GATHER || args.lengths[1] >= (size_t)rows * 4) &&
                     args.lengths[codes] >= (size_t)rows * (k / 2u) && args.lengths[codes + 1] >= (size_t)rows * words_of(k) * 4,
                 "buffer is too short");
  LLMOPT_REQUIRE(aligned(args.buffers[codes]) && ((uintptr_t)args.buffers[codes + 1] & 3u) == 0, "codes must be 16-byte aligned, scales 4-byte");
  LLMOPT_REQUIRE(((uintptr_t)args.buffers[0] & (sizeof(T) - 1)) == 0 && (!GATHER || ((uintptr_t)args.buffers[1] & 3u) == 0),
                 "x and the rows must lie at multiples of their element");
  const bool vectors = aligned(args.buffers[0]) && stride * sizeof(T) % 16u == 0;
  launch_kernel(args, quantize_kernel<T, GATHER>, tiles_of(rows, k), dim3(kWarps * 32), 0, (const T*)args.buffers[0],
                GATHER ? (const uint32_t*)args.buffers[1] : nullptr, (uint8_t*)args.buffers[codes], (uint32_t*)args.buffers[codes + 1], rows,
                source_rows, k, (size_t)stride, vectors);
  return check_launch(args);
}

template <typename T>
int launch_dequantize(const KernelArgs& args) {
  LLMOPT_REQUIRE(args.buffer_count == 3 && args.param_bytes == 8, "expects 3 buffers and 8 parameter bytes");
  const uint32_t rows = param_u32(args, 0), k = param_u32(args, 1);
  if (const int status = check_rows(args, rows, k)) return status;
  if (rows == 0) return 0;
  LLMOPT_REQUIRE(args.lengths[0] >= (size_t)rows * (k / 2u) && args.lengths[1] >= (size_t)rows * words_of(k) * 4 &&
                     args.lengths[2] / sizeof(T) >= (size_t)rows * k,
                 "buffer is too short");
  LLMOPT_REQUIRE(aligned(args.buffers[0]) && ((uintptr_t)args.buffers[1] & 3u) == 0, "codes must be 16-byte aligned, scales 4-byte");
  LLMOPT_REQUIRE(((uintptr_t)args.buffers[2] & (sizeof(T) - 1)) == 0, "out must lie at a multiple of its element");
  launch_kernel(args, dequantize_kernel<T>, tiles_of(rows, k), dim3(kWarps * 32), 0, (const uint8_t*)args.buffers[0],
                (const uint32_t*)args.buffers[1], (T*)args.buffers[2], rows, k, aligned(args.buffers[2]));
  return check_launch(args);
}

}  // namespace

template <typename T>
int launch_mxfp4_linear(const KernelArgs& args);
template <typename T>
int launch_mxfp4_expert_rows(const KernelArgs& args);

const NamedLauncher* mxfp4_launchers(size_t* count) {
  static const NamedLauncher table[] = {
      {"llmopt_mxfp4_quantize_f16", launch_quantize<__half, false>},
      {"llmopt_mxfp4_quantize_bf16", launch_quantize<bf16, false>},
      {"llmopt_mxfp4_quantize_f32", launch_quantize<float, false>},
      {"llmopt_mxfp4_quantize_rows_f16", launch_quantize<__half, true>},
      {"llmopt_mxfp4_quantize_rows_bf16", launch_quantize<bf16, true>},
      {"llmopt_mxfp4_quantize_rows_f32", launch_quantize<float, true>},
      {"llmopt_mxfp4_dequantize_f16", launch_dequantize<__half>},
      {"llmopt_mxfp4_dequantize_bf16", launch_dequantize<bf16>},
      {"llmopt_mxfp4_dequantize_f32", launch_dequantize<float>},
      {"llmopt_mxfp4_linear_f16", launch_mxfp4_linear<__half>},
      {"llmopt_mxfp4_linear_bf16", launch_mxfp4_linear<bf16>},
      {"llmopt_mxfp4_linear_f32", launch_mxfp4_linear<float>},
      {"llmopt_mxfp4_expert_rows_f16", launch_mxfp4_expert_rows<__half>},
      {"llmopt_mxfp4_expert_rows_bf16", launch_mxfp4_expert_rows<bf16>},
  };
  *count = sizeof(table) / sizeof(table[0]);
  return table;
}

}  // namespace llmopt
