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

// 32-bit values are bound by HBM, 16-bit ones by their instructions (61 % of the issue slots), few rows by the launch: 14336 x 4096 fp32 into
// codes 45 us, 5.7 TB/s, and back 45 to 49, 5.1 to 5.7; 4096 rows gathered from 2048 x 4096 bf16 10.0, and back 9.5, one behind the other 16.5;
// 1 x 4096 2.6, and back beside it.  All of a CTA's values are asked for before the first is looked at.
// A CTA takes 32 rows x 256 columns, a warp four of the rows, 16 bytes of values per lane and access: 256 columns of 16 bits at a
// time, 128 of 32.  The exponents of the 32 rows leave together, 128 bytes of a word's row.
constexpr uint32_t kTileRows = 32, kTileColumns = 256, kWarps = 8, kRowsPerWarp = kTileRows / kWarps;
template <typename T>
struct Access {
  static constexpr uint32_t kValues = 16 / sizeof(T), kColumns = 32 * kValues, kPasses = kTileColumns / kColumns;
  static constexpr uint32_t kBlockLanes = kBlock / kValues, kWordLanes = kWordValues / kValues;
};

template <typename T>
__device__ __forceinline__ uint4 load_values(const T* source, bool vectors) {
  if (vectors) return *reinterpret_cast<const uint4*>(source);
  uint4 raw;
  T* const values = reinterpret_cast<T*>(&raw);
#pragma unroll
  for (uint32_t i = 0; i < Access<T>::kValues; ++i) values[i] = source[i];
  return raw;
}
// The largest size among a lane's values, as the bits of a float: sizes compare as integers, NaN above infinity.  Sixteen-bit types
// compare two at a time and by themselves.
__device__ __forceinline__ uint32_t largest_pair(const uint4& raw) {
  uint32_t most = raw.x & 0x7fff7fffu;
  asm("max.u16x2 %0, %0, %1;" : "+r"(most) : "r"(raw.y & 0x7fff7fffu));
  asm("max.u16x2 %0, %0, %1;" : "+r"(most) : "r"(raw.z & 0x7fff7fffu));
  asm("max.u16x2 %0, %0, %1;" : "+r"(most) : "r"(raw.w & 0x7fff7fffu));
#pragma unroll
  for (uint32_t offset = 1; offset < Access<__half>::kBlockLanes; offset <<= 1) {
    const uint32_t other = __shfl_xor_sync(0xffffffffu, most, offset);
    asm("max.u16x2 %0, %0, %1;" : "+r"(most) : "r"(other));
  }
  return max(most & 0xffffu, most >> 16);
}
__device__ __forceinline__ uint32_t largest(const uint4& raw, __half) {
  return __float_as_uint(__half2float(__ushort_as_half((uint16_t)largest_pair(raw))));
}
__device__ __forceinline__ uint32_t largest(const uint4& raw, bf16) { return largest_pair(raw) << 16; }
__device__ __forceinline__ uint32_t largest(const uint4& raw, float) {
  uint32_t most = max(max(raw.x & 0x7fffffffu, raw.y & 0x7fffffffu), max(raw.z & 0x7fffffffu, raw.w & 0x7fffffffu));
#pragma unroll
  for (uint32_t offset = 1; offset < Access<float>::kBlockLanes; offset <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, offset));
  return most;
}
// Codes of eight or four values times `inverse`.
__device__ __forceinline__ uint32_t encode(const float (&v)[8], float inverse) {
  uint32_t codes;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\tcvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\tmov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(codes)
      : "f"(v[0] * inverse), "f"(v[1] * inverse), "f"(v[2] * inverse), "f"(v[3] * inverse), "f"(v[4] * inverse), "f"(v[5] * inverse),
        "f"(v[6] * inverse), "f"(v[7] * inverse));
  return codes;
}
__device__ __forceinline__ uint32_t encode(const float (&v)[4], float inverse) {
  uint16_t codes;
  asm("{\n\t.reg .b8 a, b;\n\tcvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\tmov.b16 %0, {a, b};\n\t}"
      : "=h"(codes)
      : "f"(v[0] * inverse), "f"(v[1] * inverse), "f"(v[2] * inverse), "f"(v[3] * inverse));
  return codes;
}
// The codes of a lane's values: four bytes of eight, two of four.
__device__ __forceinline__ void store_codes(uint8_t* target, uint32_t codes, __half) { *reinterpret_cast<uint32_t*>(target) = codes; }
__device__ __forceinline__ void store_codes(uint8_t* target, uint32_t codes, bf16) { *reinterpret_cast<uint32_t*>(target) = codes; }
__device__ __forceinline__ void store_codes(uint8_t* target, uint32_t codes, float) { *reinterpret_cast<uint16_t*>(target) = (uint16_t)codes; }
template <typename T>
__device__ __forceinline__ uint32_t load_codes(const uint8_t* source) {
  return sizeof(T) == 4 ? *reinterpret_cast<const uint16_t*>(source) : *reinterpret_cast<const uint32_t*>(source);
}

template <typename T, bool GATHER>
__global__ void __launch_bounds__(kWarps * 32, sizeof(T) == 4 ? 5 : 6)
quantize_kernel(const T* x, const uint32_t* index, uint8_t* codes, uint32_t* scales, uint32_t rows, uint32_t source_rows, uint32_t k, size_t stride,
                bool vectors) {
  using A = Access<T>;
  grid_chain_prologue();
  __shared__ uint32_t words[2][kTileRows];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const uint32_t row0 = blockIdx.x * kTileRows, column0 = blockIdx.y * kTileColumns + lane * A::kValues;
  uint4 raw[kRowsPerWarp][A::kPasses];
  uint32_t source[kRowsPerWarp];
#pragma unroll
  for (uint32_t i = 0; i < kRowsPerWarp; ++i) {
    const uint32_t row = row0 + warp + i * kWarps;
    source[i] = row < rows ? GATHER ? min(index[row], source_rows - 1u) : row : 0u;  // whatever the index says
  }
#pragma unroll
  for (uint32_t i = 0; i < kRowsPerWarp; ++i)
#pragma unroll
    for (uint32_t pass = 0; pass < A::kPasses; ++pass) {
      const uint32_t column = column0 + pass * A::kColumns;
      raw[i][pass] = make_uint4(0u, 0u, 0u, 0u);
      if (row0 + warp + i * kWarps < rows && column < k) raw[i][pass] = load_values(x + source[i] * stride + column, vectors);
    }
#pragma unroll
  for (uint32_t i = 0; i < kRowsPerWarp; ++i)
#pragma unroll
    for (uint32_t pass = 0; pass < A::kPasses; ++pass) {
      const uint32_t at = warp + i * kWarps, row = row0 + at, column = column0 + pass * A::kColumns;
      const T* const values = reinterpret_cast<const T*>(&raw[i][pass]);
      float v[A::kValues];
#pragma unroll
      for (uint32_t j = 0; j < A::kValues; ++j) v[j] = as_float(values[j]);
      const uint32_t most = largest(raw[i][pass], T{});
      const bool number = most < 0x7f800000u;
      const uint32_t s = number ? max(most >> 23, 2u) - 2u : 255u;
      const uint32_t packed = encode(v, __uint_as_float((254u - min(s, 253u)) << 23));
      if (row < rows && column < k) store_codes(codes + (size_t)row * (k / 2u) + column / 2u, number ? packed : 0u, T{});
      uint32_t word = column < k ? s << (8u * (lane / A::kBlockLanes & 3u)) : 0u;
#pragma unroll
      for (uint32_t offset = A::kBlockLanes; offset < A::kWordLanes; offset <<= 1) word |= __shfl_xor_sync(0xffffffffu, word, offset);
      if (lane % A::kWordLanes == 0u) words[pass * (A::kColumns / kWordValues) + lane / A::kWordLanes][at] = word;
    }
  __syncthreads();
  const uint32_t group = blockIdx.y * 2u + warp, row = row0 + lane;
  if (warp < 2u && group < words_of(k) && row < rows) scales[(size_t)group * rows + row] = words[warp][lane];
}

// The same tiles the other way.  A value has two significant bits, so its product with the power of two is exact in fp32 and leaves
// with the one rounding of its type.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32) dequantize_kernel(const uint8_t* codes, const uint32_t* scales, T* out, uint32_t rows, uint32_t k,
                                                                 bool vectors) {
  using A = Access<T>;
  grid_chain_prologue();
  __shared__ uint32_t words[2][kTileRows];
  const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31u;
  const uint32_t row0 = blockIdx.x * kTileRows, column0 = blockIdx.y * kTileColumns + lane * A::kValues;
  uint32_t packed[kRowsPerWarp][A::kPasses];
#pragma unroll
  for (uint32_t i = 0; i < kRowsPerWarp; ++i)
#pragma unroll
    for (uint32_t pass = 0; pass < A::kPasses; ++pass) {
      const uint32_t row = row0 + warp + i * kWarps, column = column0 + pass * A::kColumns;
      packed[i][pass] = row < rows && column < k ? load_codes<T>(codes + (size_t)row * (k / 2u) + column / 2u) : 0u;
    }
  const uint32_t group = blockIdx.y * 2u + warp;
  if (warp < 2u) words[warp][lane] = group < words_of(k) && row0 + lane < rows ? scales[(size_t)group * rows + row0 + lane] : 0u;
  __syncthreads();
#pragma unroll
  for (uint32_t i = 0; i < kRowsPerWarp; ++i)
#pragma unroll
    for (uint32_t pass = 0; pass < A::kPasses; ++pass) {
      const uint32_t at = warp + i * kWarps, row = row0 + at, column = column0 + pass * A::kColumns;
      if (row >= rows || column >= k) continue;
      const uint32_t word = words[pass * (A::kColumns / kWordValues) + lane / A::kWordLanes][at];
      const float scale = scale_value(word >> (8u * (lane / A::kBlockLanes & 3u)) & 255u);
      float v[A::kValues];
      elements(packed[i][pass], v);
      uint4 raw;
      T* const values = reinterpret_cast<T*>(&raw);
#pragma unroll
      for (uint32_t j = 0; j < A::kValues; ++j) values[j] = from_float<T>(v[j] * scale);
      T* const target = out + (size_t)row * k + column;
      if (vectors) {
        *reinterpret_cast<uint4*>(target) = raw;
      } else {
#pragma unroll
        for (uint32_t j = 0; j < A::kValues; ++j) target[j] = values[j];
      }
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
