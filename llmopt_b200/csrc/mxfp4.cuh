// Microscaled 4-bit floating point (MXFP4) of the OCP Microscaling specification: what its kernels share.
//
// An element is e2m1 -- a sign, two bits of exponent, one of fraction: 0, 0.5, 1, 1.5, 2, 3, 4, 6 -- and the 32 elements of a
// block along k share a power of two, e8m0: value = element * 2^(s - 127), s = 255 is no number.
//   codes   u8 [rows, k / 2]            the element of even k in the low nibble
//   scales  u32 [ceil(k / 128), rows]   byte j of word (g, r): s of block 4 g + j of row r; bytes behind k are not read
// A word is a column of the tensor cores' scale operand, and the words of neighbouring rows are neighbours wherever a tile
// of rows begins, which rows sorted by expert need.
#pragma once
#include <cuda_fp16.h>

#include "dense_linear.cuh"

namespace llmopt {

template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }
__device__ __forceinline__ float as_float(__half v) { return __half2float(v); }

namespace mxfp4 {

constexpr uint32_t kBlock = 32, kWordValues = 128;

__host__ __device__ __forceinline__ uint32_t words_of(uint32_t k) { return (k + kWordValues - 1u) / kWordValues; }

// 2^(s - 127)
__device__ __forceinline__ float scale_value(uint32_t s) {
  return __uint_as_float(s == 255u ? 0x7fffffffu : s == 0u ? 0x00400000u : s << 23);
}

// COUNT elements, the first in the lowest nibble; halves hold them exactly.
template <uint32_t COUNT>
__device__ __forceinline__ void elements(uint32_t codes, float (&v)[COUNT]) {
#pragma unroll
  for (uint32_t i = 0; i < COUNT / 2; ++i) {
    uint32_t pair;
    asm("{\n\t.reg .b8 b0, b1, b2, b3;\n\tmov.b32 {b0, b1, b2, b3}, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b0;\n\t}" : "=r"(pair) : "r"(codes >> (8 * i)));
    const float2 both = __half22float2(*reinterpret_cast<const __half2*>(&pair));
    v[2 * i] = both.x, v[2 * i + 1] = both.y;
  }
}

// y = x . w^T (+ bias): x rows [m, k], w rows [n, k] (with a plan [experts, n, k]).
struct Problem {
  const uint8_t* x;
  const uint32_t* x_scales;
  const uint8_t* w;
  const uint32_t* w_scales;
  const void* bias;        // [n] in the type of the output; null: none
  const float* row_scale;  // paired: multiplies a row's sums
  void* out;
  uint32_t m, n, k, w_rows;  // w_rows: rows of w, all experts'
  DensePlan plan;            // rows sorted by expert
};

}  // namespace mxfp4
}  // namespace llmopt
