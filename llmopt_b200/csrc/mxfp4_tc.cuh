// What the MXFP4 products on tcgen05 share: operand and instruction forms, the way sums leave, tensor maps.
//
// y[m, n] = sum over blocks b of 2^(sx + sw - 254) (x block . w block): the tensor cores take both operands as they are held, 64 elements
// of k at a time with two powers of two per row (tcgen05.mma kind::mxf4), so no weight is ever converted.  The weights are the M side
// (128 rows of a tile are the lanes of tensor memory, one output column each), the rows of x the N side: one token costs an N of 16,
// and a ragged tile of an expert costs its rows rounded up to 16.
#pragma once
#include <cuda.h>

#include <atomic>

#include "mxfp4.cuh"
#include "w4a16_tc_device.cuh"

namespace llmopt {

uint32_t* context_device_error(Context* ctx);
uint32_t context_mxfp4_wait_limit(Context* ctx);

namespace mxfp4 {
using namespace tc;

inline uint32_t* error_word_of(const KernelArgs& args) { return args.error_word ? args.error_word : context_device_error(args.ctx); }

constexpr uint32_t kColumns = 128;                              // weight rows of a tile
constexpr uint32_t kBoxDepth = 256, kRowBytes = kBoxDepth / 2;  // elements of k of a box of codes
constexpr uint32_t kAtom = 512;                                 // an atom: the words of 128 rows
constexpr uint32_t kScaleWarps = 4;                             // a warp per word of a stage

// One lane of a converged warp.  What the tensor cores and copies take lies in uniform registers: where the whole warp walks through a loop
// with values that are the same in all lanes and one lane issues, they are kept there; a loop that one lane walks through alone
// moves every operand over, which cost 750 to 1000 cycles per four products.
__device__ __forceinline__ bool elect_one() {
  uint32_t chosen;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(chosen));
  return chosen != 0;
}
__device__ __forceinline__ uint32_t uniform(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }
// A warp's wait, until all of its lanes have seen the phase end or looked `limit` times.  The limit is looked at after a look that was in vain:
// ahead of the first, which mostly is the last, it cost up to 3 % of a product (512 x 14336 x 4096 19.4, 20.0 us).
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, uint32_t limit = kWaitLimit) {
  uint32_t done = 0, looks = 0;
  do {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(bar), "r"(parity)
        : "memory");
  } while (!done && ++looks < limit);
  return __all_sync(0xffffffffu, done != 0u);
}

__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }

// kind::mxf4, e2m1 A and B (format 1), e8m0 scales, both K-major; `pair` picks the half of a scale word.
__device__ __forceinline__ uint32_t mxf4_instruction(uint32_t m, uint32_t n, uint32_t pair) {
  return (pair << 5) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | (1u << 23) | ((m >> 4) << 24) | (pair << 30);
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
// An atom (32 rows of 16 bytes, unswizzled, eight rows every 128 bytes) to four columns, the same in all four quarters of the lanes.  Scale
// operands start at multiples of four columns.
__device__ __forceinline__ uint64_t atom_descriptor(uint32_t shared_address) {
  constexpr uint64_t kForm = (uint64_t)(128 >> 4) << 16 | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
  return kForm | (uint64_t)((shared_address & 0x3ffffu) >> 4);
}
__device__ __forceinline__ void copy_atom(uint32_t columns, uint32_t shared_address) {
  asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(columns), "l"(atom_descriptor(shared_address)) : "memory");
}

enum Store : uint32_t { kStoreHalf, kStoreBf16, kStoreFloat, kStorePairHalf, kStorePairBf16 };
template <Store S> struct Element { typedef float Type; };
template <> struct Element<kStoreHalf> { typedef __half Type; };
template <> struct Element<kStorePairHalf> { typedef __half Type; };
template <> struct Element<kStoreBf16> { typedef bf16 Type; };
template <> struct Element<kStorePairBf16> { typedef bf16 Type; };

__device__ __forceinline__ uint32_t packed(__half a, __half b) { return (uint32_t)__half_as_ushort(a) | (uint32_t)__half_as_ushort(b) << 16; }
__device__ __forceinline__ uint32_t packed(bf16 a, bf16 b) { return (uint32_t)__bfloat16_as_ushort(a) | (uint32_t)__bfloat16_as_ushort(b) << 16; }

// silu(gate) up: gate up / (1 + t^3) with t = e^(-|gate| / 3), below zero times t^3.  Its exponential and quotient are off by a few steps of
// fp32: of a result in sixteen bits that is nothing, and with the exact quotient the pairs of a tile took longer than its products (9.0
// against 5.2 us).  Far below zero silu leaves fp32's normal numbers, where `up` may bring it back: so every t is a factor of its own, and
// either side has one ahead of their product, which leaves fp32's range only if the result does.  t stays normal down to a gate of
// -262, where nothing that fp32 holds is left of the product.  us of 4096 sorted rows through 4096 x 7168: 73.5; with the square of
// e^(gate / 2), which needs subnormal numbers, 74.9; silu by itself, zero from -87 on, 72.2.
__device__ __forceinline__ float silu_pair(float gate, float up) {
  float t, inverse;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(t) : "f"(fabsf(gate) * -0.48089834696f));  // log2(e) / 3
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(inverse) : "f"(fmaf(t * t, t, 1.0f)));
  const float factor = gate < 0.0f ? t : 1.0f;
  return (gate * inverse * factor) * (up * factor) * factor;
}

// Sums of COUNT rows from `row` on, of the output column that is this lane's, and its bias: fp32.
template <int COUNT>
__device__ __forceinline__ void store_floats(const Problem& p, uint32_t row, uint32_t end, uint32_t column, const uint32_t (&raw)[COUNT], float bias) {
  if (column >= p.n) return;
  float* out = reinterpret_cast<float*>(p.out) + (size_t)row * p.n + column;
  if (row + COUNT <= end) {
#pragma unroll
    for (int i = 0; i < COUNT; ++i, out += p.n) *out = __uint_as_float(raw[i]) + bias;
    return;
  }
#pragma unroll
  for (int i = 0; i < COUNT; ++i, out += p.n)
    if (row + i < end) *out = __uint_as_float(raw[i]) + bias;
}

// The same in any type, on their way out; the whole warp takes part.  Sixteen-bit
// results go two columns at a time: neighbouring lanes exchange the sums of every other row.
template <Store S, int COUNT>
__device__ __forceinline__ void store_rows(const Problem& p, uint32_t row, uint32_t end, uint32_t column, const uint32_t (&raw)[COUNT]) {
  typedef typename Element<S>::Type T;
  const bool odd = threadIdx.x & 1u;
  if constexpr (S == kStoreFloat) {
    store_floats(p, row, end, column, raw, p.bias && column < p.n ? reinterpret_cast<const float*>(p.bias)[column] : 0.0f);
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
      if (row + i >= end) break;  // the same for the whole warp
      const uint32_t away = __shfl_xor_sync(0xffffffffu, odd ? raw[i] : raw[i + 1], 1);
      const float first = __uint_as_float(odd ? away : raw[i]), second = __uint_as_float(odd ? raw[i + 1] : away);
      const uint32_t at = row + i + (odd ? 1 : 0);
      if (at >= end || even_column >= p.n) continue;
      if constexpr (kPair) {
        const float scale = p.row_scale[at];
        reinterpret_cast<T*>(p.out)[(size_t)at * (p.n / 2u) + even_column / 2u] = from_float<T>(silu_pair(first * scale, second * scale));
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

constexpr uint32_t kStagingRow = 80, kStagingBytes = 32 * kStagingRow;  // a warp's 32 rows of 64 bytes and 16 of padding

template <Store S> constexpr bool kPaired = S == kStorePairHalf || S == kStorePairBf16;

// What a lane brings to a piece of up to 32 rows from `row` on and the warp's 32 columns: of pairs the score of its row, otherwise the bias of
// its column, whatever the row.  Asked for ahead of the sums.
template <Store S>
__device__ __forceinline__ float piece_operand(const Problem& p, uint32_t row, uint32_t end, uint32_t column0) {
  const uint32_t lane = threadIdx.x & 31u;
  if constexpr (kPaired<S>) return row + lane < end ? p.row_scale[row + lane] : 0.0f;
  return p.bias && column0 + lane < p.n ? as_float(reinterpret_cast<const typename Element<S>::Type*>(p.bias)[column0 + lane]) : 0.0f;
}

// Results of sixteen bits of such a piece's `rows` rows, rounded up to eights, to shared memory, STRIDE bytes a row.  A test per row kept the
// rows' chains of operations apart: 2 us a piece of pairs, where eight rows at a time take less than a tile's products.
template <Store S, uint32_t STRIDE, uint32_t COUNT>
__device__ __forceinline__ void stage_piece(uint32_t rows, const uint32_t (&raw)[COUNT], float own, unsigned char* staging) {
  typedef typename Element<S>::Type T;
  const uint32_t lane = threadIdx.x & 31u;
  if constexpr (kPaired<S>) {
    const bool odd = lane & 1u;
#pragma unroll
    for (uint32_t i = 0; i < COUNT; i += 2) {
      if (i % 8u == 0 && i >= rows) break;  // the same for the whole warp
      const uint32_t away = __shfl_xor_sync(0xffffffffu, odd ? raw[i] : raw[i + 1], 1), at = i + (odd ? 1u : 0u);
      const float scale = __shfl_sync(0xffffffffu, own, at);
      const float gate = __uint_as_float(odd ? away : raw[i]) * scale, up = __uint_as_float(odd ? raw[i + 1] : away) * scale;
      *reinterpret_cast<T*>(staging + at * STRIDE + lane / 2u * 2u) = from_float<T>(silu_pair(gate, up));
    }
  } else {
#pragma unroll
    for (uint32_t i = 0; i < COUNT; ++i) {
      if (i % 8u == 0 && i >= rows) break;  // the same for the whole warp
      *reinterpret_cast<T*>(staging + i * STRIDE + lane * 2u) = from_float<T>(__uint_as_float(raw[i]) + own);
    }
  }
}

// Staged rows to `out`, whose rows are `stride` elements apart: lanes share the 64 bytes (of pairs 32) of a row, a V of them each.  With eight
// values per lane whatever the alignment, stored one by one, 3209 x 256 x 7126 took 114 us, with a V that fits 31 (7128 columns, in boxes: 16).
template <Store S, typename V, uint32_t COUNT, typename T>
__device__ __forceinline__ void unstage_piece(T* out, uint32_t stride, uint32_t rows, uint32_t width, const unsigned char* staging) {
  constexpr uint32_t kValues = sizeof(V) / 2, kLanes = (kPaired<S> ? 16 : 32) / kValues;  // of a V; of a row
  const uint32_t lane = threadIdx.x & 31u, first = lane % kLanes * kValues;
#pragma unroll
  for (uint32_t i = 0; i < COUNT * kLanes / 32; ++i) {
    const uint32_t at = i * (32u / kLanes) + lane / kLanes;
    if (at < rows && first < width)
      *reinterpret_cast<V*>(out + (size_t)at * stride + first) = *reinterpret_cast<const V*>(staging + at * kStagingRow + first * 2u);
  }
}

// A piece on its way out.
template <Store S, uint32_t COUNT>
__device__ __forceinline__ void store_piece(const Problem& p, uint32_t row, uint32_t end, uint32_t column0, const uint32_t (&raw)[COUNT], float own,
                                            unsigned char* staging) {
  typedef typename Element<S>::Type T;
  const uint32_t lane = threadIdx.x & 31u;
  if constexpr (S == kStoreFloat) {
    store_floats(p, row, end, column0 + lane, raw, own);
  } else {
    stage_piece<S, kStagingRow>(end - row, raw, own, staging);
    __syncwarp();
    const uint32_t columns = kPaired<S> ? p.n / 2u : p.n, column = kPaired<S> ? column0 / 2u : column0;
    T* const out = reinterpret_cast<T*>(p.out) + (size_t)row * columns + column;
    const uint32_t rows = min(end - row, COUNT), width = column < columns ? columns - column : 0u;
    if (columns % 8u == 0 && ((uintptr_t)p.out & 15u) == 0) unstage_piece<S, uint4, COUNT>(out, columns, rows, width, staging);
    else if (columns % 2u == 0 && ((uintptr_t)p.out & 3u) == 0) unstage_piece<S, uint32_t, COUNT>(out, columns, rows, width, staging);
    else unstage_piece<S, uint16_t, COUNT>(out, columns, rows, width, staging);
    __syncwarp();  // read before the next piece
  }
}

// Rows of x that a tile multiplies, its first weight row, and the output column of that row.
struct Place {
  uint32_t row, end, w_row, column;
};
// Tiles have at most `rows` rows; the plan's have no more of them than that.
__device__ __forceinline__ Place place_of(const Problem& p, uint32_t row_tile, uint32_t rows, uint32_t column) {
  if (!p.plan.tiles) return {row_tile * rows, min(p.m, (row_tile + 1u) * rows), column, column};
  const DenseTile tile = dense_tile(p.plan, row_tile);  // whatever the plan says: rows that are there, and no more than a tile's
  const uint32_t row = min(tile.first, p.m), end = max(row, min(min(tile.end, p.m), row + rows));
  return {row, end, min(tile.expert, p.plan.experts - 1u) * p.n + column, column};
}
// Bytes of the last word that lie behind k hold no exponents.
__device__ __forceinline__ uint32_t last_word_mask(uint32_t k) {
  return k % kWordValues ? (1u << (k % kWordValues / kBlock * 8u)) - 1u : 0xffffffffu;
}

typedef CUresult (*EncodeTiled)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*, const cuuint32_t*,
                                const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// Rows of `inner` elements in boxes of box_inner x box_rows.
inline bool make_map(CUtensorMap* map, CUtensorMapDataType type, uint32_t size, const void* base, uint64_t inner, uint64_t rows, uint32_t box_inner,
                     uint32_t box_rows, CUtensorMapSwizzle swizzle) {
  static EncodeTiled encode = []() -> EncodeTiled {
    void* pointer = nullptr;
    cudaDriverEntryPointQueryResult result;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &pointer, cudaEnableDefault, &result) != cudaSuccess ||
        result != cudaDriverEntryPointSuccess)
      return nullptr;
    return reinterpret_cast<EncodeTiled>(pointer);
  }();
  if (encode == nullptr) return false;
  const cuuint64_t dims[2] = {inner, rows}, strides[1] = {inner * size};
  const cuuint32_t box[2] = {box_inner, box_rows}, element_strides[2] = {1, 1};
  auto made = [&] {
    return encode(map, type, 2, const_cast<void*>(base), dims, strides, box, element_strides, CU_TENSOR_MAP_INTERLEAVE_NONE, swizzle,
                  CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
  };
  if (made()) return true;
  // a thread that has called nothing yet has no context, which this call does not give it
  int device = 0;
  return cudaGetDevice(&device) == cudaSuccess && cudaSetDevice(device) == cudaSuccess && made();
}
// Codes [rows, k / 2] read in boxes of 128 bytes x `box_rows` with the 128-byte swizzle; absent bytes read zero.
inline bool make_map(CUtensorMap* map, const void* codes, uint64_t k, uint64_t rows, uint32_t box_rows) {
  return make_map(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 1u, codes, k / 2, rows, kRowBytes, box_rows, CU_TENSOR_MAP_SWIZZLE_128B);
}

// Lets a kernel have as much shared memory as any launch of it asks for: the limit is one per kernel and device, whoever launches it, and the
// call that sets it takes 0.3 us, so it is made once.
template <auto KERNEL, uint32_t BYTES>
bool allow_shared() {
  static std::atomic<uint64_t> allowed{0};  // a bit per device
  int device = 0;
  if (cudaGetDevice(&device) != cudaSuccess) return false;
  const uint64_t bit = device < 64 ? 1ull << device : 0ull;
  if (allowed.load(std::memory_order_relaxed) & bit) return true;
  if (cudaFuncSetAttribute(KERNEL, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)BYTES) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  allowed.fetch_or(bit, std::memory_order_relaxed);
  return true;
}

inline uint32_t most_plan_tiles(uint32_t slots, uint32_t experts) { return slots / kExpertTile + (slots < experts ? slots : experts); }

// Few rows: every weight is read once and what counts is how fast (mxfp4_stream.cu).  Many: mxfp4_tiles.cu.  row_tiles: those of the
// plan there can be.
template <Store S> int run_stream(const KernelArgs& args, const Problem& p, uint32_t row_tiles);
template <Store S> int run_tiles(const KernelArgs& args, const Problem& p, uint32_t row_tiles);

}  // namespace mxfp4
}  // namespace llmopt
