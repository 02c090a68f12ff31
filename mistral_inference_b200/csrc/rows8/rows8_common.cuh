// Rows of 8-bit numbers, shared by the kernels of libmb200_rows8.so.
//
// A row of K numbers is e4m3 codes, K rounded up to 128 of them (zeros behind the K-th), and a power of two for every 128: a number is its code times its block's power.
// e4m3 is a floating-point format, so a scale between two powers would gain nothing inside a block; and powers are what the tensor cores multiply by for nothing
// (tcgen05.mma.kind::mxf8f6f4 takes one for every row and 32 entries; here four of these are the same byte).
// Scales are 8-bit exponents (e8m0: byte b is 2^(b - 127)) in the order in which tensor memory holds them: tiles of 128 rows by 4 blocks, 512 bytes, row 32 j + i and block b
// at byte 16 i + 4 j + b; [row tiles][quads of blocks][512].  Places of no row or no block hold 127.
// A block that holds a NaN or an infinity is NaN as a whole (e4m3 has no infinity, and its largest code would pass for a number).
#pragma once
#include "../../../include/mistral_b200_rows8.h"
#include "../paged/paged_common.cuh"

namespace mb200 {

constexpr int R8_BLOCK = 128, R8_TILE = 512 /* bytes of scales of 128 rows and 4 blocks */;
constexpr uint32_t R8_ONES = 0x7f7f7f7fu;  // four scales of 1

inline int64_t r8_width(int64_t K) { return (K + R8_BLOCK - 1) / R8_BLOCK * R8_BLOCK; }
inline int64_t r8_quads(int64_t K) { return (K + 4 * R8_BLOCK - 1) / (4 * R8_BLOCK); }
// the byte of row r's first block of quad q
__device__ __forceinline__ int64_t r8_scale_at(int64_t r, int q, int quads) { return ((r >> 7) * quads + q) * R8_TILE + (r & 31) * 16 + ((r >> 5) & 3) * 4; }

// Exponent of a block whose largest magnitude has these bits, as its byte; what a code is multiplied by to give a number is 2^(byte - 127), the other way 2^(127 - byte).
__device__ __forceinline__ uint32_t r8_byte(uint32_t amax_bits) { return amax_bits < 0x7f800000u ? (uint32_t)(e4m3_exponent(__uint_as_float(amax_bits)) + 127) : 127u; }
__device__ __forceinline__ float r8_inverse(uint32_t byte) { return __uint_as_float((254u - byte) << 23); }  // (27 <= byte <= 247)

// 16 numbers, |x| <= 448 after the scale, as codes; all NaN where the block's largest magnitude is no number
__device__ __forceinline__ uint4 r8_codes16(const uint64_t (&v)[8], uint32_t amax_bits) {
  const float inverse = r8_inverse(r8_byte(amax_bits));
  const uint64_t scale = pair(inverse, inverse);
  uint32_t c[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const float2 x = unpair(mul_pair(v[2 * j], scale)), y = unpair(mul_pair(v[2 * j + 1], scale));
    c[j] = to_e4m3x2(x.x, x.y) | to_e4m3x2(y.x, y.y) << 16;
  }
  return amax_bits < 0x7f800000u ? make_uint4(c[0], c[1], c[2], c[3]) : make_uint4(R8_ONES, R8_ONES, R8_ONES, R8_ONES);  // (e4m3's NaN is 0x7f)
}
__device__ __forceinline__ uint4 r8_codes16(const float (&v)[16], uint32_t amax_bits) {
  uint64_t w[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) w[j] = pair(v[2 * j], v[2 * j + 1]);
  return r8_codes16(w, amax_bits);
}
__device__ __forceinline__ uint32_t r8_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }  // (as whole numbers magnitudes order like their values, infinity and NaN above all)
// the largest of a and two numbers' magnitudes; NaN where one is
__device__ __forceinline__ float r8_larger(float a, float x, float y) {
  float r;
  asm("max.NaN.abs.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(x), "f"(y));
  return r;
}

// 2-D map of codes [rows][width] with boxes of box_rows x 128, 128-byte swizzle
inline int r8_code_map(CUtensorMap* map, const void* codes, int64_t rows, int64_t width, int box_rows) {
  PFN_encodeTiled enc = get_encode_tiled();
  if (enc == nullptr) return fail(MB200_E_CUDA, "cuTensorMapEncodeTiled entry point not available");
  const cuuint64_t dims[2] = {(cuuint64_t)width, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)width};
  const cuuint32_t box[2] = {R8_BLOCK, (cuuint32_t)box_rows}, one[2] = {1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(codes), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? MB200_OK : fail(MB200_E_CUDA, "cuTensorMapEncodeTiled (codes) failed (%d)", (int)r);
}
// 3-D map of scales [row tiles][quads][128 words]: a box is the tiles of one quad of `box_tiles` x 128 rows
inline int r8_scale_map(CUtensorMap* map, const void* scales, int64_t rows, int64_t quads, int box_tiles) {
  PFN_encodeTiled enc = get_encode_tiled();
  if (enc == nullptr) return fail(MB200_E_CUDA, "cuTensorMapEncodeTiled entry point not available");
  const cuuint64_t dims[3] = {R8_TILE / 4, (cuuint64_t)quads, (cuuint64_t)((rows + 127) / 128)}, strides[2] = {R8_TILE, (cuuint64_t)quads * R8_TILE};
  const cuuint32_t box[3] = {R8_TILE / 4, 1, (cuuint32_t)box_tiles}, one[3] = {1, 1, 1};
  const CUresult r = enc(map, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<void*>(scales), dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                         CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? MB200_OK : fail(MB200_E_CUDA, "cuTensorMapEncodeTiled (scales) failed (%d)", (int)r);
}

}  // namespace mb200
