// MXFP4 on the device: blocks of 32 E2M1 values with one E8M0 (power of two) scale.
//
//   codes   [rows][n_blocks * 16] bytes, element 2j of a row in the low nibble of byte j, 2j + 1 in the high one.
//           A code is a sign bit and a magnitude 0..7 that stands for 0, 0.5, 1, 1.5, 2, 3, 4, 6.
//   scales  one byte b per block, 2^(b - 127), 255 = NaN, in tiles of 128 rows x 4 blocks: the order in which the
//           tensor cores' block-scaled products take them (32 lanes of 16 bytes, a lane holding the four scales of
//           rows r, r + 32, r + 64 and r + 96).  Tiles of one row range follow one another along the blocks; rows
//           and blocks that only fill up a tile are zero.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "axc_device.cuh"
#include "axc_umma.cuh"

namespace axc {

constexpr int MX_BLOCK = 32;          // values per scale
constexpr int MX_BLOCK_BYTES = 16;
constexpr uint32_t MX_TILE_BYTES = 512;   // scales of 128 rows x 4 blocks

// Kernels that stream rows give a warp one segment of 256 columns at a time up to this many segments (two rounds of the
// 64 warps of each of a B200's 148 SMs), and four beyond.
constexpr uint64_t SMALL_SEGMENTS = 148u * 64u * 2u;

// Byte offset of the scales of blocks 4 * quad .. 4 * quad + 3 of a row; n_quads = ceil(n_blocks / 4).
__host__ __device__ __forceinline__ uint64_t mx_scale_at(uint64_t row, uint32_t quad, uint32_t n_quads) {
    return ((row >> 7) * n_quads + quad) * MX_TILE_BYTES + (row & 31u) * 16u + ((row >> 5) & 3u) * 4u;
}

// 2^(byte - 127); 255 is NaN.
__device__ __forceinline__ float mx_scale_value(uint32_t byte) {
    return __int_as_float(byte == 0u ? 0x00400000 : byte == 255u ? 0x7FFFFFFF : (int)(byte << 23));
}

// The two values of one byte of codes, exactly, as fp16 (low nibble first).
__device__ __forceinline__ float2 mx_code_pair(uint32_t byte) {
    uint32_t h;
    asm("{\n\t.reg .b8 b;\n\tcvt.u8.u32 b, %1;\n\tcvt.rn.f16x2.e2m1x2 %0, b;\n\t}" : "=r"(h) : "r"(byte));
    return __half22float2(*reinterpret_cast<const __half2*>(&h));
}

// One output value, rounded to nearest even.
__device__ __forceinline__ void put(float* p, float v) { *p = v; }
__device__ __forceinline__ void put(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void put(__half* p, float v) { *p = __float2half_rn(v); }

// Consecutive output values in one 16-byte store, rounded to nearest even.
__device__ __forceinline__ void store16(float* p, const float (&v)[4]) {
    *reinterpret_cast<float4*>(p) = make_float4(v[0], v[1], v[2], v[3]);
}
__device__ __forceinline__ void store16(__nv_bfloat16* p, const float (&v)[8]) {
    __nv_bfloat162 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
}
__device__ __forceinline__ void store16(__half* p, const float (&v)[8]) {
    __half2 h[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) h[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(h);
}

// kind::mxf4 instruction descriptor: both operands E2M1 (1 at bits 7 and 10), K-major, E8M0 scales (bit 23), N >> 3 at
// bit 17, M >> 7 at bit 27; sf_id (0 or 2: which two of a column's four scale bytes) at bits 4 and 29.
__device__ __forceinline__ uint32_t mx_idesc(uint32_t m, uint32_t n, uint32_t sf_id) {
    return (1u << 7) | (1u << 10) | ((n >> 3) << 17) | (1u << 23) | ((m >> 7) << 27) | (sf_id << 4) | (sf_id << 29);
}

// Shared-memory descriptor of a 512-byte scale tile: 32 rows of 16 bytes, no swizzle, 8 rows 128 bytes apart.
__device__ __forceinline__ uint64_t mx_scale_desc(uint32_t smem_addr) {
    return (uint64_t)((smem_addr >> 4) & 0x3FFFu) | (8ull << 16) | (8ull << 32) | (1ull << 46);
}

// Tensor map of a matrix' codes: boxes of 256 columns (128 bytes, 128-byte swizzle) x box_rows rows; what lies outside
// the matrix reads as zero.
inline bool mx_encode_codes(CUtensorMap* map, const uint8_t* codes, uint32_t rows, uint32_t n_blocks, uint32_t box_rows) {
    cuuint64_t dims[2] = {(uint64_t)n_blocks * MX_BLOCK_BYTES, rows};
    cuuint64_t strides[1] = {(uint64_t)n_blocks * MX_BLOCK_BYTES};
    cuuint32_t box[2] = {128u, box_rows};
    cuuint32_t estr[2] = {1, 1};
    return tensor_map_encoder()(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<uint8_t*>(codes), dims, strides, box, estr,
                                CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                                CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace axc
