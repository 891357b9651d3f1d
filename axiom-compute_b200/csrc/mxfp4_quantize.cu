// Rows of fp32 / bf16 / fp16 values to MXFP4 (layout: axc_mx.cuh).
//
// Per block of 32 columns: e = clamp(floor(log2(max |x|)) - 2, -127, 127), so that the largest value lies in
// [4, 8) * 2^e and E2M1's largest binade (4, 6) is in use; code = x * 2^-e rounded to the nearest E2M1 value, ties to
// the even code, larger magnitudes to 6.  The product x * 2^-e is exact (a power of two between 2^-125 and 2^127),
// so each value is rounded once.  A block that holds a NaN or an infinity gets the NaN scale and zero codes.
//
// One pass over x, bound by HBM: 2 or 4 bytes read and 17/32 byte written per value.  A warp takes 256 columns of a
// row, a lane 8 of them (one 16-byte load of 16-bit values): the block maximum is two shuffles over four lanes, the
// codes of a warp are 128 contiguous bytes, and its scales are two 4-byte words.
#include "axc_kernels.h"
#include "axc_mx.cuh"

namespace axc {
namespace {

__device__ __forceinline__ float widen(float v) { return v; }
__device__ __forceinline__ float widen(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float widen(__half v) { return __half2float(v); }

__device__ __forceinline__ void load8(const float* p, float (&v)[8]) {
    const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
    v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
}
template <typename T>
__device__ __forceinline__ void load8(const T* p, float (&v)[8]) {
    const uint4 raw = __ldg(reinterpret_cast<const uint4*>(p));
    const T* h = reinterpret_cast<const T*>(&raw);
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = widen(h[i]);
}

// Two values to two codes in one byte, the first in the low nibble: nearest even, saturating.
__device__ __forceinline__ uint32_t code_pair(float lo, float hi) {
    uint32_t r;
    asm("{\n\t.reg .b8 b;\n\tcvt.rn.satfinite.e2m1x2.f32 b, %2, %1;\n\tcvt.u32.u8 %0, b;\n\t}" : "=r"(r) : "f"(lo), "f"(hi));
    return r;
}

template <typename T>
__global__ void __launch_bounds__(256)
mxfp4_quantize_kernel(const T* __restrict__ x, uint64_t row_stride, uint32_t rows, uint32_t cols, uint32_t n_blocks,
                      uint8_t* __restrict__ codes, uint8_t* __restrict__ scales, uint32_t n_seg, uint64_t n_items, int wide) {
    asm volatile("griddepcontrol.wait;" ::: "memory");   // an ordered launch: see axc_tuning.pdl
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t lane = threadIdx.x & 31u;
    const uint32_t n_quads = (n_blocks + 3u) / 4u;
    const uint64_t warps = (uint64_t)gridDim.x * (blockDim.x >> 5);
    for (uint64_t item = (uint64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); item < n_items; item += warps) {
        const uint64_t row = item / n_seg;
        const uint32_t seg = (uint32_t)(item - row * n_seg);
        const uint32_t col = seg * 256u + lane * 8u;
        float v[8] = {};
        if (row < rows) {
            const T* src = x + row * row_stride + col;
            if (wide && col + 8u <= cols) {
                load8(src, v);
            } else {
#pragma unroll
                for (uint32_t i = 0; i < 8u; ++i)
                    if (col + i < cols) v[i] = widen(src[i]);
            }
        }
        // the largest magnitude as bits: NaN and infinity compare above every finite value
        uint32_t top = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) top = max(top, (uint32_t)__float_as_int(v[i]) & 0x7FFFFFFFu);
        top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
        top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
        const uint32_t ex = top >> 23;                       // biased exponent; 0 for zero and subnormal
        const bool bad = ex == 255u;
        const uint32_t byte = bad ? 255u : ex > 2u ? ex - 2u : 0u;
        // 2^-(byte - 127) = 2^(127 - byte), byte <= 252
        const float inv = __int_as_float((int)((254u - (bad ? 127u : byte)) << 23));
        uint32_t word = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) word |= code_pair(v[2 * i] * inv, v[2 * i + 1] * inv) << (8 * i);
        if (bad) word = 0;
        const uint32_t block = seg * 8u + (lane >> 2);
        if (row < rows && block < n_blocks)
            *reinterpret_cast<uint32_t*>(codes + (row * n_blocks + block) * MX_BLOCK_BYTES + (lane & 3u) * 4u) = word;
        // the four scales of 16 lanes in one word; blocks and rows that only fill up a tile are zero
        uint32_t s = row < rows && block < n_blocks ? byte << (8u * ((lane >> 2) & 3u)) : 0u;
        s |= __shfl_xor_sync(0xFFFFFFFFu, s, 4);
        s |= __shfl_xor_sync(0xFFFFFFFFu, s, 8);
        const uint32_t quad = seg * 2u + (lane >> 4);
        if ((lane & 15u) == 0u && quad < n_quads) *reinterpret_cast<uint32_t*>(scales + mx_scale_at(row, quad, n_quads)) = s;
    }
}

template <typename T>
cudaError_t launch(const void* x, uint64_t row_stride, uint32_t rows, uint32_t cols, uint8_t* codes, uint8_t* scales,
                   cudaStream_t stream) {
    const uint32_t n_blocks = (cols + 31u) / 32u, n_seg = (n_blocks + 7u) / 8u;
    const uint64_t n_items = ((uint64_t)rows + 127u) / 128u * 128u * n_seg;
    const uint64_t want = (n_items + 7u) / 8u;
    const int wide = ((uintptr_t)x & 15u) == 0 && (row_stride * sizeof(T)) % 16u == 0;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(want < 148u * 8u ? want : 148u * 8u)), cfg.blockDim = dim3(256), cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr, cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, mxfp4_quantize_kernel<T>, (const T*)x, row_stride, rows, cols, n_blocks, codes, scales,
                              n_seg, n_items, wide);
}

}  // namespace

cudaError_t launch_mxfp4_quantize(const void* x, ElemType type, uint64_t row_stride, uint32_t rows, uint32_t cols,
                                  uint8_t* codes, uint8_t* scales, cudaStream_t stream) {
    if (rows == 0 || cols == 0) return cudaSuccess;
    switch (type) {
        case ElemType::F32: return launch<float>(x, row_stride, rows, cols, codes, scales, stream);
        case ElemType::BF16: return launch<__nv_bfloat16>(x, row_stride, rows, cols, codes, scales, stream);
        case ElemType::F16: return launch<__half>(x, row_stride, rows, cols, codes, scales, stream);
    }
    return cudaErrorInvalidValue;
}

}  // namespace axc
