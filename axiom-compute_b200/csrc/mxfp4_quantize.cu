// Rows of fp32 / bf16 / fp16 values to MXFP4 (layout: axc_mx.cuh).
//
// Per block of 32 columns: e = clamp(floor(log2(max |x|)) - 2, -127, 127), so that the largest value lies in
// [4, 8) * 2^e and E2M1's largest binade (4, 6) is in use; code = x * 2^-e rounded to the nearest E2M1 value, ties to
// the even code, larger magnitudes to 6.  The product x * 2^-e is exact (a power of two between 2^-125 and 2^127),
// so each value is rounded once.  A block that holds a NaN or an infinity gets the NaN scale and zero codes.
//
// One pass over x, bound by HBM: 2 or 4 bytes read and 17/32 byte written per value.  A warp takes segments of 256 columns
// of a row, a lane 8 neighbouring columns of each (one 16-byte load of 16-bit values): the block maximum is two shuffles
// over four lanes, the codes of a segment are 128 contiguous bytes, and its scales are two 4-byte words.  Where there is
// work for it, four segments are under way at a time.  Measured over buffers that rotate beyond L2 (in brackets: the same ones
// again): 2048 x 14336 bf16 16.2 to 17.9 us (14.3 to 16.3), fp16 14.2 us (12.4), 8192 x 8192 bf16 30.4 us (5.6 TB/s), fp32 45.5 us
// (6.7 TB/s: a stream of reads, which runs faster than a copy).  Rows that do not start at multiples of 16 bytes are read
// value by value: 2048 rows of 14336, 14349 apart, bf16 27.3 us, fp16 26.5 us, fp32 34.6 us (aligned 20.9).  The 16-bit types are near the rate at which their instructions issue, which is why
// maxima are taken two at a time and scales are turned over between lanes and stored four segments at once (17.2 -> 14.4 us).
#include "axc_kernels.h"
#include "axc_mx.cuh"

namespace axc {
namespace {

// Eight values as they lie in memory, the largest magnitude among them as the bits of an fp32 (NaN and infinity compare
// above every finite value), and the values as fp32.
template <typename T>
struct Eight;

template <>
struct Eight<float> {
    float v[8];
    __device__ __forceinline__ void load(const float* p) {
        const float4* src = reinterpret_cast<const float4*>(p);
        const float4 a = src[0], b = src[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    }
    __device__ __forceinline__ void load_edge(const float* p, uint32_t count) {
#pragma unroll
        for (uint32_t i = 0; i < 8u; ++i) v[i] = i < count ? p[i] : 0.0f;
    }
    __device__ __forceinline__ uint32_t top() const {
        uint32_t t = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) t = max(t, (uint32_t)__float_as_int(v[i]) & 0x7FFFFFFFu);
        return t;
    }
    __device__ __forceinline__ float value(int i) const { return v[i]; }
};

// 16-bit types: the magnitudes of two values are compared in one instruction.
struct EightHalves {
    uint32_t w[4];
    template <typename T>
    __device__ __forceinline__ void load(const T* p) {
        const uint4 a = *reinterpret_cast<const uint4*>(p);
        w[0] = a.x, w[1] = a.y, w[2] = a.z, w[3] = a.w;
    }
    template <typename T>
    __device__ __forceinline__ void load_edge(const T* p, uint32_t count) {
        const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i)
            w[i] = (2u * i < count ? (uint32_t)h[2u * i] : 0u) | (2u * i + 1u < count ? (uint32_t)h[2u * i + 1u] << 16 : 0u);
    }
    __device__ __forceinline__ uint32_t top16() const {
        const uint32_t t = __vmaxu2(__vmaxu2(w[0] & 0x7FFF7FFFu, w[1] & 0x7FFF7FFFu), __vmaxu2(w[2] & 0x7FFF7FFFu, w[3] & 0x7FFF7FFFu));
        return max(t & 0xFFFFu, t >> 16);
    }
};
template <>
struct Eight<__nv_bfloat16> : EightHalves {
    __device__ __forceinline__ uint32_t top() const { return top16() << 16; }
    __device__ __forceinline__ float value(int i) const { return __int_as_float((int)(i & 1 ? w[i >> 1] & 0xFFFF0000u : w[i >> 1] << 16)); }
};
template <>
struct Eight<__half> : EightHalves {
    __device__ __forceinline__ uint32_t top() const { return (uint32_t)__float_as_int(f16_bits_to_f32(top16())) & 0x7FFFFFFFu; }
    __device__ __forceinline__ float value(int i) const { return f16_bits_to_f32(i & 1 ? w[i >> 1] >> 16 : w[i >> 1] & 0xFFFFu); }
};

// Eight values to eight codes, the first in the lowest nibble: nearest even, saturating.
template <typename T>
__device__ __forceinline__ uint32_t codes_of(const Eight<T>& x, float inv) {
    uint32_t r;
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
        "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
        "mov.b32 %0, {a, b, c, d};\n\t}"
        : "=r"(r)
        : "f"(x.value(0) * inv), "f"(x.value(1) * inv), "f"(x.value(2) * inv), "f"(x.value(3) * inv), "f"(x.value(4) * inv),
          "f"(x.value(5) * inv), "f"(x.value(6) * inv), "f"(x.value(7) * inv));
    return r;
}

template <typename T, uint32_t SEGS>   // segments of 256 columns that a warp has under way
__global__ void __launch_bounds__(256)
mxfp4_quantize_kernel(const T* x, uint64_t row_stride, uint32_t rows, uint32_t cols, uint32_t n_blocks,
                      uint8_t* codes, uint8_t* scales, uint32_t n_groups, uint64_t n_items, int wide) {
    asm volatile("griddepcontrol.wait;" ::: "memory");   // an ordered launch: see axc_tuning.pdl.  x may be new: no __ldg, no __restrict__
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t lane = threadIdx.x & 31u;
    const uint32_t n_quads = (n_blocks + 3u) / 4u;
    const uint64_t warps = (uint64_t)gridDim.x * (blockDim.x >> 5);
    for (uint64_t item = (uint64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); item < n_items; item += warps) {
        const uint64_t row = n_groups == 1u ? item : item >> 32 ? item / n_groups : (uint32_t)item / n_groups;
        const uint32_t seg0 = (uint32_t)(item - row * n_groups) * SEGS;
        Eight<T> v[SEGS];
        const uint32_t col0 = seg0 * 256u + lane * 8u;
        const T* src = x + row * row_stride + col0;
        const uint32_t end = row < rows ? cols : 0u;             // rows that only fill up a tile of scales read as zero
        const uint32_t left = end > col0 ? end - col0 : 0u;
#pragma unroll
        for (uint32_t k = 0; k < SEGS; ++k) {
            if (wide && k * 256u + 8u <= left) v[k].load(src + k * 256u);
            else v[k].load_edge(src + k * 256u, left > k * 256u ? left - k * 256u : 0u);
        }
        // block seg0 * 8 + k * 8 + lane / 4 of the row; how many of them k runs over
        const uint32_t block0 = seg0 * 8u + (lane >> 2), blocks = row < rows && n_blocks > block0 ? n_blocks - block0 : 0u;
        uint8_t* dst = codes + (row * n_blocks + block0) * MX_BLOCK_BYTES + (lane & 3u) * 4u;
        uint32_t bytes = 0;                                      // scale of block k in byte k; zero where there is none
#pragma unroll
        for (uint32_t k = 0; k < SEGS; ++k) {
            uint32_t top = v[k].top();
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
            const uint32_t ex = top >> 23;                       // biased exponent; 0 for zero and subnormal
            const bool bad = ex == 255u;
            uint32_t byte = max(ex, 2u) - 2u;
            const float inv = __int_as_float((int)((254u - byte) << 23));   // 2^-(byte - 127)
            uint32_t word = codes_of(v[k], inv);
            if (bad) word = 0u, byte = 255u;
            if (k * 8u < blocks) {
                *reinterpret_cast<uint32_t*>(dst + k * 8u * MX_BLOCK_BYTES) = word;
                bytes |= byte << (8u * k);
            }
        }
        // The scales of four neighbouring blocks, which lie in lanes four apart, make one word.
        const uint32_t g = (lane >> 2) & 3u, half = lane >> 4;
        uint32_t word, seg = seg0;
        bool writes;
        if constexpr (SEGS == 4) {
            // 4 x 4 bytes turned over between the lanes g = 0..3: lane g ends up with segment g
            const uint32_t q = __shfl_xor_sync(0xFFFFFFFFu, bytes, 8);
            bytes = __byte_perm(bytes, q, g & 2u ? 0x3276 : 0x5410);
            const uint32_t r = __shfl_xor_sync(0xFFFFFFFFu, bytes, 4);
            word = __byte_perm(bytes, r, g & 1u ? 0x3715 : 0x6240);
            seg += g;
            writes = (lane & 3u) == 0u;
        } else {
            word = bytes << (8u * g);
            word |= __shfl_xor_sync(0xFFFFFFFFu, word, 4);
            word |= __shfl_xor_sync(0xFFFFFFFFu, word, 8);
            writes = (lane & 15u) == 0u;
        }
        const uint32_t quad = seg * 2u + half;
        if (writes && quad < n_quads) *reinterpret_cast<uint32_t*>(scales + mx_scale_at(row, quad, n_quads)) = word;
    }
}

template <typename T, uint32_t SEGS>
cudaError_t launch_segs(const void* x, uint64_t row_stride, uint32_t rows, uint32_t cols, uint8_t* codes, uint8_t* scales,
                   cudaStream_t stream) {
    const uint32_t n_blocks = (cols + 31u) / 32u, n_groups = (n_blocks + SEGS * 8u - 1u) / (SEGS * 8u);
    const uint64_t n_items = ((uint64_t)rows + 127u) / 128u * 128u * n_groups;
    const uint64_t want = (n_items + 7u) / 8u;
    const int wide = ((uintptr_t)x & 15u) == 0 && (row_stride * sizeof(T)) % 16u == 0;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(want < (1u << 30) ? want : (1u << 30))), cfg.blockDim = dim3(256), cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr, cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, mxfp4_quantize_kernel<T, SEGS>, (const T*)x, row_stride, rows, cols, n_blocks, codes, scales,
                              n_groups, n_items, wide);
}

template <typename T>
cudaError_t launch(const void* x, uint64_t row_stride, uint32_t rows, uint32_t cols, uint8_t* codes, uint8_t* scales,
                   cudaStream_t stream) {
    const uint64_t segs = ((uint64_t)rows + 127u) / 128u * 128u * ((cols + 255u) / 256u);
    return segs <= SMALL_SEGMENTS ? launch_segs<T, 1>(x, row_stride, rows, cols, codes, scales, stream)
                                  : launch_segs<T, 4>(x, row_stride, rows, cols, codes, scales, stream);
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
