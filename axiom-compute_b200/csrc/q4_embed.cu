// Rows of a quantised matrix by number: out[i] = dequant(row ids[i]) * factor, for Q4_K_M, Q4_0 and MXFP4 tables
// (the token embedding of a checkpoint), and the dequantisation of a whole MXFP4 matrix, which is the same kernel
// without ids and factor.
//
// The dequantised value has the bits of the format's *_dequant kernel; it is multiplied by the factor in fp32 and
// rounded once to the output type.  An id outside [0, rows) reads nothing: its row of the output is zero and bit 1
// (value 2) of the status word is set.
//
// Bound by HBM: 0.53 to 0.56 byte read and 2 or 4 bytes written per value.  A warp takes 256 columns of a row (one
// Q4_K superblock, eight blocks of the other formats), a lane 8 neighbouring ones, so that a warp's stores are
// contiguous.
#include "axc_kernels.h"
#include "axc_mx.cuh"

namespace axc {
namespace {

struct TableQ4K {
    const uint8_t* q;
    uint32_t n;   // superblocks per row
    __device__ __forceinline__ uint32_t cols() const { return n * 256u; }
    __device__ __forceinline__ void read8(uint64_t row, uint32_t col, float (&v)[8]) const {
        const uint8_t* blk = q + (row * n + (col >> 8)) * Q4K_SB_BYTES;
        const uint32_t chunk = (col >> 6) & 3u, high = (col >> 5) & 1u, at = col & 31u;   // at: 0, 8, 16, 24
        const uint4 hdr = __ldg(reinterpret_cast<const uint4*>(blk));   // d, dmin, 12 scale bytes
        const uint2 qs = __ldg(reinterpret_cast<const uint2*>(blk + 16 + chunk * 32u + at));
        uint32_t sc_pair, m_pair;
        q4k_unpack_pair(hdr.y, hdr.z, hdr.w, (int)chunk, sc_pair, m_pair);
        const float d1 = __fmul_rn(f16_bits_to_f32(hdr.x & 0xFFFFu), (float)((sc_pair >> (8u * high)) & 0xFFu));
        const float m1 = __fmul_rn(f16_bits_to_f32(hdr.x >> 16), (float)((m_pair >> (8u * high)) & 0xFFu));
        const uint32_t w[2] = {qs.x >> (4u * high), qs.y >> (4u * high)};
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = __fsub_rn(__fmul_rn(d1, (float)((w[i >> 2] >> (8 * (i & 3))) & 15u)), m1);
    }
};

struct TableQ40 {
    const uint8_t* q;
    uint32_t n;   // blocks per row
    __device__ __forceinline__ uint32_t cols() const { return n * 32u; }
    __device__ __forceinline__ void read8(uint64_t row, uint32_t col, float (&v)[8]) const {
        const uint16_t* blk = reinterpret_cast<const uint16_t*>(q + (row * n + (col >> 5)) * Q4_0_BLK_BYTES);
        const uint32_t high = (col >> 4) & 1u, at = (col >> 3) & 1u;   // nibble, bytes 0..7 or 8..15
        const float d = f16_bits_to_f32(__ldg(blk));
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            const uint32_t two = (uint32_t)__ldg(blk + 1 + at * 4u + i) >> (4u * high);
            v[2 * i] = __fmul_rn(__fsub_rn((float)(two & 15u), 8.0f), d);
            v[2 * i + 1] = __fmul_rn(__fsub_rn((float)((two >> 8) & 15u), 8.0f), d);
        }
    }
};

struct TableMx {
    const uint8_t* codes;
    const uint8_t* scales;
    uint32_t n;   // blocks per row
    __device__ __forceinline__ uint32_t cols() const { return n * 32u; }
    __device__ __forceinline__ void read8(uint64_t row, uint32_t col, float (&v)[8]) const {
        const uint32_t block = col >> 5;
        const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(codes + (row * n + block) * MX_BLOCK_BYTES + ((col & 31u) >> 1)));
        const float s = mx_scale_value(__ldg(scales + mx_scale_at(row, block >> 2, (n + 3u) >> 2) + (block & 3u)));
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 p = mx_code_pair((w >> (8 * i)) & 0xFFu);
            v[2 * i] = p.x * s, v[2 * i + 1] = p.y * s;
        }
    }
};

// ids: nullptr (row i of the output is row i of the table), or 32-bit / 64-bit numbers.
template <typename Table, typename Out>
__global__ void __launch_bounds__(256)
rows_kernel(const Table table, const void* __restrict__ ids, int ids64, uint32_t n_ids, uint32_t rows, float factor,
            Out* __restrict__ out, uint32_t n_seg, uint64_t n_items, uint32_t* status) {
    asm volatile("griddepcontrol.wait;" ::: "memory");   // an ordered launch: see axc_tuning.pdl
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t lane = threadIdx.x & 31u, cols = table.cols();
    const uint64_t warps = (uint64_t)gridDim.x * (blockDim.x >> 5);
    for (uint64_t item = (uint64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); item < n_items; item += warps) {
        const uint64_t i = item / n_seg;
        const uint32_t seg = (uint32_t)(item - i * n_seg), col = seg * 256u + lane * 8u;
        int64_t row = (int64_t)i;
        if (ids) row = ids64 ? __ldg(reinterpret_cast<const long long*>(ids) + i) : (int64_t)__ldg(reinterpret_cast<const int*>(ids) + i);
        const bool fits = row >= 0 && row < (int64_t)rows;
        if (!fits && status && seg == 0u && lane == 0u) atomicOr(status, ERR_BAD_ARGUMENT);
        if (col >= cols) continue;
        float v[8] = {};
        if (fits) {
            table.read8((uint64_t)row, col, v);
            if (ids) {
#pragma unroll
                for (int j = 0; j < 8; ++j) v[j] = __fmul_rn(v[j], factor);
            }
        }
        store8(out + i * cols + col, v);
    }
}

template <typename Table, typename Out>
cudaError_t launch(const Table& table, uint32_t n, uint32_t per_block, const void* ids, int ids64, uint32_t n_ids,
                   uint32_t rows, float factor, void* out, uint32_t* status, cudaStream_t stream) {
    const uint32_t n_seg = (uint32_t)(((uint64_t)n * per_block + 255u) / 256u);
    const uint64_t n_items = (uint64_t)n_ids * n_seg;
    const uint64_t want = (n_items + 7u) / 8u;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(want < 148u * 8u ? want : 148u * 8u)), cfg.blockDim = dim3(256), cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr, cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, rows_kernel<Table, Out>, table, ids, ids64, n_ids, rows, factor, (Out*)out, n_seg,
                              n_items, status);
}

template <typename Table>
cudaError_t launch_typed(const Table& table, uint32_t n, uint32_t per_block, const void* ids, int ids64, uint32_t n_ids,
                         uint32_t rows, float factor, void* out, ElemType type, uint32_t* status, cudaStream_t stream) {
    if (n_ids == 0 || n == 0) return cudaSuccess;
    switch (type) {
        case ElemType::F32: return launch<Table, float>(table, n, per_block, ids, ids64, n_ids, rows, factor, out, status, stream);
        case ElemType::BF16: return launch<Table, __nv_bfloat16>(table, n, per_block, ids, ids64, n_ids, rows, factor, out, status, stream);
        case ElemType::F16: return launch<Table, __half>(table, n, per_block, ids, ids64, n_ids, rows, factor, out, status, stream);
    }
    return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_q4k_embed(const uint8_t* q, const void* ids, int ids64, uint32_t n_ids, uint32_t rows, uint32_t n_sb,
                             float factor, void* out, ElemType type, uint32_t* status, cudaStream_t stream) {
    return launch_typed(TableQ4K{q, n_sb}, n_sb, 256u, ids, ids64, n_ids, rows, factor, out, type, status, stream);
}

cudaError_t launch_q4_0_embed(const uint8_t* q, const void* ids, int ids64, uint32_t n_ids, uint32_t rows, uint32_t n_blocks,
                              float factor, void* out, ElemType type, uint32_t* status, cudaStream_t stream) {
    return launch_typed(TableQ40{q, n_blocks}, n_blocks, 32u, ids, ids64, n_ids, rows, factor, out, type, status, stream);
}

cudaError_t launch_mxfp4_embed(const uint8_t* codes, const uint8_t* scales, const void* ids, int ids64, uint32_t n_ids,
                               uint32_t rows, uint32_t n_blocks, float factor, void* out, ElemType type, uint32_t* status,
                               cudaStream_t stream) {
    return launch_typed(TableMx{codes, scales, n_blocks}, n_blocks, 32u, ids, ids64, n_ids, rows, factor, out, type, status, stream);
}

}  // namespace axc
