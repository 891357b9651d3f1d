// Rows of a quantised matrix by number: out[i] = dequant(row ids[i]) * factor, for Q4_K_M, Q4_0 and MXFP4 tables
// (the token embedding of a checkpoint), and the dequantisation of a whole MXFP4 matrix, which is the same kernel
// without ids and factor.
//
// The dequantised value has the bits of the format's *_dequant kernel; it is multiplied by the factor in fp32 and
// rounded once to the output type.  An id outside [0, rows) reads nothing: its row of the output is zero and bit 1
// (value 2) of the status word is set.
//
// Bound by HBM: 0.53 to 0.56 byte read and 2 or 4 bytes written per value.  A lane takes neighbouring columns that fill a
// 16-byte store (V = 8 of a 16-bit type, 4 of fp32: two stores per lane would each leave half of their 32-byte sectors to
// the other), a warp a segment of 32 * V columns; where there is work for it, four segments at a time, whose loads are all
// under way before the first value is computed.  Measured: 4096 rows of 8192 bf16 from an MXFP4 table 18.7 us, all of 2048 x
// 14336 bf16 14.3 us (5.2 TB/s), fp32 22.5 us (5.9 TB/s); one row 1.4 us.
#include <type_traits>

#include "axc_kernels.h"
#include "axc_mx.cuh"

namespace axc {
namespace {

// A table gives the raw words of V = 4 or 8 neighbouring values at a column that is a multiple of V, and their values.
// Plain loads, neither __ldg nor __restrict__: the launch before may still be writing ids and table when this one starts,
// and a load of what counts as constant could move in front of the dependency wait.  (Volatile loads are in order too but
// took 23.7 us where these take 18.9 for 2048 rows of 8192 MXFP4 values.)
template <int V>
struct TableQ4K {
    static constexpr uint32_t BLOCK = 256;
    const uint8_t* q;
    uint32_t n;   // superblocks per row
    struct Raw {
        uint4 hdr;          // d, dmin, 12 scale bytes
        uint32_t w[V / 4];  // bytes whose low or high nibbles they are
    };
    __device__ __forceinline__ Raw load(uint64_t row, uint32_t col) const {
        const uint8_t* blk = q + (row * n + (col >> 8)) * Q4K_SB_BYTES;
        Raw r;
        r.hdr = *reinterpret_cast<const uint4*>(blk);
        const uint32_t* at = reinterpret_cast<const uint32_t*>(blk + 16 + ((col >> 6) & 3u) * 32u + (col & 31u));
#pragma unroll
        for (int i = 0; i < V / 4; ++i) r.w[i] = at[i];
        return r;
    }
    __device__ __forceinline__ void values(const Raw& r, uint32_t col, float (&v)[V]) const {
        const uint32_t chunk = (col >> 6) & 3u, high = (col >> 5) & 1u;
        uint32_t sc_pair, m_pair;
        q4k_unpack_pair(r.hdr.y, r.hdr.z, r.hdr.w, (int)chunk, sc_pair, m_pair);
        const float d1 = __fmul_rn(f16_bits_to_f32(r.hdr.x & 0xFFFFu), (float)((sc_pair >> (8u * high)) & 0xFFu));
        const float m1 = __fmul_rn(f16_bits_to_f32(r.hdr.x >> 16), (float)((m_pair >> (8u * high)) & 0xFFu));
#pragma unroll
        for (int i = 0; i < V; ++i)
            v[i] = __fsub_rn(__fmul_rn(d1, (float)((r.w[i >> 2] >> (8 * (i & 3) + 4u * high)) & 15u)), m1);
    }
};

template <int V>
struct TableQ40 {
    static constexpr uint32_t BLOCK = 32;
    const uint8_t* q;
    uint32_t n;   // blocks per row
    struct Raw {
        uint16_t d, two[V / 2];   // pairs of bytes whose low or high nibbles they are
    };
    __device__ __forceinline__ Raw load(uint64_t row, uint32_t col) const {
        const uint16_t* blk = reinterpret_cast<const uint16_t*>(q + (row * n + (col >> 5)) * Q4_0_BLK_BYTES);
        Raw r;
        r.d = *blk;
#pragma unroll
        for (uint32_t i = 0; i < V / 2; ++i) r.two[i] = blk[1 + ((col & 15u) >> 1) + i];
        return r;
    }
    __device__ __forceinline__ void values(const Raw& r, uint32_t col, float (&v)[V]) const {
        const uint32_t shift = ((col >> 4) & 1u) * 4u;                   // low or high nibbles
        const float d = f16_bits_to_f32(r.d);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            const uint32_t two = (uint32_t)r.two[i] >> shift;
            v[2 * i] = __fmul_rn(__fsub_rn((float)(two & 15u), 8.0f), d);
            v[2 * i + 1] = __fmul_rn(__fsub_rn((float)((two >> 8) & 15u), 8.0f), d);
        }
    }
};

template <int V>
struct TableMx {
    static constexpr uint32_t BLOCK = 32;
    const uint8_t* codes;
    const uint8_t* scales;
    uint32_t n;   // blocks per row
    struct Raw {
        uint32_t w;
        uint8_t scale;
    };
    __device__ __forceinline__ Raw load(uint64_t row, uint32_t col) const {
        const uint32_t block = col >> 5;
        const uint8_t* at = codes + (row * n + block) * MX_BLOCK_BYTES + ((col & 31u) >> 1);
        Raw r;
        r.w = V == 8 ? *reinterpret_cast<const uint32_t*>(at) : (uint32_t)*reinterpret_cast<const uint16_t*>(at);
        r.scale = scales[mx_scale_at(row, block >> 2, (n + 3u) >> 2) + (block & 3u)];
        return r;
    }
    __device__ __forceinline__ void values(const Raw& r, uint32_t, float (&v)[V]) const {
        const float s = mx_scale_value(r.scale);
#pragma unroll
        for (int i = 0; i < V / 2; ++i) {
            const float2 p = mx_code_pair((r.w >> (8 * i)) & 0xFFu);
            v[2 * i] = p.x * s, v[2 * i + 1] = p.y * s;
        }
    }
};

// ids: nullptr (row i of the output is row i of the table), or 32-bit / 64-bit numbers.
template <template <int> class Table, typename Out, uint32_t SEGS>
__global__ void __launch_bounds__(256)
rows_kernel(const Table<16 / sizeof(Out)> table, const void* ids, int ids64, uint32_t rows,
            float factor, Out* out, uint32_t n_groups, uint64_t n_items, uint32_t* status) {
    constexpr uint32_t V = 16 / sizeof(Out), SEG = 32u * V;
    using T = Table<V>;
    asm volatile("griddepcontrol.wait;" ::: "memory");   // an ordered launch: see axc_tuning.pdl
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const uint32_t lane = threadIdx.x & 31u, cols = table.n * T::BLOCK;
    const uint64_t warps = (uint64_t)gridDim.x * (blockDim.x >> 5);
    for (uint64_t item = (uint64_t)blockIdx.x * (blockDim.x >> 5) + (threadIdx.x >> 5); item < n_items; item += warps) {
        const uint64_t i = n_groups == 1u ? item : item >> 32 ? item / n_groups : (uint32_t)item / n_groups;
        const uint32_t group = (uint32_t)(item - i * n_groups), col0 = group * (SEGS * SEG) + lane * V;
        int64_t row = (int64_t)i;
        if (ids) row = ids64 ? reinterpret_cast<const long long*>(ids)[i] : (int64_t)reinterpret_cast<const int*>(ids)[i];
        const bool fits = row >= 0 && row < (int64_t)rows;
        if (!fits && status && group == 0u && lane == 0u) atomicOr(status, ERR_BAD_ARGUMENT);
        typename T::Raw raw[SEGS];
        if (fits) {
#pragma unroll
            for (uint32_t k = 0; k < SEGS; ++k)
                if (col0 + k * SEG < cols) raw[k] = table.load((uint64_t)row, col0 + k * SEG);
        }
#pragma unroll
        for (uint32_t k = 0; k < SEGS; ++k) {
            const uint32_t col = col0 + k * SEG;
            if (col >= cols) break;
            float v[V] = {};
            if (fits) {
                table.values(raw[k], col, v);
                if (ids) {
#pragma unroll
                    for (uint32_t j = 0; j < V; ++j) v[j] = __fmul_rn(v[j], factor);
                }
            }
            store16(out + i * cols + col, v);
        }
    }
}

struct RowsArgs {
    const uint8_t* codes;
    const uint8_t* scales;      // MXFP4
    uint32_t n;                 // blocks per row
    const void* ids;
    int ids64;
    uint32_t n_ids, rows;
    float factor;
    void* out;
    uint32_t* status;
};

template <template <int> class Table, typename Out, uint32_t SEGS>
cudaError_t launch_segs(const RowsArgs& a, cudaStream_t stream) {
    constexpr uint32_t V = 16 / sizeof(Out);
    Table<V> table{};
    if constexpr (std::is_same_v<Table<V>, TableMx<V>>) table = {a.codes, a.scales, a.n};
    else table = {a.codes, a.n};
    const uint64_t cols = (uint64_t)a.n * Table<V>::BLOCK;
    const uint32_t n_groups = (uint32_t)((cols + SEGS * 32u * V - 1u) / (SEGS * 32u * V));
    const uint64_t n_items = (uint64_t)a.n_ids * n_groups;
    const uint64_t want = (n_items + 7u) / 8u;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(want < (1u << 30) ? want : (1u << 30))), cfg.blockDim = dim3(256), cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr, cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, rows_kernel<Table, Out, SEGS>, table, a.ids, a.ids64, a.rows, a.factor,
                              (Out*)a.out, n_groups, n_items, a.status);
}

// One segment per warp until all SMs have two rounds of warps (301 x 8200 fp32 to MXFP4 and back, where both kernels go by
// this rule: 8.1 us, with four segments 13.5 us), four from there on (4096 rows of 8192 columns: 22 us, with one 39 us).
template <template <int> class Table, typename Out>
cudaError_t launch(const RowsArgs& a, cudaStream_t stream) {
    constexpr uint32_t V = 16 / sizeof(Out);
    const uint64_t segs = (uint64_t)a.n_ids * (((uint64_t)a.n * Table<V>::BLOCK + 32u * V - 1u) / (32u * V));
    return segs <= SMALL_SEGMENTS ? launch_segs<Table, Out, 1>(a, stream) : launch_segs<Table, Out, 4>(a, stream);
}

template <template <int> class Table>
cudaError_t launch_typed(const RowsArgs& a, ElemType type, cudaStream_t stream) {
    if (a.n_ids == 0 || a.n == 0) return cudaSuccess;
    switch (type) {
        case ElemType::F32: return launch<Table, float>(a, stream);
        case ElemType::BF16: return launch<Table, __nv_bfloat16>(a, stream);
        case ElemType::F16: return launch<Table, __half>(a, stream);
    }
    return cudaErrorInvalidValue;
}

}  // namespace

cudaError_t launch_q4k_embed(const uint8_t* q, const void* ids, int ids64, uint32_t n_ids, uint32_t rows, uint32_t n_sb,
                             float factor, void* out, ElemType type, uint32_t* status, cudaStream_t stream) {
    return launch_typed<TableQ4K>({q, nullptr, n_sb, ids, ids64, n_ids, rows, factor, out, status}, type, stream);
}

cudaError_t launch_q4_0_embed(const uint8_t* q, const void* ids, int ids64, uint32_t n_ids, uint32_t rows, uint32_t n_blocks,
                              float factor, void* out, ElemType type, uint32_t* status, cudaStream_t stream) {
    return launch_typed<TableQ40>({q, nullptr, n_blocks, ids, ids64, n_ids, rows, factor, out, status}, type, stream);
}

cudaError_t launch_mxfp4_embed(const uint8_t* codes, const uint8_t* scales, const void* ids, int ids64, uint32_t n_ids,
                               uint32_t rows, uint32_t n_blocks, float factor, void* out, ElemType type, uint32_t* status,
                               cudaStream_t stream) {
    return launch_typed<TableMx>({codes, scales, n_blocks, ids, ids64, n_ids, rows, factor, out, status}, type, stream);
}

}  // namespace axc
