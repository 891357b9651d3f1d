// C[m][n] = sum_k A[m][k] W[n][k] for many tokens, A and W in MXFP4: the form of axc_cuda_mxfp4_prefill that reuses what it
// reads (tcgen05.mma kind::mxf4, block scales, fp32 accumulators in tensor memory).
//
// A pair of CTAs (a cluster of two) computes pieces of 256 weight rows (the MMA's M, 128 TMEM lanes in each CTA) x up to
// 256 tokens (its N, as many TMEM columns) with tcgen05.mma.cta_group::2: each CTA holds its own 128 weight rows and one
// half of the tokens, so that per SM 32 KB of codes feed 128 x 256 x 256 products.  One CTA alone would have to read 48 KB
// through the same shared-memory port.  The pairs are persistent and take the pieces in turn, tokens first, so that the
// pairs at work share the weights through L2.  (Equal contiguous parts for the pairs, cut at 128 tokens, were measured and
// are not used: 768 x 9472 x 4096 17.9 us either way, 4096 x 28672 x 8192 329 us against 442 us, where every pair reads
// weights of its own.)
//
// Measured, bf16 output: 4096 x 28672 x 8192 320 us (6.0 PFLOP/s; 377 us where the power limit has lowered the clock), 2048
// x 18944 x 4096 58 us (5.5 PFLOP/s; 67 us sustained) with the tensor pipe busy 72 % of the time.  At 0.26 us of MMAs per
// stage of a pair the first would take 201 us: the rest are stages that wait.  A stage takes 0.33 to 0.38 us where its MMAs
// take 0.26: its 35 KB arrive from L2 at 10.8 TB/s over all SMs, and issuing it costs the MMA thread about 600 cycles.
//
//   warp 0       one thread: TMA loads of this CTA's codes (128-byte swizzle, stages of 256 columns) and bulk copies
//                of the scale tiles of its rows and of all 256 tokens
//   warp 1       leader: one thread copies the stage's scales into both CTAs' tensor memory (tcgen05.cp), issues four
//                MMAs of 64 columns and the commit that frees the stage in both CTAs; peer: one thread tells the
//                leader when its stage has landed
//   warps 2..9   epilogue: 128 of the 256 columns each to registers, tensor memory is free again, then the stores,
//                while the next piece's MMAs run
//
// The accumulators truncate: each of the K / 64 MMAs of a chain cuts off at most 2^-22 of the running sum, and nothing while
// all partial sums are multiples of one unit below 2^24.  Measured on positive products with scales 24 binades apart, where
// it is worst: 2.0e-10 to 2.4e-10 of the value per column on average, always towards zero, and at most 7.0e-6 at K = 14336;
// with products of both signs 5.2e-6 of sum |A W|.  Shorter chains, emptied on the way and added in fp32, would lose less at
// the cost of an epilogue's loads for every part; they are not built.
//
// Every wait on an mbarrier is bounded; a wait that runs out sets an error bit and an abort flag, all roles fall
// through to the common exit, outstanding copies are waited for and tensor memory is freed.
#include <mutex>

#include "axc_kernels.h"
#include "axc_mx.cuh"
#include "axc_umma.cuh"

namespace axc {
namespace {

constexpr uint32_t GM_ROWS = 256, GM_TOKENS = 256;     // largest piece of a pair
constexpr uint32_t GM_STAGES = 6;
constexpr uint32_t GM_W_BYTES = 128 * 128, GM_A_BYTES = 128 * 128;       // codes of a stage in one CTA
constexpr uint32_t GM_SFW_BYTES = 1024, GM_SFA_BYTES = 2048;
constexpr uint32_t GM_STAGE_BYTES = GM_W_BYTES + GM_A_BYTES + GM_SFW_BYTES + GM_SFA_BYTES;
constexpr uint32_t GM_OFF_A = GM_W_BYTES, GM_OFF_SFW = GM_OFF_A + GM_A_BYTES, GM_OFF_SFA = GM_OFF_SFW + GM_SFW_BYTES;
constexpr uint32_t GM_OFF_BAR = GM_STAGES * GM_STAGE_BYTES;
constexpr uint32_t GM_SMEM = GM_OFF_BAR + 256 + 1024;                     // + alignment slack
constexpr uint32_t GM_EPI_WARPS = 8;
constexpr uint32_t GM_THREADS = (2 + GM_EPI_WARPS) * 32;
constexpr uint32_t GM_SF_COL = 256;                    // scale columns behind the accumulator: 24 for each stage
static_assert(GM_STAGE_BYTES % 1024 == 0, "the swizzled tiles need 1024-byte alignment");
static_assert(GM_SF_COL + GM_STAGES * 24 <= 512, "tensor memory");
static_assert(GM_SMEM <= 227 * 1024, "one CTA per SM");

struct GmArgs {
    const uint8_t* w_scales;
    const uint8_t* a_scales;
    void* c;
    uint32_t m, rows, n_blocks;
    uint32_t token_pieces, pieces;   // pieces of 256 tokens per row tile and in all
    uint32_t* status;
};

struct GmBars {
    uint64_t full[GM_STAGES], empty[GM_STAGES];
    uint64_t acc_full, acc_empty;
    uint32_t tmem_base;
    volatile uint32_t abort;
};

__device__ __forceinline__ void scales_to_tmem_pair(uint32_t taddr, uint32_t smem_addr) {
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(mx_scale_desc(smem_addr)) : "memory");
}

__device__ __forceinline__ void umma_mxf4_pair(uint32_t d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sfa,
                                               uint32_t sfb, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}

// The pieces of one pair, in order.
struct Pieces {
    uint32_t at, end, step, per_row, m;
    uint32_t row_tile, tok0, n;   // n: columns of the MMA, the tokens rounded up to 32
    __device__ __forceinline__ Pieces(const GmArgs& p, uint32_t pair, uint32_t pairs)
        : at(pair), end(p.pieces), step(pairs), per_row(p.token_pieces), m(p.m) {}
    __device__ __forceinline__ bool next() {
        if (at >= end) return false;
        row_tile = at / per_row;
        tok0 = (at - row_tile * per_row) * GM_TOKENS;
        n = (min(GM_TOKENS, m - tok0) + 31u) & ~31u;
        at += step;
        return true;
    }
    __device__ __forceinline__ bool last() const { return at >= end; }
};

template <typename Out>
__global__ void __launch_bounds__(GM_THREADS, 1)
mx_gemm_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_a, const GmArgs p) {
    extern __shared__ uint8_t smem_dyn[];
    const uint32_t raw_addr = smem_u32(smem_dyn);
    const uint32_t base = (raw_addr + 1023u) & ~1023u;
    uint8_t* sm = smem_dyn + (base - raw_addr);
    GmBars* bars = reinterpret_cast<GmBars*>(sm + GM_OFF_BAR);

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    uint32_t rank;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(rank));
    const bool leader = rank == 0;
    const uint32_t pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    const uint32_t n_st = (p.n_blocks + 7u) / 8u, n_quads = (p.n_blocks + 3u) / 4u;
    const uint32_t row_tiles = (p.rows + 127u) / 128u, tok_tiles = (p.m + 127u) / 128u;   // scale tiles of W and A

    if (tid == 0) {
        for (uint32_t s = 0; s < GM_STAGES; ++s) mbar_init(&bars->full[s], leader ? 2u : 1u), mbar_init(&bars->empty[s], 1);
        mbar_init(&bars->acc_full, 1);
        mbar_init(&bars->acc_empty, leader ? 2u * GM_EPI_WARPS : 1u);
        bars->abort = 0;
        mbar_init_fence();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem_base)),
                     "r"(512u)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    cluster_sync_all();   // both CTAs' barriers exist before anyone arrives remotely
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = bars->tmem_base;   // 0: all columns are this CTA's (the MMA loop counts on it)
    asm volatile("griddepcontrol.wait;" ::: "memory");   // an ordered launch: see axc_tuning.pdl
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    if (warp == 0) {
        // The whole warp runs the loop, an elected lane issues.
        uint32_t issued = 0, s = 0, ph = 1;
        bool ok = true;
        Pieces it(p, pair, pairs);
        while (ok && it.next()) {
            const uint32_t row0 = it.row_tile * GM_ROWS + rank * 128u, tok0 = it.tok0;
            // scale tiles that exist: the last row tile may have no rows for the second CTA, the last tokens one tile
            const bool has_rows = row0 / 128u < row_tiles;
            const uint32_t a_tiles = min(2u, tok_tiles - tok0 / 128u);
            const uint8_t* sw = p.w_scales + (uint64_t)(row0 / 128u) * n_quads * MX_TILE_BYTES;
            const uint8_t* sa = p.a_scales + (uint64_t)(tok0 / 128u) * n_quads * MX_TILE_BYTES;
            for (uint32_t st = 0; st < n_st; ++st, ++issued) {
                ok = __all_sync(0xFFFFFFFFu, mbar_wait_or_abort(&bars->empty[s], ph, &bars->abort, p.status));
                if (!ok) break;
                if (elect_one()) {
                    const uint32_t quad_bytes = min(2u, n_quads - st * 2u) * MX_TILE_BYTES;
                    uint8_t* stage = sm + s * GM_STAGE_BYTES;
                    mbar_expect_tx(&bars->full[s], GM_W_BYTES + GM_A_BYTES + ((has_rows ? 1u : 0u) + a_tiles) * quad_bytes);
                    tma_load_2d(base + s * GM_STAGE_BYTES, &tm_w, (int32_t)(st * 128u), (int32_t)row0, &bars->full[s]);
                    tma_load_2d(base + s * GM_STAGE_BYTES + GM_OFF_A, &tm_a, (int32_t)(st * 128u), (int32_t)(tok0 + rank * (it.n / 2u)),
                                &bars->full[s]);   // a whole box; the MMA takes the first half of the piece's tokens
                    if (has_rows) bulk_g2s(stage + GM_OFF_SFW, sw + (uint64_t)st * 2u * MX_TILE_BYTES, quad_bytes, &bars->full[s]);
                    bulk_g2s(stage + GM_OFF_SFA, sa + (uint64_t)st * 2u * MX_TILE_BYTES, quad_bytes, &bars->full[s]);
                    if (a_tiles > 1u)
                        bulk_g2s(stage + GM_OFF_SFA + 1024u, sa + ((uint64_t)n_quads + st * 2u) * MX_TILE_BYTES, quad_bytes,
                                 &bars->full[s]);
                }
                __syncwarp();
                if (++s == GM_STAGES) s = 0, ph ^= 1u;
            }
        }
        // nothing may still be in flight towards this CTA's shared memory at exit
        for (uint32_t j = issued > GM_STAGES ? issued - GM_STAGES : 0; j < issued; ++j)
            (void)mbar_wait(&bars->full[j % GM_STAGES], (j / GM_STAGES) & 1u, p.status);
    } else if (warp == 1) {
        if (leader) {
            bool ok = true;
            uint32_t s = 0, ph = 0, acc_ph = 1;
            Pieces it(p, pair, pairs);
            if (elect_one()) for (; ok && it.next(); acc_ph ^= 1u) {
                const uint32_t idesc = mx_idesc(256u, it.n, 0u), idesc2 = mx_idesc(256u, it.n, 2u);
                ok = mbar_wait_or_abort(&bars->acc_empty, acc_ph, &bars->abort, p.status);   // the last piece is read
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                for (uint32_t st = 0; st < n_st; ++st) {
                    ok = mbar_wait_or_abort(&bars->full[s], ph, &bars->abort, p.status);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t steps = min(4u, (p.n_blocks - st * 8u + 1u) / 2u);
                    {
                        const uint32_t sf = GM_SF_COL + s * 24u, stage = base + s * GM_STAGE_BYTES;
#pragma unroll
                        for (uint32_t g = 0; g < 2u; ++g) {
                            if (2u * g >= steps) break;
                            scales_to_tmem_pair(sf + g * 4u, stage + GM_OFF_SFW + g * MX_TILE_BYTES);
                            scales_to_tmem_pair(sf + 8u + g * 8u, stage + GM_OFF_SFA + g * MX_TILE_BYTES);
                            scales_to_tmem_pair(sf + 12u + g * 8u, stage + GM_OFF_SFA + 1024u + g * MX_TILE_BYTES);
                        }
                        const uint64_t wd = sw128_desc(stage), ad = sw128_desc(stage + GM_OFF_A);
#pragma unroll
                        for (uint32_t kk = 0; kk < 4u; ++kk) {
                            if (kk >= steps) break;
                            umma_mxf4_pair(0u, wd + 2u * kk, ad + 2u * kk, kk & 1u ? idesc2 : idesc,
                                           sf + (kk >> 1) * 4u, sf + 8u + (kk >> 1) * 8u, (st | kk) != 0u);
                        }
                        umma_commit_pair(&bars->empty[s]);
                        if (st + 1u == n_st) umma_commit_pair(&bars->acc_full);
                    }
                    if (++s == GM_STAGES) s = 0, ph ^= 1u;
                }
            }
        } else if (lane == 0) {
            // peer: tell the leader when this CTA's stage has landed
            uint32_t s = 0, ph = 0;
            bool ok = true;
            Pieces it(p, pair, pairs);
            while (ok && it.next())
                for (uint32_t st = 0; st < n_st; ++st) {
                    ok = mbar_wait_or_abort(&bars->full[s], ph, &bars->abort, p.status);
                    if (!ok) break;
                    mbar_arrive_remote(&bars->full[s], 0u);
                    if (++s == GM_STAGES) s = 0, ph ^= 1u;
                }
        }
    } else {
        // ---------------- epilogue: TMEM lane = weight row, column = token ----------------
        const uint32_t quad = warp & 3u, half = (warp - 2u) >> 2;   // warps 2..5: the first half of the tokens, 6..9: the second
        uint32_t ph = 0;
        bool ok = true, arrived = false;
        for (Pieces it(p, pair, pairs); ok && it.next(); ph ^= 1u) {
            const uint32_t row = it.row_tile * GM_ROWS + rank * 128u + quad * 32u + lane;
            const uint32_t col0 = half * (it.n / 2u), tok0 = it.tok0 + col0;
            ok = __all_sync(0xFFFFFFFFu, mbar_wait_or_abort(&bars->acc_full, ph, &bars->abort, p.status));
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            uint32_t v[8][16];
#pragma unroll
            for (uint32_t b = 0; b < 8u; ++b)
                if (b * 32u < it.n) tmem_load16(tmem + ((quad * 32u) << 16) + col0 + b * 16u, v[b]);
            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) {
                if (leader) mbar_arrive(&bars->acc_empty);
                else mbar_arrive_remote(&bars->acc_empty, 0u);
            }
            if (it.last()) {
                // this warp's part in the cluster barrier at the end, in front of the stores that then hide it (512 x 9472 x
                // 4096 with fp32 output 12.2 -> 11.7 us)
                __syncwarp();
                cluster_arrive();
                arrived = true;
            }
            if (row < p.rows && tok0 < p.m) {
                // sixteen tokens without a test per value: with tests a warp took 10 000 cycles here instead of the
                // 3 400 that fit behind the next piece's MMAs (2048 x 18944 x 4096: 68 us)
                Out* dst = reinterpret_cast<Out*>(p.c) + (uint64_t)tok0 * p.rows + row;
                const uint32_t count = min(p.m - tok0, it.n / 2u);
#pragma unroll
                for (uint32_t b = 0; b < 8u; ++b) {
                    if (b * 16u + 16u <= count) {
#pragma unroll
                        for (uint32_t j = 0; j < 16u; ++j, dst += p.rows) put(dst, __uint_as_float(v[b][j]));
                    } else {
#pragma unroll
                        for (uint32_t j = 0; j < 16u; ++j, dst += p.rows)
                            if (b * 16u + j < count) put(dst, __uint_as_float(v[b][j]));
                    }
                }
            }
        }
        if (!ok) bars->abort = 1;
        __syncwarp();
        if (!arrived) cluster_arrive();
    }
    if (warp < 2u) {
        __syncwarp();
        cluster_arrive();
    }
    cluster_wait();   // no remote arrive or multicast commit may still target a CTA that left; tensor memory is read
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

template <typename Out>
cudaError_t launch(const CUtensorMap& tm_w, const CUtensorMap& tm_a, const GmArgs& p, cudaStream_t stream, int sm_count) {
    auto kern = mx_gemm_kernel<Out>;
    cudaLaunchConfig_t cfg{};
    cfg.blockDim = dim3(GM_THREADS), cfg.dynamicSmemBytes = GM_SMEM, cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2, attr[0].val.clusterDim.y = 1, attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    int pairs = sm_count / 2;
    {   // once per device: raise the shared-memory limit, ask how many pairs fit at once
        static std::mutex mu;
        static int fits[64] = {};
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        std::lock_guard<std::mutex> lock(mu);
        if (dev < 0 || dev >= 64 || fits[dev] == 0) {
            e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)GM_SMEM);
            if (e != cudaSuccess) return e;
            int n = 0;
            cfg.gridDim = dim3(2u * (unsigned)pairs), cfg.numAttrs = 1;
            if (cudaOccupancyMaxActiveClusters(&n, kern, &cfg) != cudaSuccess || n <= 0) n = pairs, cudaGetLastError();
            if (dev >= 0 && dev < 64) fits[dev] = n;
            if (n < pairs) pairs = n;
        } else if (fits[dev] < pairs) {
            pairs = fits[dev];
        }
    }
    cfg.gridDim = dim3(2u * (p.pieces < (uint32_t)pairs ? p.pieces : (uint32_t)pairs)), cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kern, tm_w, tm_a, p);
}

}  // namespace

cudaError_t launch_mxfp4_gemm(const uint8_t* w_codes, const uint8_t* w_scales, const uint8_t* a_codes, const uint8_t* a_scales,
                              void* c, ElemType type, uint32_t m_tokens, uint32_t n_rows, uint32_t n_blocks,
                              uint32_t* status, cudaStream_t stream, int sm_count) {
    if (!tensor_map_encoder()) return cudaErrorNotSupported;
    CUtensorMap tm_w, tm_a;
    if (!mx_encode_codes(&tm_w, w_codes, n_rows, n_blocks, 128u) || !mx_encode_codes(&tm_a, a_codes, m_tokens, n_blocks, 128u))
        return cudaErrorInvalidValue;
    const uint32_t token_pieces = (m_tokens + GM_TOKENS - 1u) / GM_TOKENS;
    const uint64_t pieces = (uint64_t)((n_rows + GM_ROWS - 1u) / GM_ROWS) * token_pieces;
    if (pieces >= 1u << 31) return cudaErrorInvalidConfiguration;
    const GmArgs p{w_scales, a_scales, c, m_tokens, n_rows, n_blocks, token_pieces, (uint32_t)pieces, status};
    switch (type) {
        case ElemType::F32: return launch<float>(tm_w, tm_a, p, stream, sm_count);
        case ElemType::BF16: return launch<__nv_bfloat16>(tm_w, tm_a, p, stream, sm_count);
        case ElemType::F16: return launch<__half>(tm_w, tm_a, p, stream, sm_count);
    }
    return cudaErrorInvalidValue;
}

}  // namespace axc
