// Products with an MXFP4 matrix W on the block-scaled tensor-core path (tcgen05.mma kind::mxf4, 4-bit operands with
// one power-of-two scale per 32 values, fp32 accumulators in tensor memory).
//
//   prefill   C[m][n] = sum_k A[m][k] W[n][k], A in MXFP4 too: the operands go from memory to the tensor cores as
//             they lie there, codes through TMA (128-byte swizzle), scales through shared into tensor memory.
//   matvec    y[t][r] = sum_k W[r][k] x[t][k] for a few fp32 vectors x, without rounding them to 4 bits: within each
//             block of 32 columns x is a 23-bit integer X times a power of two, and X is written in eight digits of
//             base 8, v_0 .. v_7 in -4 .. 3, X = sum v_d 8^d.  Every digit is an E2M1 value (half of it is one of
//             0, 0.5, 1, 1.5, 2, whose codes count 0, 1, 2, 3, 4), so one token is eight rows of an MXFP4 matrix
//             that differ in their scales by factors of 8, and the product with these rows is the same tensor-core
//             product.  y is the sum of its eight columns.  A weight never passes through a register.
//
// A CTA owns up to 128 weight rows (the MMA's M, one TMEM lane each) and one token tile of up to 256 columns (the
// MMA's N), and streams K through a ring of stages of 256 columns:
//
//   warp 0       one thread: TMA loads of the codes of W (and of A), bulk copies of A's scales
//   warp 1       one thread: scales from shared into tensor memory (tcgen05.cp), four MMAs of 64 columns per stage,
//                and the commit that frees the stage; the whole warp allocates and frees tensor memory
//   warps 2..5   the scales of this CTA's rows, arranged as the MMA takes them; then the epilogue
//   warps 6..9   matvec only: digits and scales of x
//
// The rows of a CTA need not start at a multiple of 128, so that a matrix spreads over all SMs evenly; that is why
// warps 2..5 arrange the scales instead of a copy of whole tiles.
//
// The accumulators truncate: measured, a chain of K / 64 MMAs loses up to 1.2e-7 * K / 512 of its value when the
// scales of a row are far apart (and nothing while all partial sums are multiples of one unit below 2^24).  So a
// chain ends after 4096 columns; the next ones go to further accumulators as long as tensor memory has columns, and
// the parts are added in fp32 in the epilogue.
//
// Every wait on an mbarrier is bounded; a wait that runs out sets an error bit and an abort flag, all roles fall
// through to the common exit, outstanding copies are waited for and tensor memory is freed.
#include <mutex>

#include "axc_kernels.h"
#include "axc_mx.cuh"
#include "axc_umma.cuh"

namespace axc {
namespace {

constexpr uint32_t MP_ROWS = 128;
constexpr uint32_t MP_STAGE_BYTES = 128;            // one stage: 256 columns = 128 bytes of codes per row
constexpr uint32_t MP_CHAIN = 16;                   // stages per accumulator: 4096 columns
constexpr uint32_t MP_MAX_STAGES = 12;
constexpr uint32_t MP_ROW_WARPS = 4, MP_X_WARPS = 4;

__device__ __forceinline__ void scales_to_tmem(uint32_t taddr, uint32_t smem_addr) {
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(mx_scale_desc(smem_addr)) : "memory");
}

__device__ __forceinline__ void umma_mxf4(uint32_t d, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t sfa,
                                          uint32_t sfb, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %6, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%4], [%5], p;\n\t}" ::"r"(d),
        "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(sfa), "r"(sfb), "r"(accumulate)
        : "memory");
}

struct MpArgs {
    const uint8_t* w_scales;
    const uint8_t* a_scales;    // prefill
    const float* x;             // matvec
    void* out;
    uint32_t m, rows, n_blocks;
    uint32_t rows_per_cta;      // 1..128
    uint32_t n;                 // columns of the MMA = rows of the B operand per token tile
    uint32_t n_acc, tmem_cols;
    uint32_t stages;
    uint32_t off_b, off_sfa, off_sfb, off_bar, a_stage, b_stage, sfb_stage;   // shared-memory layout
    uint32_t out_type;
    uint32_t* status;
};

struct MpBars {
    uint64_t full[MP_MAX_STAGES], empty[MP_MAX_STAGES];
    uint64_t done;
    uint32_t tmem_base;
    volatile uint32_t abort;
};

// A word of eight octal digits v = -4..3, each as its low three bits in a nibble, to the eight E2M1 codes of v / 2:
// t = 0..3 is its own code, t = 4..7 stands for t - 8, code 8 | (8 - t) = 16 - t.
__device__ __forceinline__ uint32_t digit_codes(uint32_t t) {
    const uint32_t neg = (t >> 2) & 0x11111111u;
    return (t ^ (neg * 15u)) + neg;
}

// 24 bits = eight octal fields to eight nibbles.
__device__ __forceinline__ uint32_t spread_octal(uint32_t y) {
    y = (y & 0xFFFu) | ((y & 0xFFF000u) << 4);
    y = (y & 0x003F003Fu) | ((y & 0x0FC00FC0u) << 2);
    return (y & 0x07070707u) | ((y & 0x38383838u) << 1);
}

// 8 x 8 nibbles: w[e] holds digit d of element e in nibble d; afterwards w[d] holds it in nibble e.
__device__ __forceinline__ void transpose_nibbles(uint32_t (&w)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const uint32_t a = w[i], b = w[i + 1];
        w[i] = (a & 0x0F0F0F0Fu) | ((b & 0x0F0F0F0Fu) << 4);
        w[i + 1] = ((a >> 4) & 0x0F0F0F0Fu) | (b & 0xF0F0F0F0u);
    }
#pragma unroll
    for (int i = 0; i < 8; i += 4)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint32_t a = w[i + j], b = w[i + j + 2];
            w[i + j] = __byte_perm(a, b, 0x6240);
            w[i + j + 2] = __byte_perm(a, b, 0x7351);
        }
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const uint32_t a = w[j], b = w[j + 4];
        w[j] = __byte_perm(a, b, 0x5410);
        w[j + 4] = __byte_perm(a, b, 0x7632);
    }
}

__device__ __forceinline__ void store_out(const MpArgs& p, uint64_t at, float v) {
    if (p.out_type == (uint32_t)ElemType::F32) reinterpret_cast<float*>(p.out)[at] = v;
    else if (p.out_type == (uint32_t)ElemType::BF16) reinterpret_cast<__nv_bfloat16*>(p.out)[at] = __float2bfloat16_rn(v);
    else reinterpret_cast<__half*>(p.out)[at] = __float2half_rn(v);
}

template <bool DIGITS>
__global__ void __launch_bounds__((2 + MP_ROW_WARPS + (DIGITS ? MP_X_WARPS : 0)) * 32, 1)
mx_product_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_a, const MpArgs p) {
    extern __shared__ uint8_t smem_dyn[];
    const uint32_t raw_addr = smem_u32(smem_dyn);
    const uint32_t base = (raw_addr + 1023u) & ~1023u;   // the swizzled tiles need 1024-byte alignment
    uint8_t* sm = smem_dyn + (base - raw_addr);
    MpBars* bars = reinterpret_cast<MpBars*>(sm + p.off_bar);

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t row0 = blockIdx.x * p.rows_per_cta;
    const uint32_t tok0 = blockIdx.y * 256u;
    const uint32_t n_st = (p.n_blocks + 7u) / 8u, n_quads = (p.n_blocks + 3u) / 4u;
    const uint32_t b_tiles = (p.n + 127u) / 128u;
    const uint32_t a_tiles = DIGITS ? 0u : min(b_tiles, (p.m - tok0 + 127u) / 128u);   // scale tiles that A has here

    if (tid == 0) {
        for (uint32_t s = 0; s < p.stages; ++s)
            mbar_init(&bars->full[s], 1u + MP_ROW_WARPS + (DIGITS ? p.m : 0u)), mbar_init(&bars->empty[s], 1);
        mbar_init(&bars->done, 1);
        bars->abort = 0;
        mbar_init_fence();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem_base)),
                     "r"(p.tmem_cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = bars->tmem_base;
    // An ordered launch (see axc_tuning.pdl).  The weights too are read after the wait: a quantise call directly
    // before this one may have written them.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    if (warp == 0) {
        if (lane == 0) {
            uint32_t issued = 0;
            for (uint32_t st = 0; st < n_st && !bars->abort; ++st, ++issued) {
                const uint32_t s = st % p.stages, ph = (st / p.stages) & 1u;
                if (!mbar_wait(&bars->empty[s], ph ^ 1u, p.status)) {
                    bars->abort = 1;
                    break;
                }
                const uint32_t quads = min(2u, n_quads - st * 2u);   // scale tiles of this stage
                uint32_t bytes = p.rows_per_cta * MP_STAGE_BYTES;
                if (!DIGITS) bytes += p.n * MP_STAGE_BYTES + a_tiles * quads * MX_TILE_BYTES;
                mbar_expect_tx(&bars->full[s], bytes);
                tma_load_2d(base + s * p.a_stage, &tm_w, (int32_t)(st * MP_STAGE_BYTES), (int32_t)row0, &bars->full[s]);
                if constexpr (!DIGITS) {
                    tma_load_2d(base + p.off_b + s * p.b_stage, &tm_a, (int32_t)(st * MP_STAGE_BYTES), (int32_t)tok0, &bars->full[s]);
                    for (uint32_t q = 0; q < a_tiles; ++q)
                        bulk_g2s(sm + p.off_sfb + s * p.sfb_stage + q * 2u * MX_TILE_BYTES,
                                 p.a_scales + ((uint64_t)(tok0 / 128u + q) * n_quads + st * 2u) * MX_TILE_BYTES,
                                 quads * MX_TILE_BYTES, &bars->full[s]);
                }
            }
            // nothing may still be in flight towards this CTA's shared memory at exit
            for (uint32_t j = issued > p.stages ? issued - p.stages : 0; j < issued; ++j)
                (void)mbar_wait(&bars->full[j % p.stages], (j / p.stages) & 1u, p.status);
        }
    } else if (warp == 1) {
        if (lane == 0) {
            bool ok = true;
            const uint32_t sf0 = tmem + p.n_acc * p.n;     // scale columns: 2 slots x 2 tiles x (4 + 4 * b_tiles)
            for (uint32_t st = 0; st < n_st && !bars->abort; ++st) {
                const uint32_t s = st % p.stages, ph = (st / p.stages) & 1u;
                ok = mbar_wait(&bars->full[s], ph, p.status);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t slot = sf0 + (st & 1u) * (8u + 8u * b_tiles);
                const uint32_t steps = min(4u, (p.n_blocks - st * 8u + 1u) / 2u);   // MMAs of 64 columns
                for (uint32_t g = 0; g < (steps + 1u) / 2u; ++g) {
                    scales_to_tmem(slot + g * 4u, base + p.off_sfa + s * 1024u + g * MX_TILE_BYTES);
                    for (uint32_t q = 0; q < b_tiles; ++q)
                        scales_to_tmem(slot + 8u + (g * b_tiles + q) * 4u,
                                       base + p.off_sfb + s * p.sfb_stage + (q * 2u + g) * MX_TILE_BYTES);
                }
                const uint64_t ad = sw128_desc(base + s * p.a_stage), bd = sw128_desc(base + p.off_b + s * p.b_stage);
                const uint32_t chain = min(st / MP_CHAIN, p.n_acc - 1u);
                const uint32_t first = st == chain * MP_CHAIN;   // the chain's first stage overwrites its accumulator
                for (uint32_t kk = 0; kk < steps; ++kk)          // 64 codes = 32 bytes = 2 descriptor units per step
                    umma_mxf4(tmem + chain * p.n, ad + 2u * kk, bd + 2u * kk, mx_idesc(128u, p.n, (kk & 1u) * 2u),
                              slot + (kk >> 1) * 4u, slot + 8u + (kk >> 1) * b_tiles * 4u, !(first && kk == 0u));
                umma_commit(&bars->empty[s]);
            }
            if (!ok) bars->abort = 1;
            umma_commit(&bars->done);     // accumulators complete (or nothing outstanding)
        }
    } else if (warp < 2u + MP_ROW_WARPS) {
        // ---------------- scales of this CTA's rows: thread = row ----------------
        const uint32_t r = (warp & 3u) * 32u + lane;     // also the TMEM lane of the epilogue
        const uint64_t row = (uint64_t)row0 + r;
        const bool mine = r < p.rows_per_cta && row < p.rows;
        bool ok = true;
        for (uint32_t st = 0; st < n_st && ok; ++st) {
            const uint32_t s = st % p.stages, ph = (st / p.stages) & 1u;
            uint32_t w[2] = {0, 0};
#pragma unroll
            for (uint32_t g = 0; g < 2; ++g)
                if (mine && st * 2u + g < n_quads)
                    w[g] = __ldg(reinterpret_cast<const uint32_t*>(p.w_scales + mx_scale_at(row, st * 2u + g, n_quads)));
            ok = __all_sync(0xFFFFFFFFu, mbar_wait(&bars->empty[s], ph ^ 1u, p.status) && !bars->abort);
            if (!ok) break;
#pragma unroll
            for (uint32_t g = 0; g < 2; ++g)
                *reinterpret_cast<uint32_t*>(sm + p.off_sfa + s * 1024u + g * MX_TILE_BYTES + (r & 31u) * 16u + (r >> 5) * 4u) = w[g];
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // generic writes -> async proxy
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->full[s]);
        }
        if (!ok) bars->abort = 1;

        // ---------------- epilogue: TMEM lane = weight row ----------------
        ok = __all_sync(0xFFFFFFFFu, mbar_wait(&bars->done, 0u, p.status) && !bars->abort);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (ok) {
            const uint32_t used = min(p.n_acc, (n_st + MP_CHAIN - 1u) / MP_CHAIN);
            const uint32_t count = DIGITS ? p.m * 8u : min(p.n, p.m - tok0);
            for (uint32_t c = 0; c < count; c += 8u) {
                float sum[8] = {};
                for (uint32_t a = 0; a < used; ++a) {
                    uint32_t v[8];
                    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                                 : "r"(tmem + (((warp & 3u) * 32u) << 16) + a * p.n + c)
                                 : "memory");
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                    for (int j = 0; j < 8; ++j) sum[j] += __uint_as_float(v[j]);
                }
                if (!mine) continue;
                if (DIGITS) {
                    float y = sum[0];
#pragma unroll
                    for (int j = 1; j < 8; ++j) y += sum[j];
                    reinterpret_cast<float*>(p.out)[(uint64_t)(c >> 3) * p.rows + row] = y;
                } else {
#pragma unroll
                    for (uint32_t j = 0; j < 8u; ++j)
                        if (c + j < count) store_out(p, (uint64_t)(tok0 + c + j) * p.rows + row, sum[j]);
                }
            }
        }
    } else if (DIGITS) {
        // ---------------- digits of x: a warp takes 256 columns of one token, a lane 8 of them ----------------
        const uint32_t k_total = p.n_blocks * 32u;
        bool ok = true;
        for (uint64_t u = warp - (2u + MP_ROW_WARPS); u < (uint64_t)n_st * p.m && ok; u += MP_X_WARPS) {
            const uint32_t st = (uint32_t)(u / p.m), t = (uint32_t)(u - (uint64_t)st * p.m);
            const uint32_t s = st % p.stages, ph = (st / p.stages) & 1u;
            const uint32_t col = st * 256u + lane * 8u;
            float v[8] = {};
            if (col < k_total) {     // k_total is a multiple of 32
                const float4* src = reinterpret_cast<const float4*>(p.x + (uint64_t)t * k_total + col);
                const float4 a = __ldg(src), b = __ldg(src + 1);
                v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
            }
            uint32_t top = 0;
#pragma unroll
            for (int i = 0; i < 8; ++i) top = max(top, (uint32_t)__float_as_int(v[i]) & 0x7FFFFFFFu);
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
            top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
            // X = rn(x * 2^(22 - e)), e = exponent of the block's largest |x| plus one, so |X| <= 2^22; the unit of
            // digit 0, with the half that a code counts, is 2^(e - 21): scale byte e - 21 + 127.  Blocks below
            // 2^-105 keep the smallest unit 2^-127; 2^127 and above count as infinite (scale byte 255).
            const uint32_t ex = top >> 23;                               // e = ex - 126
            const bool bad = ex >= 254u;
            const uint32_t unit = bad ? 0u : ex > 20u ? ex - 20u : 0u;   // scale byte of digit 0
            // 2^(22 - e) = 2^(128 - unit): in two factors, since 2^128 is not a float
            const float f1 = __int_as_float((int)((254u - unit) << 23));  // 2^(127 - unit)
            uint32_t w[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                // + 1.5 * 2^23 rounds to an integer in the low mantissa bits; + 4 in every octal digit, then ^ 4
                // gives the digits -4..3 as three-bit two's complement fields
                const float shifted = __fmaf_rn(v[i] * f1, 2.0f, 12582912.0f);
                const uint32_t biased = (uint32_t)__float_as_int(shifted) + (0x00924924u - 0x4B400000u);
                w[i] = spread_octal((bad ? 0x00924924u : biased) ^ 0x00924924u);
            }
            transpose_nibbles(w);
            uint32_t sb = unit << (8u * ((lane >> 2) & 3u)), nan = bad ? 255u << (8u * ((lane >> 2) & 3u)) : 0u;
            sb |= __shfl_xor_sync(0xFFFFFFFFu, sb, 4), nan |= __shfl_xor_sync(0xFFFFFFFFu, nan, 4);
            sb |= __shfl_xor_sync(0xFFFFFFFFu, sb, 8), nan |= __shfl_xor_sync(0xFFFFFFFFu, nan, 8);
            ok = __all_sync(0xFFFFFFFFu, mbar_wait(&bars->empty[s], ph ^ 1u, p.status) && !bars->abort);
            if (!ok) break;
            // row d of the token's eight rows; the 16-byte chunk j of a row sits at chunk j ^ (row & 7)
            uint8_t* tile = sm + p.off_b + s * p.b_stage + t * 1024u;
#pragma unroll
            for (uint32_t d = 0; d < 8u; ++d)
                *reinterpret_cast<uint32_t*>(tile + d * 128u + (((lane >> 2) ^ d) << 4) + (lane & 3u) * 4u) = digit_codes(w[d]);
            // scales: lanes 0..7 write the first four blocks, lanes 16..23 the others; digit d is 8^d units
            if ((lane & 15u) < 8u) {
                const uint32_t d = lane & 15u, n = t * 8u + d;
                *reinterpret_cast<uint32_t*>(sm + p.off_sfb + s * p.sfb_stage + (lane >> 4) * MX_TILE_BYTES + (n & 31u) * 16u +
                                             (n >> 5) * 4u) = (sb + 0x03030303u * d) | nan;
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive(&bars->full[s]);
        }
        if (!ok) bars->abort = 1;
    }

    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.tmem_cols) : "memory");
    }
}

template <bool DIGITS>
cudaError_t launch(const uint8_t* w_codes, const uint8_t* a_codes, MpArgs p, uint32_t smem_budget, uint32_t token_tiles,
                   cudaStream_t stream) {
    if (!tensor_map_encoder()) return cudaErrorNotSupported;
    // Shared memory: W stages, B stages, row scales, B scales, barriers.  The MMA reads 128 rows of a W stage; the
    // ones behind this CTA's rows are the next stage or what follows (their results are not used), and the region
    // behind the last stage is larger than that.
    const uint32_t b_tiles = (p.n + 127u) / 128u, n_st = (p.n_blocks + 7u) / 8u;
    p.a_stage = (p.rows_per_cta + 7u) / 8u * 1024u;
    p.b_stage = p.n * MP_STAGE_BYTES;
    p.sfb_stage = b_tiles * 1024u;
    const uint32_t per_stage = p.a_stage + p.b_stage + 1024u + p.sfb_stage;
    const uint32_t fixed = 1024u + (uint32_t)sizeof(MpBars) + MP_ROWS * MP_STAGE_BYTES - p.a_stage;
    uint32_t stages = (smem_budget - fixed) / per_stage;
    if (stages > MP_MAX_STAGES) stages = MP_MAX_STAGES;
    if (stages > n_st) stages = n_st;
    if (stages < 1u) stages = 1u;
    p.stages = stages;
    p.off_b = stages * p.a_stage;
    p.off_sfa = p.off_b + stages * p.b_stage;
    p.off_sfb = p.off_sfa + stages * 1024u;
    p.off_bar = p.off_sfb + stages * p.sfb_stage;
    const uint32_t smem = fixed + stages * per_stage;
    // tensor memory: accumulators for chains of 4096 columns as far as they fit, two slots of scales
    const uint32_t sf_cols = 2u * (8u + 8u * b_tiles);
    uint32_t want = (n_st + MP_CHAIN - 1u) / MP_CHAIN;
    uint32_t cols = 32u;
    while (cols < p.n + sf_cols || (cols < 128u && cols < want * p.n + sf_cols)) cols *= 2u;
    p.tmem_cols = cols;
    p.n_acc = (cols - sf_cols) / p.n;
    if (p.n_acc > want) p.n_acc = want;
    CUtensorMap tm_w, tm_a;
    if (!mx_encode_codes(&tm_w, w_codes, p.rows, p.n_blocks, p.rows_per_cta)) return cudaErrorInvalidValue;
    if (DIGITS) tm_a = tm_w;
    else if (!mx_encode_codes(&tm_a, a_codes, p.m, p.n_blocks, p.n)) return cudaErrorInvalidValue;
    auto kern = mx_product_kernel<DIGITS>;
    {
        static std::mutex mu;
        static bool done[64] = {};
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        std::lock_guard<std::mutex> lock(mu);
        if (dev < 0 || dev >= 64 || !done[dev]) {
            e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024);
            if (e != cudaSuccess) return e;
            if (dev >= 0 && dev < 64) done[dev] = true;
        }
    }
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((p.rows + p.rows_per_cta - 1u) / p.rows_per_cta, token_tiles);
    cfg.blockDim = dim3((2u + MP_ROW_WARPS + (DIGITS ? MP_X_WARPS : 0u)) * 32u);
    cfg.dynamicSmemBytes = smem, cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr, cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kern, tm_w, tm_a, p);
}

}  // namespace

cudaError_t launch_mxfp4_matvec(const uint8_t* codes, const uint8_t* scales, const float* x, float* y, uint32_t m_tokens,
                                uint32_t rows, uint32_t n_blocks, uint32_t* status, cudaStream_t stream, int sm_count) {
    if (m_tokens == 0 || rows == 0 || n_blocks == 0) return cudaSuccess;
    MpArgs p{};
    p.w_scales = scales, p.x = x, p.out = y, p.m = m_tokens, p.rows = rows, p.n_blocks = n_blocks, p.status = status;
    p.out_type = (uint32_t)ElemType::F32;
    p.n = (m_tokens + 1u) / 2u * 16u;
    // rows spread evenly over the SMs, in as many rounds as 128 rows per CTA make necessary
    const uint32_t sms = (uint32_t)sm_count;
    const uint32_t rounds = (uint32_t)(((uint64_t)rows + 128ull * sms - 1u) / (128ull * sms));
    p.rows_per_cta = (uint32_t)(((uint64_t)rows + (uint64_t)rounds * sms - 1u) / ((uint64_t)rounds * sms));
    return launch<true>(codes, nullptr, p, 110u * 1024u, 1u, stream);
}

cudaError_t launch_mxfp4_prefill(const uint8_t* w_codes, const uint8_t* w_scales, const uint8_t* a_codes,
                                 const uint8_t* a_scales, void* c, ElemType type, uint32_t m_tokens, uint32_t n_rows,
                                 uint32_t n_blocks, uint32_t* status, cudaStream_t stream, int sm_count) {
    if (m_tokens == 0 || n_rows == 0 || n_blocks == 0) return cudaSuccess;
    if (m_tokens > 64u)
        return launch_mxfp4_gemm(w_codes, w_scales, a_codes, a_scales, c, type, m_tokens, n_rows, n_blocks, status, stream, sm_count);
    MpArgs p{};
    p.w_scales = w_scales, p.a_scales = a_scales, p.out = c, p.m = m_tokens, p.rows = n_rows, p.n_blocks = n_blocks;
    p.status = status, p.out_type = (uint32_t)type;
    p.n = m_tokens >= 256u ? 256u : (m_tokens + 15u) / 16u * 16u;
    const uint32_t sms = (uint32_t)sm_count, token_tiles = (m_tokens + 255u) / 256u;
    (void)sms;
    p.rows_per_cta = 128u;
    return launch<false>(w_codes, a_codes, p, 220u * 1024u, token_tiles, stream);
}

}  // namespace axc
