// Products with an MXFP4 matrix W on the block-scaled tensor-core path (tcgen05.mma kind::mxf4, 4-bit operands with
// one power-of-two scale per 32 values, fp32 accumulators in tensor memory).
//
//   prefill   C[m][n] = sum_k A[m][k] W[n][k], A in MXFP4 too: the operands go from memory to the tensor cores as
//             they lie there, codes through TMA (128-byte swizzle), scales through shared into tensor memory.
//   matvec    y[t][r] = sum_k W[r][k] x[t][k] for a few fp32 vectors x.  They are rounded, though not to 4 bits: within
//             each block of 32 columns x is a 23-bit integer X with sign times a power of two, off by at most 2^-22 of
//             the block's largest |x| (an fp32 is off by 2^-24 of each value: a value beside one 2^20 times as large
//             keeps two bits).  X is written in eight digits of base 8, v_0 .. v_7 in -4 .. 3, X = sum v_d 8^d, which
//             is what one step of eight columns holds; more digits would widen every MMA and double the work of
//             splitting x.  Every digit is an E2M1 value (half of it is one of
//             0, 0.5, 1, 1.5, 2, whose codes count 0, 1, 2, 3, 4), so one token is eight rows of an MXFP4 matrix
//             that differ in their scales by factors of 8, and the product with these rows is the same tensor-core
//             product.  y is the sum of its eight columns.  A weight never passes through a register.
//
// Both are bound by reading W.  A cluster of `splits` CTAs (1, 2, 4 or 8) owns one or two tiles of 128 weight rows (the
// MMA's M, one TMEM lane each) and all tokens, or 128 of them (its N columns); each CTA takes its share of K, so that small
// matrices too are spread over the SMs and a CTA has most of its share requested from memory at once.  Stages of 256 columns:
//
//   warp 0       TMA loads of the codes of W (and of A), bulk copies of the scale tiles
//   warps 1, 2   stages in turn: scales from shared into tensor memory (tcgen05.cp), four MMAs of 64 columns per tile and
//                stage, and the commit that frees the stage.  With few columns an MMA is quick (32 cycles for its 4 KB of
//                codes) and the issuing thread is the limit, about 550 cycles per stage: two take turns, each with an
//                accumulator of its own (14336 x 4096, one token: 8.2 -> 7.8 us; four are no faster than two)
//   warps 3...   matvec: digits and scales of x, a warp taking 256 columns of one token at a time; then, in both, the
//                epilogue: every CTA holds partial sums of all its cluster's rows, sends those of each 1/splits of the
//                rows to the CTA that finishes them (distributed shared memory), and adds what it got in rank order,
//                so results do not depend on timing.
//
// Measured, ordered launches back to back, weights that rotate over more than 640 MB (in brackets: the same weights again,
// which up to 126 MB lie in L2): matvec of one token 4096 x 4096 4.1 us (3.8), 14336 x 4096 7.4 us (6.6), 57344 x 8192 43.7 us
// (5.7 TB/s); five tokens 8192 x 28672 25.4 us (4.9 TB/s), eight 14336 x 4096 10.5 us; prefill of 37 tokens 4096 x 14336
// 9.1 us (8.6), of 128 12.4 us (11.5), of 256 15.8 us (15.1).  What an ordered launch adds to the time that its bytes take is
// a chain of latencies of about 3 us: x, its digits, the first stage, the MMAs, the cluster, the store.  With eight tokens the
// digits take as long again (every CTA splits x for its share of K), with more than 64 tokens the exchange of partial sums.
//
// Each place of the ring has its scale columns in tensor memory, which are free again when the place is.  The
// accumulators truncate: each MMA (64 columns) of a chain cuts off at most 2^-22 of the running sum, and nothing while all
// partial sums are multiples of one unit below 2^24.  Measured on positive products with scales 24 binades apart, where it
// is worst: 2.2e-10 of the value per column of a chain on average, always towards zero.  A chain is half of a CTA's share of
// K, and the parts are added in fp32 (300 x 1024 x 14336, chains of 1792 columns: 4.0e-7 on average, 1.1e-6 at most).
//
// Tensor memory and clusters: a CTA that waits for its cluster while another of the cluster waits for tensor memory
// could wait for good, so a CTA's shared memory is at least its share of tensor memory (columns / 512 of an SM), and
// whatever fits an SM finds its columns.  (They may lie anywhere: by their registers no more than two of these CTAs share
// an SM, and beside one power of two of columns the other's are always left in one piece.)
//
// Every wait on an mbarrier is bounded; a wait that runs out sets an error bit and an abort flag, all roles fall
// through to the common exit, outstanding copies are waited for and tensor memory is freed.
#include <mutex>

#include "axc_kernels.h"
#include "axc_mx.cuh"

namespace axc {
namespace {

constexpr uint32_t MP_ROWS = 128, MP_TOKENS = 128;   // most that a CTA takes of a tile of rows, of tokens
constexpr uint32_t MP_STAGE_BYTES = 128;            // one stage: 256 columns = 128 bytes of codes per row
constexpr uint32_t MP_W_BYTES = MP_ROWS * MP_STAGE_BYTES;
constexpr uint32_t MP_MAX_STAGES = 8;
constexpr uint32_t MP_PREFETCH = 16;                // stages requested into L2 before the dependency wait
constexpr uint32_t MP_MMA_WARPS = 2;
constexpr uint32_t MP_FIRST_X = 1 + MP_MMA_WARPS;   // the first of the warps that split x and run the epilogue
static_assert(MX_MATVEC_TOKENS * 8u <= MP_TOKENS / 2u, "eight columns per token: at most 64, see the tensor memory of two tiles");
// A unit of 256 columns of one token takes such a warp about 1500 cycles, most of them waiting: with two tiles, where a
// CTA has the SM to itself, 16 of them (8 tokens, 14336 x 4096: 10.7 us, with 8 warps 12.4 us).
__host__ __device__ constexpr uint32_t mp_x_warps(uint32_t tiles) { return 8u * tiles; }
__host__ __device__ constexpr uint32_t mp_threads(uint32_t tiles) { return (MP_FIRST_X + mp_x_warps(tiles)) * 32u; }
constexpr uint32_t MP_SMEM_SM = 228u * 1024u, MP_SMEM_MAX = 227u * 1024u;   // of an SM, of a CTA

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

__device__ __forceinline__ void tmem_load8(uint32_t taddr, uint32_t (&v)[8]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7])
                 : "r"(taddr)
                 : "memory");
}

struct MpArgs {
    const uint8_t* w_scales;
    const uint8_t* a_scales;    // prefill
    const float* x;             // matvec
    void* out;
    uint32_t m, rows, n_blocks;
    uint32_t splits, per_shift; // CTAs of a cluster; each finishes 1 << per_shift of its rows
    uint32_t n;                 // columns of the MMA = rows of the B operand
    uint32_t tmem_cols;
    uint32_t stages;
    uint32_t takers;            // matvec: warps that split x
    uint32_t off_b, off_sfw, off_sfb, off_red, off_bar;   // shared-memory layout
    uint32_t* status;
};

struct MpBars {
    uint64_t full[MP_MAX_STAGES], empty[MP_MAX_STAGES];
    uint64_t done;
    uint32_t tmem_base;
    volatile uint32_t abort;
};

// Eight octal fields f = v + 4 (v = -4..3), one per nibble, to the eight E2M1 codes of v / 2: v >= 0 is its own code,
// v < 0 has code 8 | -v = 16 - (v & 7).
__device__ __forceinline__ uint32_t digit_codes(uint32_t f) {
    const uint32_t neg = (~f >> 2) & 0x11111111u;
    return (f ^ 0x44444444u ^ (neg * 15u)) + neg;
}

// 24 bits = eight octal fields to eight nibbles: the upper half of each part moves up (hi * 2^k = hi + hi * (2^k - 1)).
__device__ __forceinline__ uint32_t spread_octal(uint32_t y) {
    y += (y & 0x00FFF000u) * 15u;
    y += (y & 0x0FC00FC0u) * 3u;
    return y + (y & 0x38383838u);
}

// 8 x 8 nibbles: w[e] holds digit d of element e in nibble d; afterwards w[d] holds it in nibble e.
__device__ __forceinline__ void transpose_nibbles(uint32_t (&w)[8]) {
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
        const uint32_t a = w[i], b = w[i + 1];
        w[i] = (a & 0x0F0F0F0Fu) | ((b << 4) & 0xF0F0F0F0u);
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

// max(a, |b|); a NaN stays.
__device__ __forceinline__ float max_abs(float a, float b) {
    float r;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(fabsf(b)));
    return r;
}

__device__ __forceinline__ void load_x(const MpArgs& p, uint32_t st, uint32_t t, uint32_t lane, float (&v)[8]) {
    const uint32_t k_total = p.n_blocks * 32u, col = st * 256u + lane * 8u;
    if (col < k_total) {     // k_total is a multiple of 32
        const float4* src = reinterpret_cast<const float4*>(p.x + (uint64_t)t * k_total + col);
        const float4 a = src[0], b = src[1];
        v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = 0.0f;
    }
}

// Digit codes w[d] of a lane's eight values, and the scale bytes of digit 0 of the four blocks of its half warp with the
// blocks that hold a value too large to count as finite.
__device__ __forceinline__ void split_x(const float (&v)[8], uint32_t lane, uint32_t (&w)[8], uint32_t& unit_bytes, uint32_t& nan) {
    float most = 0.0f;
#pragma unroll
    for (int i = 0; i < 8; ++i) most = max_abs(most, v[i]);
    uint32_t top = (uint32_t)__float_as_int(most);
    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 1));
    top = max(top, __shfl_xor_sync(0xFFFFFFFFu, top, 2));
    // X = rn(x * 2^(22 - e)), e = exponent of the block's largest |x| plus one, so |X| <= 2^22; the unit of digit 0,
    // with the half that a code counts, is 2^(e - 21): scale byte e - 21 + 127.  Blocks below 2^-105 keep digit 0 at
    // 2^-126, the unit of X at 2^-127; 2^127 and above count as infinite (scale byte 255, any digits).
    const uint32_t ex = top >> 23;                                // e = ex - 126
    const bool bad = ex >= 254u;
    const uint32_t unit = bad ? 1u : ex > 21u ? ex - 20u : 1u;    // scale byte of digit 0
    const float factor = __int_as_float((int)((255u - unit) << 23));   // 2^(22 - e) = 2^(128 - unit)
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        // + 1.5 * 2^23 rounds to an integer in the low mantissa bits; + 4 in every octal digit gives the fields v + 4
        const float shifted = __fmaf_rn(v[i], factor, 12582912.0f);
        w[i] = spread_octal((uint32_t)__float_as_int(shifted) + (0x00924924u - 0x4B400000u));
    }
    transpose_nibbles(w);
#pragma unroll
    for (int d = 0; d < 8; ++d) w[d] = digit_codes(w[d]);
    const uint32_t at = 8u * ((lane >> 2) & 3u);
    unit_bytes = unit << at, nan = bad ? 255u << at : 0u;
    unit_bytes |= __shfl_xor_sync(0xFFFFFFFFu, unit_bytes, 4), nan |= __shfl_xor_sync(0xFFFFFFFFu, nan, 4);
    unit_bytes |= __shfl_xor_sync(0xFFFFFFFFu, unit_bytes, 8), nan |= __shfl_xor_sync(0xFFFFFFFFu, nan, 8);
}

// Floats of a row of what one CTA of a cluster sends another: a value per token, or a whole number of groups of eight
// with four to spare, which spreads the 16-byte accesses of neighbouring rows over the banks.
template <bool DIGITS>
__host__ __device__ __forceinline__ uint32_t red_row(uint32_t m) {
    return DIGITS ? m : (m + 7u) / 8u * 8u + 4u;
}

template <bool DIGITS, uint32_t TILES, typename Out>
__global__ void __launch_bounds__(mp_threads(TILES), 1)
mx_product_kernel(const __grid_constant__ CUtensorMap tm_w, const __grid_constant__ CUtensorMap tm_a, const MpArgs p) {
    constexpr uint32_t W_STAGE = TILES * MP_W_BYTES, SFW_STAGE = TILES * 1024u, SFB_STAGE = 1024u;
    constexpr uint32_t X_WARPS = mp_x_warps(TILES);
    constexpr uint32_t SF_COLS = 8u * TILES + 8u;                  // scale columns of a place: B, then the tiles of W
    extern __shared__ uint8_t smem_dyn[];
    const uint32_t raw_addr = smem_u32(smem_dyn);
    const uint32_t base = (raw_addr + 1023u) & ~1023u;   // the swizzled tiles need 1024-byte alignment
    uint8_t* sm = smem_dyn + (base - raw_addr);
    MpBars* bars = reinterpret_cast<MpBars*>(sm + p.off_bar);

    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31u;
    const uint32_t group = blockIdx.x / p.splits, rank = blockIdx.x - group * p.splits;
    const uint32_t tile0 = group * TILES;                          // first tile of 128 rows
    const uint32_t n_quads = (p.n_blocks + 3u) / 4u, all_st = (p.n_blocks + 7u) / 8u;
    const uint32_t st0 = (uint32_t)((uint64_t)all_st * rank / p.splits);
    const uint32_t n_st = (uint32_t)((uint64_t)all_st * (rank + 1u) / p.splits) - st0;   // at least one
    const uint32_t tok0 = DIGITS ? 0u : blockIdx.y * MP_TOKENS, m = min(p.m - tok0, MP_TOKENS);   // this CTA's tokens
    const uint32_t b_stage = p.n * MP_STAGE_BYTES;
    const uint32_t w_tiles = min(TILES, (p.rows + 127u) / 128u - tile0);                 // tiles that exist

    if (p.splits > 1u) cluster_arrive();     // waited for before another CTA's shared memory is written
    if (tid == 0) {
        for (uint32_t s = 0; s < p.stages; ++s) mbar_init(&bars->full[s], 1u + (DIGITS ? p.m : 0u)), mbar_init(&bars->empty[s], 1);
        mbar_init(&bars->done, MP_MMA_WARPS);
        bars->abort = 0;
        mbar_init_fence();
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&bars->tmem_base)),
                     "r"(p.tmem_cols)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    // The weights too are read after the dependency wait below: a quantise call directly before this one may have
    // written them.  Until then they are brought into L2, where a later write still reaches them: the launch before
    // this one and the transfer from HBM overlap (14336 x 4096, back to back: 8.5 -> 8.2 us).
    if (warp == 0 && elect_one()) {
        for (uint32_t i = 0; i < w_tiles; ++i) {
            for (uint32_t j = 0; j < min(n_st, MP_PREFETCH); ++j)
                tma_prefetch_2d(&tm_w, (int32_t)((st0 + j) * MP_STAGE_BYTES), (int32_t)((tile0 + i) * MP_ROWS));
            bulk_prefetch(p.w_scales + ((uint64_t)(tile0 + i) * n_quads + st0 * 2u) * MX_TILE_BYTES,
                          min(n_st * 2u, n_quads - st0 * 2u) * MX_TILE_BYTES);
        }
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = bars->tmem_base;
    asm volatile("griddepcontrol.wait;" ::: "memory");   // an ordered launch: see axc_tuning.pdl
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    if (warp == 0) {
        uint32_t s = 0, ph = 1, issued = 0;
        for (; issued < n_st; ++issued) {
            if (!__all_sync(0xFFFFFFFFu, mbar_wait_or_abort(&bars->empty[s], ph, &bars->abort, p.status))) break;
            if (elect_one()) {
                const uint32_t st = st0 + issued, quad_bytes = min(2u, n_quads - st * 2u) * MX_TILE_BYTES;
                mbar_expect_tx(&bars->full[s], w_tiles * (MP_W_BYTES + quad_bytes) + (DIGITS ? 0u : b_stage + quad_bytes));
                for (uint32_t i = 0; i < w_tiles; ++i) {
                    tma_load_2d(base + s * W_STAGE + i * MP_W_BYTES, &tm_w, (int32_t)(st * MP_STAGE_BYTES),
                                (int32_t)((tile0 + i) * MP_ROWS), &bars->full[s]);
                    bulk_g2s(sm + p.off_sfw + s * SFW_STAGE + i * 1024u,
                             p.w_scales + ((uint64_t)(tile0 + i) * n_quads + st * 2u) * MX_TILE_BYTES, quad_bytes, &bars->full[s]);
                }
                if (!DIGITS) {
                    tma_load_2d(base + p.off_b + s * b_stage, &tm_a, (int32_t)(st * MP_STAGE_BYTES), (int32_t)tok0, &bars->full[s]);
                    bulk_g2s(sm + p.off_sfb + s * SFB_STAGE, p.a_scales + ((uint64_t)(tok0 / 128u) * n_quads + st * 2u) * MX_TILE_BYTES,
                             quad_bytes, &bars->full[s]);
                }
            }
            __syncwarp();
            if (++s == p.stages) s = 0, ph ^= 1u;
        }
        // nothing may still be in flight towards this CTA's shared memory at exit
        for (uint32_t j = issued > p.stages ? issued - p.stages : 0; j < issued; ++j)
            (void)mbar_wait(&bars->full[j % p.stages], (j / p.stages) & 1u, p.status);
    } else if (warp < MP_FIRST_X) {
        // ---------------- MMA: warp `turn` takes the stages turn, turn + 2, ... into its accumulators ----------------
        const uint32_t turn = warp - 1u;
        if (elect_one()) {
            const uint32_t sf0 = tmem + TILES * MP_MMA_WARPS * p.n, acc = tmem + turn * p.n;
            const uint32_t idesc = mx_idesc(128u, p.n, 0u), idesc2 = mx_idesc(128u, p.n, 2u);
            uint32_t s = turn % p.stages, ph = turn / p.stages;
            for (uint32_t i = turn; i < n_st; i += MP_MMA_WARPS) {
                if (!mbar_wait_or_abort(&bars->full[s], ph, &bars->abort, p.status)) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint32_t steps = min(4u, (p.n_blocks - (st0 + i) * 8u + 1u) / 2u);   // MMAs of 64 columns
                const uint32_t sf = sf0 + s * SF_COLS, sfw = base + p.off_sfw + s * SFW_STAGE, sfb = base + p.off_sfb + s * SFB_STAGE;
                const uint64_t wd = sw128_desc(base + s * W_STAGE), bd = sw128_desc(base + p.off_b + s * b_stage);
#pragma unroll
                for (uint32_t g = 0; g < 2u; ++g) {
                    if (2u * g >= steps) break;
                    scales_to_tmem(sf + g * 4u, sfb + g * MX_TILE_BYTES);
#pragma unroll
                    for (uint32_t t = 0; t < TILES; ++t)
                        scales_to_tmem(sf + 8u + t * 8u + g * 4u, sfw + t * 1024u + g * MX_TILE_BYTES);
                }
#pragma unroll
                for (uint32_t kk = 0; kk < 4u; ++kk) {           // 64 codes = 32 bytes = 2 descriptor units per step
                    if (kk >= steps) break;
#pragma unroll
                    for (uint32_t t = 0; t < TILES; ++t)         // the first use of an accumulator overwrites it
                        umma_mxf4(acc + t * MP_MMA_WARPS * p.n, wd + t * (MP_W_BYTES / 16u) + 2u * kk, bd + 2u * kk,
                                  kk & 1u ? idesc2 : idesc, sf + 8u + t * 8u + (kk >> 1) * 4u, sf + (kk >> 1) * 4u, (i - turn) | kk);
                }
                umma_commit(&bars->empty[s]);
                s += MP_MMA_WARPS;
                while (s >= p.stages) s -= p.stages, ph ^= 1u;
            }
            umma_commit(&bars->done);     // this warp's accumulators are complete (or nothing is outstanding)
        }
    } else {
        const uint32_t xw = warp - MP_FIRST_X;
        if constexpr (DIGITS) {
            // ---------------- digits of x: a warp takes 256 columns of one token, a lane 8 of them ----------------
            // A place of the ring (stage and token) belongs to one warp, see launch().
            const uint32_t takers = p.takers, units = xw < takers ? n_st * p.m : 0u;
            float v[8];
            if (xw < units) load_x(p, st0 + xw / p.m, xw % p.m, lane, v);
            for (uint32_t u = xw; u < units; u += takers) {
                const uint32_t i = u / p.m, t = u - i * p.m, s = i % p.stages, ph = (i / p.stages) & 1u;
                uint32_t w[8], unit_bytes, nan;
                split_x(v, lane, w, unit_bytes, nan);
                const uint32_t next = u + takers;
                if (next < units) load_x(p, st0 + next / p.m, next % p.m, lane, v);
                if (!__all_sync(0xFFFFFFFFu, mbar_wait_or_abort(&bars->empty[s], ph ^ 1u, &bars->abort, p.status))) break;
                // row d of the token's eight rows; the 16-byte chunk j of a row sits at chunk j ^ (row & 7)
                uint8_t* tile = sm + p.off_b + s * b_stage + t * 1024u;
#pragma unroll
                for (uint32_t d = 0; d < 8u; ++d)
                    *reinterpret_cast<uint32_t*>(tile + d * 128u + (((lane >> 2) ^ d) << 4) + (lane & 3u) * 4u) = w[d];
                // scales: lanes 0..7 write the first four blocks, lanes 16..23 the others; digit d is 8^d units
                if ((lane & 15u) < 8u) {
                    const uint32_t d = lane & 15u, n = t * 8u + d;
                    *reinterpret_cast<uint32_t*>(sm + p.off_sfb + s * SFB_STAGE + (lane >> 4) * MX_TILE_BYTES + (n & 31u) * 16u +
                                                 (n >> 5) * 4u) = (unit_bytes + 0x03030303u * d) | nan;
                }
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // generic writes -> async proxy
                __syncwarp();
                if (lane == 0) mbar_arrive(&bars->full[s]);
            }
        }

        // ---------------- epilogue: TMEM lane = weight row; partial sums to the CTA that finishes the row ----------------
        const bool ok = __all_sync(0xFFFFFFFFu, mbar_wait_or_abort(&bars->done, 0u, &bars->abort, p.status) && !bars->abort);
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        if (p.splits > 1u) cluster_wait();   // every CTA of the cluster has started
        if (ok) {
            // groups of four warps, two for each tile, that take turns at its columns
            const uint32_t t = xw >> 3, grp = (xw >> 2) & 1u, quad = warp & 3u;
            const uint32_t lr = t * MP_ROWS + quad * 32u + lane;          // row of the cluster's
            const uint64_t row = (uint64_t)tile0 * MP_ROWS + lr;
            const bool two = n_st > 1u;                                   // both issuing warps had a stage
            const uint32_t taddr = tmem + ((quad * 32u) << 16) + t * MP_MMA_WARPS * p.n;
            uint32_t dst = 0;
            if (p.splits > 1u) {
                asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(dst) : "r"(base + p.off_red), "r"(lr >> p.per_shift));
                const uint32_t slot = (rank << p.per_shift) | (lr & ((1u << p.per_shift) - 1u));   // [source][row]
                dst += slot * red_row<DIGITS>(m) * 4u;
            }
            const uint32_t columns = DIGITS ? m * 8u : m;
            for (uint32_t c = grp * 8u; c < columns; c += 16u) {
                uint32_t r0[8], r1[8];
                tmem_load8(taddr + c, r0);
                tmem_load8(taddr + p.n + c, r1);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                float sum[8];
#pragma unroll
                for (int j = 0; j < 8; ++j) sum[j] = __uint_as_float(r0[j]) + (two ? __uint_as_float(r1[j]) : 0.0f);
                if constexpr (DIGITS) {
                    const float y = ((sum[0] + sum[1]) + (sum[2] + sum[3])) + ((sum[4] + sum[5]) + (sum[6] + sum[7]));
                    if (p.splits > 1u)
                        asm volatile("st.shared::cluster.f32 [%0], %1;" ::"r"(dst + (c >> 3) * 4u), "f"(y) : "memory");
                    else if (row < p.rows)
                        put(reinterpret_cast<Out*>(p.out) + (uint64_t)(c >> 3) * p.rows + row, y);
                } else if (p.splits > 1u) {
#pragma unroll
                    for (int j = 0; j < 8; j += 4)
                        asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(dst + (c + j) * 4u), "f"(sum[j]),
                                     "f"(sum[j + 1]), "f"(sum[j + 2]), "f"(sum[j + 3])
                                     : "memory");
                } else if (row < p.rows) {
                    Out* out = reinterpret_cast<Out*>(p.out) + (uint64_t)(tok0 + c) * p.rows + row;
#pragma unroll
                    for (uint32_t j = 0; j < 8u; ++j)
                        if (c + j < columns) put(out + (uint64_t)j * p.rows, sum[j]);
                }
            }
        }
    }

    __syncwarp();
    if (p.splits > 1u) {
        if (warp < MP_FIRST_X) cluster_wait();
        cluster_sync_all();
        if (warp >= MP_FIRST_X) {
            const uint32_t per = 1u << p.per_shift, pitch = red_row<DIGITS>(m);
            const float* red = reinterpret_cast<const float*>(sm + p.off_red);
            const uint64_t first = (uint64_t)tile0 * MP_ROWS + rank * per;
            constexpr uint32_t WIDE = DIGITS ? 1u : 4u;            // neighbouring columns that a thread adds
            for (uint32_t i = tid - MP_FIRST_X * 32u; i < (m + WIDE - 1u) / WIDE << p.per_shift; i += X_WARPS * 32u) {
                const uint32_t r = i & (per - 1u), c = (i >> p.per_shift) * WIDE;
                float sum[WIDE] = {};
                for (uint32_t k = 0; k < p.splits; ++k) {
                    const float* src = red + ((k << p.per_shift) + r) * pitch + c;
                    if constexpr (DIGITS) {
                        sum[0] += src[0];
                    } else {
                        const float4 q = *reinterpret_cast<const float4*>(src);
                        sum[0] += q.x, sum[1] += q.y, sum[2] += q.z, sum[3] += q.w;
                    }
                }
                if (first + r < p.rows) {
                    Out* out = reinterpret_cast<Out*>(p.out) + (uint64_t)(tok0 + c) * p.rows + first + r;
#pragma unroll
                    for (uint32_t j = 0; j < WIDE; ++j)
                        if (c + j < m) put(out + (uint64_t)j * p.rows, sum[j]);
                }
            }
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.tmem_cols) : "memory");
    }
}

template <bool DIGITS, uint32_t TILES, typename Out>
cudaError_t launch(const CUtensorMap& tm_w, const CUtensorMap& tm_a, MpArgs p, cudaStream_t stream) {
    const uint32_t all_st = (p.n_blocks + 7u) / 8u;
    const uint32_t share = (all_st + p.splits - 1u) / p.splits;     // the longest share of K, in stages
    p.per_shift = 0;
    while ((p.splits << p.per_shift) < TILES * MP_ROWS) ++p.per_shift;
    // shared memory: W stages, B stages, scales of W and B, what the cluster sends, barriers
    const uint32_t w_stage = TILES * MP_W_BYTES, b_stage = p.n * MP_STAGE_BYTES, sfw_stage = TILES * 1024u;
    const uint32_t per_stage = w_stage + b_stage + sfw_stage + 1024u;
    const uint32_t red = p.splits > 1u ? TILES * MP_ROWS * red_row<DIGITS>(p.m < MP_TOKENS ? p.m : MP_TOKENS) * 4u : 0u;
    const uint32_t fixed = 1024u + (uint32_t)sizeof(MpBars) + red;
    uint32_t stages = (MP_SMEM_MAX - fixed) / per_stage;
    if (stages > MP_MAX_STAGES) stages = MP_MAX_STAGES;
    if (stages > share) stages = share;
    // Where the ring wraps, a place of it belongs to one issuing warp and, for each token, to one warp that splits x: a
    // warp that waits for a place that another used last could take the parity of a phase still to come for its own.
    p.takers = mp_x_warps(TILES);
    if (stages < share) {
        stages -= stages % MP_MMA_WARPS;
        while (stages * p.m % p.takers) --p.takers;
    }
    // tensor memory: the accumulators, and a place of scales per stage
    uint32_t cols = 32u;
    while (cols < TILES * MP_MMA_WARPS * p.n + stages * (8u * TILES + 8u)) cols *= 2u;
    p.tmem_cols = cols;
    p.stages = stages;
    p.off_b = stages * w_stage;
    p.off_sfw = p.off_b + stages * b_stage;
    p.off_sfb = p.off_sfw + stages * sfw_stage;
    p.off_red = p.off_sfb + stages * 1024u;
    p.off_bar = p.off_red + red;
    uint32_t smem = fixed + stages * per_stage;
    const uint32_t least = MP_SMEM_SM / 512u * cols;                // an SM's CTAs never ask for more than 512 columns
    if (smem < least) smem = least > MP_SMEM_MAX ? MP_SMEM_MAX : least;
    auto kern = mx_product_kernel<DIGITS, TILES, Out>;
    {
        static std::mutex mu;
        static bool done[64] = {};
        int dev = 0;
        cudaError_t e = cudaGetDevice(&dev);
        if (e != cudaSuccess) return e;
        std::lock_guard<std::mutex> lock(mu);
        if (dev < 0 || dev >= 64 || !done[dev]) {
            e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)MP_SMEM_MAX);
            if (e != cudaSuccess) return e;
            if (dev >= 0 && dev < 64) done[dev] = true;
        }
    }
    const uint32_t row_tiles = (p.rows + MP_ROWS - 1u) / MP_ROWS;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((row_tiles + TILES - 1u) / TILES * p.splits, (p.m + MP_TOKENS - 1u) / MP_TOKENS);
    cfg.blockDim = dim3(mp_threads(TILES));
    cfg.dynamicSmemBytes = smem, cfg.stream = stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = p.splits, attr[1].val.clusterDim.y = 1, attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr, cfg.numAttrs = p.splits > 1u ? 2 : 1;
    return cudaLaunchKernelEx(&cfg, kern, tm_w, tm_a, p);
}

// CTAs per cluster: K of at least `first` stages of 256 columns is split in two, again and again, as long as all clusters
// run at once and each half of a share has least / 2 stages.  A second round of CTAs costs as much as the first (14336 x 4096, one token: 112 CTAs 7.5 us, 224
// CTAs 10.8 us), and clusters of 4 and 8 do not reach every SM (15 clusters of 8 on 148 SMs; 4096 x 14336, one token: 64
// CTAs in clusters of 8 9.4 us, 128 CTAs 12.5 us).
uint32_t choose_splits(uint32_t groups, uint32_t n_blocks, uint32_t sms, uint32_t first, uint32_t least) {
    const uint32_t st = (n_blocks + 7u) / 8u;
    const uint64_t most[4] = {sms, sms, sms * 7u / 8u, sms * 13u / 16u};   // CTAs that run at once in clusters of 1, 2, 4, 8
    uint32_t shift = 0;
    while (shift < 3u && st >= first && ((uint64_t)groups << (shift + 1u)) <= most[shift + 1u] && st >= least << shift) ++shift;
    return 1u << shift;
}

}  // namespace

cudaError_t launch_mxfp4_matvec(const uint8_t* codes, const uint8_t* scales, const float* x, float* y, uint32_t m_tokens,
                                uint32_t rows, uint32_t n_blocks, uint32_t* status, cudaStream_t stream, int sm_count) {
    if (m_tokens == 0 || rows == 0 || n_blocks == 0) return cudaSuccess;
    if (!tensor_map_encoder()) return cudaErrorNotSupported;
    MpArgs p{};
    p.w_scales = scales, p.x = x, p.out = y, p.m = m_tokens, p.rows = rows, p.n_blocks = n_blocks, p.status = status;
    p.n = (m_tokens + 1u) / 2u * 16u;
    CUtensorMap tm_w;
    if (!mx_encode_codes(&tm_w, codes, rows, n_blocks, MP_ROWS)) return cudaErrorInvalidValue;
    // Two tiles per CTA halve the work of splitting x, which every CTA does for its share of K (8192 x 8192, 8 tokens: 11.2
    // us, one tile 17.2 us), and allow twice the splits (2048 x 8192, one token: 4.6 us, one tile 5.4 us).  A CTA of one
    // tile starts and ends sooner and needs less per stage.  So one tile where that allows as many splits and either the
    // share of K is short (one token, 4096 x 2048: 3.2 us, two tiles 3.5 us) or, with few tokens, there are not many CTAs
    // (2048 x 4096: 3.5 us, two tiles 3.9 us; but 4096 x 4096 4.4 us, two tiles 4.1 us) or much to read for each
    // (4096 x 14336: 8.5 us, two tiles 9.4 us).  More rows than SMs take two, but for few tokens and the shortest rows
    // (40000 x 256: 5.1 us, two tiles 5.7 us; 40000 x 2048: 15.2 us, 13.2 us).  The splits do not depend on the number of
    // tokens, so that a token's sums do not.
    const uint32_t sms = (uint32_t)sm_count, row_tiles = (rows + MP_ROWS - 1u) / MP_ROWS, st = (n_blocks + 7u) / 8u;
    const uint32_t one = choose_splits(row_tiles, n_blocks, sms, 4u, 3u), two = choose_splits((row_tiles + 1u) / 2u, n_blocks, sms, 6u, 6u);
    p.splits = one > two ? one : two;
    const uint32_t share = (st + p.splits - 1u) / p.splits;
    const bool few = m_tokens <= 4u;
    const bool one_tile = one >= two && row_tiles <= sms && (share <= 2u || (few && (share >= 8u || row_tiles * p.splits * 2u <= sms)));
    if (one_tile || (st <= 3u && few)) return launch<true, 1, float>(tm_w, tm_w, p, stream);
    return launch<true, 2, float>(tm_w, tm_w, p, stream);
}

cudaError_t launch_mxfp4_prefill(const uint8_t* w_codes, const uint8_t* w_scales, const uint8_t* a_codes,
                                 const uint8_t* a_scales, void* c, ElemType type, uint32_t m_tokens, uint32_t n_rows,
                                 uint32_t n_blocks, uint32_t* status, cudaStream_t stream, int sm_count) {
    if (m_tokens == 0 || n_rows == 0 || n_blocks == 0) return cudaSuccess;
    if (!tensor_map_encoder()) return cudaErrorNotSupported;
    // Which form: this one splits K, the one for many tokens reads W and A less often.  Up to 128 tokens this one, beyond 64
    // unless the other has a row tile for each of its pairs of CTAs (128 tokens, 28672 x 8192: 29.8 us, this form 33.8 us;
    // 4096 x 14336: 20.7 us, this form 12.5 us).  Beyond 128 this one where rows and tokens leave SMs to split long rows over
    // (256 tokens, 4096 x 14336: 15.7 us, the other 20.7 us, 1024 x 14336: 10.4 us, 20.3 us; but 4096 x 1024: 5.7 us, 5.6 us, and
    // without a split 1024 tokens, 4096 x 14336: 40.8 us, 20.9 us).
    const uint32_t sms = (uint32_t)sm_count, row_tiles = (n_rows + MP_ROWS - 1u) / MP_ROWS;
    const uint32_t chunks = (m_tokens + MP_TOKENS - 1u) / MP_TOKENS;
    // Two tiles per CTA where one each would need a second round of CTAs: 28672 x 3200, 64 tokens 15.9 -> 12.1 us.
    const bool two = row_tiles > sms && m_tokens <= 64u;
    const uint64_t groups = (uint64_t)(two ? (row_tiles + 1u) / 2u : row_tiles) * chunks;
    const uint32_t splits = groups > sms ? 1u : choose_splits((uint32_t)groups, n_blocks, sms, 8u, 4u);
    if (chunks > 1u ? splits == 1u || n_blocks < 128u : m_tokens > 64u && row_tiles >= sms)
        return launch_mxfp4_gemm(w_codes, w_scales, a_codes, a_scales, c, type, m_tokens, n_rows, n_blocks, status, stream, sm_count);
    MpArgs p{};
    p.w_scales = w_scales, p.a_scales = a_scales, p.out = c, p.m = m_tokens, p.rows = n_rows, p.n_blocks = n_blocks;
    p.status = status, p.splits = splits;
    p.n = chunks > 1u ? MP_TOKENS : (m_tokens + 15u) / 16u * 16u;
    CUtensorMap tm_w, tm_a;
    if (!mx_encode_codes(&tm_w, w_codes, n_rows, n_blocks, MP_ROWS) || !mx_encode_codes(&tm_a, a_codes, m_tokens, n_blocks, p.n))
        return cudaErrorInvalidValue;
    switch (type) {
        case ElemType::F32: return two ? launch<false, 2, float>(tm_w, tm_a, p, stream) : launch<false, 1, float>(tm_w, tm_a, p, stream);
        case ElemType::BF16: return two ? launch<false, 2, __nv_bfloat16>(tm_w, tm_a, p, stream) : launch<false, 1, __nv_bfloat16>(tm_w, tm_a, p, stream);
        case ElemType::F16: return two ? launch<false, 2, __half>(tm_w, tm_a, p, stream) : launch<false, 1, __half>(tm_w, tm_a, p, stream);
    }
    return cudaErrorInvalidValue;
}

}  // namespace axc
