// Products of microscaled 4-bit floats (mx4.cuh) on the fifth-generation tensor cores:
//
//     out[r, f] = sum over blocks b of 2^(sa[r, b] + sw[f, b]) * sum over i in b of pa[r, i] pw[f, i]
//
// by block-scaled MMAs (kind::mxf4), which take both operands' codes from shared memory and both operands' scales from
// tensor memory and add up in float32.  The weights are the M operand (128 features a tile), the rows the N operand.
//
// A CTA computes 128 features by BN rows over one part of k; the parts of a tile are the CTAs of a cluster, which add
// their sums up in the order of k through distributed shared memory, so the result comes out whole.  Warp 0 loads
// stages of 256 values of k (codes by TMA with the 128-byte swizzle, scales by plain bulk copies: they lie in memory
// as the tensor cores take them), warp 1 copies a stage's scales to tensor memory and issues its MMAs, warps 2 to 9 read
// the accumulator back.  A stage has its own columns of tensor memory for its scales, so nothing overwrites scales that
// an MMA may still read.
//
// Few rows may come as floats, in tiles of 16 or 32 rows: every CTA then brings its part of them to 4 bits itself (warps 2
// to 9, a warp a row's two chunks at a time), which saves the launch of a kernel that does it once (mx_rows_tile).
//
// Every wait on an mbarrier has a time limit, as in gemm_tc.cu; when it runs out, the error word says which.
#include "kernels.h"
#include "mx4.cuh"
#include "tc_common.cuh"

namespace jb {

constexpr int MX_TILE_M = 128;
constexpr int MX_W_BYTES = MX_TILE_M * (MX4_CHUNK / 2);
constexpr int MX_THREADS = 320;
constexpr int SM_SMEM = 228 * 1024, CTA_SMEM = 1024;        // an SM's shared memory, and what each CTA takes beside its own
constexpr int SM_TMEM_COLS = 512;

__device__ int g_gemm_mx4_error;    // 0, or the code of the first wait that ran out

template <int BN> struct MxCfg {
    static constexpr int A_BYTES = BN * (MX4_CHUNK / 2);
    static constexpr int STAGE_BYTES = MX_W_BYTES + A_BYTES + 2 * MX4_TILE;
    static constexpr int STAGES = 110 * 1024 / STAGE_BYTES > 6 ? 6 : 110 * 1024 / STAGE_BYTES;   // two CTAs fit an SM
    static constexpr int SCALE_COL = BN < 32 ? 32 : BN;
    __host__ __device__ static constexpr int tmem_cols(int stages)
    {
        const int cols = SCALE_COL + 16 * stages;
        return cols <= 64 ? 64 : cols <= 128 ? 128 : 256;
    }
    // Of the shared memory, `stages` are asked for: no more than a CTA has chunks, so that CTAs of the kernel behind this
    // one find room on the SM before this one ends.  CTAs of a cluster ask for no less than their share of the SM's as their
    // columns are of its tensor memory: a CTA that finds no columns free waits for them, while a CTA that has some keeps
    // them until its whole cluster has its own.  Where clusters (of products on several streams) could hold more columns
    // together than an SM has, they could wait for one another for good, and no time limit covers that wait.  So they
    // fit an SM's tensor memory wherever they fit its shared memory.  (A CTA without a cluster waits for nobody that waits
    // for columns: a kernel lets the one behind it start after its own CTAs have theirs.)
    static constexpr int smem_bytes(int stages, bool cluster)
    {
        const int own = stages * STAGE_BYTES + 1024 /* alignment */ + 256 /* barriers */;
        const int share = tmem_cols(stages) * (SM_SMEM / SM_TMEM_COLS) - CTA_SMEM;
        return cluster && own < share ? share : own;
    }
    static constexpr int SMEM_MOST = smem_bytes(STAGES, true);
    static_assert(SMEM_MOST <= 227 * 1024 && SCALE_COL + 16 * STAGES <= 256, "a CTA's shared memory and columns");
};

// kind::mxf4 instruction descriptor: 4-bit A and B (bits 7-9 and 10-12 = 1), both K-major, N / 8 at bit 17, scales that
// are powers of two (bit 23), M / 16 at bit 24; which two of a column's four scales: bits 4-5 (B) and 29-30 (A).
__host__ __device__ constexpr uint32_t mx_instr_desc(int n, int which)
{
    return ((uint32_t)which << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(n >> 3) << 17) | (1u << 23) |
           ((uint32_t)(MX_TILE_M >> 4) << 24) | ((uint32_t)which << 29);
}

// The descriptor of 32 rows of 16 bytes without a swizzle, 128 bytes from one group of eight rows to the next.
__device__ __forceinline__ uint64_t mx_scale_desc(uint32_t addr)
{
    return (uint64_t)((addr >> 4) & 0x3fff) | (uint64_t)(128 >> 4) << 16 | (uint64_t)(128 >> 4) << 32 | (uint64_t)1 << 46;
}

__device__ __forceinline__ void bulk_load(uint32_t dst, const void *src, uint32_t bytes, uint32_t bar)
{
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(dst), "l"(src), "r"(bytes), "r"(bar) : "memory");
}

// A stage's MMAs, by a whole warp whose lanes agree on the arguments: its scales (1,024 bytes of each operand) to tensor
// memory, eight columns each, then four MMAs of 64 values of k.
template <int BN>
__device__ __forceinline__ void mx_stage(uint32_t d, uint64_t a, uint64_t b, uint32_t sa, uint32_t sb, uint64_t sa_mem,
                                         uint64_t sb_mem, uint32_t accumulate)
{
    asm volatile(
        "{\n\t"
        ".reg .pred p, q;\n\t"
        ".reg .b64 a1, a2, a3, b1, b2, b3, ma, mb;\n\t"
        ".reg .b32 ta, tb;\n\t"
        "setp.ne.b32 p, %7, 0;\n\t"
        "add.u64 a1, %1, 2;\n\t"
        "add.u64 a2, %1, 4;\n\t"
        "add.u64 a3, %1, 6;\n\t"
        "add.u64 b1, %2, 2;\n\t"
        "add.u64 b2, %2, 4;\n\t"
        "add.u64 b3, %2, 6;\n\t"
        "add.u64 ma, %5, 32;\n\t"
        "add.u64 mb, %6, 32;\n\t"
        "add.u32 ta, %3, 4;\n\t"
        "add.u32 tb, %4, 4;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.cp.cta_group::1.32x128b.warpx4 [%3], %5;\n\t"
        "@q tcgen05.cp.cta_group::1.32x128b.warpx4 [ta], ma;\n\t"
        "@q tcgen05.cp.cta_group::1.32x128b.warpx4 [%4], %6;\n\t"
        "@q tcgen05.cp.cta_group::1.32x128b.warpx4 [tb], mb;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %8, [%3], [%4], p;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], a1, b1, %9, [%3], [%4], 1;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], a2, b2, %8, [ta], [tb], 1;\n\t"
        "@q tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], a3, b3, %9, [ta], [tb], 1;\n\t"
        "}\n"
        ::"r"(d), "l"(a), "l"(b), "r"(sa), "r"(sb), "l"(sa_mem), "l"(sb_mem), "r"(accumulate),
        "r"(mx_instr_desc(BN, 0)), "r"(mx_instr_desc(BN, 2))
        : "memory");
}

__device__ __forceinline__ float4 cluster_read4(uint32_t mine, uint32_t rank)
{
    uint32_t ra;
    float4 v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(mine), "r"(rank));
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(ra) : "memory");
    return v;
}

// Rows as floats in memory: [n, k] of bfloat16 or float, vec: whole 16-byte loads.
struct MxRows {
    const void *x;
    int k, is_bf16, vec;
};

// Eight values of row r from column col on, zeros past the row's end.
__device__ __forceinline__ void mx_fetch(const MxRows &a, size_t r, int col, float *v)
{
    const size_t at = r * (size_t)a.k + col;
    if (a.is_bf16) {
        const bf16 *p = (const bf16 *)a.x + at;
        a.vec ? load8<bf16, true>(p, a.k - col, v) : load8<bf16, false>(p, a.k - col, v);
    } else {
        const float *p = (const float *)a.x + at;
        a.vec ? load8<float, true>(p, a.k - col, v) : load8<float, false>(p, a.k - col, v);
    }
}

constexpr int ROWS_NONE = 0, ROWS_BF16 = 1, ROWS_ANY = 2;   // as codes, as bfloat16 in whole 16-byte loads, as any floats

// Sixteen bfloat16 of a lane.
struct SixteenRows : SixteenBf16 {
    __device__ __forceinline__ void fetch(const MxRows &a, size_t r, int col0, int lane)
    {
        load((const bf16 *)a.x + r * (size_t)a.k + col0 + 16 * lane, a.k - col0 - 16 * lane);
    }
};
// Eight values of a lane from anywhere.
struct AnyEight {
    float v[8];
    __device__ __forceinline__ void fetch(const MxRows &a, size_t r, int col0, int lane) { mx_fetch(a, r, col0 + 8 * lane, v); }
    __device__ __forceinline__ uint2 pack(uint32_t &code) const { return make_uint2(mx4_pack_chunk(v, code), 0); }
};

// Brings this CTA's part of the rows, chunks c0 .. c0 + nc - 1, to 4 bits and into the stages.  Eight warps share the
// (SPAN chunks, row) items; the loads of D spans are in flight.  Every warp waits for and arrives at every stage in turn,
// whether it has an item there or not: it is then never more than one use of a stage behind, so that the parity that it
// waits for names one phase.  Q: the most items of a span that a warp has.  False where a wait ran out.
template <typename Values, int SPAN, int D, int Q, int BN>
__device__ __forceinline__ bool mx_pack_rows(const MxRows &a, int rows, int c0, int nc, int stages, uint8_t *smem,
                                             uint32_t full0, uint32_t empty0, int warp, volatile int *abort)
{
    static_assert(8 * Q >= BN, "items of a span");
    constexpr int LANES = 32 / SPAN;            // lanes of a chunk
    const int lane = threadIdx.x & 31, spans = (nc + SPAN - 1) / SPAN;
    Values v[D][Q];
    auto fetch = [&](int j, Values *to) {
        const int r0 = (warp - j * rows) & 7;   // this warp's rows of span j: r0, r0 + 8, ..
#pragma unroll
        for (int q = 0; q < Q; q++)
            if (j < spans && r0 + 8 * q < rows)
                to[q].fetch(a, r0 + 8 * q, (c0 + j * SPAN) * MX4_CHUNK, lane);
    };
#pragma unroll
    for (int d = 0; d < D; d++)
        fetch(d, v[d]);
    bool ok = true;
    for (int j0 = 0; j0 < spans && ok; j0 += D) {
#pragma unroll
        for (int d = 0; d < D; d++) {
            const int j = j0 + d, r0 = (warp - j * rows) & 7;
            if (j >= spans || !ok)
                continue;
            uint2 packed[Q];
            uint32_t code[Q];
#pragma unroll
            for (int q = 0; q < Q; q++)
                if (r0 + 8 * q < rows)
                    packed[q] = v[d][q].pack(code[q]);
            fetch(j + D, v[d]);
#pragma unroll
            for (int h = 0; h < SPAN; h++) {
                const int i = j * SPAN + h, s = i % stages;
                if (i >= nc || !ok)
                    continue;
                if (i >= stages)
                    ok = __all_sync(0xffffffffu, mbar_wait(empty0 + 8 * s, ((i / stages) & 1) ^ 1, abort, &g_gemm_mx4_error, 5));
                if (!ok)
                    continue;
                uint8_t *stage = smem + s * MxCfg<BN>::STAGE_BYTES + MX_W_BYTES;
                if (lane / LANES == h) {
                    const int l = lane % LANES;
#pragma unroll
                    for (int q = 0; q < Q; q++) {
                        const int r = r0 + 8 * q;
                        if (r >= rows)
                            continue;
                        uint8_t *line = stage + r * 128, *scale = stage + MxCfg<BN>::A_BYTES + MX4_TILE + r * 16;
                        if (SPAN == 2) {
                            *reinterpret_cast<uint2 *>(line + (((l >> 1) ^ (r & 7)) << 4) + (l & 1) * 8) = packed[q];
                            if ((l & 1) == 0)
                                scale[(l >> 3) * 512 + ((l >> 1) & 3)] = (uint8_t)code[q];
                        } else {
                            *reinterpret_cast<uint32_t *>(line + (((l >> 2) ^ (r & 7)) << 4) + (l & 3) * 4) = packed[q].x;
                            if ((l & 3) == 0)
                                scale[(l >> 4) * 512 + ((l >> 2) & 3)] = (uint8_t)code[q];
                        }
                    }
                }
                fence_async_smem();
                __syncwarp();
                if (lane == 0)
                    mbar_arrive(full0 + 8 * s);
            }
        }
    }
    return ok;
}

// w_early: the weights were written before the kernel ahead of this one was launched, and may be read at once
template <int BN, typename TO, int ROWS>
__global__ void __launch_bounds__(MX_THREADS)
gemm_mx4_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a,
                const uint8_t *w_scales, const uint8_t *a_scales, const MxRows a_rows, TO *__restrict__ out, int n, int m,
                int chunks, int parts, int stages, int w_early)
{
    using Cfg = MxCfg<BN>;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    uint64_t *bars = (uint64_t *)(smem + stages * Cfg::STAGE_BYTES);
    uint32_t *tmem_slot = (uint32_t *)(bars + 2 * stages + 1);
    volatile int *abort = (volatile int *)(tmem_slot + 1);

    const int warp = (int)warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const int rank = blockIdx.x % parts, tile = blockIdx.x / parts;
    const int m0 = tile * MX_TILE_M, n0 = blockIdx.y * BN;
    const int c0 = (int)((long long)chunks * rank / parts), nc = (int)((long long)chunks * (rank + 1) / parts) - c0;
    const uint32_t full0 = smem_u32(bars), empty0 = smem_u32(bars + stages), accum = smem_u32(bars + 2 * stages);
    if (threadIdx.x == 0) {
        prefetch_tensor_map(&map_w);
        if (!ROWS)
            prefetch_tensor_map(&map_a);
        for (int s = 0; s < stages; s++) {
            mbar_init(full0 + 8 * s, ROWS ? 9 : 1);        // the loads, and the warps that pack the rows
            mbar_init(empty0 + 8 * s, 1);
        }
        mbar_init(accum, 1);
        *abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(tmem_slot)), "r"((uint32_t)Cfg::tmem_cols(stages)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = warp_uniform(*tmem_slot);
    pdl_trigger();

    const int q = warp & 3, hgrp = (warp - 2) >> 2;
    const int rows = min(n - n0, BN);
    constexpr uint32_t LOADED = ROWS ? MX_W_BYTES + MX4_TILE : Cfg::STAGE_BYTES;
    bool ok = true;
    if (warp == 0 && lane == 0) {
        // ---------------------------------------------------------- loads
        const uint8_t *ws = w_scales + ((size_t)tile * chunks + c0) * MX4_TILE;
        const uint8_t *as = a_scales + ((size_t)(n0 >> 7) * chunks + c0) * MX4_TILE;
        uint32_t armed = 0, last_parity = 0;
        auto load_w = [&](int i, uint32_t dst, uint32_t bar) {
            tma_load_2d(dst, &map_w, bar, (c0 + i) * (MX4_CHUNK / 2), m0);
            bulk_load(dst + MX_W_BYTES + Cfg::A_BYTES, ws + (size_t)i * MX4_TILE, MX4_TILE, bar);
        };
        auto load_a = [&](int i, uint32_t dst, uint32_t bar) {
            tma_load_2d(dst + MX_W_BYTES, &map_a, bar, (c0 + i) * (MX4_CHUNK / 2), n0);
            bulk_load(dst + MX_W_BYTES + Cfg::A_BYTES + MX4_TILE, as + (size_t)i * MX4_TILE, MX4_TILE, bar);
        };
        const int pre = min(nc, stages);
        if (!w_early)
            pdl_wait();
        for (int i = 0; i < pre; i++) {
            mbar_expect_tx(full0 + 8 * i, LOADED);
            load_w(i, smem_u32(smem + i * Cfg::STAGE_BYTES), full0 + 8 * i);
            armed |= 1u << i;
        }
        if (w_early && !ROWS)
            pdl_wait();
        for (int i = 0; i < pre && !ROWS; i++)
            load_a(i, smem_u32(smem + i * Cfg::STAGE_BYTES), full0 + 8 * i);
        for (int i = pre; i < nc; i++) {
            const int s = i % stages;
            const uint32_t ph = (i / stages) & 1;
            if (!mbar_wait(empty0 + 8 * s, ph ^ 1, abort, &g_gemm_mx4_error, 1))
                break;
            const uint32_t dst = smem_u32(smem + s * Cfg::STAGE_BYTES), bar = full0 + 8 * s;
            mbar_expect_tx(bar, LOADED);
            load_w(i, dst, bar);
            if (!ROWS)
                load_a(i, dst, bar);
            last_parity = (last_parity & ~(1u << s)) | (ph << s);
        }
        if (*abort) {
            // the loads in flight: wait for each stage armed last, once, with the limit
            volatile int never = 0;
            for (int s = 0; s < stages; s++)
                if (armed & (1u << s))
                    mbar_wait(full0 + 8 * s, (last_parity >> s) & 1, &never, &g_gemm_mx4_error, 4);
        }
    } else if (warp == 1) {
        // --------------------------------------------------------------- MMAs
        int s = 0;
        uint32_t ph = 0;
        for (int i = 0; i < nc; i++) {
            if (!__all_sync(0xffffffffu, mbar_wait(full0 + 8 * s, ph, abort, &g_gemm_mx4_error, 2)))
                break;
            const uint32_t base = smem_u32(smem) + s * Cfg::STAGE_BYTES, scales = base + MX_W_BYTES + Cfg::A_BYTES;
            const uint32_t col = tmem + Cfg::SCALE_COL + 16 * s;
            tc_fence_after();
            mx_stage<BN>(tmem, smem_desc_sw128(base, 16, 1024), smem_desc_sw128(base + MX_W_BYTES, 16, 1024), col, col + 8,
                         mx_scale_desc(scales), mx_scale_desc(scales + MX4_TILE), i != 0);
            tc_commit_warp(empty0 + 8 * s);
            if (++s == stages) {
                s = 0;
                ph ^= 1;
            }
        }
        tc_commit_warp(accum);
    } else if (warp >= 2) {
        // ------------------------------------------------------------ the accumulator
        pdl_wait();
        const MxRows mine{(const uint8_t *)a_rows.x + (size_t)n0 * a_rows.k * (a_rows.is_bf16 ? 2 : 4), a_rows.k, a_rows.is_bf16,
                          a_rows.vec};
        if constexpr (ROWS == ROWS_BF16)
            ok = mx_pack_rows<SixteenRows, 2, BN == 16 ? 3 : 2, BN / 8, BN>(mine, rows, c0, nc, stages, smem, full0, empty0, warp - 2, abort);
        else if constexpr (ROWS == ROWS_ANY)
            ok = mx_pack_rows<AnyEight, 1, BN == 16 ? 3 : 2, BN / 8, BN>(mine, rows, c0, nc, stages, smem, full0, empty0, warp - 2, abort);
        ok = __all_sync(0xffffffffu, mbar_wait(accum, 0, abort, &g_gemm_mx4_error, 3));
        tc_fence_after();
        const uint32_t taddr = tmem + ((uint32_t)(q * 32) << 16);
        const int fl = q * 32 + lane, f = m0 + fl;
        for (int c = 8 * hgrp; c < rows && ok; c += 16) {
            uint32_t v[8];
            tc_ld8_nowait(taddr + c, v);
            tc_ld_wait();
            if (parts > 1) {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (c + j < rows)
                        ((float *)smem)[(c + j) * MX_TILE_M + fl] = __uint_as_float(v[j]);
            } else if (f < m) {
#pragma unroll
                for (int j = 0; j < 8; j++)
                    if (c + j < rows)
                        out[(size_t)(n0 + c + j) * m + f] = from_f<TO>(__uint_as_float(v[j]));
            }
        }
    }
    if (parts > 1) {
        // ---------------------------------------------------------- the parts' sums, in the order of k
        __syncwarp();
        cluster_arrive();
        cluster_wait();
        if (warp >= 2) {
            const bool vec = m % 4 == 0;
            for (int g = rank * (MX_THREADS - 64) + (int)threadIdx.x - 64; g < rows * (MX_TILE_M / 4); g += parts * (MX_THREADS - 64)) {
                const uint32_t at = smem_u32(smem) + g * 16;
                float4 t = cluster_read4(at, 0);
                for (int p = 1; p < parts; p++) {
                    const float4 u = cluster_read4(at, p);
                    t.x += u.x, t.y += u.y, t.z += u.z, t.w += u.w;
                }
                const int f = m0 + (g % (MX_TILE_M / 4)) * 4;
                TO *o = out + (size_t)(n0 + g / (MX_TILE_M / 4)) * m + f;
                if (vec) {
                    if (f < m)
                        store4(o, t);
                } else {
                    if (f < m)
                        o[0] = from_f<TO>(t.x);
                    if (f + 1 < m)
                        o[1] = from_f<TO>(t.y);
                    if (f + 2 < m)
                        o[2] = from_f<TO>(t.z);
                    if (f + 3 < m)
                        o[3] = from_f<TO>(t.w);
                }
            }
        }
        __syncwarp();
        cluster_arrive();
        cluster_wait();             // no CTA ends while another reads its sums
    }
    tc_fence_before();
    __syncthreads();
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;"
                     ::"r"(tmem), "r"((uint32_t)Cfg::tmem_cols(stages)) : "memory");
}


// ------------------------------------------------------------------ many rows
// Pairs of CTAs (a cluster of two) that share their MMAs: 256 features by 256 rows, each CTA with 128 of the features, half
// of the rows' codes, the scales of its features and of all the rows.  The leader's warp 1 issues for both; the loads of
// both CTAs report to the leader's barriers.  A pair stays on its two SMs for all its tiles; the epilogue's warps take the
// accumulator into registers at once, so the next tile's MMAs run while they store.  (Two accumulators leave no room in
// tensor memory for scales; with 192 rows they would fit, but an MMA of 64 values of k takes 135 cycles whether it is of
// 128, 192 or 256 rows: 2,048 rows x 18,944 x 2,560 52 us with tiles of 192.)
//
// What bounds it: the MMAs (541 cycles a chunk of 256 values of k, and 96 for the copies of its scales) and, while the
// epilogue stores, what the SMs can take in from the L2 beside it.
//
// Tiles go round over the pairs; those that are left when less than a round is make up a last round in which each is
// shared out along k by as many pairs as there are for it.  These write their sums to scratch, and a kernel behind this
// one adds them up in the order of k.
constexpr int MX_PAIR_M = 2 * MX_TILE_M;
constexpr int MX_PAIR_N = 256;
constexpr int MX_GROUP = 2;         // chunks whose scales are copied together
constexpr int MX_GROUPS = 3;        // such copies in shared memory
constexpr int MX_ROW_TILES = MX_PAIR_N / 128;
constexpr int MX_PAIR_STAGES = 6;
constexpr int MX_PAIR_A_BYTES = MX_PAIR_N / 2 * (MX4_CHUNK / 2);
constexpr int MX_PAIR_STAGE_BYTES = MX_W_BYTES + MX_PAIR_A_BYTES;
constexpr int MX_PAIR_SCALE_BYTES = MX_GROUP * (1 + MX_ROW_TILES) * MX4_TILE;
constexpr int MX_SLOT_COLS = 8 + 8 * MX_ROW_TILES;      // columns of tensor memory of a stage's scales
static_assert(MX_PAIR_N + MX_PAIR_STAGES * MX_SLOT_COLS <= 512, "tensor memory");
constexpr int MX_PAIR_SMEM = MX_PAIR_STAGES * MX_PAIR_STAGE_BYTES + MX_GROUPS * MX_PAIR_SCALE_BYTES + 1024 /* alignment */ +
                             256 /* barriers */;
// (a pair has all of the tensor memory: no other CTA of a cluster fits beside it, see MxCfg::smem_bytes)
static_assert(MX_PAIR_SMEM + CTA_SMEM + MxCfg<16>::smem_bytes(1, true) + CTA_SMEM > SM_SMEM, "room beside a pair's CTA");

// Tiled loads whose bytes are counted at a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y)
{
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y)
        : "memory");
}
__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z)
{
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes"
        " [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z)
        : "memory");
}

// The MMAs so far report to the barrier at the same place of both CTAs.
__device__ __forceinline__ void tc_commit_pair(uint32_t bar)
{
    asm volatile(
        "{\n\t"
        ".reg .pred q;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;\n\t"
        "}\n"
        ::"r"(bar), "h"((uint16_t)3) : "memory");
}

__device__ __forceinline__ uint32_t cluster_addr(uint32_t mine, uint32_t rank)
{
    uint32_t ra;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(ra) : "r"(mine), "r"(rank));
    return ra;
}

// Arrives at a barrier of either CTA.  What it hands over is tensor memory, read and fenced by tcgen05's own means: an
// arrival that also released this thread's stores to the cluster would wait for them (2,000 cycles, measured).
__device__ __forceinline__ void mbar_arrive_pair(uint32_t bar)
{
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

// A chunk's scales to tensor memory of both CTAs, by a whole warp whose lanes agree on the arguments: from column sa on the
// features' eight columns, behind them the rows', a half chunk's columns of both row tiles side by side.  sa_mem, sb_mem:
// their descriptors, half chunks 512 bytes apart and row tiles MX_GROUP * 1,024.
__device__ __forceinline__ void mx_scales_pair(uint32_t sa, uint64_t sa_mem, uint64_t sb_mem)
{
    asm volatile(
        "{\n\t"
        ".reg .pred q;\n\t"
        ".reg .b64 m1, n1, n2, n3;\n\t"
        ".reg .b32 t1, u0, u1, u2, u3;\n\t"
        "add.u64 m1, %1, 32;\n\t"
        "add.u64 n1, %2, 32;\n\t"
        "add.u64 n2, %2, %3;\n\t"
        "add.u64 n3, n2, 32;\n\t"
        "add.u32 t1, %0, 4;\n\t"
        "add.u32 u0, %0, 8;\n\t"            // row tile 0, first half of the chunk
        "add.u32 u1, %0, 16;\n\t"           // and second
        "add.u32 u2, %0, 12;\n\t"           // row tile 1
        "add.u32 u3, %0, 20;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;\n\t"
        "@q tcgen05.cp.cta_group::2.32x128b.warpx4 [u0], %2;\n\t"
        "@q tcgen05.cp.cta_group::2.32x128b.warpx4 [u2], n2;\n\t"
        "@q tcgen05.cp.cta_group::2.32x128b.warpx4 [t1], m1;\n\t"
        "@q tcgen05.cp.cta_group::2.32x128b.warpx4 [u1], n1;\n\t"
        "@q tcgen05.cp.cta_group::2.32x128b.warpx4 [u3], n3;\n\t"
        "}\n"
        ::"r"(sa), "l"(sa_mem), "l"(sb_mem), "n"(MX_GROUP * MX4_TILE / 16) : "memory");
}

// A chunk's four MMAs of a pair, by a whole warp whose lanes agree on the arguments (see tc_mma4).
__device__ __forceinline__ void mx_chunk_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t sa, uint32_t accumulate)
{
    constexpr uint32_t idesc = (1u << 7) | (1u << 10) | ((uint32_t)(MX_PAIR_N >> 3) << 17) | (1u << 23) | ((uint32_t)(MX_PAIR_M >> 4) << 24);
    constexpr uint32_t idesc2 = idesc | (2u << 4) | (2u << 29);
    asm volatile(
        "{\n\t"
        ".reg .pred p, q;\n\t"
        ".reg .b64 a1, a2, a3, b1, b2, b3;\n\t"
        ".reg .b32 t1, u0, u1;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "add.u64 a1, %1, 2;\n\t"
        "add.u64 a2, %1, 4;\n\t"
        "add.u64 a3, %1, 6;\n\t"
        "add.u64 b1, %2, 2;\n\t"
        "add.u64 b2, %2, 4;\n\t"
        "add.u64 b3, %2, 6;\n\t"
        "add.u32 t1, %3, 4;\n\t"
        "add.u32 u0, %3, 8;\n\t"
        "add.u32 u1, %3, 16;\n\t"
        "elect.sync _|q, 0xffffffff;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %5, [%3], [u0], p;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], a1, b1, %6, [%3], [u0], 1;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], a2, b2, %5, [t1], [u1], 1;\n\t"
        "@q tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], a3, b3, %6, [t1], [u1], 1;\n\t"
        "}\n"
        ::"r"(d), "l"(a), "l"(b), "r"(sa), "r"(accumulate), "r"(idesc), "r"(idesc2)
        : "memory");
}

// What a pair does in its round `i`: a tile, a range of its chunks, and where its sums go.
struct MxTask {
    int tile, c0, c1, part;         // part: which of the partial sums in scratch, or -1: the output itself
};

// tiles: all tiles; whole: those that go round whole; splits: the pairs that share one of the others.
struct MxSchedule {
    int tiles_n, tiles, whole, splits;
    __device__ __forceinline__ bool task(int i, int pair, int pairs, int chunks, MxTask &t) const
    {
        const long long u = (long long)i * pairs + pair;
        if (u < whole) {
            t = MxTask{(int)u, 0, chunks, -1};
            return true;
        }
        // (whole is a multiple of the pairs wherever tiles are shared)
        const int v = (int)(u - whole), left = v / splits, part = v - left * splits;
        if (i > whole / pairs || left >= tiles - whole)
            return false;
        t = MxTask{whole + left, (int)((long long)chunks * part / splits), (int)((long long)chunks * (part + 1) / splits), v};
        return true;
    }
};

template <typename TO>
__global__ void __launch_bounds__(MX_THREADS, 1)
gemm_mx4_pair_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_a,
                     const __grid_constant__ CUtensorMap map_ws, const __grid_constant__ CUtensorMap map_as,
                     TO *__restrict__ out, float *__restrict__ partial, int n, int m, int chunks, const MxSchedule plan, int w_early)
{
    constexpr uint32_t STAGES = MX_PAIR_STAGES;
    extern __shared__ uint8_t smem_raw[];
    uint8_t *smem = (uint8_t *)(((uintptr_t)smem_raw + 1023) & ~(uintptr_t)1023);
    const uint32_t codes0 = smem_u32(smem), scales0 = codes0 + STAGES * MX_PAIR_STAGE_BYTES;
    uint64_t *bars = (uint64_t *)(smem + STAGES * MX_PAIR_STAGE_BYTES + MX_GROUPS * MX_PAIR_SCALE_BYTES);
    const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * STAGES, sc_full0 = empty0 + 8 * STAGES,
                   sc_empty0 = sc_full0 + 8 * MX_GROUPS, accum = sc_empty0 + 8 * MX_GROUPS, drained = accum + 8;
    uint32_t *tmem_slot = (uint32_t *)(bars + 2 * STAGES + 2 * MX_GROUPS + 2);
    volatile int *abort = (volatile int *)(tmem_slot + 1);

    const int warp = (int)warp_uniform(threadIdx.x >> 5), lane = threadIdx.x & 31;
    const uint32_t rank = cluster_rank();
    const int pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
    if (threadIdx.x == 0) {
        prefetch_tensor_map(&map_w);
        prefetch_tensor_map(&map_a);
        prefetch_tensor_map(&map_ws);
        prefetch_tensor_map(&map_as);
        for (uint32_t s = 0; s < 2 * (STAGES + MX_GROUPS) + 1; s++)
            mbar_init(full0 + 8 * s, 1);
        mbar_init(drained, 16);             // the epilogue's warps of both CTAs
        *abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_arrive();
    cluster_wait();
    tc_fence_after();
    const uint32_t tmem = warp_uniform(*tmem_slot);
    pdl_trigger();

    if (warp == 0 && lane == 0) {
        // ---------------------------------------------------------- loads
        uint32_t it = 0, group = 0;
        const uint32_t lead_full = cluster_addr(full0, 0), lead_sc = cluster_addr(sc_full0, 0);
        bool ok = true, waited = !w_early;
        if (waited)
            pdl_wait();
        MxTask t;
        for (int i = 0; ok && plan.task(i, pair, pairs, chunks, t); i++) {
            const int m0 = t.tile / plan.tiles_n * MX_PAIR_M + (int)rank * MX_TILE_M, n0 = t.tile % plan.tiles_n * MX_PAIR_N;
            for (int c = t.c0; c < t.c1; c++, it++) {
                const uint32_t s = it % STAGES, codes = codes0 + s * MX_PAIR_STAGE_BYTES;
                const uint32_t g = group % MX_GROUPS, scales = scales0 + g * MX_PAIR_SCALE_BYTES;
                const bool first = (c - t.c0) % MX_GROUP == 0;
                if (first) {
                    if (group >= MX_GROUPS && !mbar_wait(sc_empty0 + 8 * g, ((group / MX_GROUPS) & 1) ^ 1, abort, &g_gemm_mx4_error, 7)) {
                        ok = false;
                        break;
                    }
                    if (rank == 0)
                        mbar_expect_tx(sc_full0 + 8 * g, 2 * MX_PAIR_SCALE_BYTES);
                    tma_load_pair(scales, &map_ws, lead_sc + 8 * g, 0, 8 * c, m0 >> 7);
                    group++;
                }
                if (it >= STAGES && !mbar_wait(empty0 + 8 * s, ((it / STAGES) & 1) ^ 1, abort, &g_gemm_mx4_error, 1)) {
                    ok = false;
                    break;
                }
                if (rank == 0)
                    mbar_expect_tx(full0 + 8 * s, 2 * MX_PAIR_STAGE_BYTES);
                tma_load_pair(codes, &map_w, lead_full + 8 * s, c * (MX4_CHUNK / 2), m0);
                if (!waited) {
                    pdl_wait();
                    waited = true;
                }
                if (first)
                    tma_load_pair(scales + MX_GROUP * MX4_TILE, &map_as, lead_sc + 8 * g, 0, 8 * c, n0 >> 7);
                tma_load_pair(codes + MX_W_BYTES, &map_a, lead_full + 8 * s, c * (MX4_CHUNK / 2), n0 + (int)rank * (MX_PAIR_N / 2));
            }
        }
        if (*abort && rank == 0) {
            // the loads in flight of both CTAs: wait for each barrier's last use, once, with the limit (the other CTA then
            // waits for this one at the cluster's barrier)
            volatile int never = 0;
            for (uint32_t u = it > STAGES ? it - STAGES : 0; u < it; u++)
                mbar_wait(full0 + 8 * (u % STAGES), (u / STAGES) & 1, &never, &g_gemm_mx4_error, 4);
            for (uint32_t u = group > MX_GROUPS ? group - MX_GROUPS : 0; u < group; u++)
                mbar_wait(sc_full0 + 8 * (u % MX_GROUPS), (u / MX_GROUPS) & 1, &never, &g_gemm_mx4_error, 4);
        }
    } else if (warp == 1 && rank == 0) {
        // --------------------------------------------------------------- MMAs of both CTAs
        uint32_t it = 0, group = 0, done = 0;
        bool ok = true;
        MxTask t;
        for (; ok && plan.task(done, pair, pairs, chunks, t); done++) {
            for (int c = 0; c < t.c1 - t.c0; c++, it++) {
                const uint32_t s = it % STAGES, g = group % MX_GROUPS;
                if (c % MX_GROUP == 0)
                    ok = mbar_wait(sc_full0 + 8 * g, (group / MX_GROUPS) & 1, abort, &g_gemm_mx4_error, 8);
                ok = __all_sync(0xffffffffu, ok && mbar_wait(full0 + 8 * s, (it / STAGES) & 1, abort, &g_gemm_mx4_error, 2));
                if (!ok)
                    break;
                tc_fence_after();
                const uint32_t codes = codes0 + s * MX_PAIR_STAGE_BYTES, col = tmem + MX_PAIR_N + s * MX_SLOT_COLS;
                const uint32_t scales = scales0 + g * MX_PAIR_SCALE_BYTES + c % MX_GROUP * MX4_TILE;
                mx_scales_pair(col, mx_scale_desc(scales), mx_scale_desc(scales + MX_GROUP * MX4_TILE));
                if (c == 0 && done) {           // the accumulator of the tile before has been read
                    ok = __all_sync(0xffffffffu, mbar_wait(drained, (done - 1) & 1, abort, &g_gemm_mx4_error, 6));
                    if (!ok)
                        break;
                    tc_fence_after();
                }
                mx_chunk_pair(tmem, smem_desc_sw128(codes, 16, 1024), smem_desc_sw128(codes + MX_W_BYTES, 16, 1024), col, c != 0);
                tc_commit_pair(empty0 + 8 * s);
                if (c % MX_GROUP == MX_GROUP - 1 || c == t.c1 - t.c0 - 1) {
                    tc_commit_pair(sc_empty0 + 8 * g);
                    group++;
                }
            }
            tc_commit_pair(accum);
        }
    } else if (warp >= 2) {
        // ------------------------------------------------------------ epilogue
        constexpr int PART = MX_PAIR_N / 2;
        const int q = warp & 3, part = (warp - 2) >> 2;
        const uint32_t lead_drained = cluster_addr(drained, 0);
        uint32_t done = 0;
        pdl_wait();
        MxTask t;
        for (; plan.task(done, pair, pairs, chunks, t); done++) {
            if (!__all_sync(0xffffffffu, mbar_wait(accum, done & 1, abort, &g_gemm_mx4_error, 3)))
                break;
            tc_fence_after();
            const int fl = (int)rank * MX_TILE_M + q * 32 + lane;
            const int f = t.tile / plan.tiles_n * MX_PAIR_M + fl, r0 = t.tile % plan.tiles_n * MX_PAIR_N + part * PART;
            uint32_t v[PART];
#pragma unroll
            for (int c = 0; c < PART; c += 32)
                tc_ld32_nowait(tmem + ((uint32_t)(q * 32) << 16) + part * PART + c, v + c);
            tc_ld_wait();
            tc_fence_before();
            __syncwarp();
            if (lane == 0)
                mbar_arrive_pair(lead_drained);
            if (t.part >= 0) {
                float *o = partial + ((size_t)t.part * MX_PAIR_N + part * PART) * MX_PAIR_M + fl;
#pragma unroll
                for (int j = 0; j < PART; j++)
                    if (r0 + j < n)
                        o[j * MX_PAIR_M] = __uint_as_float(v[j]);
            } else if (f < m) {
                TO *o = out + (size_t)r0 * m + f;
                if (r0 + PART <= n) {
#pragma unroll
                    for (int j = 0; j < PART; j++, o += m)
                        *o = from_f<TO>(__uint_as_float(v[j]));
                } else {
#pragma unroll
                    for (int j = 0; j < PART; j++, o += m)
                        if (r0 + j < n)
                            *o = from_f<TO>(__uint_as_float(v[j]));
                }
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    cluster_arrive();
    cluster_wait();                 // neither CTA ends, or gives its tensor memory back, while the other's MMAs may run
    if (warp == 1)
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
}

// The sums of tiles that were shared out along k: a block per row of a tile, a thread per feature.
template <typename TO>
__global__ void __launch_bounds__(MX_PAIR_M)
mx_join_kernel(const float *partial, TO *__restrict__ out, int n, int m, const MxSchedule plan)
{
    pdl_trigger();
    const int left = blockIdx.x / MX_PAIR_N, j = blockIdx.x - left * MX_PAIR_N, tile = plan.whole + left;
    const int r = tile % plan.tiles_n * MX_PAIR_N + j, f = tile / plan.tiles_n * MX_PAIR_M + threadIdx.x;
    if (r >= n || f >= m)
        return;
    pdl_wait();
    const float *p = partial + ((size_t)left * plan.splits * MX_PAIR_N + j) * MX_PAIR_M + threadIdx.x;
    out[(size_t)r * m + f] = from_f<TO>(add_partials(0.0f, p, plan.splits, (size_t)MX_PAIR_N * MX_PAIR_M));
}

// A matrix of codes in boxes of box_rows x 128 bytes with the 128-byte swizzle; what lies outside reads as zero.
static bool mx_tensor_map(const void *codes, int rows, int k, int box_rows, CUtensorMap *out)
{
    EncodeTiled enc = tensor_map_encoder();
    if (!enc)
        return false;
    cuuint64_t dims[2] = {(cuuint64_t)mx4_row_bytes(k), (cuuint64_t)rows};
    cuuint64_t strides[1] = {(cuuint64_t)mx4_row_bytes(k)};
    cuuint32_t box[2] = {128, (cuuint32_t)box_rows}, estr[2] = {1, 1};
    return enc(out, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(codes), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// Scales as [tiles of 128 rows, chunks, 1,024 bytes], in boxes of MX_GROUP chunks of box_tiles tiles; what lies outside
// reads as zero.
static bool mx_scale_map(const void *scales, int rows, int k, int box_tiles, CUtensorMap *out)
{
    EncodeTiled enc = tensor_map_encoder();
    if (!enc)
        return false;
    const cuuint64_t chunks = mx4_chunks(k);
    cuuint64_t dims[3] = {32, 8 * chunks, (cuuint64_t)((rows + 127) / 128)};
    cuuint64_t strides[2] = {128, MX4_TILE * chunks};
    cuuint32_t box[3] = {32, 8 * MX_GROUP, (cuuint32_t)box_tiles}, estr[3] = {1, 1, 1};
    return enc(out, CU_TENSOR_MAP_DATA_TYPE_UINT32, 3, const_cast<void *>(scales), dims, strides, box, estr,
               CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
               CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// How the tiles of a product are shared out.  What is left over after whole rounds is shared out along k where that saves
// more than the partial sums' way through memory and a launch cost, about ten chunks' time (a chunk of k takes a pair 0.35
// us; 2,048 rows x 2,560 x 9,728, 80 tiles of 38 chunks: 35 us in two rounds, 26 with six tiles shared by 12 pairs each).
static MxSchedule mx_schedule(int n, int m, int k)
{
    const int pairs = sm_count() / 2, chunks = mx4_chunks(k);
    MxSchedule p;
    p.tiles_n = (n + MX_PAIR_N - 1) / MX_PAIR_N;
    p.tiles = p.tiles_n * ((m + MX_PAIR_M - 1) / MX_PAIR_M);
    p.whole = p.tiles;
    p.splits = 1;
    const int left = p.tiles % pairs;
    if (left > 0) {
        int splits = pairs / left;
        splits = splits > chunks ? chunks : splits;
        if (splits > 1 && chunks - (chunks + splits - 1) / splits > 10) {
            p.whole = p.tiles - left;
            p.splits = splits;
        }
    }
    return p;
}

static long long mx_partial_bytes(const MxSchedule &p)
{
    return p.whole == p.tiles ? 0 : (long long)(p.tiles - p.whole) * p.splits * MX_PAIR_M * MX_PAIR_N * 4;
}

template <typename TO>
static int launch_mx_pair(const void *ac, const void *as, const void *wc, const void *ws, TO *out, void *partial, int n, int m,
                          int k, int w_early, cudaStream_t st)
{
    CUtensorMap map_w, map_a, map_ws, map_as;
    if (!mx_tensor_map(wc, m, k, MX_TILE_M, &map_w) || !mx_tensor_map(ac, n, k, MX_PAIR_N / 2, &map_a) ||
        !mx_scale_map(ws, m, k, 1, &map_ws) || !mx_scale_map(as, n, k, MX_ROW_TILES, &map_as))
        return JB_EINVAL;
    auto kern = gemm_mx4_pair_kernel<TO>;
    static unsigned long long allowed = 0;
    if (!allow_dynamic_smem(kern, MX_PAIR_SMEM, allowed))
        return JB_ELAUNCH;
    const MxSchedule plan = mx_schedule(n, m, k);
    const int pairs = sm_count() / 2, shared = plan.tiles - plan.whole;
    if (shared && !partial)
        return JB_EINVAL;
    launch_cluster(kern, dim3(2u * (plan.tiles < pairs && !shared ? plan.tiles : pairs)), MX_THREADS, MX_PAIR_SMEM, st, 2u, map_w,
                   map_a, map_ws, map_as, out, (float *)partial, n, m, mx4_chunks(k), plan, w_early);
    int e = launch_status();
    if (e == JB_OK && shared) {
        launch(mx_join_kernel<TO>, (unsigned)shared * MX_PAIR_N, MX_PAIR_M, 0, st, (const float *)partial, out, n, m, plan);
        e = launch_status();
    }
    return e;
}

// Parts of k (1, 2, 4 or 8) that a product's tiles are shared out in: as many as leave every part an SM of its own, and where
// the CTAs pack the rows of floats themselves, which shorter parts shorten, two parts an SM (8 rows, 20 tiles of 16
// chunks: codes 4.1 us in 4 parts and 4.6 in 8, floats 5.4 and 5.2; 64 rows of codes 5.1 and 7.5).
static int mx_parts(int tiles, int chunks, bool few_floats)
{
    int p = 1;
    while (p < 8 && tiles * p * 2 <= (few_floats ? 2 : 1) * sm_count() && p * 2 <= chunks)
        p *= 2;
    return p;
}

// How a product with tiles of BN rows is launched: its parts of k, and each CTA's stages, shared memory and columns of
// tensor memory.
struct MxShape {
    int tiles_m, tiles_n, parts, stages, smem, cols;
};
template <int BN> static MxShape mx_shape(int n, int m, int k, bool few_floats)
{
    using Cfg = MxCfg<BN>;
    MxShape s;
    const int chunks = mx4_chunks(k);
    s.tiles_m = (m + MX_TILE_M - 1) / MX_TILE_M, s.tiles_n = (n + BN - 1) / BN;
    s.parts = mx_parts(s.tiles_m > 0x7fffff ? 0x7fffff : s.tiles_m * s.tiles_n, chunks, few_floats);
    // (a part's sums, BN x 128 floats, lie in the stages' memory when the MMAs are done)
    constexpr int SUMS = (BN * MX_TILE_M * 4 + Cfg::STAGE_BYTES - 1) / Cfg::STAGE_BYTES;
    static_assert(SUMS <= Cfg::STAGES, "room for a part's sums");
    s.stages = (chunks + s.parts - 1) / s.parts;
    s.stages = s.stages > Cfg::STAGES ? Cfg::STAGES : s.parts > 1 && s.stages < SUMS ? SUMS : s.stages;
    s.smem = Cfg::smem_bytes(s.stages, s.parts > 1);
    s.cols = Cfg::tmem_cols(s.stages);
    return s;
}

template <int BN, typename TO, int ROWS>
static int launch_mx(const void *ac, const void *as, MxRows rows, const void *wc, const void *ws, TO *out, int n, int m, int k,
                     int w_early, cudaStream_t st)
{
    CUtensorMap map_w, map_a;
    if (!mx_tensor_map(wc, m, k, MX_TILE_M, &map_w) || (!ROWS && !mx_tensor_map(ac, n, k, BN, &map_a)))
        return JB_EINVAL;
    if (ROWS)
        map_a = map_w;              // not used
    auto kern = gemm_mx4_kernel<BN, TO, ROWS>;
    static unsigned long long allowed = 0;
    if (!allow_dynamic_smem(kern, MxCfg<BN>::SMEM_MOST, allowed))
        return JB_ELAUNCH;
    const MxShape s = mx_shape<BN>(n, m, k, ROWS != ROWS_NONE);
    if (s.tiles_n > 65535)
        return JB_EINVAL;
    launch_cluster(kern, dim3((unsigned)s.tiles_m * s.parts, s.tiles_n), MX_THREADS, s.smem, st, (unsigned)s.parts, map_w, map_a,
                   (const uint8_t *)ws, (const uint8_t *)as, rows, out, n, m, mx4_chunks(k), s.parts, s.stages, w_early);
    return launch_status();
}

constexpr int MX_FEW = 128;         // rows up to which a product's tiles are single CTAs'

// Rows of a tile, 16 or 32, where the product's CTAs pack rows of floats themselves, or 0 where a kernel ahead does: up to 32
// rows always, and up to 128 where a warp has at most 12 items (a row of a chunk) to pack, as each tile along m packs the
// same rows again.  Tiles of 16 rows leave a warp the fewest; 32 where those would be over two an SM.
// The rule weighs a call from Python, in which a second launch and memory for the codes cost about 5 us: 77 rows of floats x
// 1,003 x 1,037 8.9 us, quantised by a call of its own before 15.5; 128 x 2,560 x 1,037 10.0 and 15.4; 128 x 2,560 x 2,560,
// with a kernel ahead, 14.3.  On the device alone, as a captured step pays for it, it holds for one token and for short k
// only; with more rows, tiles along m or chunks of k the kernel ahead would be faster.  Rows of bfloat16, packed by the
// product / by a kernel ahead, us (40 of the same in a graph, so with the weights in the L2):
//     1 x 2,560 x 9,728    5.7 /  6.3     8 x 2,560 x 4,096   5.1 /  5.4     77 x 1,003 x 1,037   6.2 /  6.7
//     1 x 19,456 x 2,560   6.5 /  5.9     8 x 19,456 x 2,560  8.5 /  5.9     40 x 6,144 x 2,560   8.2 /  6.5
//     16 x 6,144 x 2,560   6.4 /  5.4    32 x 6,144 x 2,560  10.0 /  6.1     77 x 6,144 x 1,037   9.6 /  7.4
//     16 x 19,456 x 2,560 10.9 /  6.0    32 x 19,456 x 2,560 21.0 /  6.4    128 x 2,560 x 1,037   9.5 /  7.5
//     16 x 2,560 x 9,728   8.6 /  6.9    32 x 2,560 x 9,728  13.9 /  7.3     32 x 19,456 x 9,728 79.8 / 19.2
static int mx_rows_tile(int n, int m, int k)
{
    if (n <= 32)
        return n <= 16 ? 16 : 32;
    if (n > MX_FEW)
        return 0;
    const int chunks = mx4_chunks(k), tiles_m = (m + MX_TILE_M - 1) / MX_TILE_M;
    for (int bn = 16; bn <= 32; bn *= 2) {
        const long long tiles = (long long)tiles_m * ((n + bn - 1) / bn);
        if (tiles > 2 * sm_count())
            continue;
        const int parts = mx_parts((int)tiles, chunks, true);
        if (bn / 8 * ((chunks + parts - 1) / parts) <= 12)
            return bn;
    }
    return 0;
}

// Rows of a tile where they come as codes, or 0: pairs' tiles.
static int mx_codes_tile(int n) { return n <= 16 ? 16 : n <= 32 ? 32 : n <= 64 ? 64 : n <= MX_FEW ? 128 : 0; }

template <typename TO>
static int any_mx(const void *ac, const void *as, MxRows rows, const void *wc, const void *ws, TO *out, void *partial, int n,
                  int m, int k, int w_early, cudaStream_t st)
{
    if (rows.x) {
        const bool wide = mx_rows_tile(n, m, k) == 32;
        if (rows.is_bf16 && rows.vec)
            return wide ? launch_mx<32, TO, ROWS_BF16>(ac, as, rows, wc, ws, out, n, m, k, w_early, st)
                        : launch_mx<16, TO, ROWS_BF16>(ac, as, rows, wc, ws, out, n, m, k, w_early, st);
        return wide ? launch_mx<32, TO, ROWS_ANY>(ac, as, rows, wc, ws, out, n, m, k, w_early, st)
                    : launch_mx<16, TO, ROWS_ANY>(ac, as, rows, wc, ws, out, n, m, k, w_early, st);
    }
    switch (mx_codes_tile(n)) {
    case 16: return launch_mx<16, TO, ROWS_NONE>(ac, as, rows, wc, ws, out, n, m, k, w_early, st);
    case 32: return launch_mx<32, TO, ROWS_NONE>(ac, as, rows, wc, ws, out, n, m, k, w_early, st);
    case 64: return launch_mx<64, TO, ROWS_NONE>(ac, as, rows, wc, ws, out, n, m, k, w_early, st);
    case 128: return launch_mx<128, TO, ROWS_NONE>(ac, as, rows, wc, ws, out, n, m, k, w_early, st);
    }
    return launch_mx_pair<TO>(ac, as, wc, ws, out, partial, n, m, k, w_early, st);
}

// Tiles and partial sums are counted in 32 bits; every address is one that 16 divides.
static bool bad_product(const void *ac, const void *as, const void *wc, const void *ws, const void *out, const void *scratch,
                        int out_dt, int n, int m, int k)
{
    return n < 0 || m < 0 || k < 1 || n > MX4_MOST || m > MX4_MOST || k > MX4_MOST || (out_dt != 0 && out_dt != 1) ||
           ((uintptr_t)ac | (uintptr_t)as | (uintptr_t)wc | (uintptr_t)ws | (uintptr_t)out | (uintptr_t)scratch) % 16 ||
           ((long long)n / 16 + 1) * ((long long)m / 128 + 1) > 0x3fffffff;
}

}  // namespace jb

using namespace jb;

// Bytes of scratch that a product needs, with n rows that come as codes (rows 0) or as floats (rows 1).
extern "C" long long jb_linear_mx4_scratch(int n, int m, int k, int rows)
{
    if (n < 1 || m < 1 || k < 1 || n > MX4_MOST || m > MX4_MOST || k > MX4_MOST)
        return 0;
    long long bytes = n > MX_FEW ? mx_partial_bytes(mx_schedule(n, m, k)) : 0;
    if (rows && mx_rows_tile(n, m, k) == 0)
        bytes += jb_mx4_code_bytes(n, k) + jb_mx4_scale_bytes(n, k);
    return bytes;
}

// How many kernels such a product launches.
extern "C" int jb_linear_mx4_launches(int n, int m, int k, int rows)
{
    if (n < 1 || m < 1 || k < 1 || n > MX4_MOST || m > MX4_MOST || k > MX4_MOST)
        return 0;
    return 1 + (rows && mx_rows_tile(n, m, k) == 0) + (n > MX_FEW && mx_partial_bytes(mx_schedule(n, m, k)) > 0);
}

// How such a product's CTAs share an SM: out = {CTAs of a cluster, shared memory of a CTA in bytes, its columns of tensor
// memory}.
extern "C" int jb_linear_mx4_cta(int n, int m, int k, int rows, int *out)
{
    if (n < 1 || m < 1 || k < 1 || n > MX4_MOST || m > MX4_MOST || k > MX4_MOST)
        return JB_EINVAL;
    const int own = rows ? mx_rows_tile(n, m, k) : 0, tile = own ? own : mx_codes_tile(n);
    const MxShape s = tile == 16 ? mx_shape<16>(n, m, k, own) : tile == 32 ? mx_shape<32>(n, m, k, own)
                    : tile == 64 ? mx_shape<64>(n, m, k, false) : tile == 128 ? mx_shape<128>(n, m, k, false)
                                 : MxShape{0, 0, 2, 0, MX_PAIR_SMEM, SM_TMEM_COLS};
    out[0] = s.parts, out[1] = s.smem, out[2] = s.cols;
    return JB_OK;
}

// out [n, m] (out_dt 0 float32, 1 bfloat16) = a [n, k] . w [m, k]^T, both as codes and scales.  scratch: see
// jb_linear_mx4_scratch.  w_early: no kernel that may still be running when this one starts writes the weights.
extern "C" int jb_linear_mx4(const void *a_codes, const void *a_scales, const void *w_codes, const void *w_scales, void *out,
                             int out_dt, int n, int m, int k, void *scratch, int w_early, cudaStream_t st)
{
    if (bad_product(a_codes, a_scales, w_codes, w_scales, out, scratch, out_dt, n, m, k))
        return JB_EINVAL;
    if (n == 0 || m == 0)
        return JB_OK;
    const MxRows none{nullptr, k, 0, 0};
    return out_dt == 1 ? any_mx(a_codes, a_scales, none, w_codes, w_scales, (bf16 *)out, scratch, n, m, k, w_early, st)
                       : any_mx(a_codes, a_scales, none, w_codes, w_scales, (float *)out, scratch, n, m, k, w_early, st);
}

// The same with a as floats (dt 0 float32, 1 bfloat16), which are brought to 4 bits on the way: in the product's own
// kernel for few rows, else by a kernel ahead of it, in scratch.
extern "C" int jb_linear_mx4_rows(const void *x, int dt, const void *w_codes, const void *w_scales, void *out, int out_dt, int n,
                                  int m, int k, void *scratch, int w_early, cudaStream_t st)
{
    if (bad_product(nullptr, nullptr, w_codes, w_scales, out, scratch, out_dt, n, m, k) || (dt != 0 && dt != 1))
        return JB_EINVAL;
    if (n == 0 || m == 0)
        return JB_OK;
    if (mx_rows_tile(n, m, k) == 0) {
        if (!scratch)
            return JB_EINVAL;
        uint8_t *codes = (uint8_t *)scratch, *scales = codes + jb_mx4_code_bytes(n, k), *rest = scales + jb_mx4_scale_bytes(n, k);
        const int e = jb_mx4_quantize(x, dt, codes, scales, n, k, 1, st);
        return e != JB_OK ? e : jb_linear_mx4(codes, scales, w_codes, w_scales, out, out_dt, n, m, k, rest, w_early, st);
    }
    const MxRows rows{x, k, dt, k % 8 == 0 && (uintptr_t)x % 16 == 0};
    return out_dt == 1 ? any_mx(nullptr, nullptr, rows, w_codes, w_scales, (bf16 *)out, nullptr, n, m, k, w_early, st)
                       : any_mx(nullptr, nullptr, rows, w_codes, w_scales, (float *)out, nullptr, n, m, k, w_early, st);
}

// Reads and clears the error word: 0, or which wait ran out first (as jb_gemm_tc_error).
extern "C" int jb_gemm_mx4_error(void)
{
    int v = 0, zero = 0;
    if (cudaMemcpyFromSymbol(&v, g_gemm_mx4_error, sizeof v) != cudaSuccess)
        return JB_ELAUNCH;
    if (v != 0)
        cudaMemcpyToSymbol(g_gemm_mx4_error, &zero, sizeof zero);
    return v;
}
