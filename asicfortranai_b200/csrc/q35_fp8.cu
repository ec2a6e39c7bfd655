// q35_fp8.cu -- matrix product in 8-bit floating point (e4m3) with a scale for each block of
// 128 along k of every row of x, and for each 128 x 128 block of w:
//   y[m][n] = sum_b xs[m][b] ws[n / 128][b] sum_{k in block b} x[m][k] w[n][k]
//
// Both kernels below run the same pipeline, per 128-k block:
//   * producer (warp 0, one thread): two 2D TMA loads, 128 bytes of k x the tile's rows of w and
//     of x, 128-byte swizzle (rows past the edges and k past K read as zero);
//   * scale loader (warp 2): the products xs * ws of the tile's rows of x into the stage;
//   * MMA issuer (warp 1, one thread): 4 x tcgen05.mma kind::f8f6f4 (K = 32 each) into one
//     of several accumulators in tensor memory.  The sum over one block is a tensor-core
//     fp32 sum of exact products;
//   * promotion (warps 4 ..): tcgen05.ld of the block's sums, acc = fma(sum, scale, acc)
//     with acc in registers, the next columns' load on its way meanwhile (packed fma.rn.f32x2
//     was slower: the pairs had to be moved together).
// A k-block's accumulator is handed over through mbarriers, so the MMAs of the next blocks
// run under the promotion of this one.
//
// fp8_gemm_kernel (up to 128 rows of x): w in the MMA's M position, 128 rows of w (one row of
// scale blocks, so ws is one number per tile and k-block) x BN <= 128 rows of x; a thread owns a
// row of w and reads the scales of x's rows as broadcast vectors.
//
// fp8_gemm_pair_kernel (more rows): two CTAs on one 256 x 256 tile (cta_group::2), x in the M
// position, each CTA holding 128 rows of x and half of the tile's rows of w, so that an SM
// reads 32 KB a k-block instead of 48; a thread owns a row of x and one scale covers its 128
// columns.  (An accumulator, issuer and hand-over of its own for each of the two blocks of w's
// rows was slower, 573 against 522 us at 2048 x 28672 x 8192: x's rows are then read twice.)
//
// Few tiles are split along k over the CTAs (pairs) of a cluster; each CTA then adds up its
// share of the tile's columns from every CTA's shared memory, in CTA order, so the result does
// not depend on timing.
//
// Measured: 1 x 10240 x 8192 20 us (84 MB of w, 4.2 TB/s), 16 x 8192 x 28672 43 us (236 MB, 5.5
// TB/s): w's bytes through HBM bound both, less the start and the cluster's exchange.
// 197 x 5120 x 13824 44 us: 20 tiles of 256 x 256 split three ways, each pair's chain of k-blocks.
// 2048 x 28672 x 8192 600 us back to back (1.6 PFLOP/s, at the power cap): the promotion, 1230
// clocks a k-block of a pair's tile, against 512 of MMAs.
//
// Every wait is bounded: a wait that gives up records Q35_ERR_TIMEOUT in the context's error
// word and raises an abort flag that ends the other roles' waits; copies and MMAs in flight
// are waited for (bounded) before the CTA leaves.
#include <cuda.h>

#include <algorithm>

#include "q35_q8.cuh"
#include "q35_tc.cuh"

namespace q35 {
namespace {

constexpr int F8_TN = 128;                 // rows of w per tile
constexpr int F8_KB = 128;                 // k per block (bytes per row of a stage)

struct F8Params {
    const float *xs, *ws;                  // [M][KB], [ceil(N/128)][KB]
    void *y;
    int64_t ldy;
    int32_t M, N, KB;
    int32_t BN, mt, nt;                    // rows of x per tile, tiles along m and n
    int32_t split;                         // CTAs (of a cluster) per tile
    int32_t stages, bufs;
    uint32_t tmem_cols, buf_cols;
    uint32_t off_sc, off_bar;
    int *err;
};

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap *map, int32_t x, int32_t y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
                 " [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void l2_prefetch_2d(const CUtensorMap *map, int32_t x, int32_t y) {
    asm volatile("cp.async.bulk.prefetch.tensor.2d.L2.global.tile [%0, {%1, %2}];"
                 ::"l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void tc_mma_f8(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// D fp32, A and B e4m3, both K-major
__host__ __device__ constexpr uint32_t idesc_f8(int m, int n) {
    return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
__device__ __forceinline__ uint32_t cluster_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    __syncwarp();
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// the address of a shared variable of this CTA in CTA rank's shared memory
__device__ __forceinline__ uint32_t at_rank(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void st_cluster(uint32_t addr, uint32_t rank, float v) {
    asm volatile("{\n\t.reg .b32 ra;\n\tmapa.shared::cluster.u32 ra, %0, %1;\n\t"
                 "st.shared::cluster.f32 [ra], %2;\n\t}" ::"r"(addr), "r"(rank), "f"(v) : "memory");
}

// NB: accumulator registers (x rows) per promotion thread; 4 or 8 promotion warps, the second
// four taking the upper half of the tile's columns (from 33 rows on: one warp per scheduler
// could not keep up).  Tiles of up to 32 rows run two CTAs on an SM (a third of the memory each,
// with the next launch's CTA set up beside them, was slower: 23.2 against 20.7 us at
// 1 x 10240 x 8192; so was one: 32).
template <typename T, int NB, int PW>
__global__ void __launch_bounds__(128 + 32 * PW, PW == 4 ? 2 : 1)
fp8_gemm_kernel(const F8Params p, const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t *sbase = smem_raw + (base - raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int S = p.stages, NBUF = p.bufs, BN = p.BN;
    const uint32_t stage_bytes = (uint32_t)(F8_TN + BN) * F8_KB;
    const uint32_t bars = base + p.off_bar;
    auto full = [&](int i) { return bars + 8u * i; };                       // TMA bytes
    auto sc_full = [&](int i) { return bars + 8u * (S + i); };              // scale loader
    auto empty = [&](int i) { return bars + 8u * (2 * S + i); };            // commit + promotion warps
    auto acc_full = [&](int i) { return bars + 8u * (3 * S + i); };         // commit
    auto acc_empty = [&](int i) { return bars + 8u * (3 * S + NBUF + i); }; // promotion warps
    const uint32_t drain = bars + 8u * (3 * S + 2 * NBUF);
    uint8_t *misc = sbase + p.off_bar + 8 * (3 * S + 2 * NBUF + 1);
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(misc);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(misc + 4);

    if (tid == 0) {
        for (int i = 0; i < S; ++i) { mbar_init(full(i), 1); mbar_init(sc_full(i), 1); mbar_init(empty(i), 1 + PW); }
        for (int i = 0; i < NBUF; ++i) { mbar_init(acc_full(i), 1); mbar_init(acc_empty(i), PW); }
        mbar_init(drain, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32((const void *)tmem_slot)), "r"(p.tmem_cols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const int rank = p.split > 1 ? (int)cluster_rank() : 0;
    const int first_tile = blockIdx.x / p.split, step = gridDim.x / p.split;
    const int tiles = p.mt * p.nt;
    const int kb0 = (int)((int64_t)p.KB * rank / p.split), kb1 = (int)((int64_t)p.KB * (rank + 1) / p.split);
    dependency_trigger();
    // (a fetch into L2 reads nothing: a kernel before this one may still write w)
    if (PW == 4 && warp == 0 && lane < S && kb0 + lane < kb1)
        l2_prefetch_2d(&wmap, (kb0 + lane) * F8_KB, first_tile / p.mt * F8_TN);
    dependency_wait();

    bool ok = true;
    auto fail = [&]() {
        ok = false;
        *abort_flag = 1;
        atomicExch(p.err, Q35_ERR_TIMEOUT);
    };

    if (warp < 4) {
        if (warp == 0) {
            if (lane == 0) {
                Ring st{};
                int64_t issued = 0;
                for (int tile = first_tile; tile < tiles && ok; tile += step) {
                    const int nt = tile / p.mt, mt = tile - nt * p.mt;
                    for (int kb = kb0; kb < kb1; ++kb) {
                        if (!mbar_wait(empty(st.i), st.ph ^ 1u, abort_flag)) { fail(); break; }
                        mbar_expect_tx(full(st.i), stage_bytes);
                        const uint32_t dst = base + (uint32_t)st.i * stage_bytes;
                        tma_load_2d(dst, &wmap, kb * F8_KB, nt * F8_TN, full(st.i));
                        tma_load_2d(dst + F8_TN * F8_KB, &xmap, kb * F8_KB, mt * BN, full(st.i));
                        st.next(S);
                        ++issued;
                    }
                }
                // every copy has landed before the CTA leaves (after a failure too)
                for (int64_t j = issued < S ? issued : S; j > 0; --j) {
                    const int i = st.i >= j ? st.i - (int)j : st.i - (int)j + S;
                    const uint32_t ph = st.i >= j ? st.ph : st.ph ^ 1u;
                    for (uint32_t n = 0; n < (1u << 20) && !mbar_try_wait(full(i), ph); ++n) {}
                }
            }
        } else if (warp == 2) {
            // scales of a stage: xs[m][kb] * ws[nt][kb], several k-blocks' loads in flight at once
            constexpr int SN = NB * (PW / 4), SL = (SN + 31) / 32, SB = SL > 4 ? 2 : 4;
            Ring st{};
            for (int tile = first_tile; tile < tiles && ok; tile += step) {
                const int nt = tile / p.mt, mt = tile - nt * p.mt;
                for (int kb = kb0; kb < kb1 && ok; kb += SB) {
                    float v[SB][SL];
#pragma unroll
                    for (int b = 0; b < SB; ++b) {
                        const bool live = kb + b < kb1;
                        const float w = live ? p.ws[(int64_t)nt * p.KB + kb + b] : 0.0f;
#pragma unroll
                        for (int i = 0; i < SL; ++i) {
                            const int j = lane + 32 * i, m = mt * BN + j;
                            v[b][i] = live && j < BN && m < p.M ? p.xs[(int64_t)m * p.KB + kb + b] * w : 0.0f;
                        }
                    }
#pragma unroll
                    for (int b = 0; b < SB; ++b) {
                        if (kb + b >= kb1) break;
                        if (!__all_sync(0xffffffffu, mbar_wait(empty(st.i), st.ph ^ 1u, abort_flag))) { fail(); break; }
                        float *sc = reinterpret_cast<float *>(sbase + p.off_sc) + st.i * SN;
#pragma unroll
                        for (int i = 0; i < SL; ++i)
                            if (lane + 32 * i < SN) sc[lane + 32 * i] = v[b][i];
                        __syncwarp();
                        if (lane == 0) mbar_arrive(sc_full(st.i));
                        st.next(S);
                    }
                }
            }
        } else if (warp == 1) {
            if (lane == 0) {
                const uint32_t idesc = idesc_f8(F8_TN, BN);
                const uint64_t a_desc = smem_desc_sw128(base), b_desc = smem_desc_sw128(base + F8_TN * F8_KB);
                Ring st{}, ab{};
                for (int tile = first_tile; tile < tiles && ok; tile += step) {
                    for (int kb = kb0; kb < kb1; ++kb) {
                        if (!mbar_wait(acc_empty(ab.i), ab.ph ^ 1u, abort_flag) || !mbar_wait(full(st.i), st.ph, abort_flag)) {
                            fail();
                            break;
                        }
                        tc_fence_after();
                        const uint64_t off = (uint64_t)st.i * (stage_bytes >> 4);
                        const uint32_t d = tmem + (uint32_t)ab.i * p.buf_cols;
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            tc_mma_f8(d, a_desc + off + 2 * j, b_desc + off + 2 * j, idesc, j > 0 ? 1u : 0u);
                        tc_commit(empty(st.i));
                        tc_commit(acc_full(ab.i));
                        st.next(S);
                        ab.next(NBUF);
                    }
                }
                // every MMA issued has completed before the CTA moves on
                tc_commit(drain);
                if (!mbar_wait(drain, 0, abort_flag)) fail();
            }
        }
        if (p.split > 1) {
            cluster_sync();
            cluster_sync();
        }
    } else {
        const int q = warp & 3, half = (warp - 4) >> 2;
        const int c0 = half * NB;                       // first column of this thread
        constexpr int W = PW == 4 ? 16 : 32, NJ = NB / W;   // columns per load, loads per k-block
        float acc[NB];
        Ring st{}, ab{};
        for (int tile = first_tile; tile < tiles && ok; tile += step) {
            const int nt = tile / p.mt, mt = tile - nt * p.mt;
#pragma unroll
            for (int i = 0; i < NB; ++i) acc[i] = 0.0f;
            // W columns at a time, the next ones on their way while these are added (columns from BN on hold whatever was there; they are not stored)
            float v[2][W];
            auto ready = [&]() {                       // the k-block at (st, ab): its scales and sums
                // (the stage cannot be refilled before this warp arrives on it, so its phase is
                // still the one to wait for)
                if (!__all_sync(0xffffffffu, mbar_wait(sc_full(st.i), st.ph, abort_flag) &&
                                                 mbar_wait(acc_full(ab.i), ab.ph, abort_flag))) { fail(); return false; }
                tc_fence_after();
                return true;
            };
            auto load = [&](int j, float (&to)[W]) {
                const uint32_t ta = tmem + ((uint32_t)(32 * q) << 16) + (uint32_t)ab.i * p.buf_cols + (uint32_t)(c0 + W * j);
                if constexpr (W == 16) tc_ld16(ta, to);
                else tc_ld32(ta, to);
            };
            if (!ready()) break;
            load(0, v[0]);
            const int nkb = kb1 - kb0;
            for (int kb = 0; kb < nkb && ok; ++kb) {
                const float *sc = reinterpret_cast<const float *>(sbase + p.off_sc) + st.i * (NB * (PW / 4)) + c0;
#pragma unroll
                for (int j = 0; j < NJ; ++j) {
                    float (&now)[W] = v[j & 1];
                    tc_wait_ld(now);
                    if (j + 1 < NJ) {
                        load(j + 1, v[(j + 1) & 1]);
                    } else {
                        // all of the accumulator has been read
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(acc_empty(ab.i));
                    }
#pragma unroll
                    for (int i = 0; i < W / 4; ++i) {
                        const float4 s = reinterpret_cast<const float4 *>(sc + W * j)[i];
                        acc[W * j + 4 * i] = fmaf(now[4 * i], s.x, acc[W * j + 4 * i]);
                        acc[W * j + 4 * i + 1] = fmaf(now[4 * i + 1], s.y, acc[W * j + 4 * i + 1]);
                        acc[W * j + 4 * i + 2] = fmaf(now[4 * i + 2], s.z, acc[W * j + 4 * i + 2]);
                        acc[W * j + 4 * i + 3] = fmaf(now[4 * i + 3], s.w, acc[W * j + 4 * i + 3]);
                    }
                }
                // (the scales have been used)
                __syncwarp();
                if (lane == 0) mbar_arrive(empty(st.i));
                st.next(S);
                ab.next(NBUF);
                if (kb + 1 < nkb && ready()) load(0, v[0]);
            }
            if (p.split == 1 && ok) {
                const int n = nt * F8_TN + 32 * q + lane;
                T *y = static_cast<T *>(p.y) + n;
#pragma unroll
                for (int j = 0; j < NB; ++j) {
                    const int m = mt * BN + c0 + j;
                    if (c0 + j < BN && m < p.M && n < p.N) y[(int64_t)m * p.ldy] = from_f32<T>(acc[j]);
                }
            }
        }
        if (p.split > 1) {
            // column j of the tile belongs to the cluster's CTA j / cols, which receives every
            // CTA's partial sums in its stage memory (each CTA has drained its copies and MMAs
            // when it passes the first barrier) and adds them in CTA order
            const int cols = (BN + p.split - 1) / p.split;
            const int nt = first_tile / p.mt, mt = first_tile - nt * p.mt;
            cluster_sync();
#pragma unroll
            for (int j = 0; j < NB; ++j) {
                const int col = c0 + j;
                if (col < BN) {
                    const int to = col / cols;
                    st_cluster(base + 4u * (uint32_t)((rank * cols + (col - to * cols)) * F8_TN + 32 * q + lane),
                               (uint32_t)to, acc[j]);
                }
            }
            cluster_sync();
            const float *part = reinterpret_cast<const float *>(sbase);
            const int mine = min(cols, BN - rank * cols);
            for (int e = tid - 128; e < mine * F8_TN; e += 32 * PW) {
                const int j = e / F8_TN, r = e - j * F8_TN;
                float v = 0.0f;
                for (int s = 0; s < p.split; ++s) v += part[(s * cols + j) * F8_TN + r];
                const int m = mt * BN + rank * cols + j, n = nt * F8_TN + r;
                if (m < p.M && n < p.N) static_cast<T *>(p.y)[(int64_t)m * p.ldy + n] = from_f32<T>(v);
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == 1) {
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(p.tmem_cols) : "memory");
    }
}

// ---- two CTAs on one tile ----------------------------------------------------------------

constexpr int F8P_T = 256;                 // rows of x and of w per tile
constexpr int F8P_STAGES = 6;
constexpr uint32_t F8P_STAGE = 2 * 128 * F8_KB;      // one CTA's bytes of a stage: 128 rows of x, 128 of w
constexpr uint32_t F8P_SC = F8P_STAGES * F8P_STAGE;  // scales: 256 floats a stage
constexpr int F8P_PITCH = 129;             // floats between columns of the split exchange: no bank conflicts either way
constexpr uint32_t F8P_BAR = F8P_SC + F8P_STAGES * 1024;
constexpr size_t F8P_SMEM = 1024 + F8P_BAR + 8 * (3 * F8P_STAGES + 4 + 1) + 16;

__device__ __forceinline__ void tma_load_pair(uint32_t dst, const CUtensorMap *map, int32_t x, int32_t y, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2"
                 " [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(bar) : "memory");
}
__device__ __forceinline__ void tc_mma_f8_pair(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\t"
                 "setp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// arrives on the barrier at this offset in the CTAs of `mask`
__device__ __forceinline__ void tc_commit_pair(uint32_t bar, uint16_t mask) {
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 ::"r"(bar), "h"(mask) : "memory");
}
// (no .release.cluster: what it would order, the tensor-memory loads, has completed, and its
// fence cost more than all of the promotion: 844 against 522 us at 2048 x 28672 x 8192)
__device__ __forceinline__ void mbar_arrive_at(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// Each pair of a cluster: its even rank leads (it issues the MMAs of both).  The leader's `full`
// barrier counts both CTAs' copies; commits arrive in both CTAs; both CTAs' promotion warps
// free an accumulator on the leader's acc_empty.  Registers: 4 x 32 x 56 + 8 x 32 x 224 = 384 x 168.
template <typename T, bool SPLIT>
__global__ void __launch_bounds__(384, 1)
fp8_gemm_pair_kernel(const F8Params p, const __grid_constant__ CUtensorMap wmap, const __grid_constant__ CUtensorMap xmap) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t *sbase = smem_raw + (base - raw);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    constexpr int S = F8P_STAGES;
    const uint32_t bars = base + F8P_BAR;
    auto full = [&](int i) { return bars + 8u * i; };                 // both CTAs' bytes (the leader's)
    auto sc_full = [&](int i) { return bars + 8u * (S + i); };        // scale loader
    auto empty = [&](int i) { return bars + 8u * (2 * S + i); };      // commit + promotion warps
    auto acc_full = [&](int b) { return bars + 8u * (3 * S + b); };       // commit
    auto acc_empty = [&](int b) { return bars + 8u * (3 * S + 2 + b); };  // both CTAs' promotion warps (the leader's)
    const uint32_t drain = bars + 8u * (3 * S + 4);
    uint8_t *misc = sbase + F8P_BAR + 8 * (3 * S + 5);
    volatile uint32_t *tmem_slot = reinterpret_cast<volatile uint32_t *>(misc);
    volatile int *abort_flag = reinterpret_cast<volatile int *>(misc + 4);
    const uint32_t crank = cluster_rank(), rank = crank & 1, leader = SPLIT ? crank & ~1u : 0u;
    const uint16_t both = (uint16_t)(3u << leader);

    if (tid == 0) {
        for (int i = 0; i < S; ++i) { mbar_init(full(i), 1); mbar_init(sc_full(i), 1); mbar_init(empty(i), 1 + 8); }
        for (int i = 0; i < 2; ++i) { mbar_init(acc_full(i), 1); mbar_init(acc_empty(i), 16); }
        mbar_init(drain, 1);
        *abort_flag = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32((const void *)tmem_slot)), "r"(512u) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();                       // every CTA's barriers stand
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    dependency_trigger();
    dependency_wait();

    const int split = SPLIT ? p.split : 1;
    const int tiles = p.mt * p.nt, step = gridDim.x / (2 * split), first_tile = blockIdx.x / (2 * split);
    const int part = SPLIT ? (int)(crank >> 1) : 0;   // this pair's share of k
    const int kb0 = SPLIT ? (int)((int64_t)p.KB * part / split) : 0, kb1 = SPLIT ? (int)((int64_t)p.KB * (part + 1) / split) : p.KB;
    bool ok = true;
    auto fail = [&]() {
        ok = false;
        *abort_flag = 1;
        atomicExch(p.err, Q35_ERR_TIMEOUT);
    };

    if (warp < 4) {
        regs_down<56>();
        if (warp == 0 && lane == 0) {
            Ring st{};
            for (int tile = first_tile; tile < tiles && ok; tile += step) {
                const int nt = tile / p.mt, mt = tile - nt * p.mt;
                for (int kb = kb0; kb < kb1; ++kb) {
                    if (!mbar_wait(empty(st.i), st.ph ^ 1u, abort_flag)) { fail(); break; }
                    if (rank == 0) mbar_expect_tx(full(st.i), 2 * F8P_STAGE);
                    const uint32_t dst = base + (uint32_t)st.i * F8P_STAGE, bar = at_rank(full(st.i), leader);
                    tma_load_pair(dst, &xmap, kb * F8_KB, mt * F8P_T + 128 * (int)rank, bar);
                    tma_load_pair(dst + 128 * F8_KB, &wmap, kb * F8_KB, nt * F8P_T + 128 * (int)rank, bar);
                    st.next(S);
                }
            }
            // (every copy has landed when the leader's MMAs have: see the end)
        } else if (warp == 2) {
            // xs[m][kb] * ws[nb][kb] for this CTA's 128 rows and the tile's two blocks of w's rows
            constexpr int SB = 2;
            const int wb = (p.N + F8_TN - 1) / F8_TN;
            Ring st{};
            for (int tile = first_tile; tile < tiles && ok; tile += step) {
                const int nt = tile / p.mt, mt = tile - nt * p.mt;
                const int n1 = min(2 * nt + 1, wb - 1);
                for (int kb = kb0; kb < kb1 && ok; kb += SB) {
                    float v[SB][4], w[SB][2];
#pragma unroll
                    for (int b = 0; b < SB; ++b) {
                        const bool live = kb + b < kb1;
                        w[b][0] = live ? p.ws[(int64_t)(2 * nt) * p.KB + kb + b] : 0.0f;
                        w[b][1] = live ? p.ws[(int64_t)n1 * p.KB + kb + b] : 0.0f;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            const int m = mt * F8P_T + 128 * (int)rank + lane + 32 * i;
                            v[b][i] = live && m < p.M ? p.xs[(int64_t)m * p.KB + kb + b] : 0.0f;
                        }
                    }
#pragma unroll
                    for (int b = 0; b < SB; ++b) {
                        if (kb + b >= kb1) break;
                        if (!__all_sync(0xffffffffu, mbar_wait(empty(st.i), st.ph ^ 1u, abort_flag))) { fail(); break; }
                        float *sc = reinterpret_cast<float *>(sbase + F8P_SC) + st.i * 256;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            sc[lane + 32 * i] = v[b][i] * w[b][0];
                            sc[128 + lane + 32 * i] = v[b][i] * w[b][1];
                        }
                        __syncwarp();
                        if (lane == 0) mbar_arrive(sc_full(st.i));
                        st.next(S);
                    }
                }
            }
        } else if (warp == 1 && lane == 0) {
            if (rank == 0) {
                const uint32_t idesc = idesc_f8(F8P_T, F8P_T);
                const uint64_t a_desc = smem_desc_sw128(base), b_desc = smem_desc_sw128(base + 128 * F8_KB);
                Ring st{}, ab{};
                for (int tile = first_tile; tile < tiles && ok; tile += step) {
                    for (int kb = kb0; kb < kb1; ++kb) {
                        if (!mbar_wait(full(st.i), st.ph, abort_flag) || !mbar_wait(acc_empty(ab.i), ab.ph ^ 1u, abort_flag)) {
                            fail();
                            break;
                        }
                        tc_fence_after();
                        const uint64_t off = (uint64_t)st.i * (F8P_STAGE >> 4);
                        const uint32_t d = tmem + (uint32_t)ab.i * 256u;
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            tc_mma_f8_pair(d, a_desc + off + 2 * j, b_desc + off + 2 * j, idesc, j > 0 ? 1u : 0u);
                        tc_commit_pair(acc_full(ab.i), both);
                        tc_commit_pair(empty(st.i), both);
                        st.next(S);
                        ab.next(2);
                    }
                }
                tc_commit_pair(drain, both);
            }
            // every MMA has completed, so every copy it read has landed, in both CTAs
            if (!mbar_wait(drain, 0, abort_flag)) fail();
        }
        if (SPLIT) {
            cluster_sync();
            cluster_sync();
        }
    } else {
        regs_up<224>();
        const int q = warp & 3, half = (warp - 4) >> 2;
        float acc[128];
        Ring st{}, ab{};
        for (int tile = first_tile; tile < tiles && ok; tile += step) {
            const int nt = tile / p.mt, mt = tile - nt * p.mt;
#pragma unroll
            for (int i = 0; i < 128; ++i) acc[i] = 0.0f;
            // 32 columns at a time; the next ones (of the next k-block too) are on their way
            // while these are added
            float v[2][32], s = 0.0f;
            auto ready = [&]() {                       // the k-block at (st, ab): its scale and sums
                if (!__all_sync(0xffffffffu, mbar_wait(sc_full(st.i), st.ph, abort_flag) &&
                                                 mbar_wait(acc_full(ab.i), ab.ph, abort_flag))) { fail(); return false; }
                tc_fence_after();
                return true;
            };
            auto columns = [&](int j) { return tmem + ((uint32_t)(32 * q) << 16) + (uint32_t)ab.i * 256u + (uint32_t)(half * 128 + 32 * j); };
            if (!ready()) break;
            tc_ld32(columns(0), v[0]);
            for (int kb = kb0; kb < kb1 && ok; ++kb) {
                s = reinterpret_cast<const float *>(sbase + F8P_SC)[st.i * 256 + half * 128 + 32 * q + lane];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    tc_wait_ld(v[j & 1]);
                    if (j < 3) {
                        tc_ld32(columns(j + 1), v[(j + 1) & 1]);
                    } else {
                        // all of the accumulator has been read
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) { mbar_arrive_at(at_rank(acc_empty(ab.i), leader)); mbar_arrive(empty(st.i)); }
                        st.next(S);
                        ab.next(2);
                        if (kb + 1 < kb1 && ready()) tc_ld32(columns(0), v[0]);
                    }
#pragma unroll
                    for (int i = 0; i < 32; ++i) acc[32 * j + i] = fmaf(v[j & 1][i], s, acc[32 * j + i]);
                }
            }
            if (!ok || SPLIT) break;
            const int m = mt * F8P_T + 128 * (int)rank + 32 * q + lane, n0 = nt * F8P_T + 128 * half;
            if (m < p.M) {
                T *y = static_cast<T *>(p.y) + (int64_t)m * p.ldy + n0;
                constexpr int V = 16 / sizeof(T);
                if (n0 + 128 <= p.N && (reinterpret_cast<uintptr_t>(y) & 15) == 0) {
#pragma unroll
                    for (int j = 0; j < 128; j += V) {
                        uint4 u;
                        if constexpr (sizeof(T) == 4)
                            u = make_uint4(__float_as_uint(acc[j]), __float_as_uint(acc[j + 1]), __float_as_uint(acc[j + 2]),
                                           __float_as_uint(acc[j + 3]));
                        else
                            u = make_uint4(pack2<T>(acc[j], acc[j + 1]), pack2<T>(acc[j + 2], acc[j + 3]),
                                           pack2<T>(acc[j + 4], acc[j + 5]), pack2<T>(acc[j + 6], acc[j + 7]));
                        *reinterpret_cast<uint4 *>(y + j) = u;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 128; ++j)
                        if (n0 + j < p.N) y[j] = from_f32<T>(acc[j]);
                }
            }
        }
        if (SPLIT) {
            // column c of the tile belongs to pair c / cols of the cluster; its CTA of this one's
            // parity receives the sums of every pair in its stage memory (each CTA has drained its
            // copies and MMAs when it passes the first barrier) and adds them in pair order
            const int cols = (F8P_T + split - 1) / split;
            const int nt = first_tile / p.mt, mt = first_tile - nt * p.mt;
            cluster_sync();
#pragma unroll
            for (int j = 0; j < 128; ++j) {
                const int col = 128 * half + j, to = col / cols;
                st_cluster(base + 4u * (uint32_t)((part * cols + (col - to * cols)) * F8P_PITCH + 32 * q + lane),
                           2u * (uint32_t)to + rank, acc[j]);
            }
            cluster_sync();
            const float *sums = reinterpret_cast<const float *>(sbase);
            const int mine = min(cols, F8P_T - part * cols);
            for (int r = warp - 4; r < 128; r += 8) {
                const int m = mt * F8P_T + 128 * (int)rank + r;
                if (m >= p.M) break;
                for (int j = lane; j < mine; j += 32) {
                    float v = 0.0f;
                    for (int s = 0; s < split; ++s) v += sums[(s * cols + j) * F8P_PITCH + r];
                    const int n = nt * F8P_T + part * cols + j;
                    if (n < p.N) static_cast<T *>(p.y)[(int64_t)m * p.ldy + n] = from_f32<T>(v);
                }
            }
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    cluster_sync();                       // no CTA leaves while another may arrive on its barriers
    tc_fence_after();
    if (warp == 1) {
        __syncwarp();
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512u) : "memory");
    }
}

// ---- host side -------------------------------------------------------------------------

using EncodeFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                              const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                              CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

// the driver entry point, looked up through the runtime (as in q35_mma.cu)
int tma_encoder(EncodeFn *out) {
    static EncodeFn encode = nullptr;
    if (!encode) {
        void *fn = nullptr;
        cudaDriverEntryPointQueryResult q = cudaDriverEntryPointSymbolNotFound;
        cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q);
        if (e != cudaSuccess || q != cudaDriverEntryPointSuccess || !fn)
            return set_error(Q35_ERR_CUDA, "fp8_gemm: cuTensorMapEncodeTiled not available");
        encode = reinterpret_cast<EncodeFn>(fn);
    }
    *out = encode;
    return Q35_OK;
}

int byte_map(EncodeFn encode, CUtensorMap *map, const void *p, int64_t rows, int64_t K, int64_t ld, int box_rows) {
    const cuuint64_t dims[2] = {(cuuint64_t)K, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)ld};
    const cuuint32_t box[2] = {(cuuint32_t)F8_KB, (cuuint32_t)box_rows};
    const cuuint32_t estr[2] = {1u, 1u};
    CUresult cr = encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void *>(p), dims, strides, box, estr,
                         CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                         CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return cr == CUDA_SUCCESS ? Q35_OK : set_error(Q35_ERR_CUDA, "fp8_gemm: cuTensorMapEncodeTiled failed");
}

struct F8Plan {
    bool pair = false;
    int NB, PW, BN, mt, nt, split, stages, bufs, grid;
    uint32_t tmem_cols, buf_cols, off_sc, off_bar;
    size_t smem;
};

F8Plan plan_f8(int32_t M, int32_t N, int32_t KB) {
    constexpr int SMS = 148;
    F8Plan pl{};
    if (M > 128) {
        // two CTAs per tile; few tiles are split so that every pair of SMs has work, at least
        // four k-blocks each
        pl.pair = true;
        pl.mt = (int)ceil_div(M, F8P_T);
        pl.nt = (int)ceil_div(N, F8P_T);
        const int64_t tiles = (int64_t)pl.mt * pl.nt;
        pl.split = (int)std::max<int64_t>(1, std::min<int64_t>({4, KB / 4, SMS / 2 / tiles}));
        pl.grid = pl.split > 1 ? (int)tiles * 2 * pl.split : (int)std::min<int64_t>(2 * tiles, SMS);
        pl.BN = 128;
        return pl;
    }
    pl.mt = 1;
    pl.BN = (int)round_up(M, 16);
    pl.nt = (int)ceil_div(N, F8_TN);
    pl.PW = pl.BN <= 32 ? 4 : 8;
    pl.NB = pl.BN <= 16 ? 16 : pl.BN <= 64 ? 32 : 64;
    const int tiles = pl.mt * pl.nt;
    const int per_sm = pl.PW == 4 ? 2 : 1;
    // as many CTAs per tile as give every slot one, at least four k-blocks each
    pl.split = std::max(1, std::min({8, KB / 4, per_sm * SMS / tiles}));
    pl.grid = pl.split > 1 ? tiles * pl.split : std::min(tiles, per_sm * SMS);
    pl.buf_cols = (uint32_t)(pl.NB * (pl.PW / 4));
    pl.bufs = std::min<int>(8, 512 / per_sm / pl.buf_cols);
    pl.tmem_cols = 32;
    while (pl.tmem_cols < pl.bufs * pl.buf_cols) pl.tmem_cols *= 2;
    const size_t stage = (size_t)(F8_TN + pl.BN) * F8_KB, sc = pl.buf_cols * 4;
    const size_t budget = (227 * 1024 - (per_sm - 1) * 1024) / per_sm - 1024 - 512;
    pl.stages = (int)std::min<size_t>(16, budget / (stage + sc));
    // the split exchange reuses the stages: split * ceil(BN / split) columns of 128 floats
    pl.off_sc = (uint32_t)(pl.stages * stage);
    pl.off_bar = (uint32_t)round_up((int64_t)(pl.off_sc + pl.stages * sc), 8);
    pl.smem = 1024 + pl.off_bar + 8 * (3 * pl.stages + 2 * pl.bufs + 1) + 16;
    return pl;
}

template <typename T, int NB, int PW>
int launch_f8(const F8Params &p, const F8Plan &pl, const CUtensorMap &wm, const CUtensorMap &xm, int dev, cudaStream_t s) {
    auto kern = fp8_gemm_kernel<T, NB, PW>;
    static bool configured[64] = {};
    if (!configured[dev]) {
        Q35_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, 227 * 1024));
        configured[dev] = true;
    }
    Q35_CUDA_TRY(launch_dependent(kern, dim3((unsigned)pl.grid), 128 + 32 * PW, pl.smem, s, pl.split, p, wm, xm));
    return Q35_OK;
}

template <typename T, bool SPLIT>
int launch_f8_pair(const F8Params &p, const F8Plan &pl, const CUtensorMap &wm, const CUtensorMap &xm, int dev, cudaStream_t s) {
    auto kern = fp8_gemm_pair_kernel<T, SPLIT>;
    static bool configured[64] = {};
    if (!configured[dev]) {
        Q35_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)F8P_SMEM));
        configured[dev] = true;
    }
    Q35_CUDA_TRY(launch_dependent(kern, dim3((unsigned)pl.grid), 384, F8P_SMEM, s, 2 * pl.split, p, wm, xm));
    return Q35_OK;
}

template <typename T>
int launch_f8(const F8Params &p, const F8Plan &pl, const CUtensorMap &wm, const CUtensorMap &xm, int dev, cudaStream_t s) {
    if (pl.pair)
        return pl.split > 1 ? launch_f8_pair<T, true>(p, pl, wm, xm, dev, s) : launch_f8_pair<T, false>(p, pl, wm, xm, dev, s);
    if (pl.NB == 16) return launch_f8<T, 16, 4>(p, pl, wm, xm, dev, s);
    if (pl.PW == 4) return launch_f8<T, 32, 4>(p, pl, wm, xm, dev, s);
    return pl.NB == 32 ? launch_f8<T, 32, 8>(p, pl, wm, xm, dev, s) : launch_f8<T, 64, 8>(p, pl, wm, xm, dev, s);
}

}  // namespace
}  // namespace q35

using namespace q35;

extern "C" int q35_fp8_gemm_dev(q35_ctx ctx, const void *x, int64_t ldx, const float *x_scales, const void *w,
                                int64_t ldw, const float *w_scales, int dtype, void *y, int64_t ldy, int32_t M,
                                int32_t N, int32_t K) {
    if (!ctx) return set_error(Q35_ERR_INVALID, "fp8_gemm: ctx is NULL");
    int st = check_dtype(dtype);
    if (st) return st;
    if (M < 0 || M > GEMM_MAX_M) return set_error(Q35_ERR_INVALID, "fp8_gemm: M must be in [0,65536]");
    if (N < 0 || N > (1 << 24)) return set_error(Q35_ERR_INVALID, "fp8_gemm: N must be in [0,2^24]");
    if (K < 1 || K > GEMM_MAX_K) return set_error(Q35_ERR_INVALID, "fp8_gemm: K must be in [1,131072]");
    if (M == 0 || N == 0) return Q35_OK;
    if (!x || !x_scales || !w || !w_scales || !y) return set_error(Q35_ERR_INVALID, "fp8_gemm: NULL argument");
    if (ldx < K || ldw < K || ldy < N) return set_error(Q35_ERR_INVALID, "fp8_gemm: a row stride is below the row's length");
    if (ldx % 16 || ldw % 16 || !aligned_to(x, 16) || !aligned_to(w, 16))
        return set_error(Q35_ERR_INVALID, "fp8_gemm: rows of x and w must start on 16-byte boundaries");
    if (!aligned_to(x_scales, 4) || !aligned_to(w_scales, 4) || !aligned_to(y, dtype_size(dtype)))
        return set_error(Q35_ERR_INVALID, "fp8_gemm: a pointer is not aligned to its elements");
    if (ctx->device < 0 || ctx->device >= 64) return set_error(Q35_ERR_INVALID, "fp8_gemm: device ordinal out of range");
    DeviceGuard g(ctx->device);
    st = ensure_workspace(ctx, 0, 0);
    if (st) return st;
    EncodeFn encode = nullptr;
    st = tma_encoder(&encode);
    if (st) return st;
    const int KB = (int)ceil_div(K, F8_KB);
    const F8Plan pl = plan_f8(M, N, KB);
    CUtensorMap wm, xm;
    st = byte_map(encode, &wm, w, N, K, ldw, F8_TN);
    if (!st) st = byte_map(encode, &xm, x, M, K, ldx, pl.BN);
    if (st) return st;
    F8Params p;
    p.xs = x_scales; p.ws = w_scales;
    p.y = y; p.ldy = ldy;
    p.M = M; p.N = N; p.KB = KB;
    p.BN = pl.BN; p.mt = pl.mt; p.nt = pl.nt;
    p.split = pl.split; p.stages = pl.stages; p.bufs = pl.bufs;
    p.tmem_cols = pl.tmem_cols; p.buf_cols = pl.buf_cols;
    p.off_sc = pl.off_sc; p.off_bar = pl.off_bar;
    p.err = ctx->ws.err;
    switch (dtype) {
    case Q35_DT_F32: return launch_f8<float>(p, pl, wm, xm, ctx->device, ctx->stream);
    case Q35_DT_BF16: return launch_f8<__nv_bfloat16>(p, pl, wm, xm, ctx->device, ctx->stream);
    default: return launch_f8<__half>(p, pl, wm, xm, ctx->device, ctx->stream);
    }
}
