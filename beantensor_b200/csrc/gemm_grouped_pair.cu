// Two-SM form of the grouped products (gemm_grouped.cu): a tile of a CTA pair is 256 rows x 256 (or 128) columns, one
// tcgen05.mma.cta_group::2 drives both SMs. Each CTA holds 128 rows of A and half of the columns of B, so a 64-deep
// k-block costs it 32 KB of loads instead of 48 KB (450 cycles instead of 670 at 73 B per cycle, for 512 of MMAs), and the
// ring holds half as many k-blocks again. Measured (bf16, 16384 rows, 4096 x 4096): 355 us in eight equal groups (1550 TFLOP/s) and
// 379 in eight uneven ones after a pause, 442 and 470 in a long run under the power cap (1250 and 1170 TFLOP/s at 1.2 GHz); 89 %
// tensor-active. Barriers as in gemm_tc2.cu: full[s] lives in the leader and counts the bytes of both CTAs; empty[s] and tmem_full[a] are signalled in
// both by multicast tcgen05.commit; tmem_empty[a] lives in the leader and collects the sixteen epilogue warps. No TMA
// multicast is used.
//
// Rows of a group are cut into slots of 256; in a group's last slot the second CTA may own no row: it then loads none of
// A and stores nothing.
//
// Products only: the weight gradient was built and measured on pairs too and was level with the one-CTA kernel at best (16384
// rows in 8 groups 505 against 504 us, in 64 groups 221 against 185 us), so it stays there.
#include <cstring>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "btm_internal.h"
#include "btm_ptx.cuh"
#include "grouped_tile.cuh"

namespace btm {

namespace gp {
constexpr int CTA_M = 128;
constexpr int PAIR_M = 256;
constexpr int BN = 256;
constexpr int BK = 64;
constexpr int CHUNK_BYTES = 64 * 128;
constexpr int A_BYTES = CTA_M * 128;
constexpr int KB_BYTES = A_BYTES + 2 * CHUNK_BYTES;
constexpr int KPS = 2; // k-blocks per stage, as in gemm_tc2.cu
constexpr int STAGE_BYTES = KPS * KB_BYTES;
constexpr int STAGES = 3;
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + EPI_SMEM_BYTES + 1024;
constexpr int TMEM_COLS = 512;
constexpr int THREADS = 320; // warp 0 TMA, 1 MMA, 2-9 epilogue
constexpr int A_BAND = 32;
} // namespace gp

template <int DT, int MODE>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(gp::THREADS, 1)
gemm_grouped_pair_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmA_band, const __grid_constant__ CUtensorMap tmB,
                         const __grid_constant__ CUtensorMap tmC, const __grid_constant__ GemmParams p, const GroupedTables tab)
{
    using namespace gp;
    constexpr bool kBMnMajor = MODE != GROUPED_NK;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bar_full[STAGES];   // used in the leader
    __shared__ __align__(8) uint64_t bar_empty[STAGES];  // per CTA
    __shared__ __align__(8) uint64_t bar_tmem_full[2];   // per CTA
    __shared__ __align__(8) uint64_t bar_tmem_empty[2];  // used in the leader
    __shared__ uint32_t tmem_base_holder;
    __shared__ int abort_flag;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = pair_rank(); // 0 = leader
    const int pair_id = blockIdx.x >> 1, num_pairs = gridDim.x >> 1;
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(smem_u32(&bar_full[s]), 1);
            mbar_init(smem_u32(&bar_empty[s]), 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(smem_u32(&bar_tmem_full[a]), 1);
            mbar_init(smem_u32(&bar_tmem_empty[a]), 2 * GROUPED_EPI_WARPS);
        }
        fence_mbar_init();
        prefetch_tmap(&tmA);
        prefetch_tmap(&tmB);
        prefetch_tmap(&tmA_band);
    }
    if (warp == 1) {
        tmem_alloc<2>(smem_u32(&tmem_base_holder), TMEM_COLS);
        tmem_relinquish<2>();
    }
    tc_fence_before();
    __syncthreads();
    pair_sync(); // the other CTA's barriers exist before anything remote can reach them
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_holder;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    GroupWalk<PAIR_M> walk;
    walk.init(tab.offsets, tab.groups, tab.rows);
    const int group_slots = walk.count_slots();
    if (blockIdx.x == 0 && warp == 0) walk.report(p.status);
    const GroupedPlan plan = plan_tiles<BN, 128>(group_slots, p.N, num_pairs);

    // Producer and issuer run as whole warps with uniform control flow; one elected lane issues (mbar_wait_uniform).
    if (warp == 0) {
        // ------------------------------------------------------------ TMA producer (both CTAs)
        int stage = 0;
        uint32_t phase = 0;
        bool ok = !p.debug_skip_loads;
        for (int tile = pair_id; ok && tile < plan.total; tile += num_pairs) {
            const GroupedTile t = grouped_tile_uniform<false, PAIR_M>(p, plan, walk, tile);
            const int half_bn = t.bn >> 1, chunks = half_bn >> 6;
            const int am = t.m0 + (int)rank * CTA_M, bn0 = t.n0 + (int)rank * half_bn;
            // 32-row bands of A that belong to the group, of this CTA and of the pair
            const int pair_bands = min(4, (t.hi - t.m0 + A_BAND - 1) / A_BAND) + min(4, max(0, t.hi - t.m0 - CTA_M + A_BAND - 1) / A_BAND);
            const int bands = min(4, max(0, t.hi - am + A_BAND - 1) / A_BAND);
            const uint32_t kb_bytes = (uint32_t)(pair_bands * A_BAND * 128 + 2 * chunks * CHUNK_BYTES);
            for (int kb = 0; kb < p.num_kb; kb += KPS) {
                ok = mbar_wait_uniform<true>(smem_u32(&bar_empty[stage]), phase ^ 1u, &abort_flag, p.status, WAIT_PRODUCER_EMPTY, p.wait_limit);
                if (!ok) break;
                const int nsub = min(KPS, p.num_kb - kb);
                if (elect_one()) {
                    const uint32_t full_local = smem_u32(&bar_full[stage]), full = map_to_leader(full_local);
                    if (rank == 0) mbar_expect_tx(full_local, kb_bytes * (uint32_t)nsub);
#pragma unroll
                    for (int sub = 0; sub < KPS; ++sub) {
                        if (sub < nsub) {
                            const uint32_t a0 = smem_base + stage * STAGE_BYTES + sub * KB_BYTES, b0 = a0 + A_BYTES;
                            const int k0 = (kb + sub) * BK;
                            if (bands == 4) {
                                tma_load_3d_2sm(a0, &tmA, k0, am, 0, full);
                            } else {
                                for (int b = 0; b < bands; ++b) tma_load_3d_2sm(a0 + b * A_BAND * 128, &tmA_band, k0, am + b * A_BAND, 0, full);
                            }
#pragma unroll
                            for (int c = 0; c < BN / 128; ++c) {
                                if (c < chunks) {
                                    if (kBMnMajor) tma_load_3d_2sm(b0 + c * CHUNK_BYTES, &tmB, bn0 + c * 64, k0, t.g, full);
                                    else tma_load_3d_2sm(b0 + c * CHUNK_BYTES, &tmB, k0, bn0 + c * 64, t.g, full);
                                }
                            }
                        }
                    }
                }
                __syncwarp();
                if (++stage == STAGES) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
    } else if (warp == 1 && rank == 0) {
        // ------------------------------------------------------------ MMA issuer (leader)
        constexpr uint32_t kFmt = DT == BTM_BF16 ? 1u : 0u;
        constexpr uint32_t a_step = 32 >> 4, b_step = (kBMnMajor ? 16 * 128 : 32) >> 4;
        const uint32_t tmem_u = uniform(tmem_base);
        int stage = 0, it = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int tile = pair_id; ok && tile < plan.total; tile += num_pairs, ++it) {
            const GroupedTile t = grouped_tile_uniform<false, PAIR_M>(p, plan, walk, tile);
            const uint32_t idesc = make_idesc(kFmt, false, kBMnMajor, PAIR_M, (uint32_t)t.bn);
            const int acc = it & 1;
            const uint32_t d_tmem = tmem_u + (uint32_t)(acc * BN);
            ok = mbar_wait_uniform<true>(smem_u32(&bar_tmem_empty[acc]), ((uint32_t)(it >> 1) & 1u) ^ 1u, &abort_flag, p.status, WAIT_MMA_TMEM_EMPTY, p.wait_limit);
            tc_fence_after();
            for (int kb = 0; ok && kb < p.num_kb; kb += KPS) {
                ok = mbar_wait_uniform<true>(smem_u32(&bar_full[stage]), phase, &abort_flag, p.status, WAIT_MMA_FULL, p.wait_limit);
                if (!ok) break;
                tc_fence_after();
                const int nsub = min(KPS, p.num_kb - kb);
                const uint32_t a0 = smem_base + stage * STAGE_BYTES, b0 = a0 + A_BYTES;
                const uint64_t ad = make_smem_desc_sw128(a0, 16, 1024);
                const uint64_t bd = kBMnMajor ? make_smem_desc_sw128(b0, CHUNK_BYTES, 1024) : make_smem_desc_sw128(b0, 16, 1024);
                if (elect_one()) {
#pragma unroll
                    for (int sub = 0; sub < KPS; ++sub) {
                        if (sub < nsub) {
#pragma unroll
                            for (int ks = 0; ks < BK / 16; ++ks)
                                umma<2, false>(d_tmem, ad + (uint64_t)((sub * KB_BYTES >> 4) + ks * a_step), bd + (uint64_t)((sub * KB_BYTES >> 4) + ks * b_step),
                                               idesc, (uint32_t)((kb | sub | ks) != 0));
                        }
                    }
                    umma_commit_2sm(smem_u32(&bar_empty[stage]), (uint16_t)3);
                }
                __syncwarp();
                if (++stage == STAGES) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            if (ok && elect_one()) umma_commit_2sm(smem_u32(&bar_tmem_full[acc]), (uint16_t)3);
            __syncwarp();
        }
    } else if (warp >= 2) {
        // ------------------------------------------------------------ epilogue (both CTAs, own 128 rows)
        const int quad = warp & 3;
        const uint32_t epi_smem = smem_base + STAGES * STAGE_BYTES + (uint32_t)(warp - 2) * EPI_TILE_BYTES;
        int it = 0;
        for (int tile = pair_id; tile < plan.total; tile += num_pairs, ++it) {
            const GroupedTile t = grouped_tile<false, PAIR_M>(p, plan, walk, tile);
            const int acc = it & 1;
            if (!mbar_wait_uniform<true>(smem_u32(&bar_tmem_full[acc]), (uint32_t)(it >> 1) & 1u, &abort_flag, p.status, WAIT_EPI_TMEM_FULL, p.wait_limit)) break;
            tc_fence_after();
            grouped_band<DT, false>(p, tmC, tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(acc * BN), t,
                                     t.m0 + (int)rank * CTA_M + quad * 32, t.hi, false, epi_smem, (warp - 2) >> 2, lane);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) {
                if (rank == 0) mbar_arrive(smem_u32(&bar_tmem_empty[acc]));
                else mbar_arrive_cluster(smem_u32(&bar_tmem_empty[acc]), 0);
            }
        }
        epilogue_drain(lane);
    }

    // ---------------------------------------------------------------- teardown
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (abort_flag) {
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) {}
        __syncthreads();
    }
    pair_sync(); // neither CTA leaves while the other may still touch its shared memory
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc<2>(tmem_base, TMEM_COLS);
    }
}

template <int DT, int MODE>
static int launch_pair_mode(const GroupedCall &c, cudaStream_t st, int sm_count, const CUtensorMap &tmA, const CUtensorMap &tmA_band,
                            const CUtensorMap &tmB, const CUtensorMap &tmC, const GemmParams &p)
{
    using namespace gp;
    // How many pairs the device holds at once (GPC boundaries can make it less than SMs / 2).
    static std::atomic<int> resident[64];
    int dev = 0;
    cudaGetDevice(&dev);
    int pairs = dev >= 0 && dev < 64 ? resident[dev].load(std::memory_order_relaxed) : 0;
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.blockDim = dim3(THREADS, 1, 1);
    cfg.dynamicSmemBytes = SMEM_BYTES;
    cfg.stream = st;
    if (pairs == 0) {
        cfg.gridDim = dim3((unsigned)(sm_count & ~1), 1, 1);
        cudaLaunchAttribute cl;
        cl.id = cudaLaunchAttributeClusterDimension;
        cl.val.clusterDim.x = 2;
        cl.val.clusterDim.y = 1;
        cl.val.clusterDim.z = 1;
        cfg.attrs = &cl;
        cfg.numAttrs = 1;
        int n = 0;
        if (cudaOccupancyMaxActiveClusters(&n, gemm_grouped_pair_kernel<DT, MODE>, &cfg) != cudaSuccess || n <= 0) {
            (void)cudaGetLastError();
            n = sm_count / 2;
        }
        pairs = n < sm_count / 2 ? n : sm_count / 2;
        if (dev >= 0 && dev < 64) resident[dev].store(pairs, std::memory_order_relaxed);
    }
    cfg.gridDim = dim3((unsigned)(2 * pairs), 1, 1);
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    const GroupedTables tab = {c.offsets, c.groups, c.rows};
    return check_cuda(cudaLaunchKernelEx(&cfg, gemm_grouped_pair_kernel<DT, MODE>, tmA, tmA_band, tmB, tmC, p, tab), "grouped matmul (pair) launch");
}

int launch_gemm_grouped_pair(const GroupedCall &c, cudaStream_t st, int sm_count, const CUtensorMap &tmA, const CUtensorMap &tmA_band,
                             const CUtensorMap &tmB, const CUtensorMap &tmC, const GemmParams &p)
{
#define BTM_GROUPED_PAIR_CASE(DT)                                                                                             \
    do {                                                                                                                      \
        if (c.b_trans) return launch_pair_mode<DT, GROUPED_NK>(c, st, sm_count, tmA, tmA_band, tmB, tmC, p);                  \
        return launch_pair_mode<DT, GROUPED_KN>(c, st, sm_count, tmA, tmA_band, tmB, tmC, p);                                 \
    } while (0)
    if (c.dtype == BTM_F16) BTM_GROUPED_PAIR_CASE(BTM_F16);
    BTM_GROUPED_PAIR_CASE(BTM_BF16);
#undef BTM_GROUPED_PAIR_CASE
}

template <int DT>
static cudaError_t raise_pair_smem()
{
    cudaError_t e = cudaFuncSetAttribute(gemm_grouped_pair_kernel<DT, GROUPED_KN>, cudaFuncAttributeMaxDynamicSharedMemorySize, gp::SMEM_BYTES);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(gemm_grouped_pair_kernel<DT, GROUPED_NK>, cudaFuncAttributeMaxDynamicSharedMemorySize, gp::SMEM_BYTES);
    return e;
}

int configure_gemm_grouped_pair_kernels()
{
    cudaError_t e = raise_pair_smem<BTM_F16>();
    if (e == cudaSuccess) e = raise_pair_smem<BTM_BF16>();
    return check_cuda(e, "cudaFuncSetAttribute(gemm_grouped_pair)");
}

} // namespace btm
