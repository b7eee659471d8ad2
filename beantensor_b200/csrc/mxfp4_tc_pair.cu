// Two-SM form of the microscaled product (mxfp4_tc.cu): a tile of a CTA pair is 256 rows x 192 (or 128) columns, each CTA
// holds 128 rows of the activations and half of the weight rows, so a 256-deep stage costs it 31 KB of loads instead of 43.
// 8192 x 11008 x 4096: 162 us after a pause (4.6 PFLOP/s), 188 in a long run under the power cap. That is 620 to 630 cycles a stage,
// where the MMAs take 384 and 31 KB of loads at the 73 B per cycle of a loaded machine 435. Which wait makes up the rest is not
// known: no unit is above 67 % (tensor pipe 59 %, its path to memory 60 %, data banks of shared memory 20 % each for reads and
// writes). Measured without effect: the scale copies in a warp of their own, no tile look-up in the MMA issuer.
//
// Every load, scales included, is a tensor-map load whose completion goes to the leader's full[s]; the scale blocks are
// one matrix of 32-bit words (a row block per row), so that both row blocks of the weights come in one box. Issuing a TMA load
// takes a thread 75 to 120 cycles, so operands and scales have a producer warp each. SFB goes to both CTAs' tensor memory:
// each SM computes all 192 columns for its own 128 rows.
// Barriers as in gemm_tc2.cu. Slots of a pair are 256 rows; the scales count slots of 128 (GroupWalk::singles_of).
#include <cstring>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "btm_internal.h"
#include "btm_ptx.cuh"
#include "grouped_tile.cuh"
#include "mxfp4.cuh"

namespace btm {

namespace mxp {
constexpr int CTA_M = 128;
constexpr int PAIR_M = 256;
constexpr int BN = 192;
constexpr int BK = 256;
constexpr int A_BYTES = CTA_M * 128;
constexpr int SFA_AT = A_BYTES + BN / 2 * 128;
constexpr int SFB_AT = SFA_AT + 2 * MX_SCALE_BYTES;
constexpr int STAGE_BYTES = SFB_AT + 4 * MX_SCALE_BYTES; // 31 KB
constexpr int SF_COL = 2 * BN;
constexpr int SF_STAGE_COLS = 24; // A 2 x 4 columns, B 2 x 8
constexpr int STAGES = 5;         // as many as there are columns for their scales
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + EPI_SMEM_BYTES + 1024;
constexpr int TMEM_COLS = 512;
constexpr int THREADS = 352; // warp 0 operands, 1 MMA, 2-9 epilogue, 10 scales
constexpr int A_BAND = 32;
static_assert(SF_COL + STAGES * SF_STAGE_COLS <= TMEM_COLS, "accumulators and scales share tensor memory");
static_assert(STAGE_BYTES % 1024 == 0, "stages start on swizzle atoms");
} // namespace mxp

struct MxPairMaps {
    CUtensorMap a, a_band, b_wide, b_narrow, sfa, sfb, c;
};

template <int DT>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(mxp::THREADS, 1)
mxfp4_gemm_pair_kernel(const __grid_constant__ MxPairMaps maps, const __grid_constant__ GemmParams p, const GroupedTables tab)
{
    using namespace mxp;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bar_full[STAGES];  // used in the leader
    __shared__ __align__(8) uint64_t bar_empty[STAGES]; // per CTA
    __shared__ __align__(8) uint64_t bar_tmem_full[2];  // per CTA
    __shared__ __align__(8) uint64_t bar_tmem_empty[2]; // used in the leader
    __shared__ uint32_t tmem_base_holder;
    __shared__ int abort_flag;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t rank = pair_rank();
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
        prefetch_tmap(&maps.a);
        prefetch_tmap(&maps.a_band);
        prefetch_tmap(&maps.b_wide);
        prefetch_tmap(&maps.b_narrow);
        prefetch_tmap(&maps.sfa);
        prefetch_tmap(&maps.sfb);
    }
    if (warp == 1) {
        tmem_alloc<2>(smem_u32(&tmem_base_holder), TMEM_COLS);
        tmem_relinquish<2>();
    }
    tc_fence_before();
    __syncthreads();
    pair_sync();
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_holder;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    GroupWalk<PAIR_M> walk;
    walk.init(tab.offsets, tab.groups, tab.rows);
    const GroupedPlan plan = plan_tiles<BN, 128>(walk.count_slots(), p.N, num_pairs);
    if (blockIdx.x == 0 && warp == 0) walk.report(p.status);

    if (warp == 0 || warp == 10) {
        // ------------------------------------------------------------ TMA producers (both CTAs): operands, scales
        int stage = 0;
        uint32_t phase = 0;
        bool ok = !p.debug_skip_loads;
        for (int tile = pair_id; ok && tile < plan.total; tile += num_pairs) {
            const GroupedTile t = grouped_tile_uniform<false, PAIR_M>(p, plan, walk, tile);
            const int am = t.m0 + (int)rank * CTA_M, bn0 = t.n0 + (int)rank * (t.bn >> 1);
            // 32-row bands of the activations that belong to the group, of this CTA and of both; without any, no scales
            const int bands0 = min(4, (t.hi - t.m0 + A_BAND - 1) / A_BAND), bands1 = min(4, max(0, t.hi - t.m0 - CTA_M + A_BAND - 1) / A_BAND);
            const int bands = rank == 0 ? bands0 : bands1;
            const uint32_t bytes = (uint32_t)((bands0 + bands1) * A_BAND * 128 + t.bn * 128 + (bands1 > 0 ? 2 : 1) * 2 * MX_SCALE_BYTES + 2 * 4 * MX_SCALE_BYTES);
            const bool wide = t.bn == BN;
            for (int kb = 0; kb < p.num_kb; ++kb) {
                ok = mbar_wait_uniform<true>(smem_u32(&bar_empty[stage]), phase ^ 1u, &abort_flag, p.status, WAIT_PRODUCER_EMPTY, p.wait_limit);
                if (!ok) break;
                if (elect_one()) {
                    const uint32_t full_local = smem_u32(&bar_full[stage]), full = map_to_leader(full_local);
                    const uint32_t a0 = smem_base + stage * STAGE_BYTES;
                    if (warp == 0) {
                        if (rank == 0) mbar_expect_tx(full_local, bytes);
                        if (bands == 4) {
                            tma_load_3d_2sm(a0, &maps.a, kb * 128, am, 0, full);
                        } else {
                            for (int b = 0; b < bands; ++b) tma_load_3d_2sm(a0 + b * A_BAND * 128, &maps.a_band, kb * 128, am + b * A_BAND, 0, full);
                        }
                        if (wide) tma_load_3d_2sm(a0 + A_BYTES, &maps.b_wide, kb * 128, bn0, t.g, full);
                        else tma_load_3d_2sm(a0 + A_BYTES, &maps.b_narrow, kb * 128, bn0, t.g, full);
                    } else {
                        if (bands > 0) tma_load_3d_2sm(a0 + SFA_AT, &maps.sfa, kb * 256, t.slot + (int)rank, 0, full);
                        tma_load_3d_2sm(a0 + SFB_AT, &maps.sfb, kb * 256, t.n0 / 128, t.g, full);
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
        const uint32_t tmem_u = uniform(tmem_base);
        int stage = 0, it = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int tile = pair_id; ok && tile < plan.total; tile += num_pairs, ++it) {
            const GroupedTile t = grouped_tile_uniform<false, PAIR_M>(p, plan, walk, tile);
            const uint32_t idesc[2] = {make_idesc_mxf4(PAIR_M, (uint32_t)t.bn, 0), make_idesc_mxf4(PAIR_M, (uint32_t)t.bn, 2)};
            const uint32_t n_skip = (uint32_t)(t.n0 & 127) >> 5; // a tile may start in the middle of a row block: two columns in
            const int acc = it & 1;
            ok = mbar_wait_uniform<true>(smem_u32(&bar_tmem_empty[acc]), ((uint32_t)(it >> 1) & 1u) ^ 1u, &abort_flag, p.status, WAIT_MMA_TMEM_EMPTY, p.wait_limit);
            tc_fence_after();
            const uint32_t d_tmem = tmem_u + (uint32_t)(acc * BN);
            for (int kb = 0; ok && kb < p.num_kb; ++kb) {
                ok = mbar_wait_uniform<true>(smem_u32(&bar_full[stage]), phase, &abort_flag, p.status, WAIT_MMA_FULL, p.wait_limit);
                if (!ok) break;
                tc_fence_after();
                const uint32_t a0 = smem_base + stage * STAGE_BYTES;
                const uint64_t ad = make_smem_desc_sw128(a0, 16, 1024), bd = make_smem_desc_sw128(a0 + A_BYTES, 16, 1024);
                const uint64_t sa = make_smem_desc_rows16(a0 + SFA_AT), sb = make_smem_desc_rows16(a0 + SFB_AT);
                const uint32_t sf = tmem_u + SF_COL + (uint32_t)(stage * SF_STAGE_COLS);
                const int steps = min(BK / 64, (p.K - kb * BK + 63) / 64);
                if (elect_one()) {
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        if (c * 2 < steps) {
                            tmem_cp_32x128b<2>(sf + c * 4, sa + (uint64_t)(c * MX_SCALE_BYTES >> 4));
                            tmem_cp_32x128b<2>(sf + 8 + c * 8, sb + (uint64_t)(c * MX_SCALE_BYTES >> 4));
                            tmem_cp_32x128b<2>(sf + 12 + c * 8, sb + (uint64_t)((2 + c) * MX_SCALE_BYTES >> 4));
                        }
                    }
#pragma unroll
                    for (int ks = 0; ks < BK / 64; ++ks)
                        if (ks < steps)
                            umma_mxf4<2>(d_tmem, ad + (uint64_t)(ks * 2), bd + (uint64_t)(ks * 2), idesc[ks & 1], sf + (ks >> 1) * 4,
                                         sf + 8 + (ks >> 1) * 8 + n_skip, (uint32_t)((kb | ks) != 0));
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
        // ------------------------------------------------------------ epilogue (warps 2..9 of both CTAs, own 128 rows)
        const int quad = warp & 3;
        const uint32_t epi_smem = smem_base + STAGES * STAGE_BYTES + (uint32_t)(warp - 2) * EPI_TILE_BYTES;
        int it = 0;
        for (int tile = pair_id; tile < plan.total; tile += num_pairs, ++it) {
            const GroupedTile t = grouped_tile<false, PAIR_M>(p, plan, walk, tile);
            const int acc = it & 1;
            if (!mbar_wait_uniform<true>(smem_u32(&bar_tmem_full[acc]), (uint32_t)(it >> 1) & 1u, &abort_flag, p.status, WAIT_EPI_TMEM_FULL, p.wait_limit)) break;
            tc_fence_after();
            grouped_band<DT, false>(p, maps.c, tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(acc * BN), t,
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

int launch_mxfp4_matmul_pair(const Mxfp4Call &c, cudaStream_t st, int sm_count, const GemmParams &p, const CUtensorMap &tmA, const CUtensorMap &tmA_band,
                             const CUtensorMap &sfa, const CUtensorMap &sfb, const CUtensorMap &tmC)
{
    using namespace mxp;
    const uint64_t pitch = (uint64_t)c.K / 2;
    MxPairMaps maps;
    memset(&maps, 0, sizeof(maps));
    maps.a = tmA;
    maps.a_band = tmA_band;
    maps.sfa = sfa;
    maps.sfb = sfb;
    maps.c = tmC;
    int rc = encode_tmap_3d(&maps.b_wide, BTM_U8, c.w, pitch, (uint64_t)c.N, (uint64_t)c.groups, pitch, pitch * (uint64_t)c.N, 128, BN / 2);
    if (!rc) rc = encode_tmap_3d(&maps.b_narrow, BTM_U8, c.w, pitch, (uint64_t)c.N, (uint64_t)c.groups, pitch, pitch * (uint64_t)c.N, 128, 64);
    if (rc) return rc;
    static std::atomic<int> resident[64]; // pairs the device holds at once (GPC boundaries can make it less than SMs / 2)
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
        if (cudaOccupancyMaxActiveClusters(&n, mxfp4_gemm_pair_kernel<BTM_BF16>, &cfg) != cudaSuccess || n <= 0) {
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
    const cudaError_t e = c.dtype == BTM_F16 ? cudaLaunchKernelEx(&cfg, mxfp4_gemm_pair_kernel<BTM_F16>, maps, p, tab)
                                             : cudaLaunchKernelEx(&cfg, mxfp4_gemm_pair_kernel<BTM_BF16>, maps, p, tab);
    return check_cuda(e, "mxfp4 matmul (pair) launch");
}

int configure_mxfp4_pair_kernels()
{
    cudaError_t e = cudaFuncSetAttribute(mxfp4_gemm_pair_kernel<BTM_F16>, cudaFuncAttributeMaxDynamicSharedMemorySize, mxp::SMEM_BYTES);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(mxfp4_gemm_pair_kernel<BTM_BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, mxp::SMEM_BYTES);
    return check_cuda(e, "cudaFuncSetAttribute(mxfp4_gemm_pair)");
}

} // namespace btm
