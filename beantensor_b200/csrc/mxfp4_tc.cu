// Product of two microscaled 4-bit operands on the tensor cores, plain or grouped by expert:
//   out[r, n] = sum_k act[r, k] w[g][n, k],  both q 2^X with one X for 32 consecutive k (mxfp4.cuh), fp32 accumulation.
//
// tcgen05.mma kind::mxf4.block_scale multiplies the 4-bit values and applies both scales; no value is ever unpacked. Both
// operands are K-major as they lie (256 k = 128 bytes, 128-byte swizzle). The scales lie in memory in the order in which
// tensor memory holds them: as a matrix of 32-bit words, one block of 128 rows per row, they come in with their stage (two
// blocks of the weights in one box) and go to tensor memory by one tcgen05.cp per 128 rows x 128 k.
// One persistent CTA per SM, warp roles and tile walk as in gemm_grouped.cu (a plain product is one group that owns every
// row), and a second producer warp for the scales: issuing a TMA load takes a thread 75 to 120 cycles, a stage has four
// to seven, and its MMAs take 384. Measured: 256 rows in 64 groups of 2048 x 2048 29 us (4.9 TB/s of weights), 8192 x 11008 x
// 4096 167 us after a pause, 193 in a long run.
#include <cstdlib>
#include <cstring>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "btm_internal.h"
#include "btm_ptx.cuh"
#include "grouped_tile.cuh"
#include "mxfp4.cuh"

namespace btm {

namespace mxt {
constexpr int BM = 128;               // token rows of a tile
constexpr int BN = 192;               // widest tile: two accumulators of 192 columns leave tensor memory for the scales
constexpr int BK = 256;               // k per stage: 128 bytes
constexpr int A_BYTES = BM * 128;
constexpr int SFA_AT = A_BYTES + BN * 128;
constexpr int SFB_AT = SFA_AT + 2 * MX_SCALE_BYTES;        // two row blocks, two k-chunks each
constexpr int STAGE_BYTES = SFB_AT + 4 * MX_SCALE_BYTES;   // 43 KB
constexpr int STAGES = 4;
constexpr int SMEM_BYTES = STAGES * STAGE_BYTES + EPI_SMEM_BYTES + 1024;
constexpr int SF_COL = 2 * BN;        // first tensor-memory column of the scales
constexpr int SF_STAGE_COLS = 32;     // per stage: A 2 x 4 columns, B 2 x 8
constexpr int TMEM_COLS = 512;
constexpr int THREADS = 352; // warp 0 operands, 1 MMA, 2-9 epilogue, 10 scales
constexpr int A_BAND = 32;
static_assert(SF_COL + STAGES * SF_STAGE_COLS <= TMEM_COLS, "accumulators and scales share tensor memory");
static_assert(STAGE_BYTES % 1024 == 0, "stages start on swizzle atoms");
} // namespace mxt

struct MxMaps {
    CUtensorMap a, a_band, b[3] /* 192, 128 and 64 weight rows per box */, sfa, sfb, c;
};

template <int DT>
__global__ void __launch_bounds__(mxt::THREADS, 1)
mxfp4_gemm_kernel(const __grid_constant__ MxMaps maps, const __grid_constant__ GemmParams p, const GroupedTables tab)
{
    using namespace mxt;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bar_full[STAGES], bar_empty[STAGES], bar_tmem_full[2], bar_tmem_empty[2];
    __shared__ uint32_t tmem_base_holder;
    __shared__ int abort_flag;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < STAGES; ++s) {
            mbar_init(smem_u32(&bar_full[s]), 1);
            mbar_init(smem_u32(&bar_empty[s]), 1);
        }
        for (int a = 0; a < 2; ++a) {
            mbar_init(smem_u32(&bar_tmem_full[a]), 1);
            mbar_init(smem_u32(&bar_tmem_empty[a]), GROUPED_EPI_WARPS);
        }
        fence_mbar_init();
        prefetch_tmap(&maps.a);
        prefetch_tmap(&maps.a_band);
        prefetch_tmap(&maps.sfa);
        prefetch_tmap(&maps.sfb);
    }
    if (warp == 1) {
        tmem_alloc<1>(smem_u32(&tmem_base_holder), TMEM_COLS);
        tmem_relinquish<1>();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_holder;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    GroupWalk<> walk;
    walk.init(tab.offsets, tab.groups, tab.rows);
    const GroupedPlan plan = plan_tiles<BN>(walk.count_slots(), p.N, gridDim.x);
    if (blockIdx.x == 0 && warp == 0) walk.report(p.status);

    if (warp == 0 || warp == 10) {
        // ------------------------------------------------------------ TMA producers: operands, scales
        int stage = 0;
        uint32_t phase = 0;
        bool ok = !p.debug_skip_loads;
        for (int tile = blockIdx.x; ok && tile < plan.total; tile += gridDim.x) {
            const GroupedTile t = grouped_tile_uniform<false, GROUP_SLOT_ROWS>(p, plan, walk, tile);
            const int bands = min(4, (t.hi - t.m0 + A_BAND - 1) / A_BAND);
            const uint32_t bytes = (uint32_t)(bands * A_BAND * 128 + t.bn * 128 + 6 * MX_SCALE_BYTES);
            const CUtensorMap *mb = &maps.b[t.bn == BN ? 0 : t.bn == 128 ? 1 : 2];
            for (int kb = 0; kb < p.num_kb; ++kb) {
                ok = mbar_wait_uniform(smem_u32(&bar_empty[stage]), phase ^ 1u, &abort_flag, p.status, WAIT_PRODUCER_EMPTY, p.wait_limit);
                if (!ok) break;
                if (elect_one()) {
                    const uint32_t full = smem_u32(&bar_full[stage]);
                    const uint32_t a0 = smem_base + stage * STAGE_BYTES;
                    if (warp == 0) {
                        mbar_expect_tx(full, bytes);
                        if (bands == 4) {
                            tma_load_3d(a0, &maps.a, kb * 128, t.m0, 0, full);
                        } else {
                            for (int b = 0; b < bands; ++b) tma_load_3d(a0 + b * A_BAND * 128, &maps.a_band, kb * 128, t.m0 + b * A_BAND, 0, full);
                        }
                        tma_load_3d(a0 + A_BYTES, mb, kb * 128, t.n0, t.g, full);
                    } else {
                        tma_load_3d(a0 + SFA_AT, &maps.sfa, kb * 256, t.slot, 0, full);
                        tma_load_3d(a0 + SFB_AT, &maps.sfb, kb * 256, t.n0 / 128, t.g, full);
                    }
                }
                __syncwarp();
                if (++stage == STAGES) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer
        const uint32_t tmem_u = uniform(tmem_base);
        int stage = 0, it = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int tile = blockIdx.x; ok && tile < plan.total; tile += gridDim.x, ++it) {
            const GroupedTile t = grouped_tile_uniform<false, GROUP_SLOT_ROWS>(p, plan, walk, tile);
            const uint32_t idesc[2] = {make_idesc_mxf4(BM, (uint32_t)t.bn, 0), make_idesc_mxf4(BM, (uint32_t)t.bn, 2)};
            const uint32_t n_skip = (uint32_t)(t.n0 & 127) >> 5; // a tile may start in the middle of a row block: two columns in
            const int acc = it & 1;
            ok = mbar_wait_uniform(smem_u32(&bar_tmem_empty[acc]), ((uint32_t)(it >> 1) & 1u) ^ 1u, &abort_flag, p.status, WAIT_MMA_TMEM_EMPTY, p.wait_limit);
            if (!ok) break;
            tc_fence_after();
            const uint32_t d_tmem = tmem_u + (uint32_t)(acc * BN);
            for (int kb = 0; kb < p.num_kb; ++kb) {
                ok = mbar_wait_uniform(smem_u32(&bar_full[stage]), phase, &abort_flag, p.status, WAIT_MMA_FULL, p.wait_limit);
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
                            tmem_cp_32x128b<1>(sf + c * 4, sa + (uint64_t)(c * MX_SCALE_BYTES >> 4));
                            tmem_cp_32x128b<1>(sf + 8 + c * 8, sb + (uint64_t)(c * MX_SCALE_BYTES >> 4));
                            tmem_cp_32x128b<1>(sf + 12 + c * 8, sb + (uint64_t)((2 + c) * MX_SCALE_BYTES >> 4));
                        }
                    }
#pragma unroll
                    for (int ks = 0; ks < BK / 64; ++ks)
                        if (ks < steps)
                            umma_mxf4<1>(d_tmem, ad + (uint64_t)(ks * 2), bd + (uint64_t)(ks * 2), idesc[ks & 1], sf + (ks >> 1) * 4,
                                         sf + 8 + (ks >> 1) * 8 + n_skip, (uint32_t)((kb | ks) != 0));
                    umma_commit(smem_u32(&bar_empty[stage]));
                }
                __syncwarp();
                if (++stage == STAGES) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
            if (ok && elect_one()) umma_commit(smem_u32(&bar_tmem_full[acc]));
            __syncwarp();
        }
    } else {
        // ------------------------------------------------------------ epilogue (warps 2..9)
        const int quad = warp & 3;
        const uint32_t epi_smem = smem_base + STAGES * STAGE_BYTES + (uint32_t)(warp - 2) * EPI_TILE_BYTES;
        int it = 0;
        for (int tile = blockIdx.x; tile < plan.total; tile += gridDim.x, ++it) {
            const GroupedTile t = grouped_tile<false, GROUP_SLOT_ROWS>(p, plan, walk, tile);
            const int acc = it & 1;
            if (!mbar_wait_uniform(smem_u32(&bar_tmem_full[acc]), (uint32_t)(it >> 1) & 1u, &abort_flag, p.status, WAIT_EPI_TMEM_FULL, p.wait_limit)) break;
            tc_fence_after();
            grouped_band<DT, false>(p, maps.c, tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(acc * BN), t, t.m0 + quad * 32, t.hi, false,
                                    epi_smem, (warp - 2) >> 2, lane);
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&bar_tmem_empty[acc]));
        }
        epilogue_drain(lane);
    }

    // ---------------------------------------------------------------- teardown
    tc_fence_before();
    __syncthreads();
    if (abort_flag) {
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) {}
        __syncthreads();
    }
    if (warp == 1) {
        __syncwarp();
        tc_fence_after();
        tmem_dealloc<1>(tmem_base, TMEM_COLS);
    }
}

// Scale blocks as a matrix of 32-bit words, one row block per row: boxes of two k-chunks x `box_rows` row blocks.
int encode_mx_scales(CUtensorMap *m, const void *scales, int K, uint64_t blocks, uint64_t groups, uint32_t box_rows)
{
    const uint64_t words = (uint64_t)mx_chunks(K) * (MX_SCALE_BYTES / 4);
    return encode_tmap_3d(m, BTM_U32, scales, words, blocks, groups, words * 4, words * 4 * blocks, 2 * MX_SCALE_BYTES / 4, box_rows, 0);
}

int configure_mxfp4_kernels()
{
    cudaError_t e = cudaFuncSetAttribute(mxfp4_gemm_kernel<BTM_F16>, cudaFuncAttributeMaxDynamicSharedMemorySize, mxt::SMEM_BYTES);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(mxfp4_gemm_kernel<BTM_BF16>, cudaFuncAttributeMaxDynamicSharedMemorySize, mxt::SMEM_BYTES);
    return check_cuda(e, "cudaFuncSetAttribute(mxfp4_gemm)");
}

int launch_mxfp4_matmul(const Mxfp4Call &c, cudaStream_t st, int sm_count, int *status)
{
    using namespace mxt;
    if (c.K == 0) { // an empty sum: the general grouped kernel writes the zeros
        GroupedCall z;
        memset(&z, 0, sizeof(z));
        z.dtype = c.dtype; z.groups = c.groups; z.rows = c.rows; z.N = c.N; z.offsets = c.offsets; z.C = c.out; z.ldc = c.ldo;
        return launch_gemm_grouped(z, st, sm_count, status);
    }
    const char *force = getenv("BTM_FORCE_KERNEL"); // 1cta, 2cta or decode: the tests run every shape on each
    bool decode = grouped_decode_fits(c.groups, c.rows, c.N, sm_count);
    if (force) decode = !strcmp(force, "decode");
    if (decode) return launch_mxfp4_decode(c, st, sm_count, status);
    const long long slots = grouped_slot_bound(c.groups, c.rows);
    const long long most = slots * ((c.N + 63) / 64);
    if (most > 0x3FFFFFFFLL) return set_error(BTM_ERR_UNSUPPORTED, "mxfp4 matmul: too many output tiles (%lld)", most);
    const uint64_t pitch = (uint64_t)c.K / 2;
    MxMaps maps;
    memset(&maps, 0, sizeof(maps));
    int rc = encode_tmap_3d(&maps.a, BTM_U8, c.act, pitch, (uint64_t)c.rows, 1, pitch, pitch, 128, BM);
    if (!rc) rc = encode_tmap_3d(&maps.a_band, BTM_U8, c.act, pitch, (uint64_t)c.rows, 1, pitch, pitch, 128, A_BAND);
    if (!rc) rc = encode_mx_scales(&maps.sfa, c.act_scales, c.K, (uint64_t)slots, 1, 1);
    if (!rc) rc = encode_mx_scales(&maps.sfb, c.w_scales, c.K, (uint64_t)((c.N + 127) / 128), (uint64_t)c.groups, 2);
    if (rc) return rc;
    GemmParams p;
    memset(&p, 0, sizeof(p));
    p.M = c.rows;
    p.N = c.N;
    p.K = c.K;
    p.batch = 1;
    p.num_kb = (c.K + BK - 1) / BK;
    p.group_m = 8;
    p.ndst = 1;
    p.C[0] = c.out;
    p.ldc = c.ldo;
    p.c_vec_ok = ((uintptr_t)c.out & 15) == 0 && (c.ldo * 2) % 16 == 0 ? 1 : 0;
    p.status = status;
    fill_wait_params(&p);
    if (p.c_vec_ok) {
        rc = encode_tmap_3d(&maps.c, c.dtype, c.out, (uint64_t)c.N, (uint64_t)c.rows, 1, (uint64_t)c.ldo * 2, (uint64_t)c.ldo * 2, 64, 32);
        if (rc) return rc;
    }
    // Pairs of CTAs for tall groups, a deep reduction and enough outputs for their larger tiles. Measured, one CTA against pairs,
    // rows / N x K, us in a run, equal groups; uneven ones (a load of rank^-0.7):
    //   8192 / 11008 x 4096: 193 / 188    2048 / 4096 x 4096: 26.7 / 23.3    4096 in 8 groups / 4096 x 4096: 47.1 / 44.1; 51.3 / 54.4
    //   1024 / 4096 x 4096: 15.9 / 15.7   8192 / 2048 x 1024: 15.9 / 18.4    12000 in 24 / 4096 x 2048: 76.9 / 70.8; 77.5 / 78.3
    bool pair = c.rows / c.groups >= 512 && c.K >= 2048 && (long long)c.rows * c.N >= 8 << 20;
    if (force) {
        if (!strcmp(force, "1cta")) pair = false;
        else if (!strcmp(force, "2cta")) pair = true;
    }
    if (pair) return launch_mxfp4_matmul_pair(c, st, sm_count, p, maps.a, maps.a_band, maps.sfa, maps.sfb, maps.c);
    static const uint32_t box_rows[3] = {BN, 128, 64};
    for (int i = 0; i < 3 && !rc; ++i) rc = encode_tmap_3d(&maps.b[i], BTM_U8, c.w, pitch, (uint64_t)c.N, (uint64_t)c.groups, pitch, pitch * (uint64_t)c.N, 128, box_rows[i]);
    if (rc) return rc;
    const GroupedTables tab = {c.offsets, c.groups, c.rows};
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3((unsigned)(most < sm_count ? most : sm_count), 1, 1);
    cfg.blockDim = dim3(THREADS, 1, 1);
    cfg.dynamicSmemBytes = SMEM_BYTES;
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    const cudaError_t e = c.dtype == BTM_F16 ? cudaLaunchKernelEx(&cfg, mxfp4_gemm_kernel<BTM_F16>, maps, p, tab)
                                             : cudaLaunchKernelEx(&cfg, mxfp4_gemm_kernel<BTM_BF16>, maps, p, tab);
    return check_cuda(e, "mxfp4 matmul launch");
}

} // namespace btm
