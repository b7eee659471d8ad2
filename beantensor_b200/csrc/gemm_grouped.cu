// Matrix products grouped by expert with ragged sizes: the rows of A are sorted by group, offsets[g] .. offsets[g + 1]
// are the rows of group g (a device-side table, grouped_rows.cuh).
//   product:          C[r, :] = A[r, :] . B[g]                   r in group g
//   weight gradient:  C[g]    = A[rows of g]^T . D[rows of g]    (all zero for a group without rows)
//
// Tensor-core kernel: one persistent CTA per SM with the warp roles of gemm_tc.cu (TMA producer, tcgen05.mma issuer with
// two accumulators in tensor memory, eight epilogue warps). What differs is where a tile's rows come from: every role
// walks the table by itself, a warp at a time, and no tile list exists in memory.
//   product    rows are cut per group into slots of 128; a tile is (slot, column range). A tile reads up to 128 rows of
//              A from the group's first row on, whatever alignment that has (a row coordinate is free), so rows of the
//              next group can be in it: each only spoils its own output row, which is not stored. Bands of 32 rows that
//              lie inside the group leave by TMA store, the band that the group's end cuts by 16-byte stores of
//              its own rows.
//   gradient   a tile is (group, row range of C, column range), its k-blocks are 64 rows of the group. Both operands are
//              MN-major as they lie. The last k-block is cut: rows behind the group's end are overwritten with zero in
//              both operands in shared memory (zero times a foreign infinity would be NaN), and only the 16-row steps that
//              hold rows of the group are multiplied.
// Few tiles or a ragged last wave: the tile width (256, 128 or 64 columns, and half of it for what would be a partly
// filled last wave) is chosen on the device from the number of slots, by the same rule in every CTA.
// Measured (bf16, 16384 rows, 4096 x 4096, this kernel, after a pause / in a long run under the power cap): product 386 / 457 us in
// one group, 391 / 468 in eight equal ones, 422 / 502 in eight uneven ones (1430, 1410, 1300 TFLOP/s after a pause), gradient
// 392 / 472 in eight; 256 rows in 64 groups of 2048 x 2048 fp16 84 us, 6.4 TB/s. With many rows the tensor core waits for its
// operands' way: 48 KB per 64-deep k-block at the 73 B per cycle that an SM of a loaded machine gets is 670 cycles, the MMAs take 512.
//
// General kernel (operands that TMA cannot address, K == 0): 64 x 64 output tiles on CUDA cores as in gemm_simt.cu, fp32
// accumulation, one rounding. A block finds its group by walking the table. 4096 rows in eight groups, 1021 x 1023 bf16 in
// pitches of that width: product 530 us, gradient 485, where 1024 x 1024 take 14 and 15 on the tensor cores.
#include <cstdlib>
#include <cstring>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "btm_internal.h"
#include "btm_ptx.cuh"
#include "gemm_epilogue.cuh"
#include "grouped_tile.cuh"

namespace btm {

namespace gg {
constexpr int BM = 128;                 // rows of an output tile = accumulator lanes
constexpr int BN = 256;                 // widest tile
constexpr int BK = 64;                  // k per stage: 128 bytes
constexpr int CHUNK_BYTES = 64 * 128;   // every TMA box of an operand is 64 rows x 128 bytes, except A of the product
constexpr int A_BYTES = BM * 128;
// The ring holds as many stages as fit at the launch's tile width: 4 at 256 columns, 6 at 128, 8 at 64, so that a launch
// of narrow tiles (few rows: the time is the latency of the weights) asks for as many bytes ahead.
constexpr int RING_BYTES = 4 * (A_BYTES + BN * 128);
constexpr int STAGES = 8;
constexpr int SMEM_BYTES = RING_BYTES + EPI_SMEM_BYTES + 1024;
constexpr int TMEM_COLS = 512;
constexpr int THREADS = 320; // warp 0 TMA, 1 MMA, 2-9 epilogue
constexpr int A_BAND = 32;              // rows of a short A box: a tile with few rows does not fetch its neighbours'
} // namespace gg

// tmA: 128-row boxes (product) or 64-row boxes (gradient); tmA_band: boxes of A_BAND rows (product only).
template <int DT, int MODE>
__global__ void __launch_bounds__(gg::THREADS, 1)
gemm_grouped_kernel(const __grid_constant__ CUtensorMap tmA, const __grid_constant__ CUtensorMap tmA_band, const __grid_constant__ CUtensorMap tmB,
                    const __grid_constant__ CUtensorMap tmC, const __grid_constant__ GemmParams p, const GroupedTables tab)
{
    using namespace gg;
    constexpr bool kWgrad = MODE == GROUPED_WGRAD;
    constexpr bool kBMnMajor = MODE != GROUPED_NK;
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
        prefetch_tmap(&tmA);
        prefetch_tmap(&tmB);
        if (!kWgrad) prefetch_tmap(&tmA_band);
    }
    if (warp == 1) {
        tmem_alloc<1>(smem_u32(&tmem_base_holder), TMEM_COLS);
        tmem_relinquish<1>();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_holder;
    // Everything behind this line reads what earlier work on the stream may have written, the table first of all; only
    // then may a successor be let in, which so can rely on this grid's predecessors.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    GroupWalk<> walk;
    walk.init(tab.offsets, tab.groups, tab.rows);
    const int group_slots = walk.count_slots();
    if (blockIdx.x == 0 && warp == 0) walk.report(p.status);
    const GroupedPlan plan = plan_tiles<gg::BN>(kWgrad ? tab.groups * p.tiles_m : group_slots, p.N, gridDim.x);

    const uint32_t stage_bytes = (uint32_t)(A_BYTES + plan.bn * 128);
    const int stages = min(STAGES, (int)((uint32_t)RING_BYTES / stage_bytes));

    // Producer and issuer run as whole warps with uniform control flow; one elected lane issues (mbar_wait_uniform).
    if (warp == 0) {
        // ------------------------------------------------------------ TMA producer
        int stage = 0;
        uint32_t phase = 0;
        bool ok = !p.debug_skip_loads;
        for (int tile = blockIdx.x; ok && tile < plan.total; tile += gridDim.x) {
            const GroupedTile t = grouped_tile_uniform<kWgrad, GROUP_SLOT_ROWS>(p, plan, walk, tile);
            const int num_kb = kWgrad ? (t.hi - t.lo + BK - 1) / BK : p.num_kb;
            const int chunks = t.bn / 64;
            const int bands = min(4, (t.hi - t.m0 + A_BAND - 1) / A_BAND); // of A rows that the tile owns (product)
            const uint32_t bytes = (uint32_t)((kWgrad || bands == 4 ? A_BYTES : bands * A_BAND * 128) + chunks * CHUNK_BYTES);
            const int zb = kWgrad ? 0 : t.g;
            for (int kb = 0; kb < num_kb; ++kb) {
                ok = mbar_wait_uniform(smem_u32(&bar_empty[stage]), phase ^ 1u, &abort_flag, p.status, WAIT_PRODUCER_EMPTY, p.wait_limit);
                if (!ok) break;
                if (elect_one()) {
                    const uint32_t full = smem_u32(&bar_full[stage]);
                    const uint32_t a0 = smem_base + (uint32_t)stage * stage_bytes, b0 = a0 + A_BYTES;
                    const int k0 = kWgrad ? t.lo + kb * BK : kb * BK;
                    mbar_expect_tx(full, bytes);
                    if constexpr (kWgrad) {
                        tma_load_3d(a0, &tmA, t.m0, k0, 0, full);
                        tma_load_3d(a0 + CHUNK_BYTES, &tmA, t.m0 + 64, k0, 0, full);
                    } else if (bands == 4) {
                        tma_load_3d(a0, &tmA, k0, t.m0, 0, full);
                    } else {
                        for (int b = 0; b < bands; ++b) tma_load_3d(a0 + b * A_BAND * 128, &tmA_band, k0, t.m0 + b * A_BAND, 0, full);
                    }
#pragma unroll
                    for (int c = 0; c < BN / 64; ++c) {
                        if (c < chunks) {
                            if (kBMnMajor) tma_load_3d(b0 + c * CHUNK_BYTES, &tmB, t.n0 + c * 64, k0, zb, full);
                            else tma_load_3d(b0 + c * CHUNK_BYTES, &tmB, k0, t.n0 + c * 64, zb, full);
                        }
                    }
                }
                __syncwarp();
                if (++stage == stages) {
                    stage = 0;
                    phase ^= 1u;
                }
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer
        constexpr uint32_t kFmt = DT == BTM_BF16 ? 1u : 0u;
        constexpr uint32_t a_step = (kWgrad ? 16 * 128 : 32) >> 4, b_step = (kBMnMajor ? 16 * 128 : 32) >> 4; // 16 k, in 16-byte units
        const uint32_t tmem_u = uniform(tmem_base);
        int stage = 0, it = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int tile = blockIdx.x; ok && tile < plan.total; tile += gridDim.x, ++it) {
            const GroupedTile t = grouped_tile_uniform<kWgrad, GROUP_SLOT_ROWS>(p, plan, walk, tile);
            const int num_kb = kWgrad ? (t.hi - t.lo + BK - 1) / BK : p.num_kb;
            const uint32_t idesc = make_idesc(kFmt, kWgrad, kBMnMajor, BM, (uint32_t)t.bn);
            const int acc = it & 1;
            ok = mbar_wait_uniform(smem_u32(&bar_tmem_empty[acc]), ((uint32_t)(it >> 1) & 1u) ^ 1u, &abort_flag, p.status, WAIT_MMA_TMEM_EMPTY, p.wait_limit);
            if (!ok) break;
            tc_fence_after();
            const uint32_t d_tmem = tmem_u + (uint32_t)(acc * BN);
            for (int kb = 0; kb < num_kb; ++kb) {
                ok = mbar_wait_uniform(smem_u32(&bar_full[stage]), phase, &abort_flag, p.status, WAIT_MMA_FULL, p.wait_limit);
                if (!ok) break;
                const uint32_t a0 = smem_base + (uint32_t)stage * stage_bytes, b0 = a0 + A_BYTES;
                int steps = BK / 16;
                if (kWgrad) {
                    const int left = t.hi - t.lo - kb * BK; // rows of the group in this k-block
                    if (left < BK) {
                        steps = (left + 15) / 16;
                        // Rows left .. 16 * steps - 1 of every 64-wide chunk: 128 contiguous bytes per row.
                        const int dirty = steps * 16 - left;
                        for (int i = lane; i < dirty * 8; i += 32) {
                            const uint32_t off = (uint32_t)(left + (i >> 3)) * 128u + (uint32_t)(i & 7) * 16u;
                            for (int c = 0; c < BM / 64; ++c) st_shared_v4(a0 + c * CHUNK_BYTES + off, 0u, 0u, 0u, 0u);
                            for (int c = 0; c < t.bn / 64; ++c) st_shared_v4(b0 + c * CHUNK_BYTES + off, 0u, 0u, 0u, 0u);
                        }
                        fence_proxy_async_smem();
                        __syncwarp();
                    }
                }
                tc_fence_after();
                const uint64_t ad = kWgrad ? make_smem_desc_sw128(a0, CHUNK_BYTES, 1024) : make_smem_desc_sw128(a0, 16, 1024);
                const uint64_t bd = kBMnMajor ? make_smem_desc_sw128(b0, CHUNK_BYTES, 1024) : make_smem_desc_sw128(b0, 16, 1024);
                if (elect_one()) {
#pragma unroll
                    for (int ks = 0; ks < BK / 16; ++ks)
                        if (!kWgrad || ks < steps)
                            umma<1, false>(d_tmem, ad + (uint64_t)(ks * a_step), bd + (uint64_t)(ks * b_step), idesc, (uint32_t)((kb | ks) != 0));
                    umma_commit(smem_u32(&bar_empty[stage]));
                }
                __syncwarp();
                if (++stage == stages) {
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
        const uint32_t epi_smem = smem_base + RING_BYTES + (uint32_t)(warp - 2) * EPI_TILE_BYTES;
        int it = 0;
        for (int tile = blockIdx.x; tile < plan.total; tile += gridDim.x, ++it) {
            const GroupedTile t = grouped_tile<kWgrad, GROUP_SLOT_ROWS>(p, plan, walk, tile);
            const int acc = it & 1;
            if (!mbar_wait_uniform(smem_u32(&bar_tmem_full[acc]), (uint32_t)(it >> 1) & 1u, &abort_flag, p.status, WAIT_EPI_TMEM_FULL, p.wait_limit)) break;
            tc_fence_after();
            grouped_band<DT, kWgrad>(p, tmC, tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(acc * BN), t, t.m0 + quad * 32,
                                   kWgrad ? p.M : t.hi, kWgrad && t.lo == t.hi, epi_smem, (warp - 2) >> 2, lane);
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
        // A wait ran out somewhere: copies in flight land within microseconds, shared memory is held that long.
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

template <int DT>
struct Half16;
template <>
struct Half16<BTM_F16> {
    using T = __half;
    static __device__ __forceinline__ float load(const T *p) { return __half2float(*p); }
    static __device__ __forceinline__ T round(float v) { return __float2half_rn(v); }
};
template <>
struct Half16<BTM_BF16> {
    using T = __nv_bfloat16;
    static __device__ __forceinline__ float load(const T *p) { return __bfloat162float(*p); }
    static __device__ __forceinline__ T round(float v) { return __float2bfloat16_rn(v); }
};

struct GroupedSimtArgs {
    const void *A, *B;
    void *C;
    long long a_rs, a_cs, b_rs, b_cs, strideB, ldc, strideC;
    int M, N, K; // M: output rows per group (weight gradient only)
    const int *offsets;
    int groups, rows;
    int tiles_m, tiles_n; // tiles_m: 64-row tiles per group (weight gradient), per slot of 128 rows (product)
    int *status;
};

// kWgrad: rows are the reduction index, output rows are A's columns. Otherwise rows are the output rows.
template <int DT, bool kWgrad>
__global__ void __launch_bounds__(256) gemm_grouped_simt_kernel(const GroupedSimtArgs p)
{
    using E = Half16<DT>;
    using T = typename E::T;
    constexpr int TM = 64, TN = 64, TK = 16;
    __shared__ float As[TK][TM + 1];
    __shared__ float Bs[TK][TN + 1];
    GroupWalk<> walk;
    walk.init(p.offsets, p.groups, p.rows);
    const long long id = blockIdx.x;
    const int n0 = (int)(id % p.tiles_n) * TN;
    const int mt = (int)(id / p.tiles_n); // tile row over all groups
    int g, lo, hi, m0;
    if (kWgrad) {
        g = mt / p.tiles_m;
        m0 = (mt - g * p.tiles_m) * TM;
        if (blockIdx.x == 0) {
            walk.count_slots();
            if (threadIdx.x < 32) walk.report(p.status);
        }
        walk.find_group(g, lo, hi);
    } else {
        const int slots = walk.count_slots();
        if (blockIdx.x == 0 && threadIdx.x < 32) walk.report(p.status);
        const int slot = mt >> 1; // a slot is two tiles high
        if (slot >= slots) return;
        int first;
        walk.find_slot(slot, g, lo, hi, first);
        m0 = lo + (slot - first) * GROUP_SLOT_ROWS + (mt & 1) * TM;
        if (m0 >= hi) return;
    }
    const int m_end = kWgrad ? p.M : hi, k_begin = kWgrad ? lo : 0, k_end = kWgrad ? hi : p.K;
    const T *A = reinterpret_cast<const T *>(p.A);
    const T *B = reinterpret_cast<const T *>(p.B) + (kWgrad ? 0 : (long long)g * p.strideB);
    T *C = reinterpret_cast<T *>(p.C) + (kWgrad ? (long long)g * p.strideC : 0);
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float acc[4][4] = {};
    for (int k0 = k_begin; k0 < k_end; k0 += TK) {
        for (int i = threadIdx.x; i < TM * TK; i += 256) {
            // neighbouring threads read neighbouring elements of A: along k for the product, along m for the gradient
            const int r = kWgrad ? i % TM : i / TK, c = kWgrad ? i / TM : i % TK;
            const int gm = m0 + r, gk = k0 + c;
            As[c][r] = (gm < m_end && gk < k_end) ? E::load(A + (long long)gm * p.a_rs + (long long)gk * p.a_cs) : 0.0f;
        }
        for (int i = threadIdx.x; i < TK * TN; i += 256) {
            const int r = i / TN, c = i % TN;
            const int gk = k0 + r, gn = n0 + c;
            Bs[r][c] = (gk < k_end && gn < p.N) ? E::load(B + (long long)gk * p.b_rs + (long long)gn * p.b_cs) : 0.0f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < TK; ++k) {
            float a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) a[i] = As[k][ty * 4 + i];
#pragma unroll
            for (int j = 0; j < 4; ++j) b[j] = Bs[k][tx * 4 + j];
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
        }
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int gm = m0 + ty * 4 + i;
        if (gm >= m_end) continue;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int gn = n0 + tx * 4 + j;
            if (gn < p.N) C[(long long)gm * p.ldc + gn] = E::round(acc[i][j]);
        }
    }
}

// Slots that `rows` rows in `groups` groups can fill: a group of m rows fills ceil(m / 128) of them.
long long grouped_slot_bound(int groups, int rows)
{
    const long long nonempty = groups < rows ? groups : rows;
    return ((long long)rows + (GROUP_SLOT_ROWS - 1) * nonempty) / GROUP_SLOT_ROWS;
}

static int launch_grouped_simt(const GroupedCall &c, cudaStream_t st, int *status)
{
    GroupedSimtArgs p;
    memset(&p, 0, sizeof(p));
    p.A = c.A; p.B = c.B; p.C = c.C;
    p.M = c.M; p.N = c.N; p.K = c.K;
    p.offsets = c.offsets; p.groups = c.groups; p.rows = c.rows;
    p.ldc = c.ldc; p.strideC = c.strideC; p.strideB = c.strideB;
    p.status = status;
    p.tiles_n = (c.N + 63) / 64;
    long long blocks;
    if (c.wgrad) {
        p.a_rs = 1; p.a_cs = c.lda;
        p.b_rs = c.ldb; p.b_cs = 1;
        p.tiles_m = (c.M + 63) / 64;
        blocks = (long long)c.groups * p.tiles_m * p.tiles_n;
    } else {
        p.a_rs = c.lda; p.a_cs = 1;
        p.b_rs = c.b_trans ? 1 : c.ldb; p.b_cs = c.b_trans ? c.ldb : 1;
        p.tiles_m = GROUP_SLOT_ROWS / 64;
        blocks = grouped_slot_bound(c.groups, c.rows) * p.tiles_m * p.tiles_n;
    }
    if (blocks == 0) return BTM_OK;
    if (blocks > 0x7FFFFFFFLL) return set_error(BTM_ERR_UNSUPPORTED, "grouped matmul: too many output tiles (%lld) for the general kernel", blocks);
    const unsigned grid = (unsigned)blocks;
    if (c.dtype == BTM_F16) {
        if (c.wgrad) gemm_grouped_simt_kernel<BTM_F16, true><<<grid, 256, 0, st>>>(p);
        else gemm_grouped_simt_kernel<BTM_F16, false><<<grid, 256, 0, st>>>(p);
    } else {
        if (c.wgrad) gemm_grouped_simt_kernel<BTM_BF16, true><<<grid, 256, 0, st>>>(p);
        else gemm_grouped_simt_kernel<BTM_BF16, false><<<grid, 256, 0, st>>>(p);
    }
    return check_cuda(cudaGetLastError(), "grouped matmul (general kernel) launch");
}

template <int DT, int MODE>
static int launch_tc(const GroupedCall &c, cudaStream_t st, int grid, const CUtensorMap &tmA, const CUtensorMap &tmA_band, const CUtensorMap &tmB,
                     const CUtensorMap &tmC, const GemmParams &p)
{
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3((unsigned)grid, 1, 1);
    cfg.blockDim = dim3(gg::THREADS, 1, 1);
    cfg.dynamicSmemBytes = gg::SMEM_BYTES;
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    GroupedTables tab = {c.offsets, c.groups, c.rows};
    return check_cuda(cudaLaunchKernelEx(&cfg, gemm_grouped_kernel<DT, MODE>, tmA, tmA_band, tmB, tmC, p, tab), "grouped matmul launch");
}

template <int DT>
static cudaError_t raise_grouped_smem()
{
    cudaError_t e = cudaFuncSetAttribute(gemm_grouped_kernel<DT, GROUPED_KN>, cudaFuncAttributeMaxDynamicSharedMemorySize, gg::SMEM_BYTES);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(gemm_grouped_kernel<DT, GROUPED_NK>, cudaFuncAttributeMaxDynamicSharedMemorySize, gg::SMEM_BYTES);
    if (e == cudaSuccess) e = cudaFuncSetAttribute(gemm_grouped_kernel<DT, GROUPED_WGRAD>, cudaFuncAttributeMaxDynamicSharedMemorySize, gg::SMEM_BYTES);
    return e;
}

int load_grouped_simt_kernels()
{
    cudaFuncAttributes a;
    cudaError_t e = cudaFuncGetAttributes(&a, gemm_grouped_simt_kernel<BTM_F16, true>);
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, gemm_grouped_simt_kernel<BTM_F16, false>);
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, gemm_grouped_simt_kernel<BTM_BF16, true>);
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, gemm_grouped_simt_kernel<BTM_BF16, false>);
    return check_cuda(e, "cudaFuncGetAttributes(grouped general kernel)");
}

int configure_gemm_grouped_kernels()
{
    cudaError_t e = raise_grouped_smem<BTM_F16>();
    if (e == cudaSuccess) e = raise_grouped_smem<BTM_BF16>();
    return check_cuda(e, "cudaFuncSetAttribute(gemm_grouped)");
}

static bool mult16(const void *p, long long ld) { return ((uintptr_t)p & 15) == 0 && (ld * 2) % 16 == 0; }

int launch_gemm_grouped(const GroupedCall &c, cudaStream_t st, int sm_count, int *status)
{
    using namespace gg;
    // Tensor maps take bases and pitches that are multiples of 16 bytes; anything else, an empty reduction and a matrix
    // without rows take the general kernel.
    const bool tc = mult16(c.A, c.lda) && mult16(c.B, c.ldb) && (c.wgrad || c.groups == 1 || (c.strideB * 2) % 16 == 0) && c.rows > 0 &&
                    (c.wgrad || c.K > 0);
    if (!tc) return launch_grouped_simt(c, st, status);
    const char *force = getenv("BTM_FORCE_KERNEL"); // 1cta, 2cta or decode: the tests run every shape on each
    bool decode = !c.wgrad && grouped_decode_fits(c.groups, c.rows, c.N, sm_count);
    if (force) decode = !c.wgrad && !strcmp(force, "decode");
    if (decode) return launch_grouped_decode(c, st, sm_count, status);
    const long long bound = c.wgrad ? (long long)c.groups * ((c.M + BM - 1) / BM) : grouped_slot_bound(c.groups, c.rows);
    const long long most = bound * ((c.N + 63) / 64); // tiles at the smallest width
    if (most > 0x3FFFFFFFLL) return set_error(BTM_ERR_UNSUPPORTED, "grouped matmul: too many output tiles (%lld)", most);

    CUtensorMap tmA, tmA_band, tmB, tmC;
    memset(&tmA_band, 0, sizeof(tmA_band));
    memset(&tmC, 0, sizeof(tmC));
    const uint64_t rows = (uint64_t)c.rows, pa = (uint64_t)c.lda * 2, pb = (uint64_t)c.ldb * 2;
    int rc;
    if (c.wgrad) {
        rc = encode_tmap_3d(&tmA, c.dtype, c.A, (uint64_t)c.M, rows, 1, pa, pa, 64, 64);
        if (!rc) rc = encode_tmap_3d(&tmB, c.dtype, c.B, (uint64_t)c.N, rows, 1, pb, pb, 64, 64);
    } else {
        rc = encode_tmap_3d(&tmA, c.dtype, c.A, (uint64_t)c.K, rows, 1, pa, pa, 64, BM);
        if (!rc) rc = encode_tmap_3d(&tmA_band, c.dtype, c.A, (uint64_t)c.K, rows, 1, pa, pa, 64, A_BAND);
        const uint64_t inner = (uint64_t)(c.b_trans ? c.K : c.N), outer = (uint64_t)(c.b_trans ? c.N : c.K);
        if (!rc) rc = encode_tmap_3d(&tmB, c.dtype, c.B, inner, outer, (uint64_t)c.groups, pb, c.groups > 1 ? (uint64_t)c.strideB * 2 : pb, 64, 64);
    }
    if (rc) return rc;
    GemmParams p;
    memset(&p, 0, sizeof(p));
    p.M = c.wgrad ? c.M : c.rows;
    p.N = c.N;
    p.K = c.K;
    p.batch = c.wgrad ? c.groups : 1;
    p.tiles_m = c.wgrad ? (c.M + BM - 1) / BM : 0;
    p.num_kb = (c.K + BK - 1) / BK;
    p.group_m = 8; // as in gemm_tc.cu
    p.ndst = 1;
    p.C[0] = c.C;
    p.ldc = c.ldc;
    p.strideC = c.strideC;
    p.c_vec_ok = mult16(c.C, c.ldc) && (!c.wgrad || c.groups == 1 || (c.strideC * 2) % 16 == 0) ? 1 : 0;
    p.status = status;
    fill_wait_params(&p, c.wgrad ? c.rows : 0);
    if (p.c_vec_ok) {
        const uint64_t pc = (uint64_t)c.ldc * 2;
        rc = encode_tmap_3d(&tmC, c.dtype, c.C, (uint64_t)c.N, (uint64_t)p.M, (uint64_t)p.batch, pc, p.batch > 1 ? (uint64_t)c.strideC * 2 : pc, 64, 32);
        if (rc) return rc;
    }
    // Pairs of CTAs for tall and deep groups. Measured, one CTA against pairs, bf16, rows / N x K, us after a pause, equal groups;
    // uneven ones (a load of rank^-0.7), in which more slots of a pair are cut:
    //   16384 in 8 groups / 4096 x 4096: 391 / 355; 418 / 379    16384 in 16 / 2048 x 4096: 205 / 186; 230 / 208
    //   12000 in 4 / 2560 x 2560: 129 / 114; 127 / 113           4096 in 16 / 2048 x 4096: 68.8 / 66.8; 94.1 / 79.2
    //   8192 in 8 / 1024 x 1024: 24.6 / 22.1; 23.9 / 24.2        16384 in 64 / 2048 x 2048: 128 / 121; 152 / 164
    //   12000 in 64 / 1024 x 1024: 45.2 / 41.4; 41.6 / 43.2
    // The table of groups is not known here, so the mean height decides.
    // The weight gradient has no pair form (gemm_grouped_pair.cu).
    const long long height = c.rows / c.groups;
    bool pair = !c.wgrad && height >= 256 && height * c.K > 512 * 1024 && (long long)(c.rows / 256) * ((c.N + 255) / 256) >= sm_count / 4;
    if (force) {
        if (!strcmp(force, "1cta")) pair = false;
        else if (!strcmp(force, "2cta")) pair = !c.wgrad;
    }
    if (pair) return launch_gemm_grouped_pair(c, st, sm_count, tmA, tmA_band, tmB, tmC, p);
    const int grid = (int)(most < sm_count ? most : sm_count);
#define BTM_GROUPED_CASE(DT)                                                                                    \
    do {                                                                                                        \
        if (c.wgrad) return launch_tc<DT, GROUPED_WGRAD>(c, st, grid, tmA, tmA_band, tmB, tmC, p);              \
        if (c.b_trans) return launch_tc<DT, GROUPED_NK>(c, st, grid, tmA, tmA_band, tmB, tmC, p);               \
        return launch_tc<DT, GROUPED_KN>(c, st, grid, tmA, tmA_band, tmB, tmC, p);                              \
    } while (0)
    if (c.dtype == BTM_F16) BTM_GROUPED_CASE(BTM_F16);
    BTM_GROUPED_CASE(BTM_BF16);
#undef BTM_GROUPED_CASE
}

} // namespace btm
