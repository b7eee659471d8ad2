// Products with few rows per group (decoding): 16-bit weights in either storage order, or microscaled 4-bit ones.
//
// What such a call costs is the weights' way from memory, and with few tiles its latency. So the product is computed
// transposed: 128 weight rows (columns of the output) are the tensor core's A operand and the token rows its B operand
// (UMMA N = the tokens of the tile rounded up to 16), no tensor-core row is spent on padding; K is split over the CTAs
// of a cluster so that all SMs pull weights, two CTAs on each. Every CTA streams its K slice through a ring, parks its
// accumulator in shared memory, and after one cluster barrier CTA r adds the columns (tokens) r, r + S, .. over all CTAs,
// in rank order, through distributed shared memory, rounds once and stores rows of 256 contiguous bytes.
// Nothing depends on which CTA is first, so a call gives the same bits every time.
//
// Groups are cut into slots of 64 tokens; one with more is read again for each further slot, from L2.
//
// Warp roles: 0 weights and tokens by TMA, 1 tcgen05.mma, 2 scales by TMA (microscaled), 4-7 park; all store.
// The weights of a plain product (microscaled only) depend on no table: they are asked into L2 before griddepcontrol.wait,
// under the kernel before (the quantiser of the activations). That is a hint only; they are read after the wait.
#include <cstring>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "btm_internal.h"
#include "btm_ptx.cuh"
#include "grouped_tile.cuh"
#include "mxfp4.cuh"

namespace btm {

enum DecodeKind { DECODE_KN = 0 /* w[g] is [K, N] */, DECODE_NK = 1 /* w[g] is [N, K] */, DECODE_MX = 2 };

namespace dec {
constexpr int BW = 128;                  // weight rows of a tile
constexpr int SLOT = 64;                 // most tokens of a tile
constexpr int W_BYTES = BW * 128;        // weights per unit: 64 k of 16 bits, 256 k of 4 bits
constexpr int CHUNK_BYTES = 64 * 128;
constexpr int SF_BYTES = 2 * MX_SCALE_BYTES;
constexpr int MAX_STAGES = 6;
constexpr int RING_BYTES = 106 * 1024;   // two CTAs per SM
constexpr int SMEM_BYTES = RING_BYTES + 1024;
constexpr int TMEM_COLS = 256;           // accumulator, scales of six stages
constexpr int SF_COL = SLOT;
constexpr int SF_STAGE_COLS = 16;        // weights 2 x 4 columns, tokens 2 x 4
constexpr int THREADS = 256;
constexpr int MAX_SPLIT = 8;
static_assert(SLOT * BW * 4 <= RING_BYTES, "the parked accumulator takes the ring's place");
static_assert(SF_COL + MAX_STAGES * SF_STAGE_COLS <= TMEM_COLS, "accumulator and scales share tensor memory");
} // namespace dec

struct DecodeMaps {
    CUtensorMap w, tok, sfw, sft;
};
struct DecodeArgs {
    int rows, groups, N, K;
    const int *offsets;
    int units;      // K in units (64 or 256 k)
    int n_blocks;   // 128-column tiles
    int box_rows;   // token rows per box: 16, 32 or 64
    int stages;
    uint32_t stage_bytes;
    void *out;
    long long ldo;
    int vec;        // 8-byte stores are legal
    int *status;
    long long wait_limit;
    int skip_loads;
    int debug_bounds;    // as GemmParams: hand-computed store addresses are compared with the extent of the output
    long long extent;
};

template <int DT, int KIND>
__global__ void __launch_bounds__(dec::THREADS, 2) grouped_decode_kernel(const __grid_constant__ DecodeMaps maps, const __grid_constant__ DecodeArgs a)
{
    using namespace dec;
    constexpr bool kMx = KIND == DECODE_MX;
    constexpr int UNIT_X = kMx ? 128 : 64; // innermost coordinate per unit
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t bar_full[MAX_STAGES], bar_empty[MAX_STAGES], bar_acc;
    __shared__ uint32_t tmem_base_holder;
    __shared__ int abort_flag;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint32_t csize, crank;
    asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(csize));
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(crank));
    const int tile = (int)(blockIdx.x / csize);
    const int slot = tile / a.n_blocks, n0 = (tile - slot * a.n_blocks) * BW;
    // This CTA's units of K.
    const int u0 = (int)((uint32_t)a.units * crank / csize), u1 = (int)((uint32_t)a.units * (crank + 1) / csize);
    const int n_units = u1 - u0;

    if (threadIdx.x == 0) {
        abort_flag = 0;
        for (int s = 0; s < a.stages; ++s) {
            mbar_init(smem_u32(&bar_full[s]), 1);
            mbar_init(smem_u32(&bar_empty[s]), 1);
        }
        mbar_init(smem_u32(&bar_acc), 1);
        fence_mbar_init();
        prefetch_tmap(&maps.tok);
        if (kMx) prefetch_tmap(&maps.sft);
    }
    if (warp == 1) {
        tmem_alloc<1>(smem_u32(&tmem_base_holder), TMEM_COLS);
        tmem_relinquish<1>();
    }
    if constexpr (kMx) { // the 16-bit products always have a table
        if (warp == 2 && a.offsets == nullptr && elect_one()) {
            for (int u = u0; u < u1; ++u) {
                tma_prefetch_3d(&maps.w, u * UNIT_X, n0, 0);
                tma_prefetch_3d(&maps.sfw, u * 256, n0 / 128, 0);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_holder;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    int g = 0, lo = 0, hi = a.rows, m0 = slot * SLOT, single = slot >> 1;
    bool live = true;
    if (a.offsets != nullptr) {
        GroupWalk<SLOT> walk;
        walk.init(a.offsets, a.groups, a.rows);
        const int total = walk.count_slots();
        if (blockIdx.x == 0 && warp == 0) walk.report(a.status);
        live = slot < total;
        if (live) {
            int first;
            walk.find_slot(slot, g, lo, hi, first);
            m0 = lo + (slot - first) * SLOT;
            single = walk.singles_of(g, hi - lo) + ((slot - first) >> 1);
        }
    }
    const int valid = live ? min(SLOT, hi - m0) : 0; // tokens of this tile
    const int n_inst = (valid + 15) & ~15;

    if (!live) {
        // The launch is sized for the most slots the rows can fill.
    } else if (warp == 0) {
        // ------------------------------------------------------------ TMA: weights and tokens
        const int gu = uniform(g), mu = uniform(m0);
        const uint32_t bytes = (uint32_t)(W_BYTES + a.box_rows * 128 + (kMx ? 2 * SF_BYTES : 0));
        int stage = 0;
        uint32_t phase = 0;
        for (int i = 0; i < n_units && !a.skip_loads; ++i) {
            if (i >= a.stages && !mbar_wait_uniform(smem_u32(&bar_empty[stage]), phase ^ 1u, &abort_flag, a.status, WAIT_PRODUCER_EMPTY, a.wait_limit)) break;
            if (elect_one()) {
                const uint32_t full = smem_u32(&bar_full[stage]), w0 = smem_base + (uint32_t)stage * a.stage_bytes;
                const int x = (u0 + i) * UNIT_X;
                mbar_expect_tx(full, bytes);
                if (KIND == DECODE_KN) {
                    tma_load_3d(w0, &maps.w, n0, x, gu, full);
                    tma_load_3d(w0 + CHUNK_BYTES, &maps.w, n0 + 64, x, gu, full);
                } else {
                    tma_load_3d(w0, &maps.w, x, n0, gu, full);
                }
                tma_load_3d(w0 + W_BYTES + (kMx ? 2 * SF_BYTES : 0), &maps.tok, x, mu, 0, full);
            }
            __syncwarp();
            if (++stage == a.stages) {
                stage = 0;
                phase ^= 1u;
            }
        }
    } else if (warp == 2 && kMx) {
        // ------------------------------------------------------------ TMA: scales
        const int gu = uniform(g), su = uniform(single);
        int stage = 0;
        uint32_t phase = 0;
        for (int i = 0; i < n_units && !a.skip_loads; ++i) {
            if (i >= a.stages && !mbar_wait_uniform(smem_u32(&bar_empty[stage]), phase ^ 1u, &abort_flag, a.status, WAIT_PRODUCER_EMPTY, a.wait_limit)) break;
            if (elect_one()) {
                const uint32_t full = smem_u32(&bar_full[stage]), s0 = smem_base + (uint32_t)stage * a.stage_bytes + W_BYTES;
                tma_load_3d(s0, &maps.sfw, (u0 + i) * 256, n0 / 128, gu, full);
                tma_load_3d(s0 + SF_BYTES, &maps.sft, (u0 + i) * 256, su, 0, full);
            }
            __syncwarp();
            if (++stage == a.stages) {
                stage = 0;
                phase ^= 1u;
            }
        }
    } else if (warp == 1) {
        // ------------------------------------------------------------ MMA issuer
        const uint32_t tmem_u = uniform(tmem_base), n_u = (uint32_t)uniform(n_inst);
        const uint32_t skip = kMx ? ((uint32_t)uniform((m0 - lo) & 64) >> 5) : 0; // second half of a 128-row scale block: two columns in
        constexpr uint32_t kFmt = DT == BTM_BF16 ? 1u : 0u;
        const uint32_t idesc0 = kMx ? make_idesc_mxf4(BW, n_u, 0) : make_idesc(kFmt, KIND == DECODE_KN, false, BW, n_u);
        const uint32_t idesc1 = make_idesc_mxf4(BW, n_u, 2);
        int stage = 0;
        uint32_t phase = 0;
        bool ok = true;
        for (int i = 0; i < n_units; ++i) {
            ok = mbar_wait_uniform(smem_u32(&bar_full[stage]), phase, &abort_flag, a.status, WAIT_MMA_FULL, a.wait_limit);
            if (!ok) break;
            tc_fence_after();
            const uint32_t w0 = smem_base + (uint32_t)stage * a.stage_bytes;
            const uint32_t t0 = w0 + W_BYTES + (kMx ? 2 * SF_BYTES : 0);
            const uint64_t wd = KIND == DECODE_KN ? make_smem_desc_sw128(w0, CHUNK_BYTES, 1024) : make_smem_desc_sw128(w0, 16, 1024);
            const uint64_t td = make_smem_desc_sw128(t0, 16, 1024);
            if (elect_one()) {
                if constexpr (kMx) {
                    const uint64_t sw = make_smem_desc_rows16(w0 + W_BYTES), stk = make_smem_desc_rows16(w0 + W_BYTES + SF_BYTES);
                    const uint32_t sf = tmem_u + SF_COL + (uint32_t)(stage * SF_STAGE_COLS);
                    const int steps = min(4, (a.K - (u0 + i) * 256 + 63) / 64);
#pragma unroll
                    for (int c = 0; c < 2; ++c) {
                        if (c * 2 < steps) {
                            tmem_cp_32x128b<1>(sf + c * 4, sw + (uint64_t)(c * MX_SCALE_BYTES >> 4));
                            tmem_cp_32x128b<1>(sf + 8 + c * 4, stk + (uint64_t)(c * MX_SCALE_BYTES >> 4));
                        }
                    }
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks)
                        if (ks < steps)
                            umma_mxf4<1>(tmem_u, wd + (uint64_t)(ks * 2), td + (uint64_t)(ks * 2), (ks & 1) ? idesc1 : idesc0, sf + (ks >> 1) * 4,
                                         sf + 8 + (ks >> 1) * 4 + skip, (uint32_t)((i | ks) != 0));
                } else {
                    constexpr uint32_t w_step = (KIND == DECODE_KN ? 16 * 128 : 32) >> 4;
#pragma unroll
                    for (int ks = 0; ks < 4; ++ks)
                        umma<1, false>(tmem_u, wd + (uint64_t)(ks * w_step), td + (uint64_t)(ks * 2), idesc0, (uint32_t)((i | ks) != 0));
                }
                umma_commit(smem_u32(&bar_empty[stage]));
            }
            __syncwarp();
            if (++stage == a.stages) {
                stage = 0;
                phase ^= 1u;
            }
        }
        if (ok && elect_one()) umma_commit(smem_u32(&bar_acc));
        __syncwarp();
    } else if (warp >= 4) {
        mbar_wait_uniform(smem_u32(&bar_acc), 0u, &abort_flag, a.status, WAIT_EPI_TMEM_FULL, a.wait_limit);
    }

    // ---------------------------------------------------------------- K reduction over the cluster, output
    __syncthreads(); // the ring is dead: its loads and MMAs are over
    tc_fence_after();
    float *park = reinterpret_cast<float *>(smem_raw + (smem_base - smem_u32(smem_raw))); // [token][128 weight rows]
    const bool acc_ok = abort_flag == 0;
    if (live && warp >= 4) {
        const int quad = warp & 3;
#pragma unroll 1
        for (int c0 = 0; c0 < valid; c0 += 32) {
            uint32_t v[32];
            tmem_ld_32x32(tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)c0, v);
            tmem_ld_wait();
#pragma unroll
            for (int c = 0; c < 32; ++c)
                if (c0 + c < valid) park[(c0 + c) * BW + quad * 32 + lane] = __uint_as_float(v[c]);
        }
    }
    if (csize > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
    else __syncthreads();
    if (live && acc_ok) {
        // A warp takes a token: lane l sums the weight rows 4 l .. 4 l + 3 over the cluster.
        const uint32_t mine = smem_base + (uint32_t)lane * 16u;
        uint32_t src[MAX_SPLIT];
#pragma unroll
        for (int r = 0; r < MAX_SPLIT; ++r) {
            asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(src[r]) : "r"(mine), "r"(r < (int)csize ? r : 0));
        }
        const int n = n0 + lane * 4;
        for (int c = (int)crank + warp * (int)csize; c < valid; c += (int)csize * (THREADS / 32)) {
            float4 x[MAX_SPLIT];
#pragma unroll
            for (int r = 0; r < MAX_SPLIT; ++r)
                if (r < (int)csize)
                    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                                 : "=f"(x[r].x), "=f"(x[r].y), "=f"(x[r].z), "=f"(x[r].w)
                                 : "r"(src[r] + (uint32_t)c * (BW * 4)));
            float4 s = x[0];
#pragma unroll
            for (int r = 1; r < MAX_SPLIT; ++r)
                if (r < (int)csize) {
                    s.x += x[r].x;
                    s.y += x[r].y;
                    s.z += x[r].z;
                    s.w += x[r].w;
                }
            uint32_t q[2];
            if constexpr (DT == BTM_F16) {
                const __half2 h0 = __floats2half2_rn(s.x, s.y), h1 = __floats2half2_rn(s.z, s.w);
                q[0] = *reinterpret_cast<const uint32_t *>(&h0);
                q[1] = *reinterpret_cast<const uint32_t *>(&h1);
            } else {
                const __nv_bfloat162 h0 = __floats2bfloat162_rn(s.x, s.y), h1 = __floats2bfloat162_rn(s.z, s.w);
                q[0] = *reinterpret_cast<const uint32_t *>(&h0);
                q[1] = *reinterpret_cast<const uint32_t *>(&h1);
            }
            const long long off = (long long)(m0 + c) * a.ldo + n;
            uint16_t *dst = reinterpret_cast<uint16_t *>(a.out) + off;
            if (a.debug_bounds && n < a.N && off + min(4, a.N - n) > a.extent) {
                atomicCAS(a.status, 0, (int)BOUNDS_STORE);
                continue;
            }
            if (a.vec && n + 4 <= a.N) {
                *reinterpret_cast<uint2 *>(dst) = make_uint2(q[0], q[1]);
            } else {
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    if (n + e < a.N) dst[e] = (uint16_t)((e & 1) ? (q[e >> 1] >> 16) : (q[e >> 1] & 0xFFFFu));
            }
        }
    }
    // Every CTA of the cluster has read what it needs of this one's parked accumulator.
    if (csize > 1) asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");

    tc_fence_before();
    __syncthreads();
    if (abort_flag) {
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) {}
        __syncthreads();
    }
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc<1>(tmem_base, TMEM_COLS);
    }
}

template <int DT, int KIND>
static int launch_decode(cudaStream_t st, const DecodeMaps &maps, const DecodeArgs &a, int split, long long blocks)
{
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3((unsigned)blocks, 1, 1);
    cfg.blockDim = dim3(dec::THREADS, 1, 1);
    cfg.dynamicSmemBytes = dec::SMEM_BYTES;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)split;
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 2;
    return check_cuda(cudaLaunchKernelEx(&cfg, grouped_decode_kernel<DT, KIND>, maps, a), "decode matmul launch");
}

static long long slot_bound(int groups, int rows)
{
    const long long nonempty = groups < rows ? groups : rows;
    return ((long long)rows + (dec::SLOT - 1) * nonempty) / dec::SLOT;
}

// Is this launch one for the decode form? As long as all its tiles are resident at once, two per SM: the split along K then
// buys parallelism, while further waves would pay this kernel's set-up again and again. Measured, persistent kernel against
// this one (rows / groups / N x K, tiles at most), us in a run, equal groups; uneven ones (a load of rank^-0.7):
//   microscaled  1 / 1 / 11008 x 4096 (86): 10.2 / 7.7            64 / 8 / 4096 x 4096 (256): 18.2 / 15.6; 18.1 / 15.6
//                1000 / 24 / 1000 x 1440 (312): 9.2 / 10.8; 10.6 / 11.2   512 / 8 / 4096 x 4096 (480): 19.3 / 18.9; 20.2 / 24.9
//                256 / 64 / 2048 x 2048 (1040): 30.4 / 35.5; 29.2 / 32.9
//   bf16         2 / 8 / 1024 x 1024 (16): 8.7 / 5.2              515 / 16 / 1024 x 512 (184): 7.3 / 6.7; 7.3 / 7.7
//                256 / 8 / 4096 x 4096 (352): 49.5 / 45.2; 49.4 / 46.9    512 / 8 / 4096 x 4096 (480): 51.2 / 48.8; 53.5 / 63.5
//                2000 / 40 / 1000 x 1416 (560): 31.6 / 37.2; 33.4 / 40.0
// Just beyond two per SM either may be ahead by some per cent; the border is where the tiles stop being resident.
bool grouped_decode_fits(int groups, int rows, int N, int sm_count) { return slot_bound(groups, rows) * ((N + dec::BW - 1) / dec::BW) <= 2LL * sm_count; }

// Fills what all kinds share; returns the launch's split and block count.
static int prepare(DecodeArgs *a, int rows, int groups, int N, int K, const int *offsets, void *out, long long ldo, int *status, int sm_count,
                   bool mx, int *split, long long *blocks)
{
    using namespace dec;
    memset(a, 0, sizeof(*a));
    a->rows = rows; a->groups = groups; a->N = N; a->K = K; a->offsets = offsets;
    a->units = mx ? (K + 255) / 256 : (K + 63) / 64;
    a->n_blocks = (N + BW - 1) / BW;
    a->box_rows = rows <= 16 ? 16 : rows <= 32 ? 32 : 64;
    a->stage_bytes = (uint32_t)(W_BYTES + a->box_rows * 128 + (mx ? 2 * SF_BYTES : 0));
    a->stages = (int)((uint32_t)RING_BYTES / a->stage_bytes);
    if (a->stages > MAX_STAGES) a->stages = MAX_STAGES;
    a->out = out; a->ldo = ldo;
    a->vec = ((uintptr_t)out & 7) == 0 && ldo % 4 == 0;
    GemmParams p;
    memset(&p, 0, sizeof(p));
    p.M = rows; p.N = N; p.K = K; p.batch = 1; p.ldc = ldo;
    fill_wait_params(&p);
    a->status = status;
    a->wait_limit = p.wait_limit;
    a->skip_loads = p.debug_skip_loads;
    a->debug_bounds = p.debug_bounds;
    a->extent = p.c_extent;
    const long long tiles = slot_bound(groups, rows) * a->n_blocks;
    // K over as many CTAs as two per SM leave room for.
    long long s = 2LL * sm_count / tiles;
    if (s > MAX_SPLIT) s = MAX_SPLIT;
    if (s > a->units) s = a->units;
    if (s < 1) s = 1;
    *split = (int)s;
    *blocks = tiles * s;
    if (*blocks > 0x7FFFFFFFLL) return set_error(BTM_ERR_UNSUPPORTED, "grouped matmul: too many output tiles (%lld)", tiles);
    return BTM_OK;
}

// Preconditions of the 16-bit form: bases and pitches are multiples of 16 bytes, rows, N, K > 0.
int launch_grouped_decode(const GroupedCall &c, cudaStream_t st, int sm_count, int *status)
{
    using namespace dec;
    DecodeArgs a;
    int split;
    long long blocks;
    int rc = prepare(&a, c.rows, c.groups, c.N, c.K, c.offsets, c.C, c.ldc, status, sm_count, false, &split, &blocks);
    if (rc) return rc;
    DecodeMaps maps;
    memset(&maps, 0, sizeof(maps));
    const uint64_t pa = (uint64_t)c.lda * 2, pb = (uint64_t)c.ldb * 2, pg = c.groups > 1 ? (uint64_t)c.strideB * 2 : pb;
    rc = encode_tmap_3d(&maps.tok, c.dtype, c.A, (uint64_t)c.K, (uint64_t)c.rows, 1, pa, pa, 64, (uint32_t)a.box_rows);
    if (!rc)
        rc = c.b_trans ? encode_tmap_3d(&maps.w, c.dtype, c.B, (uint64_t)c.K, (uint64_t)c.N, (uint64_t)c.groups, pb, pg, 64, BW)
                       : encode_tmap_3d(&maps.w, c.dtype, c.B, (uint64_t)c.N, (uint64_t)c.K, (uint64_t)c.groups, pb, pg, 64, 64);
    if (rc) return rc;
    if (c.dtype == BTM_F16)
        return c.b_trans ? launch_decode<BTM_F16, DECODE_NK>(st, maps, a, split, blocks) : launch_decode<BTM_F16, DECODE_KN>(st, maps, a, split, blocks);
    return c.b_trans ? launch_decode<BTM_BF16, DECODE_NK>(st, maps, a, split, blocks) : launch_decode<BTM_BF16, DECODE_KN>(st, maps, a, split, blocks);
}

int launch_mxfp4_decode(const Mxfp4Call &c, cudaStream_t st, int sm_count, int *status)
{
    using namespace dec;
    DecodeArgs a;
    int split;
    long long blocks;
    int rc = prepare(&a, c.rows, c.groups, c.N, c.K, c.offsets, c.out, c.ldo, status, sm_count, true, &split, &blocks);
    if (rc) return rc;
    DecodeMaps maps;
    const uint64_t pitch = (uint64_t)c.K / 2;
    rc = encode_tmap_3d(&maps.tok, BTM_U8, c.act, pitch, (uint64_t)c.rows, 1, pitch, pitch, 128, (uint32_t)a.box_rows);
    if (!rc) rc = encode_tmap_3d(&maps.w, BTM_U8, c.w, pitch, (uint64_t)c.N, (uint64_t)c.groups, pitch, pitch * (uint64_t)c.N, 128, BW);
    if (!rc) rc = encode_mx_scales(&maps.sft, c.act_scales, c.K, (uint64_t)grouped_slot_bound(c.groups, c.rows), 1, 1);
    if (!rc) rc = encode_mx_scales(&maps.sfw, c.w_scales, c.K, (uint64_t)a.n_blocks, (uint64_t)c.groups, 1);
    if (rc) return rc;
    return c.dtype == BTM_F16 ? launch_decode<BTM_F16, DECODE_MX>(st, maps, a, split, blocks) : launch_decode<BTM_BF16, DECODE_MX>(st, maps, a, split, blocks);
}

template <int DT, int KIND>
static cudaError_t raise_decode_smem()
{
    return cudaFuncSetAttribute(grouped_decode_kernel<DT, KIND>, cudaFuncAttributeMaxDynamicSharedMemorySize, dec::SMEM_BYTES);
}

int configure_grouped_decode_kernels()
{
    cudaError_t e = raise_decode_smem<BTM_F16, DECODE_KN>();
    if (e == cudaSuccess) e = raise_decode_smem<BTM_F16, DECODE_NK>();
    if (e == cudaSuccess) e = raise_decode_smem<BTM_F16, DECODE_MX>();
    if (e == cudaSuccess) e = raise_decode_smem<BTM_BF16, DECODE_KN>();
    if (e == cudaSuccess) e = raise_decode_smem<BTM_BF16, DECODE_NK>();
    if (e == cudaSuccess) e = raise_decode_smem<BTM_BF16, DECODE_MX>();
    return check_cuda(e, "cudaFuncSetAttribute(grouped_decode)");
}

} // namespace btm
