// Matrix products grouped by expert with ragged sizes: the rows of A are sorted by group, offsets[g] .. offsets[g + 1]
// are the rows of group g (a device-side table, grouped_rows.cuh).
//   product:          C[r, :] = A[r, :] . B[g]                   r in group g
//   weight gradient:  C[g]    = A[rows of g]^T . D[rows of g]    (all zero for a group without rows)
//
// General kernel (operands that TMA cannot address, K == 0): 64 x 64 output tiles on CUDA cores as in gemm_simt.cu, fp32
// accumulation, one rounding. A block finds its group by walking the table.
#include <cstring>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "btm_internal.h"
#include "btm_ptx.cuh"
#include "grouped_rows.cuh"

namespace btm {

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
    GroupWalk walk;
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

int launch_gemm_grouped(const GroupedCall &c, cudaStream_t st, int sm_count, int *status)
{
    (void)sm_count;
    return launch_grouped_simt(c, st, status);
}

} // namespace btm
