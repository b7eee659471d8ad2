// Microscaled 4-bit operands: quantisation and its inverse (format: mxfp4.cuh; the product is in mxfp4_tc.cu).
//
// Quantise: for a block of 32 values, X = floor(log2(max |x|)) - 2 (the largest E2M1 value is 1.5 * 2^2), clamped to
// [-127, 127], and q = x / 2^X rounded to nearest (ties to the even code) and saturated at 6. A division by a power of two
// is exact, so the only rounding is the one to four bits. A block that holds an infinity or a NaN has no such scale: it
// gets scale 255 (NaN) and zero codes, and everything that it enters becomes NaN. Dequantise: q 2^X, rounded once.
#include <cstring>
#include <type_traits>

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "btm_internal.h"
#include "btm_ptx.cuh"
#include "grouped_rows.cuh"
#include "mxfp4.cuh"

namespace btm {

namespace mxq {
constexpr int THREADS = 256; // 16 threads x 8 values across a scale block's 128 k, 16 rows at a time
constexpr int ROWS = 16;
constexpr int PASSES = GROUP_SLOT_ROWS / ROWS;
} // namespace mxq

// Which rows does this block's slot hold? Uniform groups by arithmetic, others through the table. False: no such slot.
__device__ __forceinline__ bool slot_rows(int slot, const int *offsets, int groups, int rows, int *status, int &row0, int &row_end)
{
    if (offsets == nullptr) {
        const int per = rows / groups, slots = (per + GROUP_SLOT_ROWS - 1) / GROUP_SLOT_ROWS;
        const int g = slot / slots, m = slot - g * slots;
        row0 = g * per + m * GROUP_SLOT_ROWS;
        row_end = (g + 1) * per;
    } else {
        GroupWalk<> walk;
        walk.init(offsets, groups, rows);
        const int total = walk.count_slots();
        if (blockIdx.x == 0 && threadIdx.x < 32) walk.report(status);
        if (slot >= total) return false;
        int g, lo, first;
        walk.find_slot(slot, g, lo, row_end, first);
        row0 = lo + (slot - first) * GROUP_SLOT_ROWS;
    }
    row_end = min(row_end, row0 + GROUP_SLOT_ROWS);
    return true;
}

template <typename T>
__device__ __forceinline__ void load8(const T *p, bool vec, float (&v)[8])
{
    if constexpr (sizeof(T) == 4) {
        if (vec) {
            const float4 a = *reinterpret_cast<const float4 *>(p), b = *reinterpret_cast<const float4 *>(p + 4);
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) v[i] = p[i];
        }
    } else {
        uint4 q;
        if (vec) {
            q = *reinterpret_cast<const uint4 *>(p);
        } else {
            const uint16_t *s = reinterpret_cast<const uint16_t *>(p);
            q.x = s[0] | ((uint32_t)s[1] << 16);
            q.y = s[2] | ((uint32_t)s[3] << 16);
            q.z = s[4] | ((uint32_t)s[5] << 16);
            q.w = s[6] | ((uint32_t)s[7] << 16);
        }
        const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (sizeof(T) == 2 && std::is_same<T, __half>::value) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&w[i]));
                v[2 * i] = f.x;
                v[2 * i + 1] = f.y;
            } else {
                v[2 * i] = __uint_as_float(w[i] << 16);
                v[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
            }
        }
    }
}

// One block of 128 rows x 128 k per CTA: its 512 bytes of scales are put together in shared memory and written whole.
template <typename T>
__global__ void __launch_bounds__(mxq::THREADS) mxfp4_quantize_kernel(const T *__restrict__ x, long long ldx, int vec, int groups, int rows, int K,
                                                                      const int *offsets, uint8_t *__restrict__ packed,
                                                                      uint8_t *__restrict__ scales, int *status)
{
    using namespace mxq;
    __shared__ __align__(16) uint8_t sc[MX_SCALE_BYTES];
    const int chunks = mx_chunks(K);
    const int slot = blockIdx.x / chunks, chunk = blockIdx.x - slot * chunks;
    int row0, row_end;
    if (!slot_rows(slot, offsets, groups, rows, status, row0, row_end)) return;
    const int tr = threadIdx.x >> 4, tk = threadIdx.x & 15;
    const int k = chunk * MX_CHUNK_K + tk * 8;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int r = i * ROWS + tr, row = row0 + r;
        const bool in = row < row_end && k < K; // K is a multiple of 32: a block's four threads agree
        float v[8] = {};
        if (in) load8(x + (long long)row * ldx + k, vec != 0, v);
        uint32_t top = 0; // largest magnitude as an integer: ordered like the values, NaN above infinity
#pragma unroll
        for (int j = 0; j < 8; ++j) top = max(top, __float_as_uint(v[j]) & 0x7FFFFFFFu);
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = max(top, __shfl_xor_sync(0xffffffffu, top, 2));
        const uint32_t e = top >> 23;
        uint32_t s = e > 2u ? e - 2u : 0u;
        float inv = __uint_as_float((254u - s) << 23); // 2^-X, a normal number for every s
        if (e == 255u) {
            s = MX_NAN;
            inv = 0.0f;
        }
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = e == 255u ? 0.0f : v[j] * inv;
        if (in) *reinterpret_cast<uint32_t *>(packed + (long long)row * (K / 2) + (k >> 1)) = mx_encode8(v);
        if ((tk & 3) == 0) sc[mx_scale_at(r, tk >> 2)] = (uint8_t)s; // 0 outside the matrix
    }
    __syncthreads();
    if (threadIdx.x < MX_SCALE_BYTES / 16)
        reinterpret_cast<uint4 *>(scales + ((long long)slot * chunks + chunk) * MX_SCALE_BYTES)[threadIdx.x] = reinterpret_cast<const uint4 *>(sc)[threadIdx.x];
}

template <typename T>
__device__ __forceinline__ T round_to(float v);
template <>
__device__ __forceinline__ float round_to<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half round_to<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 round_to<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

template <typename T>
__global__ void __launch_bounds__(mxq::THREADS) mxfp4_dequant_kernel(const uint8_t *__restrict__ packed, const uint8_t *__restrict__ scales,
                                                                     int groups, int rows, int K, const int *offsets, T *__restrict__ out,
                                                                     long long ldo, int vec, int *status)
{
    using namespace mxq;
    const int chunks = mx_chunks(K);
    const int slot = blockIdx.x / chunks, chunk = blockIdx.x - slot * chunks;
    int row0, row_end;
    if (!slot_rows(slot, offsets, groups, rows, status, row0, row_end)) return;
    const uint8_t *sc = scales + ((long long)slot * chunks + chunk) * MX_SCALE_BYTES;
    const int tr = threadIdx.x >> 4, tk = threadIdx.x & 15;
    const int k = chunk * MX_CHUNK_K + tk * 8;
    if (k >= K) return;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int r = i * ROWS + tr, row = row0 + r;
        if (row >= row_end) continue;
        const float s = mx_scale_value(sc[mx_scale_at(r, tk >> 2)]);
        uint32_t h[4];
        mx_decode8(*reinterpret_cast<const uint32_t *>(packed + (long long)row * (K / 2) + (k >> 1)), h);
        __align__(16) T v[8];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&h[j]));
            v[2 * j] = round_to<T>(f.x * s);
            v[2 * j + 1] = round_to<T>(f.y * s);
        }
        T *dst = out + (long long)row * ldo + k;
        if (vec) {
#pragma unroll
            for (int j = 0; j < (int)(sizeof(v) / 16); ++j) reinterpret_cast<uint4 *>(dst)[j] = reinterpret_cast<const uint4 *>(v)[j];
        } else {
#pragma unroll
            for (int j = 0; j < 8; ++j) dst[j] = v[j];
        }
    }
}

static int slot_grid(int groups, int rows, int K, const int *offsets, unsigned *grid)
{
    const long long slots = offsets ? grouped_slot_bound(groups, rows) : (long long)groups * (((rows / groups) + GROUP_SLOT_ROWS - 1) / GROUP_SLOT_ROWS);
    const long long blocks = slots * mx_chunks(K);
    if (blocks > 0x7FFFFFFFLL) return set_error(BTM_ERR_UNSUPPORTED, "mxfp4: operand too large (%lld scale blocks)", blocks);
    *grid = (unsigned)blocks;
    return BTM_OK;
}

int launch_mxfp4_quantize(cudaStream_t st, int src_dtype, int groups, int rows, int K, const int *offsets, const void *x, long long ldx,
                          void *packed, void *scales, int *status)
{
    unsigned grid;
    if (int rc = slot_grid(groups, rows, K, offsets, &grid)) return rc;
    if (grid == 0) return BTM_OK;
    const int es = src_dtype == BTM_F32 ? 4 : 2;
    const int vec = ((uintptr_t)x & 15) == 0 && (ldx * es) % 16 == 0;
    uint8_t *pk = (uint8_t *)packed, *sc = (uint8_t *)scales;
    if (src_dtype == BTM_F32) mxfp4_quantize_kernel<float><<<grid, mxq::THREADS, 0, st>>>((const float *)x, ldx, vec, groups, rows, K, offsets, pk, sc, status);
    else if (src_dtype == BTM_F16) mxfp4_quantize_kernel<__half><<<grid, mxq::THREADS, 0, st>>>((const __half *)x, ldx, vec, groups, rows, K, offsets, pk, sc, status);
    else mxfp4_quantize_kernel<__nv_bfloat16><<<grid, mxq::THREADS, 0, st>>>((const __nv_bfloat16 *)x, ldx, vec, groups, rows, K, offsets, pk, sc, status);
    return check_cuda(cudaGetLastError(), "mxfp4 quantise launch");
}

int launch_mxfp4_dequant(cudaStream_t st, int dst_dtype, int groups, int rows, int K, const int *offsets, const void *packed,
                         const void *scales, void *out, long long ldo, int *status)
{
    unsigned grid;
    if (int rc = slot_grid(groups, rows, K, offsets, &grid)) return rc;
    if (grid == 0) return BTM_OK;
    const int es = dst_dtype == BTM_F32 ? 4 : 2;
    const int vec = ((uintptr_t)out & 15) == 0 && (ldo * es) % 16 == 0;
    const uint8_t *pk = (const uint8_t *)packed, *sc = (const uint8_t *)scales;
    if (dst_dtype == BTM_F32) mxfp4_dequant_kernel<float><<<grid, mxq::THREADS, 0, st>>>(pk, sc, groups, rows, K, offsets, (float *)out, ldo, vec, status);
    else if (dst_dtype == BTM_F16) mxfp4_dequant_kernel<__half><<<grid, mxq::THREADS, 0, st>>>(pk, sc, groups, rows, K, offsets, (__half *)out, ldo, vec, status);
    else mxfp4_dequant_kernel<__nv_bfloat16><<<grid, mxq::THREADS, 0, st>>>(pk, sc, groups, rows, K, offsets, (__nv_bfloat16 *)out, ldo, vec, status);
    return check_cuda(cudaGetLastError(), "mxfp4 dequantise launch");
}

} // namespace btm
