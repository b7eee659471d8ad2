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

struct SlotRows {
    int first, end; // rows of the slot; empty when there is no such slot
};

// Which rows does this block's slot hold? Uniform groups by arithmetic. Ragged ones from the table, 256 groups at a time, a
// thread each: running maximum (a decreasing entry counts as the one before it) and running slot count over the block.
// A warp's walk (GroupWalk) would take its 32 groups at a time one after the other: 8.7 against 4.4 us for 64 groups.
__device__ __forceinline__ SlotRows slot_rows(int slot, const int *offsets, int groups, int rows, int *status)
{
    if (offsets == nullptr) {
        const int per = rows / groups, slots = (per + GROUP_SLOT_ROWS - 1) / GROUP_SLOT_ROWS;
        const int g = slot / slots, first = g * per + (slot - g * slots) * GROUP_SLOT_ROWS;
        return {first, min((g + 1) * per, first + GROUP_SLOT_ROWS)};
    }
    __shared__ int warp_top[mxq::THREADS / 32], warp_slots[mxq::THREADS / 32];
    __shared__ SlotRows found;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) found = {0, 0};
    const int raw0 = offsets[0];
    int floor_row = min(max(raw0, 0), rows), floor_slot = 0, bad = raw0 != floor_row;
    for (int g0 = 0; g0 < groups; g0 += mxq::THREADS) {
        const int g = g0 + (int)threadIdx.x;
        const int raw = g < groups ? offsets[g + 1] : 0;
        int hi = g < groups ? min(max(raw, floor_row), rows) : floor_row;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, hi, d);
            if (lane >= d) hi = max(hi, o);
        }
        if (lane == 31) warp_top[warp] = hi;
        __syncthreads();
        int top = floor_row, block_top = floor_row;
#pragma unroll
        for (int w = 0; w < mxq::THREADS / 32; ++w) {
            if (w < warp) top = max(top, warp_top[w]);
            block_top = max(block_top, warp_top[w]);
        }
        int lo = max(top, __shfl_up_sync(0xffffffffu, hi, 1));
        if (lane == 0) lo = top;
        hi = max(hi, top);
        bad |= g < groups && raw != hi;
        const int count = (hi - lo + GROUP_SLOT_ROWS - 1) / GROUP_SLOT_ROWS;
        int incl = count;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, incl, d);
            if (lane >= d) incl += o;
        }
        if (lane == 31) warp_slots[warp] = incl;
        __syncthreads();
        int before = floor_slot, total = floor_slot;
#pragma unroll
        for (int w = 0; w < mxq::THREADS / 32; ++w) {
            if (w < warp) before += warp_slots[w];
            total += warp_slots[w];
        }
        const int first_slot = before + incl - count;
        if (slot >= first_slot && slot < first_slot + count) {
            const int first = lo + (slot - first_slot) * GROUP_SLOT_ROWS;
            found = {first, min(hi, first + GROUP_SLOT_ROWS)};
        }
        floor_row = block_top;
        floor_slot = total;
    }
    __syncthreads();
    if (blockIdx.x == 0 && bad) atomicCAS(status, 0, (int)ROWS_OFFSETS);
    return found;
}

// Eight consecutive values as they lie: 16 bytes of a 16-bit type, 32 of fp32.
template <typename T>
struct Raw8 {
    uint4 q[sizeof(T) / 2];
};

template <typename T>
__device__ __forceinline__ Raw8<T> load8(const T *p, bool vec)
{
    Raw8<T> r;
    if (vec) {
#pragma unroll
        for (int i = 0; i < (int)(sizeof(T) / 2); ++i) r.q[i] = __ldcs(reinterpret_cast<const uint4 *>(p) + i);
    } else if constexpr (sizeof(T) == 4) {
        const uint32_t *s = reinterpret_cast<const uint32_t *>(p);
        r.q[0] = make_uint4(s[0], s[1], s[2], s[3]);
        r.q[1] = make_uint4(s[4], s[5], s[6], s[7]);
    } else {
        const uint16_t *s = reinterpret_cast<const uint16_t *>(p);
        r.q[0] = make_uint4(s[0] | ((uint32_t)s[1] << 16), s[2] | ((uint32_t)s[3] << 16), s[4] | ((uint32_t)s[5] << 16), s[6] | ((uint32_t)s[7] << 16));
    }
    return r;
}

template <typename T>
__device__ __forceinline__ void widen8(const Raw8<T> &r, float (&v)[8])
{
    if constexpr (sizeof(T) == 4) {
        v[0] = __uint_as_float(r.q[0].x); v[1] = __uint_as_float(r.q[0].y); v[2] = __uint_as_float(r.q[0].z); v[3] = __uint_as_float(r.q[0].w);
        v[4] = __uint_as_float(r.q[1].x); v[5] = __uint_as_float(r.q[1].y); v[6] = __uint_as_float(r.q[1].z); v[7] = __uint_as_float(r.q[1].w);
    } else {
        const uint32_t w[4] = {r.q[0].x, r.q[0].y, r.q[0].z, r.q[0].w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (std::is_same<T, __half>::value) {
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
// Bound by memory: 2 + 17/32 bytes per value of a 16-bit type. A thread has the loads of four rows in flight.
template <typename T>
__global__ void __launch_bounds__(mxq::THREADS) mxfp4_quantize_kernel(const T *__restrict__ x, long long ldx, int vec, int groups, int rows, int K,
                                                                      const int *offsets, uint8_t *__restrict__ packed,
                                                                      uint8_t *__restrict__ scales, int *status)
{
    using namespace mxq;
    constexpr int BATCH = 4;
    __shared__ __align__(16) uint8_t sc[MX_SCALE_BYTES];
    const int chunks = mx_chunks(K);
    const int slot = blockIdx.x / chunks, chunk = blockIdx.x - slot * chunks;
    // x may be what the kernel before writes and the output what it reads; once that is over, the product that follows
    // may set itself up.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const SlotRows s_rows = slot_rows(slot, offsets, groups, rows, status);
    if (s_rows.first >= s_rows.end) return;
    const int tr = threadIdx.x >> 4, tk = threadIdx.x & 15;
    const int k = chunk * MX_CHUNK_K + tk * 8;
#pragma unroll
    for (int i0 = 0; i0 < PASSES; i0 += BATCH) {
        Raw8<T> raw[BATCH];
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int row = s_rows.first + (i0 + i) * ROWS + tr;
            if (row < s_rows.end && k < K) raw[i] = load8(x + (long long)row * ldx + k, vec != 0); // K is a multiple of 32: a block's four threads agree
            else raw[i] = {};
        }
#pragma unroll
        for (int i = 0; i < BATCH; ++i) {
            const int r = (i0 + i) * ROWS + tr, row = s_rows.first + r;
            float v[8];
            widen8(raw[i], v);
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
            if (row < s_rows.end && k < K) *reinterpret_cast<uint32_t *>(packed + (long long)row * (K / 2) + (k >> 1)) = mx_encode8(v);
            if ((tk & 3) == 0) sc[mx_scale_at(r, tk >> 2)] = (uint8_t)s; // 0 outside the matrix
        }
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
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const SlotRows s_rows = slot_rows(slot, offsets, groups, rows, status);
    const uint8_t *sc = scales + ((long long)slot * chunks + chunk) * MX_SCALE_BYTES;
    const int tr = threadIdx.x >> 4, tk = threadIdx.x & 15;
    const int k = chunk * MX_CHUNK_K + tk * 8;
    if (k >= K) return;
    uint32_t codes[PASSES]; // of all rows in flight at once, and their scales
    uint32_t scale[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int r = i * ROWS + tr, row = s_rows.first + r;
        if (row < s_rows.end) {
            codes[i] = *reinterpret_cast<const uint32_t *>(packed + (long long)row * (K / 2) + (k >> 1));
            scale[i] = sc[mx_scale_at(r, tk >> 2)];
        }
    }
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int row = s_rows.first + i * ROWS + tr;
        if (row >= s_rows.end) continue;
        const float s = mx_scale_value(scale[i]);
        uint32_t h[4];
        mx_decode8(codes[i], h);
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

// Programmatic stream serialisation: the kernels wait for their predecessor by themselves.
template <typename... P, typename... A>
static cudaError_t launch_pdl(void (*kernel)(P...), unsigned grid, cudaStream_t st, A... args)
{
    cudaLaunchConfig_t cfg;
    memset(&cfg, 0, sizeof(cfg));
    cfg.gridDim = dim3(grid, 1, 1);
    cfg.blockDim = dim3(mxq::THREADS, 1, 1);
    cfg.stream = st;
    cudaLaunchAttribute attr;
    attr.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr.val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = &attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, static_cast<P>(args)...);
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
    cudaError_t e;
    if (src_dtype == BTM_F32) e = launch_pdl(mxfp4_quantize_kernel<float>, grid, st, (const float *)x, ldx, vec, groups, rows, K, offsets, pk, sc, status);
    else if (src_dtype == BTM_F16) e = launch_pdl(mxfp4_quantize_kernel<__half>, grid, st, (const __half *)x, ldx, vec, groups, rows, K, offsets, pk, sc, status);
    else e = launch_pdl(mxfp4_quantize_kernel<__nv_bfloat16>, grid, st, (const __nv_bfloat16 *)x, ldx, vec, groups, rows, K, offsets, pk, sc, status);
    return check_cuda(e, "mxfp4 quantise launch");
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
    cudaError_t e;
    if (dst_dtype == BTM_F32) e = launch_pdl(mxfp4_dequant_kernel<float>, grid, st, pk, sc, groups, rows, K, offsets, (float *)out, ldo, vec, status);
    else if (dst_dtype == BTM_F16) e = launch_pdl(mxfp4_dequant_kernel<__half>, grid, st, pk, sc, groups, rows, K, offsets, (__half *)out, ldo, vec, status);
    else e = launch_pdl(mxfp4_dequant_kernel<__nv_bfloat16>, grid, st, pk, sc, groups, rows, K, offsets, (__nv_bfloat16 *)out, ldo, vec, status);
    return check_cuda(e, "mxfp4 dequantise launch");
}

} // namespace btm
