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
constexpr int THREADS = 256;
constexpr int ROWS = 16; // dequantise: 16 threads x 8 values across a scale block's 128 k, 16 rows at a time
constexpr int PASSES = GROUP_SLOT_ROWS / ROWS;
} // namespace mxq

struct SlotRows {
    int first, end; // rows of the slot; empty when there is no such slot
};

// Which rows does this block's slot hold? Uniform groups by arithmetic. Ragged ones from the table, 256 groups at a time, a
// thread each: running maximum (a decreasing entry counts as the one before it) and running slot count over the block.
// (GroupWalk would take them 32 at a time, one after the other, and the table twice: 0.5 us more for 64 groups.)
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
    if (blockIdx.x == 0 && bad) report_repaired(status);
    return found;
}

// One block of 32 consecutive values as they lie, as 32-bit words.
template <typename T>
struct RawBlock {
    static constexpr int WORDS = MX_BLOCK * sizeof(T) / 4;
    uint32_t w[WORDS];
};

// Behind griddepcontrol.wait, of what the kernel before may have written (ld_dependent): volatile, or through pointers that
// nothing promises to be read-only. vec: 2 = 32-byte loads (the widest there are), 1 = 16-byte, 0 = element by element.
template <typename T>
__device__ __forceinline__ void load_block(RawBlock<T> &r, const T *p, int vec)
{
    constexpr int W = RawBlock<T>::WORDS;
    if (vec == 2) {
#pragma unroll
        for (int i = 0; i < W; i += 8)
            asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=r"(r.w[i]), "=r"(r.w[i + 1]), "=r"(r.w[i + 2]), "=r"(r.w[i + 3]), "=r"(r.w[i + 4]), "=r"(r.w[i + 5]), "=r"(r.w[i + 6]),
                           "=r"(r.w[i + 7])
                         : "l"(reinterpret_cast<const uint32_t *>(p) + i)
                         : "memory");
    } else if (vec == 1) {
#pragma unroll
        for (int i = 0; i < W; i += 4) {
            const uint4 q = ld_dependent(reinterpret_cast<const uint4 *>(reinterpret_cast<const uint32_t *>(p) + i));
            r.w[i] = q.x; r.w[i + 1] = q.y; r.w[i + 2] = q.z; r.w[i + 3] = q.w;
        }
    } else if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < W; ++i) r.w[i] = reinterpret_cast<const uint32_t *>(p)[i];
    } else {
#pragma unroll
        for (int i = 0; i < W; ++i) r.w[i] = reinterpret_cast<const uint16_t *>(p)[2 * i] | ((uint32_t) reinterpret_cast<const uint16_t *>(p)[2 * i + 1] << 16);
    }
}

// The block's scale byte and its 32 codes. Magnitudes compare like their bit patterns, a NaN above infinity; 16-bit types
// are compared two at a time.
template <typename T>
__device__ __forceinline__ uint32_t encode_block(const RawBlock<T> &r, uint4 &codes)
{
    constexpr int W = RawBlock<T>::WORDS;
    constexpr bool kHalf = std::is_same<T, __half>::value, kBf16 = std::is_same<T, __nv_bfloat16>::value;
    uint32_t top = 0;
    if constexpr (sizeof(T) == 4) {
#pragma unroll
        for (int i = 0; i < W; ++i) top = max(top, r.w[i] & 0x7FFFFFFFu);
    } else {
        uint32_t m = 0;
#pragma unroll
        for (int i = 0; i < W; ++i) m = __vmaxu2(m, r.w[i] & 0x7FFF7FFFu);
        const uint32_t h = max(m & 0xFFFFu, m >> 16);
        top = kHalf ? __float_as_uint(__half2float(__ushort_as_half((unsigned short)h))) : h << 16;
    }
    const uint32_t e = top >> 23;
    uint32_t s = e > 2u ? e - 2u : 0u;
    const float inv = __uint_as_float((254u - s) << 23); // 2^-X, a normal number for every s
    uint32_t out[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (kHalf) {
                const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(&r.w[4 * j + i]));
                v[2 * i] = f.x * inv;
                v[2 * i + 1] = f.y * inv;
            } else if constexpr (kBf16) {
                // Scaled two at a time in bf16, which has the exponents of fp32: the product with a power of two is exact, or
                // so small that its code is 0 either way.
                const __nv_bfloat162 p = __hmul2(*reinterpret_cast<const __nv_bfloat162 *>(&r.w[4 * j + i]), __float2bfloat162_rn(inv));
                const uint32_t q = *reinterpret_cast<const uint32_t *>(&p);
                v[2 * i] = __uint_as_float(q << 16);
                v[2 * i + 1] = __uint_as_float(q & 0xFFFF0000u);
            } else {
                v[2 * i] = __uint_as_float(r.w[8 * j + 2 * i]) * inv;
                v[2 * i + 1] = __uint_as_float(r.w[8 * j + 2 * i + 1]) * inv;
            }
        }
        out[j] = mx_encode8(v);
    }
    const bool finite = e != 255u; // else an infinity or a NaN
    codes = finite ? make_uint4(out[0], out[1], out[2], out[3]) : make_uint4(0, 0, 0, 0);
    return finite ? s : MX_NAN;
}

// Blocks of 128 rows x 128 k: their 512 bytes of scales are put together in shared memory and written whole. A thread takes
// whole blocks of 32 values (64 bytes of a 16-bit type in, 16 bytes and a scale out): nothing is exchanged between
// threads. The 256 threads lie across kAcross scale blocks of a slot (4 threads each) and 64 / kAcross rows (quantize_as
// chooses). A CTA takes `steps` times that many blocks, one
// after the other, so that a large operand looks its rows up once for several.
// Bound by memory (2 + 17/32 bytes per value of a 16-bit type). With eight values per thread, the largest magnitude by
// shuffles and 4-byte stores the kernel was bound by instruction issue (109 instructions per eight values, 79 % of
// the issue slots): 16384 x 11008 bf16 in 90 us; so 68 to 71 us, 6.4 to 6.7 TB/s (part of the 96 MB written stays in L2).
template <typename T, int kAcross>
__global__ void __launch_bounds__(mxq::THREADS, sizeof(T) == 4 ? 3 : 4)
mxfp4_quantize_kernel(const T *x, long long ldx, int vec, int groups, int rows, int K, int steps, const int *offsets,
                      uint8_t *packed, uint8_t *scales, int *status)
{
    using namespace mxq;
    constexpr int BATCH = sizeof(T) == 4 ? 1 : 2, LINES = 64 / kAcross; // rows per pass
    __shared__ __align__(16) uint8_t sc[2][kAcross * MX_SCALE_BYTES];
    const int chunks = mx_chunks(K), per_cta = steps * kAcross, parts = (chunks + per_cta - 1) / per_cta;
    const int slot = blockIdx.x / parts, part = blockIdx.x - slot * parts;
    // x may be what the kernel before writes and the output what it reads; once that is over, the product that follows
    // may set itself up.
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    const SlotRows s_rows = slot_rows(slot, offsets, groups, rows, status);
    const int height = s_rows.end - s_rows.first;
    if (height <= 0) return;
    const int tr = threadIdx.x / (4 * kAcross), tk = threadIdx.x % (4 * kAcross);
    const int chunk_end = min(chunks, (part + 1) * per_cta);
    int half = 0;
    for (int chunk = part * per_cta; chunk < chunk_end; chunk += kAcross, half ^= 1) {
        uint8_t *scb = sc[half]; // the blocks before may still be on their way out of the other half
        const int k = chunk * MX_CHUNK_K + tk * MX_BLOCK;
        const bool whole = height == GROUP_SLOT_ROWS && (chunk + kAcross) * MX_CHUNK_K <= K;
        if (!whole) { // bytes outside the matrix are 0
            for (int i = threadIdx.x; i < kAcross * MX_SCALE_BYTES / 16; i += THREADS) reinterpret_cast<uint4 *>(scb)[i] = make_uint4(0, 0, 0, 0);
            __syncthreads();
        }
        const T *src = x + (long long)(s_rows.first + tr) * ldx + k;
        uint8_t *dst = packed + (long long)(s_rows.first + tr) * (K / 2) + (k >> 1);
#pragma unroll 1
        for (int r0 = 0; r0 < height; r0 += BATCH * LINES) {
            RawBlock<T> raw[BATCH];
            bool in[BATCH];
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                in[i] = whole || (r0 + i * LINES + tr < height && k < K);
                if (in[i]) load_block(raw[i], src + (long long)(r0 + i * LINES) * ldx, vec);
            }
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                if (!in[i]) continue;
                uint4 codes;
                const uint32_t s = encode_block(raw[i], codes);
                *reinterpret_cast<uint4 *>(dst + (long long)(r0 + i * LINES) * (K / 2)) = codes;
                scb[(tk >> 2) * MX_SCALE_BYTES + mx_scale_at(r0 + i * LINES + tr, tk & 3)] = (uint8_t)s;
            }
        }
        __syncthreads();
        const int left = (chunk_end - chunk < kAcross ? chunk_end - chunk : kAcross) * MX_SCALE_BYTES / 16;
        for (int i = threadIdx.x; i < left; i += THREADS)
            reinterpret_cast<uint4 *>(scales + ((long long)slot * chunks + chunk) * MX_SCALE_BYTES)[i] = reinterpret_cast<const uint4 *>(scb)[i];
    }
}

template <typename T>
__device__ __forceinline__ T round_to(float v);
template <>
__device__ __forceinline__ float round_to<float>(float v) { return v; }
template <>
__device__ __forceinline__ __half round_to<__half>(float v) { return __float2half_rn(v); }
template <>
__device__ __forceinline__ __nv_bfloat16 round_to<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }

// Bound by memory: 16384 x 11008 to bf16 in 72 us (6.35 TB/s).
template <typename T>
__global__ void __launch_bounds__(mxq::THREADS) mxfp4_dequant_kernel(const uint8_t *packed, const uint8_t *scales,
                                                                     int groups, int rows, int K, const int *offsets, T *out,
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
        if (row >= s_rows.end) break;
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

static long long slot_count(int groups, int rows, const int *offsets)
{
    return offsets ? grouped_slot_bound(groups, rows) : (long long)groups * (((rows / groups) + GROUP_SLOT_ROWS - 1) / GROUP_SLOT_ROWS);
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

template <typename T>
static int quantize_as(cudaStream_t st, int sm_count, int groups, int rows, int K, const int *offsets, const void *x, long long ldx, void *packed, void *scales, int *status)
{
    const long long slots = slot_count(groups, rows, offsets), chunks = mx_chunks(K);
    // One block across, 64 rows at a time, while all CTAs are resident at once (four per SM, 16-bit types): then the time is a CTA's latency.
    // Four across, 16 rows at a time, beyond. Measured, one / four: 256 x 2048 plain (32 CTAs at one) 2.4 / 4.7 us, 3001 x 1440 in 24
    // groups (564) 4.7 / 6.6; 256 x 2048 in 64 groups (1040) 5.1 / 2.8, 2048 x 4096 in 64 (2560) 12.0 / 6.7, 16384 x 11008 71.0 / 69.7.
    // The same border serves fp32, of which three CTAs are resident: 2048 x 4096 (512 CTAs at one) 9.8 / 11.0 us.
    const long long wave = 4LL * sm_count;
    const int across = slots * chunks <= wave ? 1 : 4;
    // More than one step per CTA once there are several waves of them (four CTAs per SM).
    long long steps = slots * chunks / (across * 4 * wave);
    steps = steps < 1 ? 1 : steps > 8 ? 8 : steps;
    const long long blocks = slots * ((chunks + steps * across - 1) / (steps * across));
    if (blocks > 0x7FFFFFFFLL) return set_error(BTM_ERR_UNSUPPORTED, "mxfp4 quantise: operand too large (%lld scale blocks)", slots * chunks);
    const long long pitch = ldx * (long long)sizeof(T);
    const int vec = (((uintptr_t)x | (uintptr_t)pitch) & 31) == 0 ? 2 : (((uintptr_t)x | (uintptr_t)pitch) & 15) == 0 ? 1 : 0;
    const cudaError_t e = launch_pdl(across == 1 ? mxfp4_quantize_kernel<T, 1> : mxfp4_quantize_kernel<T, 4>, (unsigned)blocks, st, (const T *)x, ldx, vec, groups,
                                     rows, K, (int)steps, offsets, (uint8_t *)packed, (uint8_t *)scales, status);
    return check_cuda(e, "mxfp4 quantise launch");
}

int launch_mxfp4_quantize(cudaStream_t st, int sm_count, int src_dtype, int groups, int rows, int K, const int *offsets, const void *x, long long ldx,
                          void *packed, void *scales, int *status)
{
    if (src_dtype == BTM_F32) return quantize_as<float>(st, sm_count, groups, rows, K, offsets, x, ldx, packed, scales, status);
    if (src_dtype == BTM_F16) return quantize_as<__half>(st, sm_count, groups, rows, K, offsets, x, ldx, packed, scales, status);
    return quantize_as<__nv_bfloat16>(st, sm_count, groups, rows, K, offsets, x, ldx, packed, scales, status);
}

int launch_mxfp4_dequant(cudaStream_t st, int dst_dtype, int groups, int rows, int K, const int *offsets, const void *packed,
                         const void *scales, void *out, long long ldo, int *status)
{
    const long long blocks = slot_count(groups, rows, offsets) * mx_chunks(K);
    if (blocks > 0x7FFFFFFFLL) return set_error(BTM_ERR_UNSUPPORTED, "mxfp4 dequantise: operand too large (%lld scale blocks)", blocks);
    const unsigned grid = (unsigned)blocks;
    const int es = dst_dtype == BTM_F32 ? 4 : 2;
    const int vec = ((uintptr_t)out & 15) == 0 && (ldo * es) % 16 == 0;
    const uint8_t *pk = (const uint8_t *)packed, *sc = (const uint8_t *)scales;
    cudaError_t e;
    if (dst_dtype == BTM_F32) e = launch_pdl(mxfp4_dequant_kernel<float>, grid, st, pk, sc, groups, rows, K, offsets, (float *)out, ldo, vec, status);
    else if (dst_dtype == BTM_F16) e = launch_pdl(mxfp4_dequant_kernel<__half>, grid, st, pk, sc, groups, rows, K, offsets, (__half *)out, ldo, vec, status);
    else e = launch_pdl(mxfp4_dequant_kernel<__nv_bfloat16>, grid, st, pk, sc, groups, rows, K, offsets, (__nv_bfloat16 *)out, ldo, vec, status);
    return check_cuda(e, "mxfp4 dequantise launch");
}

template <typename T>
static cudaError_t load_convert()
{
    cudaFuncAttributes a;
    cudaError_t e = cudaFuncGetAttributes(&a, mxfp4_quantize_kernel<T, 1>);
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, mxfp4_quantize_kernel<T, 4>);
    if (e == cudaSuccess) e = cudaFuncGetAttributes(&a, mxfp4_dequant_kernel<T>);
    return e;
}

int load_mxfp4_convert_kernels()
{
    cudaError_t e = load_convert<float>();
    if (e == cudaSuccess) e = load_convert<__half>();
    if (e == cudaSuccess) e = load_convert<__nv_bfloat16>();
    return check_cuda(e, "cudaFuncGetAttributes(mxfp4)");
}

} // namespace btm
