// Tiles of grouped products: how the slots and columns of all groups are cut into tiles, which rows and columns a tile
// has, and its way from tensor memory to C. Used by the 16-bit kernels (gemm_grouped.cu) and by the microscaled one
// (mxfp4_tc.cu).
#pragma once
#include "gemm_epilogue.cuh"
#include "grouped_rows.cuh"

namespace btm {

enum GroupedMode { GROUPED_KN = 0 /* B[g] is [K, N] */, GROUPED_NK = 1 /* B[g] is [N, K] */, GROUPED_WGRAD = 2 };

struct GroupedTables {
    const int *offsets;
    int groups, rows;
};

// How the tiles of a launch are cut, from the number of slots: the same in every warp of the grid.
struct GroupedPlan {
    int bn, tiles_n;  // tile width and tiles per slot
    int full, total;  // tiles of that width, then (total - full) of half of it
};

// Cost of a tile in units of B columns: its columns plus kTileOverhead for what does not shrink with the width (the A
// rows, the hand-offs). Waves are counted whole, a last one that fits twice over is run as half-width tiles.
template <int kWidth, int kNarrowest>
__device__ __forceinline__ void try_width(GroupedPlan &best, long long &best_cost, int slots, int N, int ctas)
{
    constexpr int kTileOverhead = 64;
    const unsigned tiles_n = (unsigned)(N + kWidth - 1) / kWidth;
    const unsigned tiles = (unsigned)slots * tiles_n;
    const unsigned waves = tiles / (unsigned)ctas, rem = tiles - waves * (unsigned)ctas;
    const bool halves = kWidth % 128 == 0 && kWidth / 2 >= kNarrowest && rem > 0 && 2 * rem <= (unsigned)ctas;
    const long long cost = (long long)waves * (kWidth + kTileOverhead) + (rem == 0 ? 0 : (halves ? kWidth / 2 : kWidth) + kTileOverhead);
    if (cost < best_cost) {
        best_cost = cost;
        best.bn = kWidth;
        best.tiles_n = (int)tiles_n;
        best.full = (int)(halves ? tiles - rem : tiles);
        best.total = (int)(halves ? tiles + rem : tiles);
    }
}
// Widths kWidest, 128 and 64, none below kNarrowest.
template <int kWidest, int kNarrowest = 64>
__device__ __forceinline__ GroupedPlan plan_tiles(int slots, int N, int ctas)
{
    GroupedPlan best;
    long long best_cost = 0x7FFFFFFFFFFFFFFFLL;
    try_width<kWidest, kNarrowest>(best, best_cost, slots, N, ctas);
    if (kWidest > 128) try_width<128, kNarrowest>(best, best_cost, slots, N, ctas);
    if (kNarrowest < 128) try_width<64, kNarrowest>(best, best_cost, slots, N, ctas);
    best.total = uniform(best.total);
    best.bn = uniform(best.bn);
    return best;
}

struct GroupedTile {
    int g, lo, hi; // group and its rows
    int slot;      // its slot, counted over all groups (product)
    int m0;        // first output row (row of A for the product, row of C[g] for the gradient)
    int n0, bn;    // columns
};

template <bool kWgrad, int kSlot>
__device__ __forceinline__ GroupedTile grouped_tile(const GemmParams &p, const GroupedPlan &pl, GroupWalk<kSlot> &walk, int t)
{
    GroupedTile o;
    int tile = t, half = -1;
    if (t >= pl.full) {
        const int s = t - pl.full;
        tile = pl.full + (s >> 1);
        half = s & 1;
    }
    const int slot = (int)((unsigned)tile / (unsigned)pl.tiles_n);
    int first, count; // the group's slots
    if (kWgrad) {
        o.g = (int)((unsigned)slot / (unsigned)p.tiles_m);
        first = o.g * p.tiles_m;
        count = p.tiles_m;
        walk.find_group(o.g, o.lo, o.hi);
    } else {
        walk.find_slot(slot, o.g, o.lo, o.hi, first);
        count = (o.hi - o.lo + kSlot - 1) / kSlot;
    }
    // Within a group: bands of group_m row tiles, row tiles innermost, so that neighbouring CTAs share columns of B.
    const int r0 = tile - first * pl.tiles_n;
    int first_m = 0, height = count, r = r0;
    if (count > p.group_m) {
        const int per_band = p.group_m * pl.tiles_n;
        const int band = (int)((unsigned)r0 / (unsigned)per_band);
        first_m = band * p.group_m;
        height = min(count - first_m, p.group_m);
        r = r0 - band * per_band;
    }
    const int rn = height == 1 ? r : (int)((unsigned)r / (unsigned)height), rm = r - rn * height;
    // slot: of GROUP_SLOT_ROWS rows, for a pair that of its first CTA
    if (!kWgrad && kSlot != GROUP_SLOT_ROWS) o.slot = walk.singles_of(o.g, o.hi - o.lo) + (first_m + rm) * (kSlot / GROUP_SLOT_ROWS);
    else o.slot = first + first_m + rm;
    o.m0 = (kWgrad ? 0 : o.lo) + (first_m + rm) * kSlot;
    o.bn = half < 0 ? pl.bn : pl.bn / 2;
    o.n0 = rn * pl.bn + (half > 0 ? pl.bn / 2 : 0);
    return o;
}

// The same with every field in uniform registers, for the warps that issue TMA and tcgen05 instructions.
template <bool kWgrad, int kSlot>
__device__ __forceinline__ GroupedTile grouped_tile_uniform(const GemmParams &p, const GroupedPlan &pl, GroupWalk<kSlot> &walk, int t)
{
    GroupedTile o = grouped_tile<kWgrad, kSlot>(p, pl, walk, t);
    o.g = uniform(o.g);
    o.lo = uniform(o.lo);
    o.hi = uniform(o.hi);
    o.slot = uniform(o.slot);
    o.m0 = uniform(o.m0);
    o.n0 = uniform(o.n0);
    o.bn = uniform(o.bn);
    return o;
}

// Rows of 64 values from a staging tile to rows of C that start anywhere (multiples of two bytes). Lane l holds the values
// 2 l and 2 l + 1 of a row: where the row starts on four bytes it stores them as they are, where it starts between, the pair
// 2 l - 1, 2 l with its neighbour's second value, and the ends alone. So a warp instruction writes one row's 128 contiguous
// bytes; 16-byte pieces stored in parts would touch every sector four or five times, and the store path takes about a
// sector per cycle.
__device__ __forceinline__ void store_rows_unaligned(uint32_t buf, uint16_t *c, long long ldc, int rows, int cols, int lane)
{
    uint16_t *q = c + 2 * lane;
    if (cols == 64) {
#pragma unroll 1
        for (int r0 = 0; r0 < rows; r0 += 8) {
            uint32_t w[8], pair[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[i]) : "r"(buf + (uint32_t)(r0 + i) * 128u + ((((uint32_t)lane >> 2) ^ (uint32_t)i) << 4) + (uint32_t)(lane & 3) * 4u));
#pragma unroll
            for (int i = 0; i < 8; ++i) pair[i] = __funnelshift_r(__shfl_up_sync(0xffffffffu, w[i], 1), w[i], 16);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (r0 + i < rows) {
                    if ((reinterpret_cast<uintptr_t>(q) & 2) == 0) { // the same in all lanes
                        *reinterpret_cast<uint32_t *>(q) = w[i];
                    } else {
                        if (lane > 0) *reinterpret_cast<uint32_t *>(q - 1) = pair[i];
                        else *q = (uint16_t)w[i];
                        if (lane == 31) q[1] = (uint16_t)(w[i] >> 16);
                    }
                }
                q += ldc;
            }
        }
        return;
    }
    for (int r = 0; r < rows; ++r, q += ldc) { // the last columns of the matrix
        uint32_t w;
        asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w) : "r"(buf + (uint32_t)r * 128u + ((((uint32_t)lane >> 2) ^ (uint32_t)(r & 7)) << 4) + (uint32_t)(lane & 3) * 4u));
        if (2 * lane < cols) q[0] = (uint16_t)w;
        if (2 * lane + 1 < cols) q[1] = (uint16_t)(w >> 16);
    }
}

// Eight epilogue warps, two per tensor-memory quadrant: they take alternate 64-column chunks of a band, each with a staging
// tile of its own. (One per quadrant with two tiles drained a 128 x 256 tile in about 2600 cycles, more than the main
// loop of a shallow product takes.)
constexpr int GROUPED_EPI_WARPS = 8;
static_assert(GROUPED_EPI_WARPS * EPI_TILE_BYTES == EPI_SMEM_BYTES, "one staging tile per epilogue warp");

// One 32-row band of a finished tile to C, the chunks first_chunk, first_chunk + 2, .. of it. `rows_end`: rows from here on are
// not this tile's. zero: the sum is empty.
template <int DT, bool kWgrad>
__device__ __forceinline__ void grouped_band(const GemmParams &p, const CUtensorMap &tmC, uint32_t tmem_band, const GroupedTile &t, int row0,
                                             int rows_end, bool zero, uint32_t buf, int first_chunk, int lane)
{
    if (row0 >= rows_end) return;
    const int z = kWgrad ? t.g : 0;
    const long long base = (long long)z * p.strideC;
    const uint32_t swz = (uint32_t)(lane & 7);
    const bool whole = p.c_vec_ok && (kWgrad || row0 + 32 <= rows_end); // C[g] is clipped by its tensor map
#pragma unroll 1
    for (int c = first_chunk; c < t.bn / 64; c += 2) {
        const int col = t.n0 + c * 64;
        if (col >= p.N) break;
        uint32_t v0[32], v1[32];
        tmem_ld_32x32(tmem_band + (uint32_t)(c * 64), v0);
        tmem_ld_32x32(tmem_band + (uint32_t)(c * 64 + 32), v1);
        if (lane == 0) bulk_wait_read<0>(); // the store before has read the staging tile
        __syncwarp();
        tmem_ld_wait();
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            uint32_t q[16];
            pack16<DT>(h == 0 ? v0 : v1, q);
            if (zero) {
#pragma unroll
                for (int j = 0; j < 16; ++j) q[j] = 0u;
            }
#pragma unroll
            for (int j = 0; j < 4; ++j)
                st_shared_v4(buf + (uint32_t)lane * 128u + (((uint32_t)(h * 4 + j) ^ swz) << 4), q[4 * j], q[4 * j + 1], q[4 * j + 2], q[4 * j + 3]);
        }
        // A TMA store clips rows where the matrix ends, but columns only to whole 16 bytes: up to seven values behind N, which may
        // be another matrix's columns, would be overwritten with zeros. Chunks that end inside 16 bytes go the other way.
        if (whole && (col + 64 <= p.N || (p.N & 7) == 0)) {
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
                tma_store_3d(&tmC, buf, col, row0, z);
                bulk_commit();
            }
        } else if (!p.c_vec_ok || col + 64 > p.N) {
            __syncwarp();
            const int cols = min(64, p.N - col);
            const long long off = base + (long long)row0 * p.ldc + col;
            int rows = min(32, rows_end - row0);
            while (p.debug_bounds && rows > 0 && !store_in_bounds(p, off + (long long)(rows - 1) * p.ldc, cols)) --rows;
            store_rows_unaligned(buf, reinterpret_cast<uint16_t *>(p.C[0]) + off, p.ldc, rows, cols, lane);
        } else {
            // The group ends inside the band: 16-byte pieces of its own rows, all of a lane's in flight.
            __syncwarp();
            uint16_t *dst = reinterpret_cast<uint16_t *>(p.C[0]);
            const int j = lane & 7, r_first = lane >> 3;
            uint4 v[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int r = i * 4 + r_first;
                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                             : "=r"(v[i].x), "=r"(v[i].y), "=r"(v[i].z), "=r"(v[i].w)
                             : "r"(buf + (uint32_t)r * 128u + (((uint32_t)(j ^ (r & 7))) << 4)));
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const int row = row0 + i * 4 + r_first;
                const long long off = base + (long long)row * p.ldc + col + j * 8;
                if (row < rows_end && store_in_bounds(p, off, 8)) *reinterpret_cast<uint4 *>(dst + off) = v[i];
            }
        }
    }
}

} // namespace btm
