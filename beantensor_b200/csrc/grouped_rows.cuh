// Rows grouped by a device-side offsets table: group g owns rows offsets[g] .. offsets[g + 1].
//
// The table is written by the GPU (a router's counts), so the host never sees it: it sizes a launch from bounds, and
// every warp that needs to know which rows a tile covers walks the table itself, 32 groups at a time, one per lane.
// Nothing in the table can lead outside the operands: an entry is clamped to [0, rows], and one that is smaller than an
// earlier one counts as that earlier one (its group is empty). A table that needed such repair is reported through a
// device status word of its own (report_repaired).
#pragma once
#include "btm_internal.h"
#include "btm_ptx.cuh"

namespace btm {

constexpr int GROUP_SLOT_ROWS = 128; // a group's rows are cut into slots, the last one short: of so many rows, or twice
                                     // as many for a pair of CTAs

// To the word behind the one that waits and bounds checks report to: a repaired table is no failure of the kernel, and must
// neither hide one nor be hidden by it.
__device__ __forceinline__ void report_repaired(int *status) { status[STATUS_OFFSETS_WORD] = ROWS_OFFSETS; }

// All members are used by a whole warp at once. Without a table there is one group that owns every row.
template <int kSlot = GROUP_SLOT_ROWS>
struct GroupWalk {
    const int *offsets;
    int groups, rows;
    int lane;
    // The window: groups g0 .. g0 + 31, lane l holding group g0 + l.
    int g0, floor_row, slots_before; // rows and slots in front of the window
    int lo, hi, incl;                // this lane's rows and the inclusive count of slots within the window
    // For pairs also in single slots of GROUP_SLOT_ROWS, which is how the scales of a microscaled operand are counted.
    int singles_before, incl_singles;
    int bad;

    __device__ __forceinline__ void load(int first, int floor_at, int slots, int singles)
    {
        singles_before = singles;
        g0 = first;
        floor_row = floor_at;
        slots_before = slots;
        int raw = floor_at;
        if (first + lane < groups) raw = offsets ? offsets[first + lane + 1] : rows;
        hi = min(max(raw, floor_at), rows);
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, hi, d);
            if (lane >= d) hi = max(hi, o);
        }
        bad |= first + lane < groups && raw != hi ? 1 : 0;
        lo = __shfl_up_sync(0xffffffffu, hi, 1);
        if (lane == 0) lo = floor_at;
        incl = (hi - lo + kSlot - 1) / kSlot;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int o = __shfl_up_sync(0xffffffffu, incl, d);
            if (lane >= d) incl += o;
        }
        if (kSlot == GROUP_SLOT_ROWS) {
            incl_singles = incl;
        } else {
            incl_singles = (hi - lo + GROUP_SLOT_ROWS - 1) / GROUP_SLOT_ROWS;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const int o = __shfl_up_sync(0xffffffffu, incl_singles, d);
                if (lane >= d) incl_singles += o;
            }
        }
    }
    __device__ __forceinline__ void next()
    {
        load(g0 + 32, __shfl_sync(0xffffffffu, hi, 31), slots_before + __shfl_sync(0xffffffffu, incl, 31),
             singles_before + __shfl_sync(0xffffffffu, incl_singles, 31));
    }

    __device__ __forceinline__ void first_window()
    {
        const int raw = offsets ? offsets[0] : 0, at = min(max(raw, 0), rows);
        bad |= raw != at ? 1 : 0;
        load(0, at, 0, 0);
    }
    __device__ __forceinline__ void init(const int *offs, int n_groups, int n_rows)
    {
        offsets = offs;
        groups = n_groups;
        rows = n_rows;
        lane = threadIdx.x & 31;
        bad = 0;
        first_window();
    }
    // Slots of all groups; the walk stands on the first window afterwards.
    __device__ __forceinline__ int count_slots()
    {
        while (g0 + 32 < groups) next();
        const int total = slots_before + __shfl_sync(0xffffffffu, incl, 31);
        if (g0 != 0) first_window();
        return total;
    }
    // The group that holds `slot`, which must be below count_slots() and not below the slot of an earlier call.
    __device__ __forceinline__ void find_slot(int slot, int &group, int &row_lo, int &row_hi, int &first_slot)
    {
        // (The walk ends with the table whatever happens to it meanwhile; lane 0 then stands in for a group not found.)
        while (g0 + 32 < groups && slot >= slots_before + __shfl_sync(0xffffffffu, incl, 31)) next();
        const int l = max(0, __ffs(__ballot_sync(0xffffffffu, slots_before + incl > slot)) - 1);
        group = g0 + l;
        row_lo = __shfl_sync(0xffffffffu, lo, l);
        row_hi = __shfl_sync(0xffffffffu, hi, l);
        first_slot = slots_before + __shfl_sync(0xffffffffu, incl, l) - (row_hi - row_lo + kSlot - 1) / kSlot;
    }
    // Single slots of the groups in front of `group`, which the last find_slot returned.
    __device__ __forceinline__ int singles_of(int group, int rows_of_group) const
    {
        return singles_before + __shfl_sync(0xffffffffu, incl_singles, group - g0) - (rows_of_group + GROUP_SLOT_ROWS - 1) / GROUP_SLOT_ROWS;
    }
    // The rows of `group`, which must not be below that of an earlier call.
    __device__ __forceinline__ void find_group(int group, int &row_lo, int &row_hi)
    {
        while (group >= g0 + 32) next();
        row_lo = __shfl_sync(0xffffffffu, lo, group - g0);
        row_hi = __shfl_sync(0xffffffffu, hi, group - g0);
    }
    // Reports a repaired table once (call after count_slots, from one warp of the grid).
    __device__ __forceinline__ void report(int *status) const
    {
        if (bad) report_repaired(status);
    }
};

} // namespace btm
