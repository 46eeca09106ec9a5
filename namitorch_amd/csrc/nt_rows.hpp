// nt_rows.hpp — how a row of layer norm lies over lanes: which tilings the
// launches choose, which kernels are therefore built, and which lane owns
// which column.  It also builds on the host for its unit test.
#pragma once

#include <stdint.h>

#include <initializer_list>

#include "../../include/namitorch_amd.h"

#if defined(__HIPCC__)
#define NT_ROWS_FN __host__ __device__ __forceinline__
#else
#define NT_ROWS_FN inline
#endif

namespace nt {

constexpr int kGroup = 8;               // consecutive elements that a lane holds at a time
constexpr int kRowThreads = 512;        // lanes of a workgroup, for rows of at most as many
constexpr int kBackwardThreads = 512;   // the same of the backward pass
constexpr int kWideThreads = 1024;      // of a workgroup, for rows of more
constexpr uint32_t kSimds = 256 * 4;

// A forward launch of at most this many lanes at one group a lane (16 waves a
// CU) takes one group a lane: 1 x 768 2.8 us (three groups 3.6), 512 x 760 4.3
// (5.5), 2048 x 744 5.2 (5.6); past it the idle lanes cost more, 8192 x 768
// 10.2 (6.6).
constexpr uint64_t kFewLanes = kSimds * 4 * 64;

// The group of a lane: eight columns from `column` on (the width where the
// lane has none).  The last group of a row whose width is no multiple of
// eight ends at the row's end and starts inside the group before it: its
// elements below `first` are the other lane's, computed alike by both.  So it
// too is loaded and stored whole; only rows of less than eight go element by
// element.  Element loads at every end made each wave wait before it asked for
// its next row (10006 x 1001 bfloat16: norm 14.4 -> 12.8 us, edge 26.0 -> 22.6).
struct Columns {
    uint32_t column, first;
    NT_ROWS_FN Columns() {}
    NT_ROWS_FN Columns(uint32_t c, uint32_t width)
        : column(c < width && c + kGroup > width && width >= kGroup ? width - kGroup : c < width ? c : width),
          first(c - column) {}
    template <bool EVEN>
    NT_ROWS_FN bool has(uint32_t k, uint32_t width) const {
        return EVEN ? column < width : k >= first && column + k < width;
    }
};

inline bool aligned16(std::initializer_list<const void *> arrays) {
    uintptr_t bits = 0;
    for (const void *p : arrays) bits |= (uintptr_t)p;
    return bits % 16 == 0;
}

// Whether every group of every row lies on 16 bytes, in any dtype: arrays that
// start there are not enough where rows do not end on a whole group.
inline bool aligned_rows(uint32_t width, std::initializer_list<const void *> arrays) {
    return width % kGroup == 0 && aligned16(arrays);
}

// How a row is laid over lanes; parts == 0: it does not fit.
struct RowTiling {
    uint32_t lanes, parts, threads;
};

// The forward pass: the tiling that leaves the fewest lanes idle, of equals
// the one with the fewest lanes.  Where the rows do not fill the chip, one
// group a lane: a row's latency counts, not its share of a workgroup.  Float32
// takes one group (32 bytes) a lane as far as that reaches: edge 8192 x 2048
// 52.9 us, with two 58.9 (before its stores went through the caches).
inline RowTiling forward_tiling(uint64_t rows, uint32_t width, int32_t dtype) {
    const uint32_t groups = (width + kGroup - 1) / kGroup;
    RowTiling best{0, 0, 0};
    for (uint32_t parts = dtype == NT_F32 ? 2 : 3; parts >= 1; --parts) {
        uint32_t lanes = 1;
        while (lanes * parts < groups) lanes <<= 1;
        if (lanes > (uint32_t)kWideThreads || (lanes > (uint32_t)kRowThreads && parts > 2)) continue;
        const bool one = parts == 1 && (dtype == NT_F32 || rows * lanes <= kFewLanes);
        if (best.parts == 0 || one || lanes * parts < best.lanes * best.parts)
            best = RowTiling{lanes, parts, uint32_t(lanes <= (uint32_t)kRowThreads ? kRowThreads : kWideThreads)};
    }
    return best;
}

// Whether it makes such a tiling, over all numbers and widths of rows: the
// launches build a kernel for no other.
template <int32_t DTYPE, int PARTS, int THREADS>
constexpr bool forward_makes() {
    return THREADS == kRowThreads ? PARTS == 1 || DTYPE != NT_F32 : PARTS <= 2;
}

// The backward pass: as above with at most two groups a lane (8192 x 768
// bfloat16: 12.7 us, with three groups 14.5), and one of float32 (8192 x 2048:
// 39.4 us, with two 41.4).  128 registers hold them but for the float32 edge of
// 8193 to 16384 columns, two groups a lane: 8 registers are spilled where it
// drops, on ragged rows 129 (1 without dropout).  2048 x 12288 takes 122 us, x
// 12289 147; float16, which spills none, 84 there.
inline RowTiling backward_tiling(uint32_t width, int32_t dtype) {
    const uint32_t groups = (width + kGroup - 1) / kGroup;
    RowTiling best{0, 0, 0};
    for (uint32_t parts = 2; parts >= 1; --parts) {
        uint32_t lanes = 1;
        while (lanes * parts < groups) lanes <<= 1;
        if (lanes > (uint32_t)kWideThreads) continue;
        if (best.parts == 0 || lanes * parts < best.lanes * best.parts || dtype == NT_F32)
            best = RowTiling{lanes, parts,
                             uint32_t(lanes <= (uint32_t)kBackwardThreads ? kBackwardThreads : kWideThreads)};
    }
    return best;
}

// As forward_makes.
template <int32_t DTYPE, int PARTS, int THREADS>
constexpr bool backward_makes() {
    return THREADS == kBackwardThreads ? PARTS == 1 || DTYPE != NT_F32 : PARTS == 2 || DTYPE == NT_F32;
}

}  // namespace nt
