// nt_tiles.hpp — how the loss's matrix products are cut for the sizes of a
// problem: steps along k, shapes of tiles, pieces of the vocabulary and splits.
// It also builds on the host for its unit test.
#pragma once

#include <stdint.h>

#include <algorithm>

#if defined(__HIPCC__)
#define NT_TILES_FN __host__ __device__ __forceinline__
#else
#define NT_TILES_FN inline
#endif

namespace nt {

constexpr uint32_t kDepth = 64;             // elements along k in a step
constexpr uint32_t kUnits = 256;            // compute units
constexpr uint64_t kPieceBytes = 1ull << 30;       // of dz, and of packed weights, at a time

NT_TILES_FN uint32_t whole_steps(uint32_t n) { return (n + kDepth - 1u) / kDepth * kDepth; }
inline uint32_t tiles_of(uint64_t n, uint32_t each) { return (uint32_t)((n + each - 1) / each); }

// Shapes of a workgroup's tile: elements of p (classes, or columns) and of q (rows, or classes).
enum TileShape {
    kLarge,                                 // 256 x 256
    kMiddle,                                // 128 x 128
    kTall,                                  // 256 x 128: logits of 65 to 256 rows
    kFew                                    // 128 x 64: up to 64 rows, or too few tiles of the others
};
constexpr uint32_t size_p(TileShape t) { return t == kLarge || t == kTall ? 256u : 128u; }
constexpr uint32_t size_q(TileShape t) { return t == kLarge ? 256u : t == kFew ? 64u : 128u; }

// The logits of `rows` and `classes`: the largest of which each unit gets one.
// 1920 x 718 x 6208 bfloat16, 23 large tiles or 90 of 128 x 128 or 180 small
// ones: forward 96 us with the second, 63 with the last; 777 x 10007 x 1001
// float32, 160 or 553: 129 us and 90.  Up to 256 rows tall ones, where half of
// the units get one (they wait for the weights, which larger tiles ask for
// sooner): 129 rows of 50304 x 2048 float16 forward 48.4 us, with small ones
// 58.7, and 256 rows 79 and with 128 x 128 85; but 200 rows of 10007 x 1001
// float32, 80 tiles, 104 and 71.
inline TileShape logits_tile(uint64_t classes, uint64_t rows) {
    const auto tiles = [&](TileShape t) { return (uint64_t)tiles_of(classes, size_p(t)) * tiles_of(rows, size_q(t)); };
    if (rows <= 64u) return kFew;
    if (rows <= 256u && tiles(kTall) >= kUnits / 2u) return kTall;
    if (tiles(kLarge) >= kUnits) return kLarge;
    return tiles(kMiddle) >= kUnits ? kMiddle : kFew;
}

// The two products of dz.  Large tiles, where each unit gets 64 steps of them
// (whose ends are then a small part): 8192 x 50257 x 768 bfloat16, 590 steps, a
// call 1.74 ms and with 128 x 128 1.88; 512 x 32000 x 4096, 125 steps, 475 us
// and 507; 200 x 128000 x 4096 947 and 1042; but 1500 x 10007 x 1001, 30 steps,
// 161 and 146, and 300 x 50257 x 768 155 and 130.  They leave half of
// themselves idle up to 128 rows: 70 x 128000 x 4096 739 and 723.
inline TileShape grads_tile(uint64_t classes, uint64_t rows, uint64_t pitch) {
    const uint64_t steps = tiles_of(pitch, 256) * ((uint64_t)tiles_of(rows, 256) * tiles_of(classes, kDepth) +
                                                   (uint64_t)tiles_of(classes, 256) * tiles_of(rows, kDepth));
    if (rows <= 64u) return kFew;
    return rows > 128u && steps >= 64u * kUnits ? kLarge : kMiddle;
}

// How the two products of dz are split along k.  dx: such that no workgroup has
// more than half of what each compute unit gets, nor less than four steps.  dW,
// whose tiles are many as a rule, likewise, but only where one would be longer
// than twice that (11127 rows of 720 x 64 bfloat16 have three tiles of dW: a
// call 251 us in one piece, 72 split; but 777 x 10007 x 1001 float32, 13 steps
// beside 18 on each unit: 423 split, 362 not; both in large tiles).
struct Splits {
    uint32_t input, weight;
};
inline Splits splits_of(uint64_t input_tiles, uint32_t input_steps, uint64_t weight_tiles, uint32_t weight_steps) {
    const uint64_t share =
        std::max<uint64_t>((input_tiles * input_steps + weight_tiles * weight_steps) / (2u * kUnits), 4u);
    const auto of = [&](uint32_t steps) { return (uint32_t)std::max<uint64_t>(1u, (steps + share - 1) / share); };
    return Splits{of(input_steps), weight_steps > 4u * share ? of(weight_steps) : 1u};
}

// The pieces of the vocabulary: as few as keep dz and the packed weights
// within their bytes, and a launch below 2**32 work-items (512 for each large
// tile, twice as many for as much in tall ones); of whole tiles.
inline uint32_t piece_of(uint32_t rows, uint32_t classes, uint32_t pitch, int planes, bool packed, bool backward) {
    uint64_t most = (1ull << 21) / tiles_of(rows, 256) * 256u;
    if (backward) most = std::min<uint64_t>(most, kPieceBytes / (2ull * planes * whole_steps(rows)));
    if (packed) most = std::min<uint64_t>(most, kPieceBytes / (2ull * planes * pitch));
    most = std::max<uint64_t>(most / 256u * 256u, 256u);
    if (most >= classes) return classes;
    const uint64_t pieces = (classes + most - 1) / most, each = (classes + pieces - 1) / pieces;
    return (uint32_t)((each + 255u) / 256u * 256u);
}

// A pass of one problem.  `aligned`: the weights start on 16 bytes.
struct LossPlan {
    uint32_t pitch;                         // elements of a packed line
    bool packed;                            // weights are, because they cannot be read in place
    uint32_t piece, pieces;                 // classes of a piece, the last of which may have fewer
    TileShape logits, grads;
    Splits splits;                          // of the backward pass
};
inline LossPlan loss_plan(uint32_t rows, uint32_t classes, uint32_t width, int planes, bool aligned, bool backward) {
    LossPlan plan{};
    plan.pitch = whole_steps(width);
    plan.packed = planes > 1 || plan.pitch != width || !aligned;
    plan.piece = piece_of(rows, classes, plan.pitch, planes, plan.packed, backward);
    plan.pieces = tiles_of(classes, plan.piece);
    plan.splits = Splits{1, 1};
    if (!backward) {
        plan.logits = logits_tile(plan.piece, rows);
        return plan;
    }
    plan.logits = logits_tile(plan.piece, whole_steps(rows));
    plan.grads = grads_tile(plan.piece, rows, plan.pitch);
    const uint64_t across = tiles_of(plan.pitch, size_p(plan.grads));
    plan.splits = splits_of(across * tiles_of(rows, size_q(plan.grads)), tiles_of(plan.piece, kDepth),
                            across * tiles_of(plan.piece, size_q(plan.grads)), tiles_of(rows, kDepth));
    return plan;
}

}  // namespace nt
