// nt_product.hpp — matrix products of 16-bit operands on the matrix cores,
// with what becomes of a product's tile left to the caller.
//
//   C[q][p] = sum over k of Q(q, k) P(p, k)
//
// Either operand lies in memory as [row][k] ("deep": k runs along a line) or
// as [k][row].  A workgroup makes one tile of BP x BQ elements, in steps of 64
// along k: a step's slices of both operands go straight from memory to LDS
// while the slices before are multiplied, so there are two rooms for them, or
// three.  Sums are float32 in the matrix cores' accumulators.
//
// What bounds it: 8192 counted rows of 32000 x 4096 bfloat16 take 1.57 ms with
// the loss's end, 1.69 with dz's, and the two products of dz 3.28 together, 1.27
// to 1.37 PFLOP/s, where a library's plain product of that size takes 1.61 ms
// (1.33); 7373 rows, whose last round of tiles is nearly empty, run at 1.18 to
// 1.25.  The matrix cores are busy 60 % of the cycles, at clocks that fall to 1.5
// to 1.8 GHz under the load.  Tried and not kept: 32 x 32 instead of 16 x 16
// instructions (6 to 14 % longer), the two waves of a SIMD taking turns at LDS
// and the matrix cores (11 to 22 %), four waves of 128 x 64 (38 to 50 %),
// workgroups that stride over tiles with the next one's first slice on its way
// (spills), and steps in another order for each XCD (no difference).
// Few rows are bound by the one read of the weights, at 4 to 5 TB/s.
//
// A 16-byte group of a slice does not lie where its place in memory says, but
// with its index in the line changed by an exclusive or, so that the lanes
// that read a column of groups at once find them in different banks.  The
// change is made in the address that a lane loads from, since a wave's loads
// into LDS lie in the order of its lanes.
//
// Float32 operands come as three bfloat16 planes whose sum they are (8 + 8 + 8
// significand bits): of the nine products of planes the six largest are made,
// and what is left out is below 2^-24 of the product.  The five small ones of
// all steps come first, so that only a sixth of the additions round at the
// result's size: the gradients of 777 x 10007 x 1001 are 7.9e-7 off instead of
// 1.6e-6 with all six at each step, for 2 to 5 % of the time, since the first
// planes are then read twice.  They run at 100 to 175 TFLOP/s; the matrix
// cores' own float32 instructions have 157 at their peak, and a library reaches
// 154 with them.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "nt_common.hpp"
#include "nt_tiles.hpp"

namespace nt {

typedef __bf16 bf16x8_t __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x4_t __attribute__((ext_vector_type(4)));
typedef _Float16 f16x4_t __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef short s16x8_t __attribute__((ext_vector_type(8)));

constexpr uint32_t kMostPitch = 1u << 22;   // elements of a line: a tile's offsets stay below 2**32 bytes

// There is no end of k inside a step: deep lines are padded with zeros to
// whole steps, and so is one operand's number of lines otherwise, where the
// other has `tail`, a copy of its last lines that fills a step.
struct Operand {
    const uint16_t *base;       // 16-byte aligned
    const uint16_t *tail;       // lines of the last step, if that is not whole in `base`; or null
    uint64_t pitch;             // elements from line to line, a multiple of 8
    uint64_t plane;             // elements from plane to plane
    uint32_t rows;              // deep: rows; otherwise columns, a multiple of 8
};

// How many rows there are may be known on the device alone (`live`, at most
// what the grid is made for): then they are operand q's rows, or, with
// `live_depth`, the length of k of both.
struct Product {
    Operand p, q;
    uint32_t tiles_p, tiles_q, splits, depth;   // depth: along k, in steps of 64 that are shared out among the splits
    const uint32_t *live;
    bool live_depth;
    bool pad;                   // tiles of q reach to a whole step
};

// Shape of a workgroup's tile and of the waves in it.
template <int BP_, int BQ_, int WP_, int WQ_, int ROOMS_ = 2>
struct Tile {
    static constexpr int BP = BP_, BQ = BQ_, WP = WP_, WQ = WQ_;
    static constexpr int ROOMS = ROOMS_;                            // slices in LDS: one is multiplied, the rest are on their way
    static constexpr int kWaves = WP * WQ, kThreads = kWaves * 64;
    static constexpr int kWaveP = BP / WP, kWaveQ = BQ / WQ;        // a wave's part
    static constexpr int TP = kWaveP / 16, TQ = kWaveQ / 16;        // in tiles of the matrix instruction
};

// The exclusive or of a line of the [k][row] slices, in 32-byte groups: the 16
// lines that a wave's transposed read touches at once get different ones.
__device__ __forceinline__ uint32_t turn_of(uint32_t k) { return (k & 3u) | (((k >> 3) & 3u) << 2); }

// One operand's way into LDS.
template <int B, int WAVES, bool DEEP>
struct Loader {
    static constexpr int kLoads = B * 128 / 1024 / WAVES;       // 1 KB each, a wave's share
    static_assert(kLoads * WAVES * 1024 == B * 128, "a slice is shared out among the waves");
    const char *base, *tail;
    uint64_t pitch, plane;
    uint32_t offset[kLoads];

    __device__ __forceinline__ void init(const Operand &o, uint32_t first, uint32_t wave, uint32_t lane) {
        pitch = o.pitch * 2u;
        plane = o.plane * 2u;
        const uint64_t start = DEEP ? first * pitch : (uint64_t)first * 2u;
        base = reinterpret_cast<const char *>(o.base) + start;
        tail = o.tail == nullptr ? nullptr : reinterpret_cast<const char *>(o.tail) + start;
#pragma unroll
        for (int j = 0; j < kLoads; ++j) {
            const uint32_t part = (uint32_t)j * WAVES + wave;
            if constexpr (DEEP) {
                // Rows past the last are the last again: what they give is not kept.
                uint32_t row = part * 8u + (lane >> 3);
                const uint32_t last = o.rows > first ? o.rows - 1u - first : 0u;
                row = row < last ? row : last;
                offset[j] = row * (uint32_t)pitch + ((lane & 7u) ^ (lane >> 3)) * 16u;
            } else {
                constexpr uint32_t lanes = B / 8;               // of a line
                const uint32_t k = part * (64u / lanes) + lane / lanes;
                const uint32_t group = lane % lanes;
                const uint32_t turned = (((group >> 1) ^ (turn_of(k) & (B / 16u - 1u))) << 1) | (group & 1u);
                uint32_t column = turned * 8u;
                const uint32_t last = o.rows - 8u - first;
                column = column < last ? column : last;
                offset[j] = k * (uint32_t)pitch + column * 2u;
            }
        }
    }

    // Queue the slice of step `step`, of which there are `steps`.
    __device__ __forceinline__ void load(uint16_t *room, uint32_t step, uint32_t steps, uint32_t which,
                                         uint32_t wave) const {
        const char *from = base + (DEEP ? (uint64_t)step * (2u * kDepth) : step * (kDepth * pitch)) + which * plane;
        if constexpr (!DEEP) from = tail != nullptr && step + 1u == steps ? tail : from;
        // A buffer from the tile's place on: 32-bit offsets of the lanes, and no address arithmetic in them.
        const auto buffer = __builtin_amdgcn_make_buffer_rsrc(const_cast<char *>(from), 0, -1, 0x00027000);
#pragma unroll
        for (int j = 0; j < kLoads; ++j)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(
                buffer, (__attribute__((address_space(3))) void *)(room + (j * WAVES + wave) * 512u), 16, (int)offset[j],
                0, 0, 0);
    }
};

// The eight elements along k of a lane, one for each matrix instruction: lane
// l has row l % 16 of a 16-row tile and k = 8 (l / 16) on.
template <int B, bool DEEP>
struct Reader {
    uint32_t at;                // byte of the wave's first tile; otherwise than deep, before its exclusive or
    __device__ __forceinline__ Reader(uint32_t first, uint32_t lane) {
        const uint32_t g = lane >> 4;
        if constexpr (DEEP) {
            at = (first + (lane & 15u)) * 128u + ((g ^ (lane & 7u)) << 4);
        } else {
            // A transposed read: the 16 lanes of a group bring 4 lines of 16 elements, and each gets a column.
            const uint32_t k = g * 8u + ((lane & 15u) >> 2);
            at = k * (2u * B) + (((first / 16u) ^ (turn_of(k) & (B / 16u - 1u))) << 5) + (lane & 3u) * 8u;
        }
    }
    // Keeps the compiler from holding every tile's address in a register of its own.
    __device__ __forceinline__ void hide() { __asm__ volatile("" : "+v"(at)); }
    __device__ __forceinline__ s16x8_t read(const uint16_t *room, int t, int half) const {
        const auto *from = (const __attribute__((address_space(3))) char *)room;
        if constexpr (DEEP) {
            // The second half's group is the first's with bit 2 changed.
            return *(const __attribute__((address_space(3))) s16x8_t *)(from + (half ? at ^ 64u : at) + t * 2048);
        } else {
            const auto *place = from + (at ^ ((uint32_t)t << 5)) + half * (64 * B);
            const s16x4_t low = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t *)place);
            const s16x4_t high =
                __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t *)(place + 8 * B));
            return __builtin_shufflevector(low, high, 0, 1, 2, 3, 4, 5, 6, 7);
        }
    }
};

template <bool HALF>
__device__ __forceinline__ f32x4 multiply(s16x8_t a, s16x8_t b, f32x4 c) {
    if constexpr (HALF)
        return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c,
                                                      0, 0, 0);
    else
        return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b),
                                                       c, 0, 0, 0);
}

// Workgroup b of n as a place in the order of the tiles: the ones that an XCD
// gets (every eighth) are neighbours there, so that they share its L2.
__device__ __forceinline__ uint32_t xcd_order(uint32_t b, uint32_t n) {
    const uint32_t xcd = b & 7u, left = n & 7u;
    return xcd * (n >> 3) + (xcd < left ? xcd : left) + (b >> 3);
}

// The slices of both operands of a step.
template <class T>
struct Room {
    alignas(16) uint16_t at[(T::BP + T::BQ) * kDepth];
};

// How many workgroups a product takes at most.
inline uint32_t workgroups_of(const Product &a) { return a.tiles_p * a.tiles_q * a.splits; }

// Workgroup `block` of a product.  PLANES: 1, or 3 of float32.  `finish` gets
// the wave's accumulators: element [tp][tq][r] is p = p_first + 16 tp + 4 (lane
// / 16) + r, q = q_first + 16 tq + lane % 16.  The rooms are arrays of their
// own: the compiler then knows that a read of one need not wait for what is on
// its way to another.
template <bool HALF, class T, bool P_DEEP, bool Q_DEEP, int PLANES, class Finish>
__device__ __forceinline__ void product(Product a, const Finish &finish, uint32_t block, uint16_t *room0,
                                        uint16_t *room1, uint16_t *room2) {
    const uint32_t lane = threadIdx.x & 63u, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);

    // Tiles go in bands of 8 along q, in each band along p.
    if (a.live != nullptr) {
        const uint32_t live = __builtin_amdgcn_readfirstlane(*a.live);
        if (a.live_depth) {
            a.depth = live;
        } else {
            a.q.rows = live;
            a.tiles_q = ((a.pad ? whole_steps(live) : live) + T::BQ - 1u) / T::BQ;
        }
    }
    const uint32_t tiles = a.tiles_p * a.tiles_q;
    if (block >= tiles * a.splits) return;
    const uint32_t place = xcd_order(block, tiles * a.splits), split = place / tiles, tile = place % tiles;
    const uint32_t band = tile / (8u * a.tiles_p), in_band = tile % (8u * a.tiles_p);
    const uint32_t high = a.tiles_q - band * 8u < 8u ? a.tiles_q - band * 8u : 8u;
    const uint32_t tile_q = band * 8u + in_band % high, tile_p = in_band / high;

    Loader<T::BP, T::kWaves, P_DEEP> load_p;
    Loader<T::BQ, T::kWaves, Q_DEEP> load_q;
    load_p.init(a.p, tile_p * T::BP, wave, lane);
    load_q.init(a.q, tile_q * T::BQ, wave, lane);
    const uint32_t wave_p = wave % T::WP, wave_q = wave / T::WP;
    Reader<T::BP, P_DEEP> read_p(wave_p * T::kWaveP, lane);
    Reader<T::BQ, Q_DEEP> read_q(wave_q * T::kWaveQ, lane);

    f32x4 acc[T::TP][T::TQ];
#pragma unroll
    for (int i = 0; i < T::TP; ++i)
#pragma unroll
        for (int j = 0; j < T::TQ; ++j) acc[i][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};

    constexpr uint32_t products = PLANES == 1 ? 1u : 6u;
    const uint32_t steps = (a.depth + kDepth - 1u) / kDepth;
    const uint32_t begin = (uint32_t)((uint64_t)steps * split / a.splits);
    const uint32_t end = (uint32_t)((uint64_t)steps * (split + 1u) / a.splits);
    const uint32_t total = (end - begin) * products;
    // Past the last step the last is queued again, so that the loop has no branches.
    const auto stage = [&](uint16_t *room, uint32_t s) {
        s = s < total ? s : total - 1u;
        uint32_t k = begin + s, plane_p = 0, plane_q = 0;
        if constexpr (PLANES == 3) {
            // (0,2) (2,0) (1,1) (0,1) (1,0) of all steps, then (0,0) of all.
            const uint32_t small = (end - begin) * 5u, which = s < small ? s % 5u : 5u;
            k = begin + (s < small ? s / 5u : s - small);
            plane_p = (0x010120u >> (4u * which)) & 15u;
            plane_q = (0x001102u >> (4u * which)) & 15u;
        }
        load_p.load(room, k, steps, plane_p, wave);
        load_q.load(room + T::BP * kDepth, k, steps, plane_q, wave);
    };
    const auto compute = [&](const uint16_t *room) {
        read_p.hide();
        read_q.hide();
        s16x8_t fp[2][T::TP], fq[2][T::TQ];
#pragma unroll
        for (int half = 0; half < 2; ++half) {
#pragma unroll
            for (int j = 0; j < T::TQ; ++j) fq[half][j] = read_q.read(room + T::BP * kDepth, j, half);
#pragma unroll
            for (int i = 0; i < T::TP; ++i) fp[half][i] = read_p.read(room, i, half);
        }
#pragma unroll
        for (int half = 0; half < 2; ++half)
#pragma unroll
            for (int i = 0; i < T::TP; ++i)
#pragma unroll
                for (int j = 0; j < T::TQ; ++j) acc[i][j] = multiply<HALF>(fp[half][i], fq[half][j], acc[i][j]);
        // The order of both: a tile of p is read while the one two before it is multiplied.
        constexpr int rp = P_DEEP ? 1 : 2, rq = T::TQ * (Q_DEEP ? 1 : 2);
        if constexpr (T::TP > 2) {
            __builtin_amdgcn_sched_group_barrier(0x100, rq + 2 * rp, 0);        // reads of LDS
#pragma unroll
            for (int half = 0; half < 2; ++half) {
#pragma unroll
                for (int i = 0; i < T::TP - 2; ++i) {
                    __builtin_amdgcn_sched_group_barrier(0x008, T::TQ, 0);      // matrix instructions
                    __builtin_amdgcn_sched_group_barrier(0x100, rp, 0);
                }
                __builtin_amdgcn_sched_group_barrier(0x008, T::TQ, 0);
                if (half == 0) __builtin_amdgcn_sched_group_barrier(0x100, rq, 0);
                __builtin_amdgcn_sched_group_barrier(0x008, T::TQ, 0);
                if (half == 0) __builtin_amdgcn_sched_group_barrier(0x100, 2 * rp, 0);
            }
        }
    };
    // One step: its slice is there, in every wave's part, once the loads before the last ROOMS - 2 slices are
    // done and all waves say so.  Each has then also ended its reads of the room that is loaded next: the wait
    // before the barrier is for those too.
    const auto step = [&](const uint16_t *room, uint16_t *free, uint32_t s) {
        constexpr int ahead = (T::ROOMS - 2) * (decltype(load_p)::kLoads + decltype(load_q)::kLoads);
        static_assert(ahead < 64, "the counter of loads on their way has six bits");
        __asm__ volatile("" ::: "memory");
        __builtin_amdgcn_s_waitcnt((ahead & 15) | (ahead >> 4) << 14 | 0x0070);     // vmcnt(ahead) lgkmcnt(0)
        __builtin_amdgcn_s_barrier();
        __builtin_amdgcn_sched_barrier(0);
        __asm__ volatile("" ::: "memory");
        stage(free, s + T::ROOMS - 1);
        __builtin_amdgcn_sched_barrier(0);              // the loads are under way first
        compute(room);
    };
    if (total > 0) {
        stage(room0, 0);
        if constexpr (T::ROOMS == 2) {
            uint32_t s = 0;
            for (; s + 1 < total; s += 2) {
                step(room0, room1, s);
                step(room1, room0, s + 1);
            }
            if (s < total) step(room0, room1, s);
        } else {
            stage(room1, 1);
            uint32_t s = 0;
            for (; s + 2 < total; s += 3) {
                step(room0, room2, s);
                step(room1, room0, s + 1);
                step(room2, room1, s + 2);
            }
            if (s < total) step(room0, room2, s);
            if (s + 1 < total) step(room1, room0, s + 1);
        }
        __builtin_amdgcn_s_waitcnt(0x0f70);             // nothing is on its way to LDS when it is given up
    }
    finish.template operator()<T>(acc, tile_p * T::BP + wave_p * T::kWaveP, tile_q * T::BQ + wave_q * T::kWaveQ, split,
                                  lane);
}

template <bool HALF, class T, bool P_DEEP, bool Q_DEEP, int PLANES, class Finish>
__global__ __launch_bounds__(T::kThreads, 2) void product_kernel(Product a, Finish finish) {
    __shared__ Room<T> room0, room1;
    if constexpr (T::ROOMS == 2) {
        product<HALF, T, P_DEEP, Q_DEEP, PLANES>(a, finish, blockIdx.x, room0.at, room1.at, nullptr);
    } else {
        __shared__ Room<T> room2;
        product<HALF, T, P_DEEP, Q_DEEP, PLANES>(a, finish, blockIdx.x, room0.at, room1.at, room2.at);
    }
}

// Two products in one launch, the first's workgroups first: the second's fill
// the units that the first leaves idle at its end.  Both have [k][row] lines
// for p; the first has deep lines for q.
template <bool HALF, class T, int PLANES, class FinishA, class FinishB>
__global__ __launch_bounds__(T::kThreads, 2) void two_products_kernel(Product a, FinishA finish_a, uint32_t first,
                                                                     Product b, FinishB finish_b) {
    __shared__ Room<T> room0, room1;
    const auto run = [&](uint16_t *room2) {
        if (blockIdx.x < first)
            product<HALF, T, false, true, PLANES>(a, finish_a, blockIdx.x, room0.at, room1.at, room2);
        else
            product<HALF, T, false, false, PLANES>(b, finish_b, blockIdx.x - first, room0.at, room1.at, room2);
    };
    if constexpr (T::ROOMS == 2) {
        run(nullptr);
    } else {
        __shared__ Room<T> room2;
        run(room2.at);
    }
}

template <bool HALF, class T, bool P_DEEP, bool Q_DEEP, int PLANES, class Finish>
static void launch_product(const Product &a, const Finish &finish, hipStream_t s) {
    product_kernel<HALF, T, P_DEEP, Q_DEEP, PLANES, Finish>
        <<<dim3(workgroups_of(a)), dim3(T::kThreads), 0, s>>>(a, finish);
}

template <bool HALF, class T, int PLANES, class FinishA, class FinishB>
static void launch_two_products(const Product &a, const FinishA &finish_a, const Product &b, const FinishB &finish_b,
                                hipStream_t s) {
    const uint32_t first = (workgroups_of(a) + 7u) / 8u * 8u;       // whole rounds of the XCDs
    two_products_kernel<HALF, T, PLANES, FinishA, FinishB>
        <<<dim3(first + workgroups_of(b)), dim3(T::kThreads), 0, s>>>(a, finish_a, first, b, finish_b);
}

}  // namespace nt
