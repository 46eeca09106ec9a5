// nt_loss.hip — softmax cross entropy of a linear layer's outputs over a large
// vocabulary, whose logits are never in memory, and its backward pass.
//
// With x of N rows and W of V, both H wide, z = x W^T, target t_i:
//   lse_i  = log sum_v exp z_iv,   loss_i = lse_i - z_i,t
//   dz_iv  = g_i (exp(z_iv - lse_i) - [v = t_i])
//   dx     = dz W,   dW = dz^T x
// with g_i the gradient of row i's loss (that of the mean over the counted
// rows, divided by their number).  Rows with the ignored target are taken out
// before anything else: what they hold is never multiplied.
//
// Forward: the product's tiles end as a maximum and a sum of exponentials of
// each row (and the target's logit), from which a second kernel makes lse and
// loss.  Backward: the product is made once more, a piece of the vocabulary at
// a time, and its tiles end as dz in the operands' type; two products of the
// piece follow.  The sums over the vocabulary that dx needs are float32 in
// memory from piece to piece.
//
// dz is rounded once, to the operands' type: half a unit in its last place,
// as the stored gradients themselves are.  A factor that all rows share is
// multiplied into the products instead, so that dz is exp(z - lse) - [v = t]
// and most targets' -1 is exact: rounded together with that factor, which is
// as far off for each of them, the gradient of 8192 rows by 50257 classes was
// 1.7 times as far from the 64-bit one as a single rounding.  In float16 dz is
// multiplied by a power of two first, such that the largest finite |g_i| comes
// to 2**14 to 2**15: exp(z - lse) is some 1 / V, which float16 alone would hold
// with few digits or none; row gradients of the other types are brought below
// one likewise.  Float32 is three bfloat16 planes (nt_product.hpp).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "nt_entry.hpp"
#include "nt_internal.hpp"
#include "nt_pool.hpp"
#include "nt_product.hpp"
#include "nt_row_ops.hpp"
#include "nt_tiles.hpp"

namespace nt {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;
constexpr float kInfinity = __builtin_huge_valf();

enum Reduction { kEach = 0, kMean = 1, kSum = 2 };

// What the rows' targets are; class_of gives the class, kIgnored or kOutside.
struct Targets {
    const void *at;
    int64_t ignored;
    uint32_t classes;
    int32_t size;               // bytes of a target: 4 or 8
};
constexpr int32_t kIgnored = -1, kOutside = -2;

__device__ __forceinline__ int32_t class_of(const Targets &t, uint64_t i) {
    const int64_t v = t.size == 8 ? reinterpret_cast<const int64_t *>(t.at)[i]
                                  : (int64_t) reinterpret_cast<const int32_t *>(t.at)[i];
    if (v == t.ignored) return kIgnored;
    return v >= 0 && v < (int64_t)t.classes ? (int32_t)v : kOutside;
}

// The counted rows in order, made by rows_kernel.
struct Rows {
    uint32_t *count;            // how many
    float *unscale;             // what the products of dz are multiplied by
    uint32_t *place;            // (backward) of each row: which counted row it is, or ~0
    uint32_t *row;              // of counted row j: its row,
    int32_t *target;            // its class or kOutside,
    float *weight;              // (backward) what its dz is multiplied by
};

// ---- counted rows ----------------------------------------------------------------------------------
constexpr int kRowsBlock = 1024;

// One workgroup, 8192 rows at a time: eight rows of a lane lie 1024 apart, so
// that reads and writes are whole lines, and the counts of all waves are summed
// at once.  Forward, the lse and loss of rows that are not counted are set to
// zero here.  8192 rows 7.1 us, backward 9.3: one pass, bound by its latency.
constexpr int kRowsAtOnce = 8;

template <bool BACKWARD>
__global__ __launch_bounds__(kRowsBlock) void rows_kernel(Targets t, uint32_t rows, Rows out, const float *grad,
                                                          float grad_value, int32_t reduction, bool half, float *lse,
                                                          float *loss) {
    constexpr uint32_t waves = kRowsBlock / 64, slots = waves * kRowsAtOnce;
    __shared__ uint32_t counts[slots];
    __shared__ float most[waves];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    // A power of two: float16's as said above; with row gradients of the other types, such that the largest
    // comes to 0.5 to 1, since a product of 2^-122 and a probability would have few digits, or none.
    float scale = 1.0f;
    if (BACKWARD && (half || reduction == kEach)) {
        float largest = reduction == kEach ? 0.0f : 1.0f;
        if (reduction == kEach) {
            // Of rows whose gradients are finite: the others are NaN or infinite at any scale.
            for (uint32_t i = threadIdx.x; i < rows; i += kRowsBlock) {
                const float size = fabsf(grad[i]);
                if (class_of(t, i) >= 0 && size < kInfinity) largest = fmaxf(largest, size);
            }
#pragma unroll
            for (int off = 32; off > 0; off >>= 1) largest = fmaxf(largest, __shfl_xor(largest, off, 64));
            if (lane == 0u) most[wave] = largest;
            __syncthreads();
            for (uint32_t k = 0; k < waves; ++k) largest = fmaxf(largest, most[k]);
        }
        if (largest > 0.0f) {
            int exponent;
            frexpf(largest, &exponent);
            exponent = (half ? 15 : 0) - exponent;
            scale = ldexpf(1.0f, exponent > 126 ? 126 : exponent < -126 ? -126 : exponent);
        }
    }
    uint32_t done = 0;                                      // counted rows of the rounds before
    for (uint64_t first = 0; first < rows; first += kRowsBlock * kRowsAtOnce) {
        int32_t c[kRowsAtOnce];
        uint64_t votes[kRowsAtOnce];
#pragma unroll
        for (int k = 0; k < kRowsAtOnce; ++k) {
            const uint64_t i = first + (uint32_t)k * kRowsBlock + threadIdx.x;
            c[k] = i < rows ? class_of(t, i) : kIgnored;
        }
        __syncthreads();                                    // the last round's counts are read
#pragma unroll
        for (int k = 0; k < kRowsAtOnce; ++k) {
            votes[k] = __builtin_amdgcn_ballot_w64(c[k] != kIgnored);
            if (lane == 0u) counts[(uint32_t)k * waves + wave] = (uint32_t)__builtin_popcountll(votes[k]);
        }
        __syncthreads();
        // Every wave sums them alike: before each slot, and all.
        static_assert(slots == 128, "two slots a lane");
        const uint32_t mine = counts[2u * lane], pair = mine + counts[2u * lane + 1u];
        uint32_t upto = pair;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t other = __shfl_up(upto, off, 64);
            if (lane >= (uint32_t)off) upto += other;
        }
#pragma unroll
        for (int k = 0; k < kRowsAtOnce; ++k) {
            const uint64_t i = first + (uint32_t)k * kRowsBlock + threadIdx.x;
            const uint32_t slot = (uint32_t)k * waves + wave;
            const uint32_t before = __shfl(upto - pair, (int)(slot / 2u), 64);
            const uint32_t half = __shfl(mine, (int)(slot / 2u), 64);
            if (i >= rows) continue;
            const uint32_t j = done + before + (slot % 2u ? half : 0u) +
                               (uint32_t)__builtin_popcountll(votes[k] & ((1ull << lane) - 1ull));
            if (BACKWARD) out.place[i] = c[k] == kIgnored ? ~0u : j;
            if (c[k] == kIgnored) {
                if (lse != nullptr) lse[i] = 0.0f;
                if (loss != nullptr) loss[i] = 0.0f;
                continue;
            }
            out.row[j] = (uint32_t)i;
            out.target[j] = c[k];
            if constexpr (BACKWARD)
                out.weight[j] = c[k] == kOutside ? __builtin_nanf("") : (reduction == kEach ? grad[i] : 1.0f) * scale;
        }
        done += __shfl(upto, 63, 64);
    }
    if (threadIdx.x != 0u) return;
    *out.count = done;
    if constexpr (BACKWARD) {
        float common = 1.0f;
        if (reduction != kEach) common = grad != nullptr ? *grad : grad_value;
        if (reduction == kMean) common = common / (float)(done > 0u ? done : 1u);
        *out.unscale = done > 0u ? common / scale : 0.0f;   // rows that do not count give none of an infinity either
    }
}

// ---- operands as the products take them --------------------------------------------------------------
// Float32 as three bfloat16 values whose sum it is (or nearly: the last is
// rounded where float32's exponent ends).  What is not finite is the first
// alone.
__device__ __forceinline__ void three_planes(float v, uint16_t (&plane)[3]) {
    uint32_t high = f32_to_bf16(v);
    if ((high & 0x7fffu) == 0x7f80u) high = f32_bits(v) >> 16;           // rounded up to infinity, or infinite
    const bool finite = (f32_bits(v) & 0x7f800000u) != 0x7f800000u;
    plane[0] = (uint16_t)high;
    const float left = v - bf16_to_f32((uint16_t)high);
    plane[1] = finite ? f32_to_bf16(left) : (uint16_t)0;
    plane[2] = finite ? f32_to_bf16(left - bf16_to_f32(plane[1])) : (uint16_t)0;
}

// Rows of `width` elements at any address to rows of `pitch` (a multiple of
// 64), the end of each zero, and to the next multiple of 64 rows of zeros.
// `row` and `live`: a row each from there, as many as `live` says.  8192 x 4096
// bfloat16 21.8 us (5.5 TB/s of what it reads and writes), 10007 x 1001 float32
// 18.3.
template <class T>
__global__ __launch_bounds__(kBlock) void pack_kernel(const void *from, uint32_t width, uint16_t *to, uint32_t pitch,
                                                      uint64_t plane, uint32_t rows, const uint32_t *row,
                                                      const uint32_t *live) {
    if (live != nullptr) rows = *live;
    const uint64_t groups = pitch / 8u, all = whole_steps(rows) * groups;
    for (uint64_t g = blockIdx.x * (uint64_t)kBlock + threadIdx.x; g < all; g += (uint64_t)gridDim.x * kBlock) {
        const uint32_t r = (uint32_t)(g / groups), c = (uint32_t)(g % groups) * 8u;
        const uint64_t source = (row == nullptr || r >= rows ? r : row[r]) * (uint64_t)width + c;
        const uint32_t end = r < rows ? width : 0u;
        Raw8<T> in;
        if (c + 8u <= end) load8<T, false>(in, from, source);
        else load_end<T>(in, from, source, c < end ? end - c : 0u);
        uint16_t *out = to + r * (uint64_t)pitch + c;
        if constexpr (T::code == NT_F32) {
            float v[8];
            widen8<T>(v, in);
            uint16_t planes[3][8];
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) {
                uint16_t one[3];
                three_planes(v[k], one);
                planes[0][k] = one[0];
                planes[1][k] = one[1];
                planes[2][k] = one[2];
            }
            for (int k = 0; k < 3; ++k)
                *reinterpret_cast<u32x4_t *>(out + k * plane) = __builtin_bit_cast(u32x4_t, planes[k]);
        } else {
            *reinterpret_cast<u32x4_t *>(out) = in.w[0];
        }
    }
}

// ---- what becomes of the products' tiles ------------------------------------------------------------------
// Of a difference that is made first.  With log2(e) multiplied into both sides
// of it, for one operation less (a forward call of 8192 x 50257 x 768 bfloat16
// 512 us, so 518, a backward call the same), the rounding of a product stayed
// in the exponent, 2^-24 of a logit: exp(z - lse) - 1 of a target at 1536 was
// off by 9e-5 where it is zero, and of logits past 2^32 sums were zero or
// infinite.
__device__ __forceinline__ float exp_of(float d) { return __builtin_amdgcn_exp2f(d * kLog2e); }

// Two halves' maximum m and sum of exp(z - m), joined.
struct Partial2 {
    float most, sum;
};
__device__ __forceinline__ Partial2 join(Partial2 a, Partial2 b) {
    const float most = fmaxf(a.most, b.most);
    const float fa = a.most == most ? 1.0f : exp_of(a.most - most), fb = b.most == most ? 1.0f : exp_of(b.most - most);
    return Partial2{most, a.sum * fa + b.sum * fb};
}

// Logits to a maximum and sum of each row's part of a wave's tile, and the
// target's logit: a lane has four classes of a row in each of its tiles, and 8
// bytes a row and 128 classes (of large tiles) are stored for what would be 256.
// 8192 x 50257 x 768 bfloat16, a tenth ignored: 531 us with the product, 1.07
// PFLOP/s; the product's 12 steps are short for these ends.
struct FinishLoss {
    Partial2 *partials;         // [slot][rows]
    float *target_logit;        // [rows]
    const int32_t *target;
    const uint32_t *live;
    uint32_t first, classes;    // of the piece: its first class, and their number
    uint32_t first_slot;
    uint64_t rows;              // length of a slot

    template <class T>
    __device__ __forceinline__ void operator()(const f32x4 (&acc)[T::TP][T::TQ], uint32_t p_first, uint32_t q_first,
                                               uint32_t, uint32_t lane) const {
        const uint32_t count = *live, slot = first_slot + p_first / T::kWaveP, up = p_first + 4u * (lane >> 4);
        const bool whole = p_first + T::kWaveP <= classes;
#pragma unroll
        for (int j = 0; j < T::TQ; ++j) {
            const uint32_t q = q_first + 16u * j + (lane & 15u);
            const uint32_t place = q < count ? (uint32_t)target[q] - first - up : ~0u;
            float most = -kInfinity;
            f32x4 z[T::TP];
#pragma unroll
            for (int i = 0; i < T::TP; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    z[i][r] = whole || up + 16u * i + r < classes ? acc[i][j][r] : -kInfinity;
                    most = fmaxf(most, z[i][r]);
                }
            if (__builtin_amdgcn_ballot_w64(place < 16u * T::TP) != 0) {
#pragma unroll
                for (int i = 0; i < T::TP; ++i)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (place == 16u * i + r) target_logit[q] = z[i][r];
            }
            most = fmaxf(most, __shfl_xor(most, 16, 64));
            most = fmaxf(most, __shfl_xor(most, 32, 64));
            const float from = most == -kInfinity ? 0.0f : most;
            float sum = 0.0f;
#pragma unroll
            for (int i = 0; i < T::TP; ++i)
#pragma unroll
                for (int r = 0; r < 4; ++r) sum += exp_of(z[i][r] - from);
            sum += __shfl_xor(sum, 16, 64);
            sum += __shfl_xor(sum, 32, 64);
            if (lane < 16u && q < count) partials[slot * rows + q] = Partial2{most, sum};
        }
    }
};

// Four values rounded to a 16-bit type, one rounding to nearest even each (the
// packed conversions of gfx950).
template <bool HALF>
__device__ __forceinline__ u32x2 narrow4(f32x4 v) {
    if constexpr (HALF) return __builtin_bit_cast(u32x2, __builtin_convertvector(v, f16x4_t));
    else return __builtin_bit_cast(u32x2, __builtin_convertvector(v, bf16x4_t));
}

// Two tiles' four values a lane, along p, to eight consecutive ones: lanes 16
// to 31 exchange with the first 16, the last 16 with those before them, so
// that rows of 16 lanes 0 and 2 hold the first tile's halves and 1 and 3 the
// second's.  A lane's 16 bytes then lie beside the next lanes' (64 bytes of a
// line at a time instead of 32).
struct Pair {
    u32x4_t words;
    __device__ __forceinline__ Pair(u32x2 first, u32x2 second) {
        const auto x = __builtin_amdgcn_permlane16_swap(first.x, second.x, false, false);
        const auto y = __builtin_amdgcn_permlane16_swap(first.y, second.y, false, false);
        words = u32x4_t{x[0], y[0], x[1], y[1]};
    }
    // Where a lane's elements begin, from the first tile's first on.
    static __device__ __forceinline__ uint32_t place(uint32_t lane) { return ((lane >> 4) & 1u) * 16u + (lane >> 5) * 8u; }
};

// Logits to dz, stored 16 bytes a lane.  8192 x 32000 x 4096 bfloat16, a tenth
// ignored: 1.64 ms with the product, 1.18 PFLOP/s; 50257 x 768 0.69 ms, 0.82
// with 0.74 GB stored.  The columns from the piece's last class to the line's
// end and the rows from the last counted one to a whole step are zero.
template <bool HALF, int PLANES>
struct FinishGrad {
    uint16_t *dz;
    uint64_t plane;
    uint32_t pitch;
    const float *lse, *weight;  // lse by row, the others by counted row
    const int32_t *target;
    const uint32_t *row, *live;
    uint32_t first, classes;

    template <class T>
    __device__ __forceinline__ void operator()(const f32x4 (&acc)[T::TP][T::TQ], uint32_t p_first, uint32_t q_first,
                                               uint32_t, uint32_t lane) const {
        const uint32_t count = *live, padded = whole_steps(count), up = p_first + 4u * (lane >> 4);
        const bool whole = p_first + T::kWaveP <= classes;
#pragma unroll
        for (int j = 0; j < T::TQ; ++j) {
            const uint32_t q = q_first + 16u * j + (lane & 15u);
            if (q >= padded) continue;
            const bool there = q < count;
            // A row of padding: exp(z - infinity) is zero, as its sums z are finite.
            const float from = there ? lse[row[q]] : kInfinity;
            const float by = there ? weight[q] : 0.0f;
            const uint32_t place = there ? (uint32_t)target[q] - first - up : ~0u;
            const bool any = __builtin_amdgcn_ballot_w64(place < 16u * T::TP) != 0;
            uint16_t *line = dz + q * (uint64_t)pitch;
            const auto tile = [&](int i) {
                f32x4 v;
#pragma unroll
                for (int r = 0; r < 4; ++r) v[r] = exp_of(acc[i][j][r] - from);
                if (any) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[r] = place == 16u * i + r ? v[r] - 1.0f : v[r];
                }
                v *= by;
                if (!whole) {
#pragma unroll
                    for (int r = 0; r < 4; ++r) v[r] = up + 16u * i + r < classes ? v[r] : 0.0f;
                }
                return v;
            };
            if constexpr (PLANES == 1) {
#pragma unroll
                for (int i = 0; i < T::TP; i += 2) {
                    const Pair pair(narrow4<HALF>(tile(i)), narrow4<HALF>(tile(i + 1)));
                    const uint32_t c = p_first + 16u * i + Pair::place(lane);
                    if (whole || c < pitch) *reinterpret_cast<u32x4_t *>(line + c) = pair.words;
                }
            } else {
#pragma unroll
                for (int i = 0; i < T::TP; ++i) {
                    const f32x4 v = tile(i);
                    if (!whole && up + 16u * i >= pitch) continue;
                    uint16_t e[3][4];
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        uint16_t one[3];
                        three_planes(v[r], one);
                        e[0][r] = one[0];
                        e[1][r] = one[1];
                        e[2][r] = one[2];
                    }
                    for (int k = 0; k < 3; ++k)
                        *reinterpret_cast<u32x2 *>(line + k * plane + up + 16 * i) = __builtin_bit_cast(u32x2, e[k]);
                }
            }
        }
    }
};

// Sums in float32 of a product that is split along k, or goes on with the next
// piece of the vocabulary: stored, or added to those before.  A split's sums
// cost 8 bytes an element to write and read again, splits_of when that pays.
struct FinishSum {
    float *sums;                // [split][rows][width]
    uint64_t split_stride;
    uint32_t width;             // a multiple of 8
    uint32_t rows;
    const uint32_t *live;       // how many of the rows there are; or null, all
    bool add;

    template <class T>
    __device__ __forceinline__ void operator()(const f32x4 (&acc)[T::TP][T::TQ], uint32_t p_first, uint32_t q_first,
                                               uint32_t split, uint32_t lane) const {
        const uint32_t count = live != nullptr ? *live : rows, up = p_first + 4u * (lane >> 4);
#pragma unroll
        for (int j = 0; j < T::TQ; ++j) {
            const uint32_t q = q_first + 16u * j + (lane & 15u);
            if (q >= count) continue;
            float *line = sums + split * split_stride + q * (uint64_t)width + up;
#pragma unroll
            for (int i = 0; i < T::TP; ++i) {
                if (up + 16u * i >= width) continue;
                f32x4 v = acc[i][j];
                if (add) v += *reinterpret_cast<const f32x4 *>(line + 16 * i);
                *reinterpret_cast<f32x4 *>(line + 16 * i) = v;
            }
        }
    }
};

// A piece's rows of dW.  Both products of 8192 x 32000 x 4096 bfloat16, a tenth
// of the rows ignored: 3.10 ms, 1.25 PFLOP/s; of 50257 x 768 0.98 ms, 1.16.
template <class S>
struct FinishWeight {
    typename S::raw *to;
    const float *unscale;
    uint32_t width, classes;
    bool even;                  // 16 bytes can be stored at once

    template <class T>
    __device__ __forceinline__ void operator()(const f32x4 (&acc)[T::TP][T::TQ], uint32_t p_first, uint32_t q_first,
                                               uint32_t, uint32_t lane) const {
        const float by = *unscale;
        const uint32_t up = p_first + 4u * (lane >> 4);
#pragma unroll
        for (int j = 0; j < T::TQ; ++j) {
            const uint32_t q = q_first + 16u * j + (lane & 15u);
            if (q >= classes) continue;
            typename S::raw *line = to + q * (uint64_t)width;
            if (even && S::code != NT_F32) {
#pragma unroll
                for (int i = 0; i < T::TP; i += 2) {
                    const Pair pair(narrow4<S::code == NT_F16>(acc[i][j] * by),
                                    narrow4<S::code == NT_F16>(acc[i + 1][j] * by));
                    const uint32_t c = p_first + 16u * i + Pair::place(lane);
                    if (c < width) *reinterpret_cast<u32x4_t *>(line + c) = pair.words;
                }
                continue;
            }
#pragma unroll
            for (int i = 0; i < T::TP; ++i) {
                const uint32_t c = up + 16u * i;
                const f32x4 v = acc[i][j] * by;
                if (even) {
                    if (c < width) *reinterpret_cast<f32x4 *>(line + c) = v;
                } else {
#pragma unroll
                    for (int r = 0; r < 4; ++r)
                        if (c + r < width) store1<S>(line, c + r, v[r]);
                }
            }
        }
    }
};

// ---- the ends of both passes -----------------------------------------------------------------------------
// lse and loss of ROWS rows a workgroup, over which the lanes share out their
// slots: 16 rows (7373 rows of 394 slots 7.9 us, 2.9 TB/s), or one where there
// are few, whose slots are read at once.
template <int ROWS, int THREADS>
__global__ __launch_bounds__(THREADS) void loss_rows_kernel(const Partial2 *partials, uint32_t slots, uint64_t stride,
                                                            const float *target_logit, Rows rows, float *lse,
                                                            float *loss) {
    constexpr uint32_t slices = THREADS / ROWS;
    __shared__ Partial2 shared[slices][ROWS + 1];
    const uint32_t count = *rows.count, r = threadIdx.x % ROWS, slice = threadIdx.x / ROWS;
    for (uint32_t first = blockIdx.x * ROWS; first < count; first += gridDim.x * ROWS) {
        const uint32_t j = first + r;
        Partial2 p{-kInfinity, 0.0f};
        if (j < count) {
            uint32_t k = slice;
            for (; k + 7u * slices < slots; k += 8u * slices) {
                Partial2 part[8];
#pragma unroll
                for (int u = 0; u < 8; ++u) part[u] = partials[(k + u * slices) * stride + j];
#pragma unroll
                for (int u = 0; u < 8; ++u) p = join(p, part[u]);
            }
            for (; k < slots; k += slices) p = join(p, partials[k * stride + j]);
        }
        __syncthreads();
        shared[slice][r] = p;
        __syncthreads();
        for (uint32_t half = slices / 2u; half > 0u; half /= 2u) {
            if (slice < half) shared[slice][r] = join(shared[slice][r], shared[slice + half][r]);
            __syncthreads();
        }
        if (slice == 0 && j < count) {
            p = shared[0][r];
            const float value = p.most + __builtin_amdgcn_logf(p.sum) * kLn2;
            const uint32_t row = rows.row[j];
            if (lse != nullptr) lse[row] = value;
            if (loss != nullptr) loss[row] = rows.target[j] == kOutside ? __builtin_nanf("") : value - target_logit[j];
        }
    }
}

// Sum or mean of the rows' losses, in 64 bits and a fixed order.
__global__ __launch_bounds__(kRowsBlock) void loss_sum_kernel(const float *each, uint32_t rows, const uint32_t *count,
                                                              bool mean, float *loss) {
    __shared__ double shared[kRowsBlock / 64];
    double sum = 0.0;
    for (uint32_t i = threadIdx.x; i < rows; i += kRowsBlock) sum += (double)each[i];
    sum = wave_sum(sum);
    if ((threadIdx.x & 63u) == 0u) shared[threadIdx.x >> 6] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int k = 1; k < kRowsBlock / 64; ++k) sum += shared[k];
        const uint32_t n = *count;
        *loss = (float)(mean ? sum / (double)(n > 0 ? n : 1u) : sum);
    }
}

// ---- a few rows -----------------------------------------------------------------------------------------
// Scoring a token or a few: bound by the one read of the weights, which a tile
// of the matrix cores would spend on rows that are not there, after launches
// that gather and pack.  A wave takes a run of classes, four at a time, and
// holds its lanes' part of the sums of all rows; the weights are read where
// and as they lie.  Two launches.  A call of one row of 50257 x 768 float16:
// 20.5 us (with 1024 workgroups 23.7), as a tile 27.9; 32000 x 4096 45.1 and
// 53.4.  Of two rows 29.5 and 27.8, four 41.5 and 27.8: so one row only, but up
// to four of what the tiles would have to pack first (float32, and widths that
// are not whole steps), five times the weights' bytes.
constexpr uint32_t kFewRows = 4, kFewAtOnce = 4, kFewBlocks = 2048;

template <class T>
__device__ __forceinline__ void load_group(float (&out)[8], const void *base, uint64_t row, uint32_t c, uint32_t width) {
    Raw8<T> raw;
    if (c + kGroup <= width) load8<T, false>(raw, base, row + c);
    else load_end<T>(raw, base, row + c, c < width ? width - c : 0u);
    widen8<T>(out, raw);
}

template <class T, int ROWS>
__global__ __launch_bounds__(kBlock) void few_rows_kernel(const void *x, const void *w, Targets t, uint32_t width,
                                                          Partial2 *partials, float *target_logit) {
    __shared__ Partial2 shared[kBlock / 64][ROWS];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint64_t place = blockIdx.x * (uint64_t)(kBlock / 64) + wave, waves = gridDim.x * (uint64_t)(kBlock / 64);
    const uint32_t begin = (uint32_t)(t.classes * place / waves), end = (uint32_t)(t.classes * (place + 1u) / waves);
    Partial2 part[ROWS];
    int32_t target[ROWS];
#pragma unroll
    for (int n = 0; n < ROWS; ++n) {
        part[n] = Partial2{-kInfinity, 0.0f};
        target[n] = class_of(t, n);
    }
    for (uint32_t v = begin; v < end; v += kFewAtOnce) {
        float z[kFewAtOnce][ROWS];
#pragma unroll
        for (uint32_t k = 0; k < kFewAtOnce; ++k)
#pragma unroll
            for (int n = 0; n < ROWS; ++n) z[k][n] = 0.0f;
        for (uint32_t first = 0; first < width; first += 64u * kGroup) {
            const uint32_t c = first + lane * kGroup;
            float weights[kFewAtOnce][8];
#pragma unroll
            for (uint32_t k = 0; k < kFewAtOnce; ++k)
                load_group<T>(weights[k], w, (v + k < end ? v + k : end - 1u) * (uint64_t)width, c, width);
#pragma unroll
            for (int n = 0; n < ROWS; ++n) {
                float values[8];
                load_group<T>(values, x, n * (uint64_t)width, c, width);
#pragma unroll
                for (uint32_t k = 0; k < kFewAtOnce; ++k)
#pragma unroll
                    for (int e = 0; e < 8; ++e) z[k][n] = __builtin_fmaf(weights[k][e], values[e], z[k][n]);
            }
        }
#pragma unroll
        for (int n = 0; n < ROWS; ++n) {
            float most = part[n].most;
#pragma unroll
            for (uint32_t k = 0; k < kFewAtOnce; ++k) {
                z[k][n] = lanes_sum(z[k][n], 64u);
                if (v + k >= end) z[k][n] = -kInfinity;
                else if ((int32_t)(v + k) == target[n] && lane == 0u) target_logit[n] = z[k][n];
                most = fmaxf(most, z[k][n]);
            }
            const float from = most == -kInfinity ? 0.0f : most;
            float sum = part[n].sum * (part[n].most == most ? 1.0f : exp_of(part[n].most - from));
#pragma unroll
            for (uint32_t k = 0; k < kFewAtOnce; ++k) sum += exp_of(z[k][n] - from);
            part[n] = Partial2{most, sum};
        }
    }
    if (lane == 0u)
#pragma unroll
        for (int n = 0; n < ROWS; ++n) shared[wave][n] = part[n];
    __syncthreads();
    if (threadIdx.x >= ROWS) return;
    Partial2 all = shared[0][threadIdx.x];
    for (uint32_t k = 1; k < kBlock / 64; ++k) all = join(all, shared[k][threadIdx.x]);
    partials[blockIdx.x * (uint64_t)ROWS + threadIdx.x] = all;
}

// lse, loss and their reduction for those rows: one workgroup, a lane a slot.
__global__ __launch_bounds__(kRowsBlock) void few_loss_kernel(const Partial2 *partials, uint32_t slots, Targets t,
                                                              uint32_t rows, const float *target_logit,
                                                              int32_t reduction, float *lse, float *loss) {
    __shared__ Partial2 shared[kRowsBlock / 64];
    double total = 0.0;
    uint32_t counted = 0;
    for (uint32_t n = 0; n < rows; ++n) {
        Partial2 p{-kInfinity, 0.0f};
        for (uint32_t k = threadIdx.x; k < slots; k += kRowsBlock) p = join(p, partials[k * (uint64_t)rows + n]);
#pragma unroll
        for (int off = 32; off > 0; off >>= 1)
            p = join(p, Partial2{__shfl_xor(p.most, off, 64), __shfl_xor(p.sum, off, 64)});
        __syncthreads();
        if ((threadIdx.x & 63u) == 0u) shared[threadIdx.x >> 6] = p;
        __syncthreads();
        if (threadIdx.x != 0u) continue;
        for (uint32_t k = 1; k < kRowsBlock / 64; ++k) p = join(p, shared[k]);
        const int32_t c = class_of(t, n);
        const float value = p.most + __builtin_amdgcn_logf(p.sum) * kLn2;
        const float each = c == kIgnored ? 0.0f : c == kOutside ? __builtin_nanf("") : value - target_logit[n];
        if (lse != nullptr) lse[n] = c == kIgnored ? 0.0f : value;
        if (reduction == kEach) loss[n] = each;
        total += (double)each;
        counted += c != kIgnored;
    }
    if (threadIdx.x == 0u && reduction != kEach)
        *loss = (float)(reduction == kMean ? total / (double)(counted > 0 ? counted : 1u) : total);
}

// ---- dx -------------------------------------------------------------------------------------------------
// dx (or split rows of dW, with no `place`) from its sums, eight columns a
// lane; rows that are not counted are zero.  8192 x 4096 bfloat16 of one split
// 31.2 us, 6.0 TB/s.
template <class T>
__global__ __launch_bounds__(kBlock) void grad_kernel(const float *sums, uint64_t split_stride, uint32_t splits,
                                                      uint32_t pitch, const uint32_t *place, const float *unscale,
                                                      uint32_t all, uint32_t width, bool even, typename T::raw *dx) {
    const float by = *unscale;
    const uint32_t groups = (width + 7u) / 8u;
    const uint64_t items = all * (uint64_t)groups;
    for (uint64_t g = blockIdx.x * (uint64_t)kBlock + threadIdx.x; g < items; g += (uint64_t)gridDim.x * kBlock) {
        const uint32_t i = (uint32_t)(g / groups), c = (uint32_t)(g % groups) * 8u, j = place != nullptr ? place[i] : i;
        f32x4 v[2] = {{0.0f, 0.0f, 0.0f, 0.0f}, {0.0f, 0.0f, 0.0f, 0.0f}};
        if (j != ~0u) {
            const float *from = sums + j * (uint64_t)pitch + c;
#pragma unroll 4
            for (uint32_t s = 0; s < splits; ++s) {
                v[0] += *reinterpret_cast<const f32x4 *>(from + s * split_stride);
                v[1] += *reinterpret_cast<const f32x4 *>(from + s * split_stride + 4);
            }
            v[0] *= by;
            v[1] *= by;
        }
        typename T::raw *out = dx + i * (uint64_t)width + c;
        if (even) {
            if constexpr (T::code == NT_F32) {
                *reinterpret_cast<f32x4 *>(out) = v[0];
                *reinterpret_cast<f32x4 *>(out + 4) = v[1];
            } else {
                const u32x2 low = narrow4<T::code == NT_F16>(v[0]), high = narrow4<T::code == NT_F16>(v[1]);
                *reinterpret_cast<u32x4_t *>(out) = u32x4_t{low.x, low.y, high.x, high.y};
            }
        } else {
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k)
                if (c + k < width) store1<T>(out, k, v[k >> 2][k & 3]);
        }
    }
}

// ---- launches ----------------------------------------------------------------------------------------
template <TileShape SHAPE, class T>
constexpr bool is_shape() { return T::BP == size_p(SHAPE) && T::BQ == size_q(SHAPE); }

using Large = Tile<256, 256, 2, 4>;
using Middle = Tile<128, 128, 2, 2>;
using Tall = Tile<256, 128, 4, 2, 3>;
using Few = Tile<128, 64, 4, 1, 3>;
static_assert(is_shape<kLarge, Large>() && is_shape<kMiddle, Middle>() && is_shape<kTall, Tall>() &&
              is_shape<kFew, Few>(), "nt_tiles.hpp counts tiles of these");

// Calls launch(shape) with the tile of the logits, or of the two products of dz.
template <class F>
static void with_logits_tile(TileShape shape, F &&launch) {
    if (shape == kLarge) launch(Large{});
    else if (shape == kMiddle) launch(Middle{});
    else if (shape == kTall) launch(Tall{});
    else launch(Few{});
}
template <class F>
static void with_grads_tile(TileShape shape, F &&launch) {
    if (shape == kLarge) launch(Large{});
    else if (shape == kMiddle) launch(Middle{});
    else launch(Few{});
}

struct Problem {
    const void *x, *w;
    int32_t dtype;
    uint32_t rows, classes, width;
    Targets targets;
    int32_t reduction;
};

static uint32_t blocks_of(uint64_t items, uint32_t each) {
    const uint64_t blocks = (items + each - 1) / each;
    return blocks < 1 ? 1u : blocks > 8192u ? 8192u : (uint32_t)blocks;
}

template <class T> struct Kind {            // how the products take a type
    static constexpr bool kHalf = T::code == NT_F16;
    static constexpr int kPlanes = T::code == NT_F32 ? 3 : 1;
};

template <class T>
static int32_t few_rows_of(const Problem &a, int32_t device, float *loss, float *lse, void *stream) {
    hipStream_t s = (hipStream_t)stream;
    const uint32_t blocks = std::min(kFewBlocks, (a.classes + kBlock / 64 - 1) / (kBlock / 64));
    Partial2 *partials = nullptr;
    float *target_logit = nullptr;
    Workspace room;
    room.want(&partials, (uint64_t)blocks * a.rows);
    room.want(&target_logit, a.rows);
    const int32_t rc = room.allocate(device, stream);
    if (rc != NT_OK) return rc;
    const auto launch = [&](auto rows) {
        few_rows_kernel<T, decltype(rows)::value><<<blocks, kBlock, 0, s>>>(a.x, a.w, a.targets, a.width, partials,
                                                                            target_logit);
    };
    if (a.rows == 1u) launch(std::integral_constant<int, 1>{});
    else if (a.rows == 2u) launch(std::integral_constant<int, 2>{});
    else if (a.rows == 3u) launch(std::integral_constant<int, 3>{});
    else launch(std::integral_constant<int, 4>{});
    few_loss_kernel<<<1, kRowsBlock, 0, s>>>(partials, blocks, a.targets, a.rows, target_logit, a.reduction, lse, loss);
    return hip_check(hipGetLastError(), "linear cross entropy launch");
}

template <class T>
static int32_t forward_of(const Problem &a, int32_t device, float *loss, float *lse, void *stream) {
    constexpr int planes = Kind<T>::kPlanes;
    constexpr bool half = Kind<T>::kHalf;
    hipStream_t s = (hipStream_t)stream;
    const LossPlan plan = loss_plan(a.rows, a.classes, a.width, planes, (uintptr_t)a.w % 16u == 0, false);
    const uint32_t pitch = plan.pitch, padded = whole_steps(a.rows), piece = plan.piece, pieces = plan.pieces;
    const bool pack_w = plan.packed;
    if (a.rows <= (planes > 1 || pitch != a.width ? kFewRows : 1u)) return few_rows_of<T>(a, device, loss, lse, stream);
    uint32_t slots_piece = 0, slots = 0;                  // of a whole piece, of all
    with_logits_tile(plan.logits, [&](auto shape) {
        using Shape = decltype(shape);
        slots_piece = tiles_of(piece, Shape::BP) * Shape::WP;
        slots = (pieces - 1) * slots_piece + tiles_of(a.classes - (pieces - 1) * piece, Shape::BP) * Shape::WP;
    });

    Rows rows{};
    uint16_t *px = nullptr, *pw = nullptr;
    Partial2 *partials = nullptr;
    float *target_logit = nullptr, *each = nullptr;
    Workspace room;
    room.want(&rows.count, 1);
    room.want(&rows.row, a.rows);
    room.want(&rows.target, a.rows);
    room.want(&target_logit, a.rows);
    room.want(&partials, (uint64_t)slots * a.rows);
    room.want(&px, (uint64_t)planes * padded * pitch);
    if (pack_w) room.want(&pw, (uint64_t)planes * whole_steps(piece) * pitch);
    if (a.reduction != kEach) room.want(&each, a.rows);
    int32_t rc = room.allocate(device, stream);
    if (rc != NT_OK) return rc;
    float *to = a.reduction == kEach ? loss : each;

    rows_kernel<false><<<1, kRowsBlock, 0, s>>>(a.targets, a.rows, rows, nullptr, 0.0f, a.reduction, false, lse, to);
    const uint64_t plane_x = (uint64_t)padded * pitch, plane_w = (uint64_t)whole_steps(piece) * pitch;
    pack_kernel<T><<<blocks_of(padded * (uint64_t)(pitch / 8u), kBlock), kBlock, 0, s>>>(
        a.x, a.width, px, pitch, plane_x, a.rows, rows.row, rows.count);
    for (uint32_t k = 0; k < pieces; ++k) {
        const uint32_t first = k * piece, classes = std::min(piece, a.classes - first);
        const void *weights = static_cast<const typename T::raw *>(a.w) + (uint64_t)first * a.width;
        if (pack_w)
            pack_kernel<T><<<blocks_of(classes * (uint64_t)(pitch / 8u), kBlock), kBlock, 0, s>>>(
                weights, a.width, pw, pitch, plane_w, classes, nullptr, nullptr);
        Product product{};
        product.p = Operand{pack_w ? pw : static_cast<const uint16_t *>(weights), nullptr, pitch, plane_w, classes};
        product.q = Operand{px, nullptr, pitch, plane_x, a.rows};
        product.splits = 1;
        product.depth = pitch;
        product.live = rows.count;
        const FinishLoss finish{partials, target_logit, rows.target, rows.count, first, classes, k * slots_piece, a.rows};
        with_logits_tile(plan.logits, [&](auto shape) {
            using Shape = decltype(shape);
            product.tiles_p = tiles_of(classes, Shape::BP);
            product.tiles_q = tiles_of(a.rows, Shape::BQ);
            launch_product<half, Shape, true, true, planes>(product, finish, s);
        });
    }
    if (a.rows <= kUnits)
        loss_rows_kernel<1, 1024><<<a.rows, 1024, 0, s>>>(partials, slots, a.rows, target_logit, rows, lse, to);
    else
        loss_rows_kernel<16, 512><<<blocks_of(a.rows, 16), 512, 0, s>>>(partials, slots, a.rows, target_logit, rows, lse,
                                                                        to);
    if (a.reduction != kEach)
        loss_sum_kernel<<<1, kRowsBlock, 0, s>>>(each, a.rows, rows.count, a.reduction == kMean, loss);
    return hip_check(hipGetLastError(), "linear cross entropy launch");
}

template <class T>
static int32_t backward_of(const Problem &a, int32_t device, const float *grad, float grad_value, const float *lse,
                           void *dx, void *dw, void *stream) {
    constexpr int planes = Kind<T>::kPlanes;
    constexpr bool half = Kind<T>::kHalf;
    using Raw = typename T::raw;
    hipStream_t s = (hipStream_t)stream;
    const LossPlan plan = loss_plan(a.rows, a.classes, a.width, planes, (uintptr_t)a.w % 16u == 0, true);
    const uint32_t pitch = plan.pitch, padded = whole_steps(a.rows), piece = plan.piece, pieces = plan.pieces;
    const bool pack_w = plan.packed;
    const uint32_t dz_pitch = whole_steps(piece);
    const Splits splits = plan.splits;

    Rows rows{};
    uint16_t *px = nullptr, *pw = nullptr, *dz = nullptr;
    float *sums = nullptr, *weight_sums = nullptr;
    Workspace room;
    room.want(&rows.count, 1);
    room.want(&rows.unscale, 1);
    room.want(&rows.row, a.rows);
    room.want(&rows.target, a.rows);
    room.want(&rows.weight, a.rows);
    room.want(&rows.place, a.rows);
    room.want(&px, (uint64_t)planes * padded * pitch);
    // The weights' last lines, where those are read in place and do not fill a step.
    const bool ragged = !pack_w && a.classes % kDepth != 0;
    if (pack_w) room.want(&pw, (uint64_t)planes * whole_steps(piece) * pitch);
    else if (ragged) room.want(&pw, (uint64_t)kDepth * pitch);
    room.want(&dz, (uint64_t)planes * padded * dz_pitch);
    room.want(&sums, (uint64_t)splits.input * a.rows * pitch);
    if (splits.weight > 1u) room.want(&weight_sums, (uint64_t)splits.weight * piece * pitch);
    int32_t rc = room.allocate(device, stream);
    if (rc != NT_OK) return rc;

    rows_kernel<true><<<1, kRowsBlock, 0, s>>>(a.targets, a.rows, rows, grad, grad_value, a.reduction, half, nullptr,
                                               nullptr);
    const uint64_t plane_x = (uint64_t)padded * pitch, plane_w = (uint64_t)whole_steps(piece) * pitch;
    const uint64_t plane_dz = (uint64_t)padded * dz_pitch;
    pack_kernel<T><<<blocks_of(padded * (uint64_t)(pitch / 8u), kBlock), kBlock, 0, s>>>(
        a.x, a.width, px, pitch, plane_x, a.rows, rows.row, rows.count);
    if (ragged) {
        const uint32_t lines = a.classes % kDepth;
        pack_kernel<T><<<blocks_of(kDepth * (uint64_t)(pitch / 8u), kBlock), kBlock, 0, s>>>(
            static_cast<const Raw *>(a.w) + (uint64_t)(a.classes - lines) * a.width, a.width, pw, pitch, 0, lines,
            nullptr, nullptr);
    }
    for (uint32_t k = 0; k < pieces; ++k) {
        const uint32_t first = k * piece, classes = std::min(piece, a.classes - first);
        const uint32_t line = whole_steps(classes);
        const void *weights = static_cast<const Raw *>(a.w) + (uint64_t)first * a.width;
        if (pack_w)
            pack_kernel<T><<<blocks_of(classes * (uint64_t)(pitch / 8u), kBlock), kBlock, 0, s>>>(
                weights, a.width, pw, pitch, plane_w, classes, nullptr, nullptr);
        const uint16_t *w = pack_w ? pw : static_cast<const uint16_t *>(weights);
        Product logits{};
        logits.p = Operand{w, nullptr, pitch, plane_w, classes};
        logits.q = Operand{px, nullptr, pitch, plane_x, a.rows};
        logits.splits = 1;
        logits.pad = true;
        logits.depth = pitch;
        logits.live = rows.count;
        const FinishGrad<half, planes> grads{dz,         plane_dz,    line,     lse, rows.weight, rows.target,
                                             rows.row, rows.count, first, classes};
        with_logits_tile(plan.logits, [&](auto shape) {
            using Shape = decltype(shape);
            logits.tiles_p = tiles_of(line, Shape::BP);
            logits.tiles_q = tiles_of(padded, Shape::BQ);
            launch_product<half, Shape, true, true, planes>(logits, grads, s);
        });

        Product input{};                    // dx[i][h] = sum over v of dz[i][v] W[v][h]
        input.p = Operand{w, ragged && k + 1u == pieces ? pw : nullptr, pitch, plane_w, pitch};
        input.q = Operand{dz, nullptr, line, plane_dz, a.rows};
        input.splits = splits.input;
        input.depth = line;
        input.live = rows.count;
        const FinishSum sum{sums, (uint64_t)a.rows * pitch, pitch, a.rows, rows.count, k > 0};

        Product weight{};                   // dW[v][h] = sum over i of dz[i][v] x[i][h]
        weight.p = Operand{px, nullptr, pitch, plane_x, pitch};
        weight.q = Operand{dz, nullptr, line, plane_dz, line};
        weight.splits = splits.weight;
        weight.depth = a.rows;
        weight.live = rows.count;
        weight.live_depth = true;
        Raw *to = static_cast<Raw *>(dw) + (uint64_t)first * a.width;
        const bool even_weight = a.width % 8u == 0 && (uintptr_t)dw % 16u == 0;
        with_grads_tile(plan.grads, [&](auto shape) {
            using Shape = decltype(shape);
            input.tiles_p = weight.tiles_p = tiles_of(pitch, Shape::BP);
            input.tiles_q = tiles_of(a.rows, Shape::BQ);
            weight.tiles_q = tiles_of(classes, Shape::BQ);
            if (weight_sums == nullptr) {
                const FinishWeight<T> last{to, rows.unscale, a.width, classes, even_weight};
                launch_two_products<half, Shape, planes>(input, sum, weight, last, s);
            } else {
                const FinishSum last{weight_sums, (uint64_t)piece * pitch, pitch, classes, nullptr, false};
                launch_two_products<half, Shape, planes>(input, sum, weight, last, s);
            }
        });
        if (weight_sums != nullptr)
            grad_kernel<T><<<blocks_of(classes * (uint64_t)((a.width + 7u) / 8u), kBlock), kBlock, 0, s>>>(
                weight_sums, (uint64_t)piece * pitch, splits.weight, pitch, nullptr, rows.unscale, classes, a.width,
                even_weight, to);
    }
    const bool even = a.width % 8u == 0 && (uintptr_t)dx % 16u == 0;
    grad_kernel<T><<<blocks_of(a.rows * (uint64_t)((a.width + 7u) / 8u), kBlock), kBlock, 0, s>>>(
        sums, (uint64_t)a.rows * pitch, splits.input, pitch, rows.place, rows.unscale, a.rows, a.width, even,
        static_cast<Raw *>(dx));
    return hip_check(hipGetLastError(), "linear cross entropy backward launch");
}

// ---- argument checks -----------------------------------------------------------------------------------
static int32_t check_problem(const char *entry, int32_t dtype, int32_t target_size, int32_t reduction, uint64_t rows,
                             uint64_t classes, uint64_t width) {
    const std::string name(entry);
    if (!half_or_float(dtype))
        return fail(NT_ERR_TYPE, name + ": input and weight must be float32, float16 or bfloat16");
    if (target_size != 4 && target_size != 8) return fail(NT_ERR_TYPE, name + ": targets must be int32 or int64");
    if (reduction < kEach || reduction > kSum) return fail(NT_ERR_VALUE, name + ": unknown reduction");
    if (width == 0 || width > kMostPitch / 2u) return fail(NT_ERR_VALUE, name + ": the width must be 1..2**21");
    if (classes == 0 || classes >= 1u << 30) return fail(NT_ERR_VALUE, name + ": there must be 1..2**30 - 1 classes");
    if (rows >= 1u << 24) return fail(NT_ERR_VALUE, name + ": there must be fewer than 2**24 rows");
    return NT_OK;
}

}  // namespace nt

using namespace nt;

extern "C" {

int32_t nt_linear_cross_entropy(int32_t device, const void *x, const void *weight, int32_t dtype, const void *target,
                                int32_t target_size, int64_t ignore_index, int32_t reduction, float *loss, float *lse,
                                uint64_t rows, uint64_t classes, uint64_t width, void *stream) {
    clear_error();
    const char *entry = "nt_linear_cross_entropy";
    int32_t rc = check_problem(entry, dtype, target_size, reduction, rows, classes, width);
    if (rc != NT_OK) return rc;
    const int32_t index = target_size == 8 ? kInt64 : kInt32;
    rc = check_arrays(entry, {{x, dtype, rows * width, false, rows > 0},
                              {weight, dtype, classes * width, false, true},
                              {target, index, rows, false, rows > 0},
                              {loss, NT_F32, reduction == kEach ? rows : 1, true, reduction != kEach || rows > 0},
                              {lse, NT_F32, rows, true, false}});
    if (rc != NT_OK) return rc;
    if (rows == 0 && reduction == kEach) return NT_OK;
    DeviceGuard guard(device);
    if (!guard.ok()) return hip_check(guard.error(), "hipSetDevice");
    rc = refuse_capture(entry, stream);
    if (rc != NT_OK) return rc;
    if (rows == 0) return nt_fill(loss, 1, 4, 0, stream);
    const Problem a{x, weight, dtype, (uint32_t)rows, (uint32_t)classes, (uint32_t)width,
                    {target, ignore_index, (uint32_t)classes, target_size}, reduction};
    switch (dtype) {
        case NT_F32: return forward_of<TF32>(a, device, loss, lse, stream);
        case NT_F16: return forward_of<TF16>(a, device, loss, lse, stream);
        default: return forward_of<TBF16>(a, device, loss, lse, stream);
    }
}

int32_t nt_linear_cross_entropy_backward(int32_t device, const float *grad_loss, float grad_value, const void *x,
                                         const void *weight, int32_t dtype, const void *target, int32_t target_size,
                                         int64_t ignore_index, int32_t reduction, const float *lse, void *dx,
                                         void *dweight, uint64_t rows, uint64_t classes, uint64_t width, void *stream) {
    clear_error();
    const char *entry = "nt_linear_cross_entropy_backward";
    int32_t rc = check_problem(entry, dtype, target_size, reduction, rows, classes, width);
    if (rc != NT_OK) return rc;
    const int32_t index = target_size == 8 ? kInt64 : kInt32;
    rc = check_arrays(entry, {{grad_loss, NT_F32, reduction == kEach ? rows : 1, false, reduction == kEach && rows > 0},
                              {x, dtype, rows * width, false, rows > 0},
                              {weight, dtype, classes * width, false, true},
                              {target, index, rows, false, rows > 0},
                              {lse, NT_F32, rows, false, rows > 0},
                              {dx, dtype, rows * width, true, rows > 0},
                              {dweight, dtype, classes * width, true, true}});
    if (rc != NT_OK) return rc;
    DeviceGuard guard(device);
    if (!guard.ok()) return hip_check(guard.error(), "hipSetDevice");
    rc = refuse_capture(entry, stream);
    if (rc != NT_OK) return rc;
    if (rows == 0) return nt_fill(dweight, classes * width, dtype == NT_F32 ? 4 : 2, 0, stream);
    const Problem a{x, weight, dtype, (uint32_t)rows, (uint32_t)classes, (uint32_t)width,
                    {target, ignore_index, (uint32_t)classes, target_size}, reduction};
    switch (dtype) {
        case NT_F32: return backward_of<TF32>(a, device, grad_loss, grad_value, lse, dx, dweight, stream);
        case NT_F16: return backward_of<TF16>(a, device, grad_loss, grad_value, lse, dx, dweight, stream);
        default: return backward_of<TBF16>(a, device, grad_loss, grad_value, lse, dx, dweight, stream);
    }
}

}  // extern "C"
