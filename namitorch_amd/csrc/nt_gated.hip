// nt_gated.hip — the edge after a block that is normalized before and after
// it: the norm of the block's output, its gate, the residual stream's scale
// and sum, and the norm for the next block; with the backward pass.
//
// N(x; w, b) = (x - mean) rstd w + b is layer norm, or with mean 0 and rstd of
// the root mean square.  With s the residual's scale and a the gate:
//   n = N(x; u, k),   t = s r + a n,   y = N(t; w, b)
// and, with h and i the normalized t and x, g = dy w,
//   dt = rstd (g - sum g / W - h sum(g h) / W) + what t gets from elsewhere
//   dr = s dt,   da = dt n,   q = a dt u
//   dx = rstd' (q - sum q / W - i sum(q i) / W)
//   dw = sum dy h, db = sum dy, du = sum a dt i, dk = sum a dt  over rows
// (no sums of g and q where the norm takes no mean).
//
// The gate has a row for all rows, one for each run of rows (a sequence), or
// one for each row.  In the first two cases the sums over rows that du, dk and
// da need are the same two, sum(dt i) and sum(dt) of each run:
//   da = u sum(dt i) + k sum(dt),   du = a sum(dt i),   dk = a sum(dt),
// the last two added over the runs.
//
// Sums and statistics are float32 (a lane's share of a row 64 bits in the
// kernels for rows of any width), over rows in a fixed order; each result is
// rounded once.  y is of t before its rounding; the backward pass reads t.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <string>
#include <type_traits>

#include "nt_entry.hpp"
#include "nt_internal.hpp"
#include "nt_pool.hpp"
#include "nt_row_ops.hpp"
#include "nt_rows.hpp"

namespace nt {

struct Gate {
    const void *at;             // may be null
    int32_t dtype;
    uint32_t runs;              // its rows
    uint64_t run;               // rows of the stream that share one
    __device__ __forceinline__ uint64_t row(uint64_t r) const { return runs == 1u ? 0u : r / run; }
};

struct GatedForward {
    const void *x, *residual, *inner_weight, *inner_bias, *weight, *bias;
    Gate gate;
    void *total, *y;
    float *inner_mean, *inner_rstd, *mean, *rstd;      // each may be null
    uint64_t rows;
    uint32_t width;
    int32_t weight_dtype;
    float scale, eps;
    uint32_t first_block;       // of this launch
};

struct GatedBackward {
    const void *dy, *dtotal, *x, *t, *inner_weight, *inner_bias, *weight;
    Gate gate;
    const float *inner_mean, *inner_rstd, *mean, *rstd;
    void *dx, *dresidual, *dgate;
    float *row_sums;            // [rows][2]: of g and g h over each row (rows of any width)
    float *partials;            // [blocks][4][width]: sums of dt i, dt, dy h, dy
    uint64_t rows;
    uint32_t width;
    int32_t weight_dtype;
    float scale;
    uint32_t run_blocks;        // workgroups, or groups of rows, of each run
    uint32_t first_block;       // of this launch
};

// Sum of a value of 64 bits over the workgroup, as float32 on every lane.
__device__ __forceinline__ float block_total(double v, double *shared) {
    v = wave_sum(v);
    __syncthreads();
    if ((threadIdx.x & 63u) == 0u) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    double total = 0.0;
    for (uint32_t k = 0; k < blockDim.x / 64u; ++k) total += shared[k];
    return (float)total;
}

// ---- rows that fit in registers ---------------------------------------------------------------------
// A row lies over lanes, eight consecutive elements (nt_rows.hpp) a lane, is
// read once, and variances are of centred values; rows share workgroups, which
// make as many turns as they need, and the next row is on its way while this
// one is summed.  (Three groups a lane, which the residual path's norms take
// for 768 columns: 8192 x 768 bfloat16 25 us, with one 17.5.)  The vectors wait
// in LDS as float32; a gate that a workgroup's rows share is multiplied into
// the first norm's weight and bias there.  Rows of less than eight, or of more
// than 8192 (whose vectors LDS does not hold), take the kernels for any width.
//
// Bound by memory where rows are long: 16384 x 4096 bfloat16 with root mean
// squares 96 us (5.6 TB/s), layer norms 114 (two sums more in turn); 8192 x 2048
// float32 55 (4.9).  Narrow rows are bound by the vector units: 8192 x 768
// bfloat16 17.3 us (2.9 TB/s), 387 instructions of each of a row's two waves, of
// four cycles each, which keep a SIMD busy 79 % of the time that its four waves
// live; they wait half of it, in turn, at the four sums over lanes.
constexpr uint32_t kGatedWaves = 4;     // per SIMD

enum GateKind { kFolded = 0, kOwn = 1, kOwnFloat = 2 };   // none or shared; a row's own, of the data's type or float32

template <class T, int KIND> struct GateType { using type = T; };
template <class T> struct GateType<T, kOwnFloat> { using type = TF32; };

template <class T>
__device__ __forceinline__ void store_row(void *base, uint64_t i, bool even, const float (&v)[8]) {
    Raw8<T> out;
    narrow8<T>(out, v);
    if (T::code == NT_F32 && even) store8<T, true>(base, i, out);
    else store8<T, false>(base, i, out);
}

// Sums of one value, or of two, over the lanes of a row, the same on each: as
// RowSum, for rows of any number of waves.
template <int MAX_WAVES>
struct GatedSum {
    float (*shared)[MAX_WAVES];
    uint32_t lanes, in_block;
    uint32_t half = 0;
    __device__ __forceinline__ float operator()(float v) {
        v = lanes_sum(v, lanes);
        if (lanes <= 64u) return v;
        float *slot = shared[half];
        half ^= 1u;
        if ((threadIdx.x & 63u) == 0u) slot[threadIdx.x >> 6] = v;
        __syncthreads();
        float total = 0.0f;
        const uint32_t waves = lanes / 64u, first = in_block * waves;
        for (uint32_t k = first; k < first + waves; ++k) total += slot[k];
        return total;
    }
};
template <int MAX_WAVES>
struct GatedSum2 {
    float (*shared)[2][MAX_WAVES];
    uint32_t lanes, in_block;
    uint32_t half = 0;
    __device__ __forceinline__ void operator()(float &u, float &v) {
        u = lanes_sum(u, lanes);
        v = lanes_sum(v, lanes);
        if (lanes <= 64u) return;
        float (*slot)[MAX_WAVES] = shared[half];
        half ^= 1u;
        if ((threadIdx.x & 63u) == 0u) {
            slot[0][threadIdx.x >> 6] = u;
            slot[1][threadIdx.x >> 6] = v;
        }
        __syncthreads();
        u = v = 0.0f;
        const uint32_t waves = lanes / 64u, first = in_block * waves;
        for (uint32_t k = first; k < first + waves; ++k) {
            u += slot[0][k];
            v += slot[1][k];
        }
    }
};

// The vectors of a lane's columns in LDS: [vector][half of a group][lane].
struct Vectors {
    float4 *room;
    uint32_t lanes, lane;
    __device__ __forceinline__ void keep(int vector, const float (&v)[8]) const {
        float4 *to = room + vector * 2 * lanes + lane;
        to[0] = make_float4(v[0], v[1], v[2], v[3]);
        to[lanes] = make_float4(v[4], v[5], v[6], v[7]);
    }
    __device__ __forceinline__ void get(float (&v)[8], int vector) const {
        const float4 *from = room + vector * 2 * lanes + lane;
        const float4 a = from[0], b = from[lanes];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
};

// Four waves per SIMD; at six (80 registers) 16384 x 4096 bfloat16 takes 121 us
// instead of 102, 8192 x 768 as long as at four (17.5 us a call).
template <class T, int KIND, bool EVEN, int THREADS>
__global__ __launch_bounds__(THREADS, kGatedWaves)
void gated_kernel(GatedForward a, uint32_t lanes, uint32_t run_blocks, bool rms, bool even) {
    using G = typename GateType<T, KIND>::type;
    extern __shared__ float4 room[];
    __shared__ float shared[2][THREADS / 64];
    const uint32_t in_block = threadIdx.x / lanes, lane = threadIdx.x - in_block * lanes, per_block = blockDim.x / lanes;
    const float width = (float)a.width;
    GatedSum<THREADS / 64> row_sum{shared, lanes, in_block};
    const Vectors vectors{room, lanes, lane};
    const Columns at(lane * kGroup, a.width);
    const uint32_t c = at.column;
    // Rows of one run; with gates of their own all rows are one.
    const uint32_t block = a.first_block + blockIdx.x, run = block / run_blocks;
    const uint64_t count = KIND == kFolded ? a.gate.run : a.rows, before = run * count;
    const uint64_t stride = (uint64_t)run_blocks * per_block;
    uint64_t r = (uint64_t)(block % run_blocks) * per_block + in_block;
    const bool mine = c < a.width;
    Raw8<T> x, residual;
    Raw8<G> gate;
    const auto fetch = [&](uint64_t which) {
        if (which >= count || !mine) return;
        const uint64_t base = (before + which) * a.width;
        load8<T, false>(x, a.x, base + c);
        load8<T, false>(residual, a.residual, base + c);
        if constexpr (KIND != kFolded) load8<G, false>(gate, a.gate.at, a.gate.row(which) * a.width + c);
    };
    fetch(r);
    // The vectors: the first norm's weight and bias, times a shared gate, the second's.
    for (uint32_t which = in_block; which < 4u; which += per_block) {
        float v[8];
        uint32_t column = c;
        __asm__ volatile("" : "+v"(column));            // no addresses kept from one vector for the next
        const void *from[4] = {a.inner_weight, a.inner_bias, a.weight, a.bias};
        load_params(v, from[which], a.weight_dtype, column, a.width, which % 2 == 0 ? 1.0f : 0.0f);
        if (KIND == kFolded && which < 2 && a.gate.at != nullptr) {
            float g[8];
            const char *line = static_cast<const char *>(a.gate.at) +
                               (uint64_t)run * a.width * (a.gate.dtype == NT_F32 ? 4u : 2u);
            load_params(g, line, a.gate.dtype, column, a.width, 1.0f);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] *= g[k];
        }
        vectors.keep((int)which, v);
    }
    __syncthreads();
    const auto norm = [&](const float (&t)[8], float &mean, float &rstd) {
        mean = 0.0f;
        if (!rms) {
            float sum = 0.0f;
#pragma unroll
                for (int k = 0; k < 8; ++k) sum = at.template has<EVEN>(k, a.width) ? sum + t[k] : sum;
            mean = row_sum(sum) / width;
        }
        float squares = 0.0f;
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float d = t[k] - mean;
                squares = at.template has<EVEN>(k, a.width) ? __builtin_fmaf(d, d, squares) : squares;
            }
        rstd = 1.0f / __builtin_sqrtf(row_sum(squares) / width + a.eps);
    };
    for (uint64_t round = (uint64_t)(block % run_blocks) * per_block; round < count; round += stride) {
        const uint64_t base = (before + r) * a.width;
        const bool active = r < count;
        float t[8];
        widen8<T>(t, x);
        float inner_mean, inner_rstd, mean, rstd;
        norm(t, inner_mean, inner_rstd);
        {
            float u[8], b[8], add[8];
            vectors.get(u, 0);
            vectors.get(b, 1);
            widen8<T>(add, residual);
#pragma unroll
            for (int k = 0; k < 8; ++k) t[k] = __builtin_fmaf((t[k] - inner_mean) * inner_rstd, u[k], b[k]);
            if constexpr (KIND != kFolded) {
                float g[8];
                widen8<G>(g, gate);
#pragma unroll
                for (int k = 0; k < 8; ++k) t[k] *= g[k];
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) t[k] = __builtin_fmaf(a.scale, add[k], t[k]);
        }
        fetch(r + stride);
        norm(t, mean, rstd);
        if (active && mine) {
            store_row<T>(a.total, base + c, even, t);
            float w[8], b[8];
            vectors.get(w, 2);
            vectors.get(b, 3);
#pragma unroll
            for (int k = 0; k < 8; ++k) t[k] = __builtin_fmaf((t[k] - mean) * rstd, w[k], b[k]);
            store_row<T>(a.y, base + c, even, t);
        }
        if (active && lane == 0u && a.rstd != nullptr) {
            a.inner_rstd[before + r] = inner_rstd;
            a.rstd[before + r] = rstd;
            if (!rms) {
                a.inner_mean[before + r] = inner_mean;
                a.mean[before + r] = mean;
            }
        }
        r += stride;
    }
}

// The backward pass, a group of eight a lane.  The four sums over rows of a
// lane's columns stay in registers over all rows of the workgroup, which are
// of one run; rows that share a workgroup are joined at the end, in order, and
// each workgroup writes one row of partial sums for each.
//
// Waves per SIMD: float32, and a gate of the rows' own, take more than the 128
// registers of four (with four, 5003 x 1001 float32 with such gates 70 us, with
// two 46; 8192 x 2048 bfloat16 84 and 65, float32 with a shared one 119 and 91).
//
// 16384 x 4096 bfloat16 with root mean squares 176 us: four reads and two
// writes at 4.7 TB/s, each row two exchanges over eight waves, the vector units
// busy 74 % of the time; 8192 x 768 23.8 us (3.2 TB/s), 83 %.
static constexpr uint32_t gated_backward_waves(int32_t dtype, int kind, uint32_t threads) {
    return threads > (uint32_t)kRowThreads || (dtype != NT_F32 && kind == kFolded) ? 4u : 2u;
}
template <class T, int KIND, bool EVEN, int THREADS>
__global__ __launch_bounds__(THREADS, gated_backward_waves(T::code, KIND, THREADS))
void gated_backward_kernel(GatedBackward a, uint32_t lanes, bool rms, bool even) {
    using G = typename GateType<T, KIND>::type;
    extern __shared__ float4 room[];
    __shared__ float shared[2][2][THREADS / 64];
    const uint32_t in_block = threadIdx.x / lanes, lane = threadIdx.x - in_block * lanes, per_block = blockDim.x / lanes;
    const float width = (float)a.width;
    GatedSum2<THREADS / 64> row_sum{shared, lanes, in_block};
    const Vectors vectors{room, lanes, lane};
    const Columns at(lane * kGroup, a.width);
    const uint32_t block = a.first_block + blockIdx.x, c = at.column, run = block / a.run_blocks;
    const uint64_t count = KIND == kFolded ? a.gate.run : a.rows, before = run * count;
    const uint64_t stride = (uint64_t)a.run_blocks * per_block;
    uint64_t r = (uint64_t)(block % a.run_blocks) * per_block + in_block;
    const bool mine = c < a.width;
    Raw8<T> dy, t, dtotal, x;
    Raw8<G> gate;
    const auto fetch_outer = [&](uint64_t which) {
        if (which >= count || !mine) return;
        const uint64_t base = (before + which) * a.width;
        load8<T, false>(dy, a.dy, base + c);
        load8<T, false>(t, a.t, base + c);
        if (a.dtotal != nullptr) load8<T, false>(dtotal, a.dtotal, base + c);
    };
    const auto fetch_inner = [&](uint64_t which) {
        if (which >= count || !mine) return;
        const uint64_t base = (before + which) * a.width;
        load8<T, false>(x, a.x, base + c);
        if constexpr (KIND != kFolded) load8<G, false>(gate, a.gate.at, base + c);
    };
    float next[4] = {0.0f, 0.0f, 0.0f, 0.0f};           // mean, rstd, inner mean, inner rstd
    const auto fetch_stats = [&](uint64_t which) {
        if (which >= count) return;
        if (!rms) {
            next[0] = a.mean[before + which];
            next[2] = a.inner_mean[before + which];
        }
        next[1] = a.rstd[before + which];
        next[3] = a.inner_rstd[before + which];
    };
    fetch_outer(r);
    fetch_inner(r);
    fetch_stats(r);
    // 0: the second norm's weight; 1: the first's, times a shared gate; 2: the first's bias, where rows have gates.
    for (uint32_t which = in_block; which < (KIND == kFolded ? 2u : 3u); which += per_block) {
        float v[8];
        uint32_t column = c;
        __asm__ volatile("" : "+v"(column));            // no addresses kept from one vector for the next
        load_params(v, which == 0u ? a.weight : which == 1u ? a.inner_weight : a.inner_bias, a.weight_dtype, column,
                    a.width, which == 2u ? 0.0f : 1.0f);
        if (KIND == kFolded && which == 1u && a.gate.at != nullptr) {
            float g[8];
            const char *line = static_cast<const char *>(a.gate.at) +
                               (uint64_t)run * a.width * (a.gate.dtype == NT_F32 ? 4u : 2u);
            load_params(g, line, a.gate.dtype, column, a.width, 1.0f);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] *= g[k];
        }
        vectors.keep((int)which, v);
    }
    __syncthreads();
    float sums[4][8];
#pragma unroll
    for (int v = 0; v < 4; ++v)
#pragma unroll
        for (int k = 0; k < 8; ++k) sums[v][k] = 0.0f;
    const auto has = [&](int k) { return EVEN || at.template has<false>((uint32_t)k, a.width); };
    for (uint64_t round = (uint64_t)(block % a.run_blocks) * per_block; round < count; round += stride) {
        const uint64_t base = (before + r) * a.width;
        const bool active = r < count && mine;
        const float mean = next[0], rstd = next[1], inner_mean = next[2], inner_rstd = next[3];
        float g[8], h[8], w[8];
        float level = 0.0f, along = 0.0f;
        vectors.get(w, 0);
        widen8<T>(g, dy);
        widen8<T>(h, t);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const bool in_row = active && has(k);
            h[k] = (h[k] - mean) * rstd;
            sums[2][k] = in_row ? __builtin_fmaf(g[k], h[k], sums[2][k]) : sums[2][k];
            sums[3][k] = in_row ? sums[3][k] + g[k] : sums[3][k];
            g[k] *= w[k];
            level = in_row ? level + g[k] : level;
            along = in_row ? __builtin_fmaf(g[k], h[k], along) : along;
        }
        row_sum(level, along);
        level = rms ? 0.0f : level / width;
        along /= width;
        float add[8];
        widen8<T>(add, dtotal);
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            g[k] = rstd * (g[k] - level - h[k] * along);
            g[k] = a.dtotal != nullptr ? g[k] + add[k] : g[k];
            w[k] = a.scale * g[k];
        }
        fetch_outer(r + stride);                        // into the registers that were just read
        if (active) store_row<T>(a.dresidual, base + c, even, w);
        level = along = 0.0f;
        widen8<T>(h, x);
        vectors.get(w, 1);
        if constexpr (KIND != kFolded) {
            float own[8], bias[8], by_gate[8];
            widen8<G>(own, gate);
            vectors.get(bias, 2);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                h[k] = (h[k] - inner_mean) * inner_rstd;
                by_gate[k] = g[k] * __builtin_fmaf(h[k], w[k], bias[k]);
                g[k] *= own[k];
            }
            if (active && a.dgate != nullptr) store_row<G>(a.dgate, base + c, even, by_gate);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k) h[k] = (h[k] - inner_mean) * inner_rstd;
        }
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const bool in_row = active && has(k);
            sums[0][k] = in_row ? __builtin_fmaf(g[k], h[k], sums[0][k]) : sums[0][k];
            sums[1][k] = in_row ? sums[1][k] + g[k] : sums[1][k];
            g[k] *= w[k];
            level = in_row ? level + g[k] : level;
            along = in_row ? __builtin_fmaf(g[k], h[k], along) : along;
        }
        fetch_inner(r + stride);
        fetch_stats(r + stride);
        row_sum(level, along);
        level = rms ? 0.0f : level / width;
        along /= width;
#pragma unroll
        for (int k = 0; k < 8; ++k) g[k] = inner_rstd * (g[k] - level - h[k] * along);
        if (active) store_row<T>(a.dx, base + c, even, g);
        r += stride;
    }

    // Rows of one wave, then the workgroup's waves or wider rows in order.
    for (uint32_t off = lanes; off < 64u; off <<= 1)
#pragma unroll
        for (int v = 0; v < 4; ++v)
#pragma unroll
            for (int k = 0; k < 8; ++k) sums[v][k] += __shfl_xor(sums[v][k], (int)off, 64);
    const uint32_t span = lanes < 64u ? 64u : lanes, members = blockDim.x / span, member = threadIdx.x / span;
    const uint32_t place = threadIdx.x - member * span;
    for (uint32_t half = members / 2u; half > 0u; half >>= 1) {
        __syncthreads();                                // the vectors, or the last half, are read
        if (member >= half && member < 2u * half && place < lanes)
#pragma unroll
            for (int q = 0; q < 8; ++q)
                room[((member - half) * 8 + q) * lanes + place] =
                    make_float4(sums[q >> 1][4 * (q & 1)], sums[q >> 1][4 * (q & 1) + 1], sums[q >> 1][4 * (q & 1) + 2],
                                sums[q >> 1][4 * (q & 1) + 3]);
        __syncthreads();
        if (member < half && place < lanes)
#pragma unroll
            for (int q = 0; q < 8; ++q) {
                const float4 other = room[(member * 8 + q) * lanes + place];
                sums[q >> 1][4 * (q & 1)] += other.x;
                sums[q >> 1][4 * (q & 1) + 1] += other.y;
                sums[q >> 1][4 * (q & 1) + 2] += other.z;
                sums[q >> 1][4 * (q & 1) + 3] += other.w;
            }
    }
    if (member != 0u || place >= lanes || !mine) return;
    float *out = a.partials + block * 4ull * a.width;
#pragma unroll
    for (int v = 0; v < 4; ++v) {
        if (at.first == 0u && c + kGroup <= a.width) {
            Raw8<TF32> raw;
            narrow8<TF32>(raw, sums[v]);
            store8<TF32, false>(out, (uint64_t)v * a.width + c, raw);
        } else {
#pragma unroll
            for (int k = 0; k < 8; ++k)
                if (has(k)) out[(uint64_t)v * a.width + c + k] = sums[v][k];
        }
    }
}

// ---- rows of any width: a workgroup a row ----------------------------------------------------------
// Rows of less than eight elements or more than 8192: a workgroup goes over the
// row once for each statistic, eight elements a lane, from the caches; a lane's
// share is added in 64 bits, since its chain grows with the row.
constexpr int kLongThreads = 512;

// Elements [c, c + 8) of an array from element `row` on; what lies past the width reads as zero.
template <class T>
__device__ __forceinline__ void long_load(float (&out)[8], const void *base, uint64_t row, uint32_t c, uint32_t width) {
    Raw8<T> raw;
    if (c + kGroup <= width) load8<T, false>(raw, base, row + c);
    else load_end<T>(raw, base, row + c, width - c);
    widen8<T>(out, raw);
}
template <class T>
__device__ __forceinline__ void long_store(void *base, uint64_t row, uint32_t c, uint32_t width, const float (&v)[8]) {
    Raw8<T> raw;
    narrow8<T>(raw, v);
    if (c + kGroup <= width) store8<T, false>(base, row + c, raw);
    else store_end<T>(base, row + c, raw, width - c);
}
__device__ __forceinline__ void long_gate(float (&out)[8], const Gate &gate, uint64_t row, uint32_t c, uint32_t width) {
    if (gate.at == nullptr) {
#pragma unroll
        for (int k = 0; k < 8; ++k) out[k] = 1.0f;
    } else if (gate.dtype == NT_F32) {
        long_load<TF32>(out, gate.at, row, c, width);
    } else if (gate.dtype == NT_F16) {
        long_load<TF16>(out, gate.at, row, c, width);
    } else {
        long_load<TBF16>(out, gate.at, row, c, width);
    }
}
template <class F>
__device__ __forceinline__ void long_groups(uint32_t width, F &&use) {
    for (uint32_t c = threadIdx.x * kGroup; c < width; c += kLongThreads * kGroup) use(c);
}

template <class T>
__device__ __forceinline__ void total_of(float (&t)[8], const GatedForward &a, uint64_t base, uint64_t gate_row, uint32_t c,
                                         float mean, float rstd) {
    float u[8], k[8], gate[8], r[8];
    long_load<T>(t, a.x, base, c, a.width);
    load_params(u, a.inner_weight, a.weight_dtype, c, a.width, 1.0f);
    load_params(k, a.inner_bias, a.weight_dtype, c, a.width, 0.0f);
    long_gate(gate, a.gate, gate_row, c, a.width);
    long_load<T>(r, a.residual, base, c, a.width);
#pragma unroll
    for (int e = 0; e < 8; ++e)
        t[e] = __builtin_fmaf(gate[e], __builtin_fmaf((t[e] - mean) * rstd, u[e], k[e]), a.scale * r[e]);
}

template <class T, bool RMS>
__global__ __launch_bounds__(kLongThreads) void gated_rows_kernel(GatedForward a) {
    __shared__ double shared[kLongThreads / 64];
    const float width = (float)a.width;
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const uint64_t base = row * a.width, gate_row = a.gate.row(row) * a.width;
        float means[2] = {0.0f, 0.0f}, rstds[2];
        const auto value = [&](float (&t)[8], int which, uint32_t c) {
            if (which == 0) long_load<T>(t, a.x, base, c, a.width);
            else total_of<T>(t, a, base, gate_row, c, means[0], rstds[0]);
        };
        for (int which = 0; which < 2; ++which) {
            if constexpr (!RMS) {
                double sum = 0.0;
                long_groups(a.width, [&](uint32_t c) {
                    float t[8];
                    value(t, which, c);
#pragma unroll
                    for (uint32_t k = 0; k < 8; ++k) sum += c + k < a.width ? t[k] : 0.0f;
                });
                means[which] = block_total(sum, shared) / width;
            }
            double squares = 0.0;
            long_groups(a.width, [&](uint32_t c) {
                float t[8];
                value(t, which, c);
#pragma unroll
                for (uint32_t k = 0; k < 8; ++k) {
                    const float d = c + k < a.width ? t[k] - means[which] : 0.0f;
                    squares = __builtin_fma((double)d, (double)d, squares);
                }
            });
            rstds[which] = 1.0f / __builtin_sqrtf(block_total(squares, shared) / width + a.eps);
        }
        long_groups(a.width, [&](uint32_t c) {
            float t[8], w[8], b[8];
            value(t, 1, c);
            long_store<T>(a.total, base, c, a.width, t);
            load_params(w, a.weight, a.weight_dtype, c, a.width, 1.0f);
            load_params(b, a.bias, a.weight_dtype, c, a.width, 0.0f);
#pragma unroll
            for (int k = 0; k < 8; ++k) t[k] = __builtin_fmaf((t[k] - means[1]) * rstds[1], w[k], b[k]);
            long_store<T>(a.y, base, c, a.width, t);
        });
        if (threadIdx.x == 0 && a.rstd != nullptr) {
            a.inner_rstd[row] = rstds[0];
            a.rstd[row] = rstds[1];
            if constexpr (!RMS) {
                a.inner_mean[row] = means[0];
                a.mean[row] = means[1];
            }
        }
    }
}

// dt of a group, and of the second norm dy and its normalized input, from the row's sums of g and g h over W.
template <class T>
__device__ __forceinline__ void total_grad(float (&dt)[8], float (&dy)[8], float (&h)[8], const GatedBackward &a,
                                           uint64_t base, uint32_t c, float mean, float rstd, float level, float along) {
    float w[8];
    long_load<T>(dy, a.dy, base, c, a.width);
    long_load<T>(h, a.t, base, c, a.width);
    load_params(w, a.weight, a.weight_dtype, c, a.width, 1.0f);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
        h[k] = (h[k] - mean) * rstd;
        dt[k] = rstd * (dy[k] * w[k] - level - h[k] * along);
    }
    if (a.dtotal == nullptr) return;
    float add[8];
    long_load<T>(add, a.dtotal, base, c, a.width);
#pragma unroll
    for (int k = 0; k < 8; ++k) dt[k] += add[k];
}

template <class T, bool RMS>
__global__ __launch_bounds__(kLongThreads) void gated_rows_backward_kernel(GatedBackward a) {
    __shared__ double shared[kLongThreads / 64];
    const float width = (float)a.width;
    const bool each = a.dgate != nullptr;
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const uint64_t base = row * a.width, gate_row = a.gate.row(row) * a.width;
        const float mean = RMS ? 0.0f : a.mean[row], rstd = a.rstd[row];
        const float inner_mean = RMS ? 0.0f : a.inner_mean[row], inner_rstd = a.inner_rstd[row];
        double levels = 0.0, alongs = 0.0;
        long_groups(a.width, [&](uint32_t c) {
            float g[8], h[8], w[8];
            long_load<T>(g, a.dy, base, c, a.width);
            long_load<T>(h, a.t, base, c, a.width);
            load_params(w, a.weight, a.weight_dtype, c, a.width, 1.0f);
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) {
                g[k] = c + k < a.width ? g[k] * w[k] : 0.0f;
                levels += g[k];
                alongs = __builtin_fma((double)g[k], (double)((h[k] - mean) * rstd), alongs);
            }
        });
        const float along = block_total(alongs, shared) / width;
        const float level = RMS ? 0.0f : block_total(levels, shared) / width;
        if (threadIdx.x == 0) {
            a.row_sums[2 * row] = level;
            a.row_sums[2 * row + 1] = along;
        }
        // dt and, of the first norm, its normalized input, its gradient by gate and weight.
        const auto inner = [&](float (&dt)[8], float (&i)[8], float (&q)[8], float (&u)[8], uint32_t c) {
            float dy[8], h[8], gate[8];
            total_grad<T>(dt, dy, h, a, base, c, mean, rstd, level, along);
            long_load<T>(i, a.x, base, c, a.width);
            load_params(u, a.inner_weight, a.weight_dtype, c, a.width, 1.0f);
            long_gate(gate, a.gate, gate_row, c, a.width);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                i[k] = (i[k] - inner_mean) * inner_rstd;
                q[k] = dt[k] * gate[k] * u[k];
            }
        };
        levels = alongs = 0.0;
        long_groups(a.width, [&](uint32_t c) {
            float dt[8], i[8], q[8], u[8];
            inner(dt, i, q, u, c);
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) {
                q[k] = c + k < a.width ? q[k] : 0.0f;
                levels += q[k];
                alongs = __builtin_fma((double)q[k], (double)i[k], alongs);
            }
        });
        const float inner_along = block_total(alongs, shared) / width;
        const float inner_level = RMS ? 0.0f : block_total(levels, shared) / width;
        long_groups(a.width, [&](uint32_t c) {
            float dt[8], i[8], q[8], u[8];
            inner(dt, i, q, u, c);
#pragma unroll
            for (int k = 0; k < 8; ++k) q[k] = inner_rstd * (q[k] - inner_level - i[k] * inner_along);
            long_store<T>(a.dx, base, c, a.width, q);
            if (each) {
                float bias[8];
                load_params(bias, a.inner_bias, a.weight_dtype, c, a.width, 0.0f);
#pragma unroll
                for (int k = 0; k < 8; ++k) q[k] = dt[k] * __builtin_fmaf(i[k], u[k], bias[k]);
                if (a.gate.dtype == NT_F32) long_store<TF32>(a.dgate, base, c, a.width, q);
                else if (a.gate.dtype == NT_F16) long_store<TF16>(a.dgate, base, c, a.width, q);
                else long_store<TBF16>(a.dgate, base, c, a.width, q);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) dt[k] *= a.scale;
            long_store<T>(a.dresidual, base, c, a.width, dt);
        });
    }
}

// The four column sums over a group of a run's rows, eight columns a lane.
// Where each row has a gate of its own, dt is taken with it.
template <class T, bool RMS>
__global__ __launch_bounds__(kBlock) void gated_columns_kernel(GatedBackward a, uint32_t groups, bool each) {
    const uint32_t c = (blockIdx.x * kBlock + threadIdx.x) * kGroup;
    if (c >= a.width) return;
    const uint64_t run = each ? a.rows : a.gate.run;
    for (uint32_t group = blockIdx.y; group < groups; group += gridDim.y) {
        const uint64_t first = group / a.run_blocks * run;
        float sums[4][8] = {};
        for (uint64_t r = group % a.run_blocks; r < run; r += a.run_blocks) {
            const uint64_t row = first + r, base = row * a.width;
            float dt[8], dy[8], h[8], i[8];
            total_grad<T>(dt, dy, h, a, base, c, RMS ? 0.0f : a.mean[row], a.rstd[row], a.row_sums[2 * row],
                          a.row_sums[2 * row + 1]);
            long_load<T>(i, a.x, base, c, a.width);
            const float inner_mean = RMS ? 0.0f : a.inner_mean[row], inner_rstd = a.inner_rstd[row];
            if (each) {
                float gate[8];
                long_gate(gate, a.gate, base, c, a.width);
#pragma unroll
                for (int k = 0; k < 8; ++k) dt[k] *= gate[k];
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                sums[0][k] = __builtin_fmaf(dt[k], (i[k] - inner_mean) * inner_rstd, sums[0][k]);
                sums[1][k] += dt[k];
                sums[2][k] = __builtin_fmaf(dy[k], h[k], sums[2][k]);
                sums[3][k] += dy[k];
            }
        }
        float *out = a.partials + group * 4ull * a.width;
#pragma unroll
        for (int v = 0; v < 4; ++v) long_store<TF32>(out, (uint64_t)v * a.width, c, a.width, sums[v]);
    }
}

// The vectors' gradients from the partial sums: 16 columns and 64 slices a
// workgroup, of one norm's two; of 4096 columns and more 32 and 32 (512
// workgroups' sums: 768 columns 8.7 and 12.5 us, with 8 columns 8.8; 4096 17.1
// and 13.7; a backward call of 8192 x 2048 56.8 and 59.7).  Slices
// share out the runs, and where those are fewer, the blocks of each; a run's
// sums are joined before its gate, slices in order.
struct GatedVectors {
    void *inner_weight, *inner_bias, *gate, *weight, *bias;     // each may be null
};
template <uint32_t kVectorColumns>
__global__ __launch_bounds__(1024) void gated_vectors_kernel(GatedBackward a, GatedVectors to, uint32_t runs, bool each) {
    constexpr uint32_t kVectorSlices = 1024u / kVectorColumns;
    __shared__ float shared[2][kVectorSlices][kVectorColumns + 1];
    const uint32_t column = threadIdx.x % kVectorColumns, slice = threadIdx.x / kVectorColumns;
    const uint32_t c = blockIdx.x * kVectorColumns + column;
    const bool inner = blockIdx.y == 0u;                    // the first norm's two sums, or the second's
    const uint64_t line = a.width, block = 4u * line;
    const bool there = c < a.width;
    const float u = there ? load_param(a.inner_weight, a.weight_dtype, c, 1.0f) : 0.0f;
    const float bias = there ? load_param(a.inner_bias, a.weight_dtype, c, 0.0f) : 0.0f;
    uint32_t subs = kVectorSlices;
    while (subs > 1u && kVectorSlices / subs < runs) subs >>= 1;
    const uint32_t at_once = kVectorSlices / subs, sub = slice % subs;
    float sums[2] = {0.0f, 0.0f};
    for (uint32_t first = 0; first < runs; first += at_once) {
        const uint32_t run = first + slice / subs;
        float own[2] = {0.0f, 0.0f};
        if (there && run < runs) {
            const float *from = a.partials + run * (uint64_t)a.run_blocks * block + c + (inner ? 0u : 2u * line);
#pragma unroll 8
            for (uint32_t b = sub; b < a.run_blocks; b += subs) {
                own[0] += from[b * block];
                own[1] += from[b * block + line];
            }
        }
        if (!inner) {
            sums[0] += own[0];
            sums[1] += own[1];
            continue;
        }
        if (subs > 1u) {
            __syncthreads();
            shared[0][slice][column] = own[0];
            shared[1][slice][column] = own[1];
            __syncthreads();
            if (sub == 0u)
                for (uint32_t k = 1; k < subs; ++k) {
                    own[0] += shared[0][slice + k][column];
                    own[1] += shared[1][slice + k][column];
                }
        }
        if (!there || run >= runs || sub != 0u) continue;
        if (to.gate != nullptr)
            store_param(to.gate, a.gate.dtype, run * line + c, __builtin_fmaf(u, own[0], bias * own[1]));
        const float gate = each ? 1.0f : load_param(a.gate.at, a.gate.dtype, run * line + c, 1.0f);
        sums[0] = __builtin_fmaf(gate, own[0], sums[0]);
        sums[1] = __builtin_fmaf(gate, own[1], sums[1]);
    }
    __syncthreads();
    shared[0][slice][column] = sums[0];
    shared[1][slice][column] = sums[1];
    __syncthreads();
    if (slice >= 2u || !there) return;
    float sum = 0.0f;
#pragma unroll 8
    for (uint32_t s = 0; s < kVectorSlices; ++s) sum += shared[slice][s][column];
    void *out = inner ? (slice == 0u ? to.inner_weight : to.inner_bias) : slice == 0u ? to.weight : to.bias;
    if (out != nullptr) store_param(out, a.weight_dtype, c, sum);
}

// ---- launches ----------------------------------------------------------------------------------------
constexpr uint32_t kMostBlocks = 8192;
constexpr uint32_t kUnits = 256;                        // compute units
constexpr uint32_t kRunGroups = 256;                    // groups of rows of the column sums of long rows, over all runs
constexpr uint64_t kMostWidth = 1ull << 24;
// A shared gate's runs of fewer rows than this many workgroups hold at a time
// are taken as gates of the rows' own: each run's workgroups load the vectors.
// Runs of 2, 4, 8, 16 and 32 rows of 8192 x 768 bfloat16, four to a workgroup:
// 39.1, 22.9, 19.6, 17.9 and 18.7 us apart, 18 to 19 as the rows' own; of 8192 x
// 4096, one to a workgroup: 83.5, 68.5, 62.1, 59.0 and 58.8, and 61 to 66.
constexpr uint32_t kShortRun = 4;

// Workgroups of each run: as many as are resident at a time, where there are
// rows for them; those past them would have a turn of their own.  `waves` of a
// SIMD's are counted by whole workgroups, over a unit where the kernel leaves
// registers for a wave more (16-bit forward), otherwise over each SIMD: of five
// waves a unit of 16 then holds two workgroups, not three.  16384 x 2560
// bfloat16 forward 78 to 85 us (two: 101; counted by waves alone, 819 workgroups
// in 768 places: 115), backward 140 (three: 177; by waves: 220); 8192 x 2560
// float32 forward 85 (three: 94); 4096 x 7168 bfloat16 67 and 100 instead of 113
// and 153.
static uint32_t run_blocks_of(uint64_t run, uint64_t runs, const RowTiling &g, uint32_t waves, bool each_simd) {
    const uint32_t of_block = (g.threads + 63u) / 64u, simds = kSimds / kUnits;
    const uint32_t per_unit = each_simd ? waves / ((of_block + simds - 1u) / simds) : waves * simds / of_block;
    const uint64_t most = std::max<uint64_t>(1u, kUnits * (uint64_t)std::max(1u, per_unit) / runs);
    const uint32_t per_block = g.threads / g.lanes;
    return (uint32_t)std::min<uint64_t>((run + per_block - 1) / per_block, most);
}

// How the forward pass takes the gate, and how many runs keep their rows apart.
static int gate_kind(const GatedForward &a, int32_t dtype, uint32_t per_block, uint64_t &runs) {
    runs = a.gate.runs;
    if (runs == 1u || a.gate.run >= (uint64_t)kShortRun * per_block) return kFolded;
    runs = 1u;
    return a.gate.dtype == dtype ? kOwn : kOwnFloat;
}

// A group a lane: a power of two of lanes up to 32, then whole waves, and as
// many rows (a power of two of them) as fit in 512 lanes, or one.  Rows of three
// waves share no workgroup in the forward pass: a unit holds five alone and four
// in pairs (8192 x 1536 bfloat16 25.3 us and 29.9; backward, with partial sums
// for each workgroup, 55.6 and 51.7).  No parts: rows that the tilings do not
// take.
static RowTiling gated_tiling(uint32_t width, bool backward) {
    const uint32_t groups = (width + kGroup - 1) / kGroup;
    if (width < kGroup || groups > (uint32_t)kWideThreads) return RowTiling{0, 0, 0};
    uint32_t lanes = 1, rows = 1;
    while (lanes < groups && lanes < 64u) lanes <<= 1;
    if (groups > 64u) lanes = (groups + 63u) / 64u * 64u;
    if (lanes != 192u || backward)
        while (lanes * rows * 2u <= (uint32_t)kRowThreads) rows <<= 1;
    return RowTiling{lanes, 1, lanes * rows};
}

// Calls launch(grid, args) for all blocks, below 2**32 work-items at a time.
template <class Args, class F>
static void in_launches(Args a, uint64_t blocks, F &&launch) {
    constexpr uint64_t most = 1ull << 21;               // of at most 1024 lanes
    for (uint64_t first = 0; first < blocks; first += most) {
        a.first_block = (uint32_t)first;
        launch(dim3((unsigned)std::min(most, blocks - first)), a);
    }
}

template <class T, int KIND, int THREADS>
static void launch_gated_tiled(const GatedForward &args, const RowTiling &g, uint64_t runs, bool rms, hipStream_t s) {
    const bool aligned = aligned_rows(args.width, {args.total, args.y});
    const uint32_t blocks = run_blocks_of(args.rows / runs, runs, g, kGatedWaves, T::code == NT_F32);
    const uint32_t room = g.lanes * kGroup * 16u;
    in_launches(args, runs * blocks, [&](dim3 grid, const GatedForward &a) {
        if (a.width % kGroup == 0)
            gated_kernel<T, KIND, true, THREADS><<<grid, dim3(g.threads), room, s>>>(a, g.lanes, blocks, rms, aligned);
        else gated_kernel<T, KIND, false, THREADS><<<grid, dim3(g.threads), room, s>>>(a, g.lanes, blocks, rms, aligned);
    });
}

template <class T>
static void launch_gated(const GatedForward &a, bool rms, hipStream_t s) {
    const RowTiling g = gated_tiling(a.width, false);
    if (g.parts == 0) {
        const dim3 grid((unsigned)std::min<uint64_t>(a.rows, kMostBlocks));
        if (rms) gated_rows_kernel<T, true><<<grid, dim3(kLongThreads), 0, s>>>(a);
        else gated_rows_kernel<T, false><<<grid, dim3(kLongThreads), 0, s>>>(a);
        return;
    }
    uint64_t runs = 1;
    const int kind = gate_kind(a, T::code, g.threads / g.lanes, runs);
    const auto launch = [&](auto k) {
        constexpr int KIND = decltype(k)::value;
        if (g.threads > (uint32_t)kRowThreads) launch_gated_tiled<T, KIND, kWideThreads>(a, g, runs, rms, s);
        else launch_gated_tiled<T, KIND, kRowThreads>(a, g, runs, rms, s);
    };
    if (kind == kFolded) launch(std::integral_constant<int, kFolded>{});
    else if (kind == kOwn) launch(std::integral_constant<int, kOwn>{});
    else if constexpr (T::code != NT_F32) launch(std::integral_constant<int, kOwnFloat>{});
}

template <class T, int KIND, int THREADS>
static void launch_gated_backward_tiled(const GatedBackward &args, const RowTiling &g, bool rms, uint32_t groups,
                                        hipStream_t s) {
    const bool aligned = aligned_rows(args.width, {args.dx, args.dresidual, args.dgate});
    // The vectors, or half of the rows that are joined.
    const uint32_t span = g.lanes < 64u ? 64u : g.lanes;
    const uint32_t room = std::max(g.lanes * kGroup * (KIND == kFolded ? 8u : 12u), g.threads / span / 2u * g.lanes * 128u);
    in_launches(args, groups, [&](dim3 grid, const GatedBackward &a) {
        if (a.width % kGroup == 0)
            gated_backward_kernel<T, KIND, true, THREADS><<<grid, dim3(g.threads), room, s>>>(a, g.lanes, rms, aligned);
        else gated_backward_kernel<T, KIND, false, THREADS><<<grid, dim3(g.threads), room, s>>>(a, g.lanes, rms, aligned);
    });
}

template <class T>
static void launch_gated_backward(const GatedBackward &a, bool rms, bool each, uint32_t groups, hipStream_t s) {
    const RowTiling g = gated_tiling(a.width, true);
    if (g.parts != 0) {
        const auto launch = [&](auto kind) {
            constexpr int KIND = decltype(kind)::value;
            if (g.threads > (uint32_t)kRowThreads) launch_gated_backward_tiled<T, KIND, kWideThreads>(a, g, rms, groups, s);
            else launch_gated_backward_tiled<T, KIND, kRowThreads>(a, g, rms, groups, s);
        };
        if (!each) launch(std::integral_constant<int, kFolded>{});
        else if (a.gate.dtype == T::code) launch(std::integral_constant<int, kOwn>{});
        else if constexpr (T::code != NT_F32) launch(std::integral_constant<int, kOwnFloat>{});
        return;
    }
    const dim3 grid((unsigned)std::min<uint64_t>(a.rows, kMostBlocks));
    const dim3 columns((a.width + kBlock * kGroup - 1) / (kBlock * kGroup), std::min(groups, 65535u));
    if (rms) gated_rows_backward_kernel<T, true><<<grid, dim3(kLongThreads), 0, s>>>(a);
    else gated_rows_backward_kernel<T, false><<<grid, dim3(kLongThreads), 0, s>>>(a);
    if (rms) gated_columns_kernel<T, true><<<columns, dim3(kBlock), 0, s>>>(a, groups, each);
    else gated_columns_kernel<T, false><<<columns, dim3(kBlock), 0, s>>>(a, groups, each);
}

static int32_t check_gated(const char *entry, int32_t dtype, int32_t weight_dtype, bool has_params, const void *gate,
                           int32_t gate_dtype, uint64_t gate_rows, uint64_t rows, uint64_t width) {
    const std::string name(entry);
    if (!half_or_float(dtype)) return fail(NT_ERR_TYPE, name + ": activations must be float32, float16 or bfloat16");
    if (has_params && weight_dtype != dtype && weight_dtype != NT_F32)
        return fail(NT_ERR_TYPE, name + ": weights and biases must have the activations' dtype or float32");
    if (gate != nullptr && gate_dtype != dtype && gate_dtype != NT_F32)
        return fail(NT_ERR_TYPE, name + ": the gate must have the activations' dtype or float32");
    if (width == 0 || width > kMostWidth) return fail(NT_ERR_VALUE, name + ": the width must be 1..2**24");
    if (rows > 0xffffffffffffull / width || rows >= 1ull << 31)
        return fail(NT_ERR_VALUE, name + ": too many rows or elements");
    if (gate != nullptr && rows > 0 && (gate_rows == 0 || rows % gate_rows != 0))
        return fail(NT_ERR_VALUE, name + ": the gate's rows must divide the rows");
    return NT_OK;
}

}  // namespace nt

using namespace nt;

extern "C" {

int32_t nt_norm_gate_add_norm(int32_t device, const void *x, const void *residual, int32_t dtype,
                              const void *inner_weight, const void *inner_bias, const void *gate, int32_t gate_dtype,
                              uint64_t gate_rows, const void *weight, const void *bias, int32_t weight_dtype,
                              float residual_scale, float eps, int32_t rms, void *total, void *y, float *inner_mean,
                              float *inner_rstd, float *mean, float *rstd, uint64_t rows, uint64_t width,
                              void *stream) {
    clear_error();
    const char *entry = "nt_norm_gate_add_norm";
    const bool params = inner_weight != nullptr || inner_bias != nullptr || weight != nullptr || bias != nullptr;
    int32_t rc = check_gated(entry, dtype, weight_dtype, params, gate, gate_dtype, gate_rows, rows, width);
    if (rc != NT_OK) return rc;
    if (rows == 0) return NT_OK;
    const uint64_t n = rows * width;
    rc = check_arrays(entry, {{x, dtype, n, false, true}, {residual, dtype, n, false, true},
                              {inner_weight, weight_dtype, width, false, false},
                              {inner_bias, weight_dtype, width, false, false},
                              {gate, gate_dtype, gate_rows * width, false, false},
                              {weight, weight_dtype, width, false, false}, {bias, weight_dtype, width, false, false},
                              {total, dtype, n, true, true}, {y, dtype, n, true, true},
                              {inner_mean, NT_F32, rows, true, false}, {inner_rstd, NT_F32, rows, true, false},
                              {mean, NT_F32, rows, true, false}, {rstd, NT_F32, rows, true, false}});
    if (rc != NT_OK) return rc;
    const bool stats = rstd != nullptr;
    if ((inner_rstd != nullptr) != stats || (inner_mean != nullptr) != (stats && !rms) ||
        (mean != nullptr) != (stats && !rms))
        return fail(NT_ERR_VALUE, std::string(entry) + ": statistics are given together, means where the norm has them");
    DeviceGuard guard(device);
    if (!guard.ok()) return hip_check(guard.error(), "hipSetDevice");
    const uint64_t runs = gate == nullptr ? 1u : gate_rows;
    const GatedForward a{x, residual, inner_weight, inner_bias, weight, bias,
                         {gate, gate_dtype, (uint32_t)runs, rows / runs}, total, y, inner_mean, inner_rstd, mean, rstd,
                         rows, (uint32_t)width, weight_dtype, residual_scale, eps, 0};
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
        case NT_F32: launch_gated<TF32>(a, rms != 0, s); break;
        case NT_F16: launch_gated<TF16>(a, rms != 0, s); break;
        default: launch_gated<TBF16>(a, rms != 0, s); break;
    }
    NT_LAUNCH_CHECK("gated norm launch");
    return NT_OK;
}

int32_t nt_norm_gate_add_norm_backward(int32_t device, const void *dy, const void *dtotal, const void *x,
                                       const void *total, int32_t dtype, const float *inner_mean,
                                       const float *inner_rstd, const float *mean, const float *rstd,
                                       const void *inner_weight, const void *inner_bias, const void *gate,
                                       int32_t gate_dtype, uint64_t gate_rows, const void *weight, int32_t weight_dtype,
                                       float residual_scale, void *dx, void *dresidual, void *dinner_weight,
                                       void *dinner_bias, void *dgate, void *dweight, void *dbias, uint64_t rows,
                                       uint64_t width, void *stream) {
    clear_error();
    const char *entry = "nt_norm_gate_add_norm_backward";
    const bool params = inner_weight != nullptr || inner_bias != nullptr || weight != nullptr ||
                        dinner_weight != nullptr || dinner_bias != nullptr || dweight != nullptr || dbias != nullptr;
    int32_t rc = check_gated(entry, dtype, weight_dtype, params, gate, gate_dtype, gate_rows, rows, width);
    if (rc != NT_OK) return rc;
    if (gate == nullptr && dgate != nullptr) return fail(NT_ERR_VALUE, std::string(entry) + ": there is no gate");
    const uint64_t n = rows * width, gate_size = gate == nullptr ? 0 : gate_rows * width;
    const bool any = rows > 0;
    rc = check_arrays(entry, {{dy, dtype, n, false, any}, {dtotal, dtype, n, false, false}, {x, dtype, n, false, any},
                              {total, dtype, n, false, any}, {inner_mean, NT_F32, rows, false, false},
                              {inner_rstd, NT_F32, rows, false, any}, {mean, NT_F32, rows, false, false},
                              {rstd, NT_F32, rows, false, any}, {inner_weight, weight_dtype, width, false, false},
                              {inner_bias, weight_dtype, width, false, false}, {gate, gate_dtype, gate_size, false, false},
                              {weight, weight_dtype, width, false, false}, {dx, dtype, n, true, any},
                              {dresidual, dtype, n, true, any}, {dinner_weight, weight_dtype, width, true, false},
                              {dinner_bias, weight_dtype, width, true, false}, {dgate, gate_dtype, gate_size, true, false},
                              {dweight, weight_dtype, width, true, false}, {dbias, weight_dtype, width, true, false}});
    if (rc != NT_OK) return rc;
    if ((inner_mean != nullptr) != (mean != nullptr))
        return fail(NT_ERR_VALUE, std::string(entry) + ": both means are given or none");
    DeviceGuard guard(device);
    if (!guard.ok()) return hip_check(guard.error(), "hipSetDevice");
    rc = refuse_capture(entry, stream);
    if (rc != NT_OK) return rc;
    hipStream_t s = (hipStream_t)stream;
    if (!any) {
        for (void *vector : {dinner_weight, dinner_bias, dweight, dbias})
            if (vector != nullptr && (rc = nt_fill(vector, width, weight_dtype == NT_F32 ? 4 : 2, 0, stream)) != NT_OK)
                return rc;
        return dgate == nullptr ? NT_OK : nt_fill(dgate, gate_size, gate_dtype == NT_F32 ? 4 : 2, 0, stream);
    }
    const bool rms = mean == nullptr, each = gate != nullptr && gate_rows == rows && rows > 1;
    const uint64_t gate_runs = gate == nullptr ? 1u : gate_rows;
    const uint32_t runs = each ? 1u : (uint32_t)gate_runs;          // whose sums are kept apart
    GatedBackward a{dy, dtotal, x, total, inner_weight, inner_bias, weight,
                    {gate, gate_dtype, (uint32_t)gate_runs, rows / gate_runs}, inner_mean, inner_rstd, mean, rstd,
                    dx, dresidual, each ? dgate : nullptr, nullptr, nullptr, rows, (uint32_t)width, weight_dtype,
                    residual_scale, 1, 0};
    const RowTiling tiling = gated_tiling((uint32_t)width, true);
    const uint32_t waves = gated_backward_waves(dtype, each ? kOwn : kFolded, tiling.threads);
    a.run_blocks = tiling.parts != 0 ? run_blocks_of(rows / runs, runs, tiling, waves, true)
                                     : (uint32_t)std::min<uint64_t>(rows / runs, std::max(1u, kRunGroups / runs));
    Workspace room;
    if (tiling.parts == 0) room.want(&a.row_sums, 2u * rows);
    room.want(&a.partials, 4ull * width * runs * a.run_blocks);
    rc = room.allocate(device, stream);
    if (rc != NT_OK) return rc;
    const uint32_t groups = runs * a.run_blocks;
    switch (dtype) {
        case NT_F32: launch_gated_backward<TF32>(a, rms, each, groups, s); break;
        case NT_F16: launch_gated_backward<TF16>(a, rms, each, groups, s); break;
        default: launch_gated_backward<TBF16>(a, rms, each, groups, s); break;
    }
    const GatedVectors vectors{dinner_weight, dinner_bias, each ? nullptr : dgate, dweight, dbias};
    if (width < 4096u) gated_vectors_kernel<16><<<dim3((a.width + 15u) / 16u, 2), dim3(1024), 0, s>>>(a, vectors, runs, each);
    else gated_vectors_kernel<32><<<dim3((a.width + 31u) / 32u, 2), dim3(1024), 0, s>>>(a, vectors, runs, each);
    return hip_check(hipGetLastError(), "gated norm backward launch");
}

}  // extern "C"
