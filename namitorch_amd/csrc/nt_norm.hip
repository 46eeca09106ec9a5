// nt_norm.hip — the operators between a transformer's matrix products: layer
// norm, dropout, and the residual edge that joins them (dropout of a branch,
// added to the residual stream, then the norm of the sum), each with its
// backward pass.
//
// With t a row of W elements (the input, or dropout(x) + residual):
//   mean = sum t / W, var = sum (t - mean)^2 / W, rstd = 1 / sqrt(var + eps)
//   y    = (t - mean) rstd w + b
// and with h = (t - mean) rstd, g = dy w:
//   dt   = rstd (g - sum g / W - h sum(g h) / W)   (+ the gradient that the sum gets from elsewhere)
//   dw   = sum over rows of dy h,   db = sum over rows of dy.
//
// Every sum and statistic is float32 (a lane's share of a very long row 64
// bits); values are rounded once, when stored.
// The sums over rows run in a fixed order, so gradients do not change from
// run to run.
//
// All of it is bound by memory once a launch is large: 8 to 35 vector
// operations per element (the generator is half of the latter) against 4 to 20
// bytes.  Times here are kernel times on one MI355X, by kernel trace over
// three sets of tensors in turn; a stream of one read and one write of the
// same size runs at 6.6 TB/s, one of two and two at 6.0 (268 MB) to 6.3 TB/s.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <initializer_list>
#include <type_traits>

#include "nt_internal.hpp"
#include "nt_philox.hpp"
#include "nt_pool.hpp"
#include "nt_rows.hpp"

namespace nt {

// What the edge does to its input before the norm.
enum Edge { kNone = 0, kAdd = 1, kDropAdd = 2 };

struct NormForward {
    const void *x, *residual, *weight, *bias;
    void *total, *y;
    float *mean, *rstd;         // may be null (both)
    uint64_t rows;
    uint32_t width;
    int32_t weight_dtype;
    float eps;
    Mask mask;
};

struct NormBackward {
    const void *dy, *dtotal, *t, *weight;
    const float *mean, *rstd;
    void *dx, *dresidual;       // the edge writes both, the norm dx alone
    float *partials;            // [row_blocks][2][width], or null
    uint64_t rows;
    uint32_t width;
    int32_t weight_dtype;
    Mask mask;
    uint32_t row_blocks;        // workgroups of the launch that take rows; the others take columns (few rows)
    void *dw, *db;              // what those write
};

__device__ __forceinline__ float load_param(const void *base, int32_t dtype, uint64_t i, float absent) {
    if (base == nullptr) return absent;
    switch (dtype) {
        case NT_F32: return reinterpret_cast<const float *>(base)[i];
        case NT_F16: return f16_to_f32(reinterpret_cast<const uint16_t *>(base)[i]);
        default: return bf16_to_f32(reinterpret_cast<const uint16_t *>(base)[i]);
    }
}

__device__ __forceinline__ float drop_one(float v, uint64_t i, const Mask &m) {
    const PhiloxWords words = philox(i >> 3, m.offset, m.seed);
    return philox_half(words, (int)(i & 7)) >= m.threshold ? v * m.factor : 0.0f;
}

__device__ __forceinline__ float wave_sum_f32(float v) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
    return v;
}

// Sum over the workgroup, the same value on every lane; `shared` holds one
// float per wave.
__device__ __forceinline__ float block_sum_f32(float v, float *shared) {
    v = wave_sum_f32(v);
    __syncthreads();                                    // the last reader of `shared` is done
    if ((threadIdx.x & 63u) == 0u) shared[threadIdx.x >> 6] = v;
    __syncthreads();
    float total = 0.0f;
    for (uint32_t k = 0; k < blockDim.x / 64u; ++k) total += shared[k];
    return total;
}

// ---- eight consecutive elements ------------------------------------------------------------------
// What a lane holds of a row at a time: one 16-byte access of a 16-bit type,
// two of float32, and one call of the mask's generator.  Where rows do not
// start on 16 bytes the same accesses run unaligned (gfx950 takes any
// alignment).  Norms read through the caches: their inputs were just written
// by a product or an earlier edge (8192 x 768 bfloat16 forward: 6.9 us, with
// nontemporal loads 10.8), and store around them (temporal stores 8.2 us).
// Float32's two accesses each leave half of a line, which the caches join:
// its aligned stores go through them (edge 8192 x 2048: 49.4 us, around them
// 53.6; dropout of 25 MB 10.8 and 12.4), unaligned ones do not (norm backward
// 8192 x 1001: 23.0 us through them, 19.8 around).
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_any __attribute__((aligned(2)));
typedef __attribute__((address_space(1))) u32x4 gu32x4;
typedef __attribute__((address_space(1))) u32x4_any gu32x4_any;
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

template <class T> struct Raw8 {
    static constexpr int kWords = sizeof(typename T::raw) / 2;      // 16-byte words
    u32x4 w[kWords];
};

template <class T, bool EVEN, bool NT = false>
__device__ __forceinline__ void load8(Raw8<T> &out, const void *base, uint64_t i) {
    const auto *p = reinterpret_cast<const typename T::raw *>(base) + i;
#pragma unroll
    for (int k = 0; k < Raw8<T>::kWords; ++k) {
        if constexpr (EVEN) out.w[k] = gload<NT, u32x4, gu32x4>(p + k * 4);
        else out.w[k] = gload<NT, u32x4, gu32x4_any>(p + k * 4);
    }
}

template <class T, bool EVEN>
__device__ __forceinline__ void store8(void *base, uint64_t i, const Raw8<T> &in) {
    auto *p = reinterpret_cast<typename T::raw *>(base) + i;
#pragma unroll
    for (int k = 0; k < Raw8<T>::kWords; ++k) {
        if constexpr (EVEN) gstore<T::code != NT_F32, u32x4, gu32x4>(p + k * 4, in.w[k]);
        else gstore<true, u32x4, gu32x4_any>(p + k * 4, in.w[k]);
    }
}

template <class T>
__device__ __forceinline__ void widen8(float (&out)[8], const Raw8<T> &in) {
    if constexpr (T::code == NT_F32) {
#pragma unroll
        for (int k = 0; k < 8; ++k) out[k] = bits_f32(in.w[k >> 2][k & 3]);
    } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            const uint32_t w = in.w[0][k >> 1];
            if constexpr (T::code == NT_BF16) out[k] = bits_f32(k & 1 ? w & 0xffff0000u : w << 16);
            else out[k] = f16_to_f32((uint16_t)(k & 1 ? w >> 16 : w & 0xffffu));
        }
    }
}

// One rounding to nearest even each (v_cvt_pk_bf16_f32, v_cvt_pk_f16_f32).
template <class T>
__device__ __forceinline__ void narrow8(Raw8<T> &out, const float (&in)[8]) {
    if constexpr (T::code == NT_F32) {
#pragma unroll
        for (int k = 0; k < 8; ++k) out.w[k >> 2][k & 3] = f32_bits(in[k]);
    } else {
        f32x8 v;
#pragma unroll
        for (int k = 0; k < 8; ++k) v[k] = in[k];
        if constexpr (T::code == NT_BF16) out.w[0] = __builtin_bit_cast(u32x4, __builtin_convertvector(v, bf16x8));
        else out.w[0] = __builtin_bit_cast(u32x4, __builtin_convertvector(v, f16x8));
    }
}

// The `left` (< 8) elements of a ragged end; the others read as zero.
template <class T>
__device__ __forceinline__ void load_end(Raw8<T> &out, const void *base, uint64_t i, uint32_t left) {
    const auto *p = reinterpret_cast<const typename T::raw *>(base) + i;
#pragma unroll
    for (int k = 0; k < Raw8<T>::kWords; ++k) out.w[k] = u32x4{0u, 0u, 0u, 0u};
#pragma unroll
    for (uint32_t k = 0; k < 8; ++k) {
        if (k >= left) continue;
        if constexpr (T::code == NT_F32) out.w[k >> 2][k & 3] = f32_bits(p[k]);
        else out.w[0][k >> 1] |= (uint32_t)p[k] << (16 * (k & 1));
    }
}

template <class T>
__device__ __forceinline__ void store_end(void *base, uint64_t i, const Raw8<T> &in, uint32_t left) {
    auto *p = reinterpret_cast<typename T::raw *>(base) + i;
#pragma unroll
    for (uint32_t k = 0; k < 8; ++k) {
        if (k >= left) continue;
        if constexpr (T::code == NT_F32) p[k] = bits_f32(in.w[k >> 2][k & 3]);
        else p[k] = (uint16_t)(in.w[0][k >> 1] >> (16 * (k & 1)));
    }
}

template <class T, bool EVEN>
__device__ __forceinline__ void load_part(Raw8<T> &out, const void *base, uint64_t row, uint32_t c, uint32_t width) {
    if (EVEN || width >= kGroup) load8<T, EVEN>(out, base, row + c);
    else load_end<T>(out, base, row + c, width - c);
}
template <class T, bool EVEN>
__device__ __forceinline__ void store_part(void *base, uint64_t row, uint32_t c, uint32_t width, const Raw8<T> &in) {
    if (EVEN || width >= kGroup) store8<T, EVEN>(base, row + c, in);
    else store_end<T>(base, row + c, in, width - c);
}

// Elements [c, c + 8) of weight or bias; `absent` where there is none.
__device__ __forceinline__ void load_params(float (&out)[8], const void *base, int32_t dtype, uint32_t c,
                                            uint32_t width, float absent) {
    if (base == nullptr || c + kGroup > width) {
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k) out[k] = c + k < width ? load_param(base, dtype, c + k, absent) : 0.0f;
    } else if (dtype == NT_F32) {
        Raw8<TF32> raw;
        load8<TF32, false>(raw, base, c);
        widen8<TF32>(out, raw);
    } else if (dtype == NT_F16) {
        Raw8<TF16> raw;
        load8<TF16, false>(raw, base, c);
        widen8<TF16>(out, raw);
    } else {
        Raw8<TBF16> raw;
        load8<TBF16, false>(raw, base, c);
        widen8<TBF16>(out, raw);
    }
}

// Numbers of the eight elements from flat index i on: one call where i is a
// multiple of eight, else the two groups they straddle, shifted together.
// (Taking the second group from the next lane, and the last lane's from a call
// on the scalar unit, was no faster: 26.8 against 26.0 us for the edge above.)
template <bool EVEN>
__device__ __forceinline__ PhiloxWords numbers8(uint64_t i, const Mask &m) {
    PhiloxWords words = philox(i >> 3, m.offset, m.seed);
    if constexpr (!EVEN) {
        const PhiloxWords next = philox((i >> 3) + 1, m.offset, m.seed);
        const uint32_t shift = (uint32_t)i & 7u;
        const bool by4 = shift & 4u, by2 = shift & 2u, by1 = shift & 1u;
        const uint32_t a = by4 ? words.w[2] : words.w[0], b = by4 ? words.w[3] : words.w[1];
        const uint32_t c = by4 ? next.w[0] : words.w[2], d = by4 ? next.w[1] : words.w[3];
        const uint32_t e = by4 ? next.w[2] : next.w[0], f = by4 ? next.w[3] : next.w[1];
        const uint32_t p = by2 ? b : a, q = by2 ? c : b, r = by2 ? d : c, s = by2 ? e : d, t = by2 ? f : e;
        words.w[0] = by1 ? __builtin_amdgcn_alignbit(q, p, 16) : p;
        words.w[1] = by1 ? __builtin_amdgcn_alignbit(r, q, 16) : q;
        words.w[2] = by1 ? __builtin_amdgcn_alignbit(s, r, 16) : r;
        words.w[3] = by1 ? __builtin_amdgcn_alignbit(t, s, 16) : s;
    }
    return words;
}

__device__ __forceinline__ void drop8(float (&v)[8], const PhiloxWords &words, const Mask &m) {
#pragma unroll
    for (int k = 0; k < 8; ++k) v[k] = philox_half(words, k) >= m.threshold ? v[k] * m.factor : 0.0f;
}

// ---- rows that fit in registers ----------------------------------------------------------------------
// `lanes` (a power of two) lanes hold a row in `parts` groups of eight each,
// group k of lane l at column 8 (k lanes + l).  Several rows share a workgroup
// (and a wave, below 64 lanes), which makes as many rounds as its rows need; a
// round past the last row computes nothing that is kept.  The row is read
// once, the variance is that of centred values in registers, and the next row
// is on its way while this one is summed.  Weight and bias wait in LDS: in
// registers they left room for five waves per SIMD instead of eight (16384 x
// 4096 float16 forward: 59 us with them, 49 without).

// Sum over the `lanes` lanes of a row, the same on each.  Rows of several
// waves go through `shared`, of which consecutive sums use the two halves in
// turn: a wave that writes a half again has passed the barrier of the sum in
// between, which no wave reaches before it has read that half.
//
// Within a wave the halves of 2, 4, 8 and 16 lanes are exchanged by the
// operand paths of the vector ALU (quad permutations, then mirrors: all lanes
// of a half hold the same sum by then), those of 32 and 64 by the row swaps
// (64 rows of 2048 in the forward pass: 4.8 us with permutes through LDS, 4.4 so).
template <int CTRL>
__device__ __forceinline__ float add_moved(float v) {
    return v + bits_f32((uint32_t)__builtin_amdgcn_mov_dpp((int)f32_bits(v), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float lanes_sum(float v, uint32_t lanes) {
    if (lanes > 1u) v = add_moved<0xB1>(v);             // lane ^ 1
    if (lanes > 2u) v = add_moved<0x4E>(v);             // lane ^ 2
    if (lanes > 4u) v = add_moved<0x141>(v);            // 7 - lane of eight
    if (lanes > 8u) v = add_moved<0x140>(v);            // 15 - lane of sixteen
    if (lanes > 16u) {
        const auto pair = __builtin_amdgcn_permlane16_swap(f32_bits(v), f32_bits(v), false, false);
        v = bits_f32(pair[0]) + bits_f32(pair[1]);
    }
    if (lanes > 32u) {
        const auto pair = __builtin_amdgcn_permlane32_swap(f32_bits(v), f32_bits(v), false, false);
        v = bits_f32(pair[0]) + bits_f32(pair[1]);
    }
    return v;
}

template <int MAX_WAVES>
struct RowSum {
    float (*shared)[MAX_WAVES];
    uint32_t lanes;
    uint32_t half = 0;
    __device__ __forceinline__ float operator()(float v) {
        v = lanes_sum(v, lanes);
        if (lanes <= 64u) return v;
        float *slot = shared[half];
        half ^= 1u;
        const uint32_t wave = threadIdx.x >> 6, waves = lanes / 64u, first = wave & ~(waves - 1u);
        if ((threadIdx.x & 63u) == 0u) slot[wave] = v;
        __syncthreads();
        float total = 0.0f;
        for (uint32_t k = first; k < first + waves; ++k) total += slot[k];
        return total;
    }
};

// Waves per SIMD that the compiler leaves registers for, and that the grid of
// a launch is made for: more only queue up, each loading weight and bias again
// (65536 x 768 float16: 38.9 us with the resident waves, 41.6 with twice as
// many).  It is a floor: edges of one group a lane take 64 to 78 registers,
// room for 6 or 7.  It does not look at LDS, of which weight and bias take 8
// bytes a column: 16-bit norms of 6145 to 8192 columns (64 KB) run 4 waves per
// SIMD, 16-bit rows of 8193 to 12288 (96 KB, 512 lanes) 2 and 16-bit norms of
// 12289 to 16384 4, on grids made for twice as many and more (2048 rows of
// bfloat16: 6144 columns 11.1 us, 8192 17.9, 12288 30.1, 16384 37.8).
template <class T, int EDGE, int PARTS>
constexpr int forward_waves() {
    return EDGE != kNone || PARTS > 2 || (T::code == NT_F32 && PARTS == 2) ? 4 : 8;
}

template <class T, int EDGE, int PARTS, bool EVEN, int THREADS>
__global__ __launch_bounds__(THREADS, (forward_waves<T, EDGE, PARTS>())) void norm_kernel(NormForward a,
                                                                                       uint32_t lanes) {
    extern __shared__ float4 room[];                    // weight, then bias
    __shared__ float shared[2][THREADS / 64];
    RowSum<THREADS / 64> row_sum{shared, lanes};
    const uint32_t lane = threadIdx.x & (lanes - 1u), in_block = threadIdx.x / lanes, per_block = THREADS / lanes;
    const float width = (float)a.width;
    Columns at[PARTS];
#pragma unroll
    for (int p = 0; p < PARTS; ++p) at[p] = Columns(((uint32_t)p * lanes + lane) * kGroup, a.width);
    const uint64_t stride = (uint64_t)gridDim.x * per_block;
    uint64_t row = (uint64_t)blockIdx.x * per_block + in_block;
    Raw8<T> x[PARTS], r[PARTS];
    const auto fetch = [&](uint64_t which) {
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
            if (which >= a.rows || at[p].column >= a.width) continue;
            load_part<T, EVEN>(x[p], a.x, which * a.width, at[p].column, a.width);
            if constexpr (EDGE != kNone) load_part<T, EVEN>(r[p], a.residual, which * a.width, at[p].column, a.width);
        }
    };
    // The first row's lanes bring the weight, the second's the bias (or the
    // first's again), asked for before the rows: they are there before them.
    float param[PARTS][8];
    const auto ask = [&](bool is_bias) {
#pragma unroll
        for (int p = 0; p < PARTS; ++p)
            load_params(param[p], is_bias ? a.bias : a.weight, a.weight_dtype, at[p].column, a.width,
                        is_bias ? 0.0f : 1.0f);
    };
    const auto keep = [&](bool is_bias) {
        float4 *to = room + (is_bias ? 2 * PARTS * lanes : 0u) + lane;
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
            to[2 * p * lanes] = make_float4(param[p][0], param[p][1], param[p][2], param[p][3]);
            to[(2 * p + 1) * lanes] = make_float4(param[p][4], param[p][5], param[p][6], param[p][7]);
        }
    };
    if (in_block < 2u) ask(in_block == 1u);
    fetch(row);
    if (in_block < 2u) keep(in_block == 1u);
    if (per_block == 1u) {
        ask(true);
        keep(true);
    }
    __syncthreads();
    for (uint64_t first = (uint64_t)blockIdx.x * per_block; first < a.rows; first += stride) {
        const uint64_t base = row * a.width;
        const bool active = row < a.rows;
        float t[PARTS][8];
        float sum = 0.0f;
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
            const bool mine = active && at[p].column < a.width;
            if (mine) {
                widen8<T>(t[p], x[p]);
                if constexpr (EDGE == kDropAdd) drop8(t[p], numbers8<EVEN>(base + at[p].column, a.mask), a.mask);
                if constexpr (EDGE != kNone) {
                    float add[8];
                    widen8<T>(add, r[p]);
#pragma unroll
                    for (int k = 0; k < 8; ++k) t[p][k] += add[k];
                }
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const bool in_row = active && at[p].template has<EVEN>(k, a.width);
                t[p][k] = mine ? t[p][k] : 0.0f;
                sum += EVEN || in_row ? t[p][k] : 0.0f;
            }
        }
        fetch(row + stride);
        const float mean = row_sum(sum) / width;
        float squares = 0.0f;
#pragma unroll
        for (int p = 0; p < PARTS; ++p)
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const bool in_row = at[p].template has<EVEN>(k, a.width);
                const float d = t[p][k] - mean;
                squares = in_row ? __builtin_fmaf(d, d, squares) : squares;
            }
        const float rstd = 1.0f / __builtin_sqrtf(row_sum(squares) / width + a.eps);
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
            if (!active || at[p].column >= a.width) continue;
            Raw8<T> out;
            if constexpr (EDGE != kNone) {
                narrow8<T>(out, t[p]);
                store_part<T, EVEN>(a.total, base, at[p].column, a.width, out);
            }
            float y[8];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const float4 w = room[(2 * p + q) * lanes + lane], b = room[(2 * PARTS + 2 * p + q) * lanes + lane];
                y[4 * q] = __builtin_fmaf((t[p][4 * q] - mean) * rstd, w.x, b.x);
                y[4 * q + 1] = __builtin_fmaf((t[p][4 * q + 1] - mean) * rstd, w.y, b.y);
                y[4 * q + 2] = __builtin_fmaf((t[p][4 * q + 2] - mean) * rstd, w.z, b.z);
                y[4 * q + 3] = __builtin_fmaf((t[p][4 * q + 3] - mean) * rstd, w.w, b.w);
            }
            narrow8<T>(out, y);
            store_part<T, EVEN>(a.y, base, at[p].column, a.width, out);
        }
        if (active && a.mean != nullptr && lane == 0) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
        row += stride;
    }
}

// Sums of two values over the lanes of a row, for workgroups that hold
// several rows of more than a wave: as RowSum, with a slot per wave and half.
template <int WAVES>
struct RowSum2 {
    float (*shared)[2][WAVES];
    uint32_t lanes;
    uint32_t half = 0;
    __device__ __forceinline__ void operator()(float &u, float &v) {
        u = lanes_sum(u, lanes);
        v = lanes_sum(v, lanes);
        if (lanes <= 64u) return;
        float (*slot)[WAVES] = shared[half];
        half ^= 1u;
        const uint32_t wave = threadIdx.x >> 6, waves = lanes / 64u, first = wave & ~(waves - 1u);
        if ((threadIdx.x & 63u) == 0u) {
            slot[0][wave] = u;
            slot[1][wave] = v;
        }
        __syncthreads();
        u = v = 0.0f;
        for (uint32_t k = first; k < first + waves; ++k) {
            u += slot[0][k];
            v += slot[1][k];
        }
    }
};

__device__ __forceinline__ void store_param(void *base, int32_t dtype, uint64_t i, float v) {
    switch (dtype) {
        case NT_F32: reinterpret_cast<float *>(base)[i] = v; break;
        case NT_F16: reinterpret_cast<uint16_t *>(base)[i] = f32_to_f16(v); break;
        default: reinterpret_cast<uint16_t *>(base)[i] = f32_to_bf16(v); break;
    }
}

// dw and db of 64 columns over all rows, for few rows: eight lanes to a row's
// columns, the rows over the rest of the workgroup, joined in a fixed order.
template <class T, bool EVEN, int THREADS>
__device__ __forceinline__ void column_tile(const NormBackward &a, uint32_t tile, float4 *room) {
    const Columns at(tile * 64u + (threadIdx.x & 7u) * kGroup, a.width);
    const uint32_t c = at.column;
    float dw[8] = {}, db[8] = {};
    if (c < a.width) {
#pragma unroll 2
        for (uint64_t row = threadIdx.x >> 3; row < a.rows; row += THREADS / 8) {
            Raw8<T> dy, t;
            load_part<T, EVEN>(dy, a.dy, row * a.width, c, a.width);
            load_part<T, EVEN>(t, a.t, row * a.width, c, a.width);
            const float mean = a.mean[row], rstd = a.rstd[row];
            float g[8], h[8];
            widen8<T>(g, dy);
            widen8<T>(h, t);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                dw[k] = __builtin_fmaf(g[k], (h[k] - mean) * rstd, dw[k]);
                db[k] += g[k];
            }
        }
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
#pragma unroll
        for (int off = 8; off < 64; off <<= 1) {
            dw[k] += __shfl_xor(dw[k], off, 64);
            db[k] += __shfl_xor(db[k], off, 64);
        }
    }
    float *sums = reinterpret_cast<float *>(room);      // [wave][dw, db][64]
    if ((threadIdx.x & 63u) < 8u) {
        const uint32_t place = (threadIdx.x >> 6) * 128u + (threadIdx.x & 7u) * 8u;
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k) {
            if (k < at.first) continue;                 // a last group's element `first` is the first of its place
            sums[place + k - at.first] = dw[k];
            sums[place + 64u + k - at.first] = db[k];
        }
    }
    __syncthreads();
    if (threadIdx.x >= 128u) return;
    float sum = 0.0f;
#pragma unroll
    for (uint32_t k = 0; k < THREADS / 64; ++k) sum += sums[k * 128u + threadIdx.x];
    const uint32_t column = tile * 64u + (threadIdx.x & 63u);
    void *out = threadIdx.x < 64u ? a.dw : a.db;
    if (out != nullptr && column < a.width) store_param(out, a.weight_dtype, column, sum);
}

// The backward pass of the same tiling.  dw and db of a lane's columns stay
// in registers over all rows of the workgroup; the rows that share a
// workgroup are joined at the end, halving them in turn, and each workgroup
// writes one row of partial sums, which norm_finalize_kernel adds.  With few
// rows, partial sums would be as large as the rows themselves: then workgroups
// of the same launch take columns instead (column_tile), and read the rows
// once more from the caches.
//
// Four waves per SIMD (128 registers) hide the loads; a row's successor is
// read into the registers of each group as soon as that group is done.  Twice
// the registers for it were no faster (norm 16384 x 4096 float16: 80 against
// 77 us), nor were 256 (136 us for the edge of that size, against 126) or 1024
// lanes (129).  It runs at what its accesses allow: with the sums and the
// arithmetic taken out the same kernel takes 73 us instead of 76 (norm, 16384 x
// 4096 float16, no weights), 39.1 instead of 39.5 (8192 x 2048 float32) and 124
// instead of 119 (edge, p = 0), that is 5.2 to 5.5 TB/s.
template <class T, int EDGE, int PARTS, bool EVEN, int THREADS>
__global__ __launch_bounds__(THREADS, 4) void norm_backward_kernel(NormBackward a, uint32_t lanes) {
    extern __shared__ float4 room[];                    // the weights, then the rows that are joined
    __shared__ float shared[2][2][THREADS / 64];
    if (blockIdx.x >= a.row_blocks) {
        column_tile<T, EVEN, THREADS>(a, blockIdx.x - a.row_blocks, room);
        return;
    }
    RowSum2<THREADS / 64> row_sum{shared, lanes};
    const uint32_t lane = threadIdx.x & (lanes - 1u), in_block = threadIdx.x / lanes, per_block = THREADS / lanes;
    const float width = (float)a.width;
    Columns at[PARTS];
#pragma unroll
    for (int p = 0; p < PARTS; ++p) at[p] = Columns(((uint32_t)p * lanes + lane) * kGroup, a.width);
    const uint64_t stride = (uint64_t)a.row_blocks * per_block;
    uint64_t row = (uint64_t)blockIdx.x * per_block + in_block;
    Raw8<T> dy[PARTS], t[PARTS], dt[PARTS];
    const auto fetch = [&](uint64_t which, int p) {
        if (which >= a.rows || at[p].column >= a.width) return;
        load_part<T, EVEN>(dy[p], a.dy, which * a.width, at[p].column, a.width);
        load_part<T, EVEN>(t[p], a.t, which * a.width, at[p].column, a.width);
        if constexpr (EDGE != kNone)
            if (a.dtotal != nullptr) load_part<T, EVEN>(dt[p], a.dtotal, which * a.width, at[p].column, a.width);
    };
#pragma unroll
    for (int p = 0; p < PARTS; ++p) fetch(row, p);
    float next_mean = row < a.rows ? a.mean[row] : 0.0f, next_rstd = row < a.rows ? a.rstd[row] : 0.0f;
    float dw[PARTS][8], db[PARTS][8];
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
#pragma unroll
        for (int k = 0; k < 8; ++k) dw[p][k] = db[p][k] = 0.0f;
        if (in_block == 0u) {
            float w[8];
            load_params(w, a.weight, a.weight_dtype, at[p].column, a.width, 1.0f);
            room[(2 * p) * lanes + lane] = make_float4(w[0], w[1], w[2], w[3]);
            room[(2 * p + 1) * lanes + lane] = make_float4(w[4], w[5], w[6], w[7]);
        }
    }
    __syncthreads();
    const auto weights = [&](float (&w)[8], int p) {
        const float4 low = room[(2 * p) * lanes + lane], high = room[(2 * p + 1) * lanes + lane];
        w[0] = low.x; w[1] = low.y; w[2] = low.z; w[3] = low.w;
        w[4] = high.x; w[5] = high.y; w[6] = high.z; w[7] = high.w;
    };
    for (uint64_t first = (uint64_t)blockIdx.x * per_block; first < a.rows; first += stride) {
        const uint64_t base = row * a.width, next = row + stride;
        const bool active = row < a.rows;
        const float mean = next_mean, rstd = next_rstd;
        float level = 0.0f, along = 0.0f;
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
            if (!active || at[p].column >= a.width) continue;
            float g[8], h[8], w[8];
            weights(w, p);
            widen8<T>(g, dy[p]);
            widen8<T>(h, t[p]);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const bool in_row = EVEN || at[p].template has<EVEN>(k, a.width);
                g[k] = in_row ? g[k] : 0.0f;
                h[k] = in_row ? (h[k] - mean) * rstd : 0.0f;
                dw[p][k] = __builtin_fmaf(g[k], h[k], dw[p][k]);
                db[p][k] += g[k];
                g[k] *= w[k];
                level += g[k];
                along = __builtin_fmaf(g[k], h[k], along);
            }
        }
        if (next < a.rows) {
            next_mean = a.mean[next];
            next_rstd = a.rstd[next];
        }
        row_sum(level, along);
        level /= width;
        along /= width;
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
            if (!active || at[p].column >= a.width) continue;
            float g[8], h[8], w[8];
            weights(w, p);
            widen8<T>(g, dy[p]);
            widen8<T>(h, t[p]);
#pragma unroll
            for (int k = 0; k < 8; ++k) g[k] = rstd * (g[k] * w[k] - level - (h[k] - mean) * rstd * along);
            if constexpr (EDGE != kNone) {
                if (a.dtotal != nullptr) {
                    widen8<T>(h, dt[p]);
#pragma unroll
                    for (int k = 0; k < 8; ++k) g[k] += h[k];
                }
            }
            fetch(next, p);                             // into the registers that were just read
            Raw8<T> out;
            if constexpr (EDGE != kNone) {
                narrow8<T>(out, g);
                store_part<T, EVEN>(a.dresidual, base, at[p].column, a.width, out);
                if constexpr (EDGE == kDropAdd) drop8(g, numbers8<EVEN>(base + at[p].column, a.mask), a.mask);
            }
            narrow8<T>(out, g);
            store_part<T, EVEN>(a.dx, base, at[p].column, a.width, out);
        }
        row = next;
    }
    if (a.partials == nullptr) return;
    const auto each = [&](auto &&use) {                 // the lane's sums, four at a time
#pragma unroll
        for (int p = 0; p < PARTS; ++p) {
            use(4 * p, dw[p][0], dw[p][1], dw[p][2], dw[p][3]);
            use(4 * p + 1, dw[p][4], dw[p][5], dw[p][6], dw[p][7]);
            use(4 * p + 2, db[p][0], db[p][1], db[p][2], db[p][3]);
            use(4 * p + 3, db[p][4], db[p][5], db[p][6], db[p][7]);
        }
    };
    for (uint32_t off = lanes; off < 64u; off <<= 1)    // rows of one wave
        each([&](int, float &x, float &y, float &z, float &w) {
            x += __shfl_xor(x, (int)off, 64);
            y += __shfl_xor(y, (int)off, 64);
            z += __shfl_xor(z, (int)off, 64);
            w += __shfl_xor(w, (int)off, 64);
        });
    const uint32_t span = lanes < 64u ? 64u : lanes, member = threadIdx.x / span, place = threadIdx.x & (span - 1u);
    for (uint32_t half = THREADS / span / 2u; half > 0u; half >>= 1) {
        __syncthreads();                                // the weights, or the last half, are read
        if (member >= half && member < 2u * half && place < lanes)
            each([&](int q, float x, float y, float z, float w) {
                room[((member - half) * 4 * PARTS + q) * lanes + place] = make_float4(x, y, z, w);
            });
        __syncthreads();
        if (member < half && place < lanes)
            each([&](int q, float &x, float &y, float &z, float &w) {
                const float4 other = room[(member * 4 * PARTS + q) * lanes + place];
                x += other.x;
                y += other.y;
                z += other.z;
                w += other.w;
            });
    }
    if (member != 0u || place >= lanes) return;
    float *out = a.partials + (uint64_t)blockIdx.x * 2u * a.width;
#pragma unroll
    for (int p = 0; p < PARTS; ++p) {
        if (at[p].column >= a.width) continue;
        Raw8<TF32> sums;
        if (!EVEN && (at[p].first != 0u || at[p].column + kGroup > a.width)) {
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) {
                if (!at[p].template has<false>(k, a.width)) continue;
                out[at[p].column + k] = dw[p][k];
                out[a.width + at[p].column + k] = db[p][k];
            }
            continue;
        }
        narrow8<TF32>(sums, dw[p]);
        store8<TF32, false>(out, at[p].column, sums);
        narrow8<TF32>(sums, db[p]);
        store8<TF32, false>(out, a.width + at[p].column, sums);
    }
}

// ---- rows of any width: a workgroup per row, the row read once per pass ---------------------
// For rows past the tilings (16384 columns).  Bound by the three passes over
// the row, an element at a time, from the caches, and in edges that drop by a
// whole call of the generator for every element of every pass (512 x 32768
// bfloat16: norm 115 us, backward 142, edge 185 and 182).  A lane's share of a
// row is summed in 64 bits: it is one chain of width / 256 additions (65536 at
// the widest), which in float32 put the mean of 2^20 values of 0.1 off by 4e-5
// of it, and the outputs of 2^24 of them, which are the bias, off by 0.02.
template <class T, int EDGE>
__device__ __forceinline__ float row_value(const NormForward &a, uint64_t i) {
    float v = load1<T>(reinterpret_cast<const typename T::raw *>(a.x), i);
    if constexpr (EDGE == kDropAdd) v = drop_one(v, i, a.mask);
    if constexpr (EDGE != kNone) v += load1<T>(reinterpret_cast<const typename T::raw *>(a.residual), i);
    return v;
}

template <class T, int EDGE>
__global__ __launch_bounds__(kBlock) void norm_rows_kernel(NormForward a) {
    __shared__ float shared[kBlock / 64];
    const float width = (float)a.width;
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const uint64_t base = row * a.width;
        double sum = 0.0;
        for (uint32_t c = threadIdx.x; c < a.width; c += kBlock) {
            const float v = row_value<T, EDGE>(a, base + c);
            if constexpr (EDGE != kNone) store1<T>(reinterpret_cast<typename T::raw *>(a.total), base + c, v);
            sum += v;
        }
        const float mean = block_sum_f32((float)sum, shared) / width;
        double squares = 0.0;
        for (uint32_t c = threadIdx.x; c < a.width; c += kBlock) {
            const float d = row_value<T, EDGE>(a, base + c) - mean;
            squares = __builtin_fma((double)d, (double)d, squares);
        }
        const float rstd = 1.0f / __builtin_sqrtf(block_sum_f32((float)squares, shared) / width + a.eps);
        for (uint32_t c = threadIdx.x; c < a.width; c += kBlock) {
            const float h = (row_value<T, EDGE>(a, base + c) - mean) * rstd;
            store1<T>(reinterpret_cast<typename T::raw *>(a.y), base + c,
                      __builtin_fmaf(h, load_param(a.weight, a.weight_dtype, c, 1.0f),
                                     load_param(a.bias, a.weight_dtype, c, 0.0f)));
        }
        if (a.mean != nullptr && threadIdx.x == 0) {
            a.mean[row] = mean;
            a.rstd[row] = rstd;
        }
    }
}

template <class T, int EDGE>
__global__ __launch_bounds__(kBlock) void norm_rows_backward_kernel(NormBackward a) {
    __shared__ float shared[kBlock / 64];
    const auto *dy = reinterpret_cast<const typename T::raw *>(a.dy);
    const auto *t = reinterpret_cast<const typename T::raw *>(a.t);
    const auto *dtotal = reinterpret_cast<const typename T::raw *>(a.dtotal);
    const float width = (float)a.width;
    for (uint64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
        const uint64_t base = row * a.width;
        const float mean = a.mean[row], rstd = a.rstd[row];
        double levels = 0.0, alongs = 0.0;
        for (uint32_t c = threadIdx.x; c < a.width; c += kBlock) {
            const float g = load1<T>(dy, base + c) * load_param(a.weight, a.weight_dtype, c, 1.0f);
            levels += g;
            alongs = __builtin_fma((double)g, (double)((load1<T>(t, base + c) - mean) * rstd), alongs);
        }
        const float level = block_sum_f32((float)levels, shared) / width;
        const float along = block_sum_f32((float)alongs, shared) / width;
        for (uint32_t c = threadIdx.x; c < a.width; c += kBlock) {
            const float g = load1<T>(dy, base + c) * load_param(a.weight, a.weight_dtype, c, 1.0f);
            const float h = (load1<T>(t, base + c) - mean) * rstd;
            float d = rstd * (g - level - h * along);
            if constexpr (EDGE != kNone) {
                if (dtotal != nullptr) d += load1<T>(dtotal, base + c);
                store1<T>(reinterpret_cast<typename T::raw *>(a.dresidual), base + c, d);
                if constexpr (EDGE == kDropAdd) d = drop_one(d, base + c, a.mask);
            }
            store1<T>(reinterpret_cast<typename T::raw *>(a.dx), base + c, d);
        }
    }
}

// Column sums of dy h and dy over the rows that this workgroup's y index
// strides over, one column per lane.
template <class T>
__global__ __launch_bounds__(kBlock) void norm_columns_kernel(NormBackward a) {
    const uint32_t c = blockIdx.x * kBlock + threadIdx.x;
    if (c >= a.width) return;
    const auto *dy = reinterpret_cast<const typename T::raw *>(a.dy);
    const auto *t = reinterpret_cast<const typename T::raw *>(a.t);
    float dw = 0.0f, db = 0.0f;
    for (uint64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
        const float g = load1<T>(dy, row * a.width + c);
        dw = __builtin_fmaf(g, (load1<T>(t, row * a.width + c) - a.mean[row]) * a.rstd[row], dw);
        db += g;
    }
    float *out = a.partials + (uint64_t)blockIdx.y * 2u * a.width;
    out[c] = dw;
    out[a.width + c] = db;
}

// dw and db from the partial sums, rounded to the weight's dtype: 32 columns
// and 32 slices of the groups per workgroup, the slices joined in order.  3.9
// us for 512 groups of 768 columns, of which a launch alone is near 3; 64
// columns to a workgroup took 4.4, 16 took 4.0 (and 8.0 instead of 5.1 at 4096).
constexpr uint32_t kFinalColumns = 32, kFinalSlices = 32;

template <class T>
__global__ __launch_bounds__(kFinalColumns * kFinalSlices) void norm_finalize_kernel(const float *partials,
                                                                                      uint32_t groups, uint32_t width,
                                                                                      typename T::raw *dw,
                                                                                      typename T::raw *db) {
    __shared__ float shared[kFinalSlices][kFinalColumns + 1];
    const uint32_t column = threadIdx.x % kFinalColumns, slice = threadIdx.x / kFinalColumns;
    const uint64_t c = (uint64_t)blockIdx.x * kFinalColumns + column;
    float sum = 0.0f;
    if (c < 2u * (uint64_t)width) {
#pragma unroll 8
        for (uint32_t k = slice; k < groups; k += kFinalSlices) sum += partials[(uint64_t)k * 2u * width + c];
    }
    shared[slice][column] = sum;
    __syncthreads();
    if (slice != 0 || c >= 2u * (uint64_t)width) return;
    sum = 0.0f;
#pragma unroll
    for (uint32_t k = 0; k < kFinalSlices; ++k) sum += shared[k][column];
    typename T::raw *out = c < width ? dw : db;
    if (out != nullptr) store1<T>(out, c < width ? c : c - width, sum);
}

// ---- dropout over a flat tensor ----------------------------------------------------------------
// 8192 x 8192 bfloat16: 45 us, 5.9 TB/s.  The generator's 18 wide multiplies per
// eight elements take some 34 us of the vector ALU, which the accesses hide.
// Two groups of eight per lane, a workgroup's width apart: 44.6 us, with one
// 46.7, with four 47.0 (16384 x 4096 float16).
constexpr int kDropGroups = 2;
// A 16-bit input larger than this is read around the caches, where little of
// it would be found: 134 MB 45.0 against 46.3 us, but 67 MB 24.5 against 22.0
// and 13 MB 7.2 against 6.4.  Float32, whose lanes touch a line twice, always
// reads through them (134 MB: 51.2 against 53.0 us).
constexpr uint64_t kCachedBytes = 96ull << 20;

template <class T, bool EVEN, bool NT>
__global__ __launch_bounds__(kBlock) void dropout_kernel(const void *x, void *y, uint64_t n, Mask mask) {
    constexpr uint64_t kDropTile = (uint64_t)kBlock * kGroup * kDropGroups;
    for (uint64_t start = blockIdx.x * kDropTile; start < n; start += gridDim.x * kDropTile) {
        Raw8<T> raw[kDropGroups];
#pragma unroll
        for (int u = 0; u < kDropGroups; ++u) {
            const uint64_t i = start + ((uint64_t)u * kBlock + threadIdx.x) * kGroup;
            if (i + kGroup <= n) load8<T, EVEN, NT>(raw[u], x, i);
            else if (i < n) load_end<T>(raw[u], x, i, (uint32_t)(n - i));
        }
#pragma unroll
        for (int u = 0; u < kDropGroups; ++u) {
            const uint64_t i = start + ((uint64_t)u * kBlock + threadIdx.x) * kGroup;
            if (i >= n) continue;
            float v[8];
            widen8<T>(v, raw[u]);
            drop8(v, philox(i >> 3, mask.offset, mask.seed), mask);
            narrow8<T>(raw[u], v);
            if (i + kGroup <= n) store8<T, EVEN>(y, i, raw[u]);
            else store_end<T>(y, i, raw[u], (uint32_t)(n - i));
        }
    }
}

// ---- launches ------------------------------------------------------------------------------------
constexpr uint32_t kColumnGroups = 256;                 // row groups of the column sums of rows past the tilings
constexpr uint64_t kMaxPartials = 256ull << 20;         // bytes of their workspace
constexpr uint64_t kMaxWidth = 1ull << 24;              // exact in float32, and the finalize stays below 2**32 lanes
constexpr uint32_t kBackwardWaves = 4;                  // per SIMD; with 2, the edge of 16384 x 4096: 145 us, not 126
// Up to this many rows the backward launch sums columns in workgroups of its
// own.  Kernel times with them and with partial sums: 129 x 8192 float16 5.8
// and 13.6 us, 512 x 776 bfloat16 5.5 and 10.1, 512 x 4096 9.2 and 13.7; but
// 1024 x 784 11.3 and 10.1.  The rule looks at rows alone, and wider ones would
// gain past it: a workgroup holds one row of more than 4096 columns, so that
// 513 x 8192 float16 has 512 rows of partial sums, 34 MB beside 25 MB of data
// (a whole call 25.0 us; with 512 rows 12.6).
constexpr uint64_t kFewRows = 512;
// LDS of norm_backward_kernel: the weights, half of the rows that are joined,
// or a column tile's sums of each wave.
static uint32_t backward_room(const RowTiling &g) {
    const uint32_t span = g.lanes < 64u ? 64u : g.lanes;
    const uint32_t weights = g.lanes * g.parts * kGroup * 4u;
    const uint32_t joined = g.threads / span / 2u * g.lanes * g.parts * 2u * kGroup * 4u;
    const uint32_t tile = g.threads / 64u * 128u * 4u;
    return std::max(weights, std::max(joined, tile));
}

// Whether the backward launch of `rows` rows sums columns in workgroups of its own.
static bool takes_columns(uint64_t rows, const RowTiling &g) { return g.parts != 0 && rows <= kFewRows; }

// Workgroups for `rows` rows, `per_block` at a time: as many as the registers
// leave resident (`most`) where there is work for them.  Fewer with the same
// number of rounds each leave some CUs a workgroup short: 5003 x 1001 float32
// 11.3 us with 626, 10.5 with 1024; 40001 x 512 float16 15.3 and 14.1.
static uint32_t row_grid(uint64_t rows, uint32_t per_block, uint32_t most) {
    const uint64_t blocks = (rows + per_block - 1) / per_block;
    return blocks > most ? most : blocks < 1 ? 1u : (uint32_t)blocks;
}

static uint32_t column_groups(uint64_t rows, uint64_t width) {
    uint64_t groups = rows < kColumnGroups ? rows : kColumnGroups;
    const uint64_t most = kMaxPartials / (2u * sizeof(float) * width);
    if (groups > most) groups = most;
    return groups < 1 ? 1u : (uint32_t)groups;
}

static uint32_t partial_groups(uint64_t rows, uint32_t width, int32_t dtype) {
    const RowTiling g = backward_tiling(width, dtype);
    if (g.parts == 0) return column_groups(rows, width);
    return row_grid(rows, g.threads / g.lanes, kSimds * kBackwardWaves * 64u / g.threads);
}

static bool aligned16(std::initializer_list<const void *> arrays) {
    uintptr_t bits = 0;
    for (const void *p : arrays) bits |= (uintptr_t)p;
    return bits % 16 == 0;
}

template <class T, int EDGE, int PARTS, bool EVEN>
static void launch_norm(const NormForward &a, const RowTiling &g, hipStream_t s) {
    constexpr uint32_t waves = kSimds * (uint32_t)forward_waves<T, EDGE, PARTS>();
    const dim3 grid(row_grid(a.rows, g.threads / g.lanes, waves * 64u / g.threads)), block(g.threads);
    const uint32_t room = g.lanes * g.parts * kGroup * 8u;
    if (g.threads == (uint32_t)kRowThreads) {
        if constexpr (forward_makes<T::code, PARTS, kRowThreads>())
            norm_kernel<T, EDGE, PARTS, EVEN, kRowThreads><<<grid, block, room, s>>>(a, g.lanes);
    } else {
        if constexpr (forward_makes<T::code, PARTS, kWideThreads>())
            norm_kernel<T, EDGE, PARTS, EVEN, kWideThreads><<<grid, block, room, s>>>(a, g.lanes);
    }
}

template <class T, int EDGE, int PARTS, bool EVEN>
static void launch_norm_backward(const NormBackward &a, const RowTiling &g, hipStream_t s) {
    const bool columns = a.partials == nullptr && (a.dw != nullptr || a.db != nullptr);
    const dim3 grid(a.row_blocks + (columns ? (a.width + 63u) / 64u : 0u)), block(g.threads);
    const uint32_t room = backward_room(g);
    if (g.threads == (uint32_t)kBackwardThreads) {
        if constexpr (backward_makes<T::code, PARTS, kBackwardThreads>())
            norm_backward_kernel<T, EDGE, PARTS, EVEN, kBackwardThreads><<<grid, block, room, s>>>(a, g.lanes);
    } else {
        if constexpr (backward_makes<T::code, PARTS, kWideThreads>())
            norm_backward_kernel<T, EDGE, PARTS, EVEN, kWideThreads><<<grid, block, room, s>>>(a, g.lanes);
    }
}

// Calls launch(parts, even) with both as constants.
template <int MAX_PARTS, class F>
static void with_tiling(const RowTiling &g, bool even, F &&launch) {
    using std::integral_constant;
    const auto with_parts = [&](auto e) {
        if (g.parts == 1) launch(integral_constant<int, 1>{}, e);
        else if (g.parts == 2) launch(integral_constant<int, 2>{}, e);
        else if constexpr (MAX_PARTS > 2) launch(integral_constant<int, 3>{}, e);
    };
    if (even) with_parts(integral_constant<bool, true>{});
    else with_parts(integral_constant<bool, false>{});
}

template <class T, int EDGE>
static void launch_forward_edge(const NormForward &a, hipStream_t s) {
    const RowTiling g = forward_tiling(a.rows, a.width, T::code);
    if (g.parts == 0) {
        norm_rows_kernel<T, EDGE><<<dim3(strided_grid(a.rows, kBlock)), dim3(kBlock), 0, s>>>(a);
        return;
    }
    const bool even = a.width % kGroup == 0 && aligned16({a.x, a.residual, a.total, a.y});
    with_tiling<T::code == NT_F32 ? 2 : 3>(
        g, even, [&](auto parts, auto e) { launch_norm<T, EDGE, parts.value, e.value>(a, g, s); });
}

template <class T, int EDGE>
static void launch_backward_edge(const NormBackward &a, hipStream_t s) {
    const RowTiling g = backward_tiling(a.width, T::code);
    if (g.parts == 0) {
        norm_rows_backward_kernel<T, EDGE><<<dim3(strided_grid(a.rows, kBlock)), dim3(kBlock), 0, s>>>(a);
        if (a.partials != nullptr)
            norm_columns_kernel<T><<<dim3((a.width + kBlock - 1) / kBlock, a.row_blocks), dim3(kBlock), 0, s>>>(a);
        return;
    }
    const bool even = a.width % kGroup == 0 && aligned16({a.dy, a.dtotal, a.t, a.dx, a.dresidual});
    with_tiling<2>(g, even,
                   [&](auto parts, auto e) { launch_norm_backward<T, EDGE, parts.value, e.value>(a, g, s); });
}

template <class T>
static void launch_forward(const NormForward &a, int edge, hipStream_t s) {
    if (edge == kNone) launch_forward_edge<T, kNone>(a, s);
    else if (edge == kAdd) launch_forward_edge<T, kAdd>(a, s);
    else launch_forward_edge<T, kDropAdd>(a, s);
}

template <class T>
static void launch_backward(const NormBackward &a, int edge, hipStream_t s) {
    if (edge == kNone) launch_backward_edge<T, kNone>(a, s);
    else if (edge == kAdd) launch_backward_edge<T, kAdd>(a, s);
    else launch_backward_edge<T, kDropAdd>(a, s);
}

template <class T>
static void launch_finalize(const NormBackward &a, hipStream_t s) {
    const dim3 grid((unsigned)((2u * (uint64_t)a.width + kFinalColumns - 1) / kFinalColumns));
    norm_finalize_kernel<T><<<grid, dim3(kFinalColumns * kFinalSlices), 0, s>>>(
        a.partials, a.row_blocks, a.width, static_cast<typename T::raw *>(a.dw), static_cast<typename T::raw *>(a.db));
}

template <class T>
static void launch_dropout(const void *x, void *y, uint64_t n, const Mask &mask, hipStream_t s) {
    const uint64_t tile = (uint64_t)kBlock * kGroup * kDropGroups;
    const dim3 grid(strided_grid((n + tile - 1) / tile, kBlock)), block(kBlock);
    const bool even = aligned16({x, y});
    if constexpr (T::code != NT_F32) {
        if (n * sizeof(typename T::raw) > kCachedBytes) {
            if (even) dropout_kernel<T, true, true><<<grid, block, 0, s>>>(x, y, n, mask);
            else dropout_kernel<T, false, true><<<grid, block, 0, s>>>(x, y, n, mask);
            return;
        }
    }
    if (even) dropout_kernel<T, true, false><<<grid, block, 0, s>>>(x, y, n, mask);
    else dropout_kernel<T, false, false><<<grid, block, 0, s>>>(x, y, n, mask);
}

// ---- argument checks --------------------------------------------------------------------------------
static bool half_or_float(int32_t dtype) { return dtype == NT_F32 || dtype == NT_F16 || dtype == NT_BF16; }

static int32_t check_rows(const char *entry, int32_t dtype, int32_t weight_dtype, bool has_params, uint64_t rows,
                          uint64_t width, uint32_t threshold) {
    const std::string name(entry);
    if (!half_or_float(dtype)) return fail(NT_ERR_TYPE, name + ": activations must be float32, float16 or bfloat16");
    if (has_params && weight_dtype != dtype && weight_dtype != NT_F32)
        return fail(NT_ERR_TYPE, name + ": weight and bias must have the activations' dtype or float32");
    if (width == 0 || width > kMaxWidth) return fail(NT_ERR_VALUE, name + ": the width must be 1..2**24");
    if (rows > 0xffffffffffffull / width) return fail(NT_ERR_VALUE, name + ": too many elements");
    if (threshold > 65536u) return fail(NT_ERR_VALUE, name + ": the drop threshold must be 0..65536");
    return NT_OK;
}

// One array argument: `count` elements of `dtype`, written or only read.
struct Array {
    const void *ptr;
    int32_t dtype;
    uint64_t count;
    bool written, needed;
};

// Needed arrays are there, all are aligned to their dtype, and what is
// written overlaps nothing else.
static int32_t check_arrays(const char *entry, std::initializer_list<Array> arrays) {
    for (const Array &a : arrays) {
        const uint64_t size = a.dtype == NT_F32 ? 4u : 2u;
        if (a.ptr == nullptr) {
            if (a.needed) return fail(NT_ERR_VALUE, std::string(entry) + ": NULL array");
            continue;
        }
        const uintptr_t start = (uintptr_t)a.ptr;
        if (start % size != 0) return fail(NT_ERR_VALUE, std::string(entry) + ": an array is not aligned to its dtype");
        if (!a.written) continue;
        for (const Array &b : arrays) {
            if (&a == &b || b.ptr == nullptr) continue;
            const uintptr_t other = (uintptr_t)b.ptr;
            if (start < other + b.count * (b.dtype == NT_F32 ? 4u : 2u) && other < start + a.count * size)
                return fail(NT_ERR_VALUE, std::string(entry) + ": an output overlaps another array");
        }
    }
    return NT_OK;
}

// NT_ERR_RUNTIME while `stream` is captured: a replay would repeat a mask, or
// use a workspace that the pool has handed to others since.
static int32_t refuse_capture(const char *entry, void *stream) {
    int32_t capturing = 0;
    const int32_t rc = nt_stream_capturing(stream, &capturing);
    if (rc != NT_OK) return rc;
    return capturing ? fail(NT_ERR_RUNTIME, std::string(entry) + ": not supported in stream capture") : NT_OK;
}

static int32_t forward(const char *entry, int32_t device, const NormForward &a, int32_t dtype, int edge, void *stream) {
    if ((a.mean == nullptr) != (a.rstd == nullptr))
        return fail(NT_ERR_VALUE, std::string(entry) + ": mean and rstd are given together");
    if (a.rows == 0) return NT_OK;
    DeviceGuard guard(device);
    if (!guard.ok()) return hip_check(guard.error(), "hipSetDevice");
    if (edge == kDropAdd) {
        const int32_t rc = refuse_capture(entry, stream);
        if (rc != NT_OK) return rc;
    }
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
        case NT_F32: launch_forward<TF32>(a, edge, s); break;
        case NT_F16: launch_forward<TF16>(a, edge, s); break;
        default: launch_forward<TBF16>(a, edge, s); break;
    }
    NT_LAUNCH_CHECK("norm_rows_kernel launch");
    return NT_OK;
}

static int32_t backward(const char *entry, int32_t device, NormBackward a, int32_t dtype, int edge, void *stream) {
    DeviceGuard guard(device);
    if (!guard.ok()) return hip_check(guard.error(), "hipSetDevice");
    const int32_t refused = refuse_capture(entry, stream);
    if (refused != NT_OK) return refused;
    hipStream_t s = (hipStream_t)stream;
    a.row_blocks = partial_groups(a.rows, a.width, dtype);
    const bool partial =
        (a.dw != nullptr || a.db != nullptr) && !takes_columns(a.rows, backward_tiling(a.width, dtype));
    if (partial) {
        // Goes back to the pool as soon as the kernels are queued: the pool reuses it on this stream only.
        void *workspace = nullptr;
        std::string error;
        const int32_t rc = device_pool().allocate(device, (uint64_t)a.row_blocks * 2u * a.width * sizeof(float),
                                                  stream, &workspace, error);
        if (rc != NT_OK) return fail(rc, error);
        a.partials = static_cast<float *>(workspace);
    }
    switch (dtype) {
        case NT_F32: launch_backward<TF32>(a, edge, s); break;
        case NT_F16: launch_backward<TF16>(a, edge, s); break;
        default: launch_backward<TBF16>(a, edge, s); break;
    }
    hipError_t status = hipGetLastError();
    if (!partial) return hip_check(status, "layer norm backward launch");
    if (status == hipSuccess) {
        switch (a.weight_dtype) {
            case NT_F32: launch_finalize<TF32>(a, s); break;
            case NT_F16: launch_finalize<TF16>(a, s); break;
            default: launch_finalize<TBF16>(a, s); break;
        }
        status = hipGetLastError();
    }
    std::string error;
    (void)device_pool().release(a.partials, error);
    return hip_check(status, "layer norm backward launch");
}

}  // namespace nt

using namespace nt;

extern "C" {

int32_t nt_layer_norm(int32_t device, const void *x, int32_t dtype, const void *weight, const void *bias,
                      int32_t weight_dtype, float eps, void *y, float *mean, float *rstd, uint64_t rows,
                      uint64_t width, void *stream) {
    clear_error();
    int32_t rc = check_rows("nt_layer_norm", dtype, weight_dtype, weight != nullptr || bias != nullptr, rows, width, 0);
    if (rc != NT_OK) return rc;
    if (rows == 0) return NT_OK;
    const uint64_t n = rows * width;
    rc = check_arrays("nt_layer_norm", {{x, dtype, n, false, true}, {weight, weight_dtype, width, false, false},
                                        {bias, weight_dtype, width, false, false}, {y, dtype, n, true, true},
                                        {mean, NT_F32, rows, true, false}, {rstd, NT_F32, rows, true, false}});
    if (rc != NT_OK) return rc;
    const NormForward a{x, nullptr, weight, bias, nullptr, y, mean, rstd, rows, (uint32_t)width, weight_dtype, eps, {}};
    return forward("nt_layer_norm", device, a, dtype, kNone, stream);
}

int32_t nt_layer_norm_backward(int32_t device, const void *dy, const void *x, int32_t dtype, const float *mean,
                               const float *rstd, const void *weight, int32_t weight_dtype, void *dx, void *dweight,
                               void *dbias, uint64_t rows, uint64_t width, void *stream) {
    clear_error();
    int32_t rc = check_rows("nt_layer_norm_backward", dtype, weight_dtype,
                            weight != nullptr || dweight != nullptr || dbias != nullptr, rows, width, 0);
    if (rc != NT_OK) return rc;
    const uint64_t n = rows * width;
    const bool any = rows > 0;
    rc = check_arrays("nt_layer_norm_backward",
                      {{dy, dtype, n, false, any}, {x, dtype, n, false, any}, {mean, NT_F32, rows, false, any},
                       {rstd, NT_F32, rows, false, any}, {weight, weight_dtype, width, false, false},
                       {dx, dtype, n, true, any}, {dweight, weight_dtype, width, true, false},
                       {dbias, weight_dtype, width, true, false}});
    if (rc != NT_OK) return rc;
    const NormBackward a{dy, nullptr, x, weight, mean, rstd, dx, nullptr, nullptr, rows, (uint32_t)width,
                         weight_dtype, {}, 0, dweight, dbias};
    return backward("nt_layer_norm_backward", device, a, dtype, kNone, stream);
}

int32_t nt_dropout(int32_t device, const void *x, int32_t dtype, void *y, uint64_t count, uint32_t threshold,
                   uint64_t seed, uint64_t offset, void *stream) {
    clear_error();
    if (!half_or_float(dtype)) return fail(NT_ERR_TYPE, "nt_dropout: activations must be float32, float16 or bfloat16");
    if (threshold > 65536u) return fail(NT_ERR_VALUE, "nt_dropout: the drop threshold must be 0..65536");
    if (count == 0) return NT_OK;
    if (count > 0xffffffffffffull) return fail(NT_ERR_VALUE, "nt_dropout: too many elements");
    // In place (y == x) each lane reads its elements before it writes them.
    int32_t rc = check_arrays("nt_dropout",
                              {{x, dtype, x == y ? 0 : count, false, true}, {y, dtype, count, true, true}});
    if (rc != NT_OK) return rc;
    DeviceGuard guard(device);
    if (!guard.ok()) return hip_check(guard.error(), "hipSetDevice");
    if (threshold != 0 && (rc = refuse_capture("nt_dropout", stream)) != NT_OK) return rc;
    const Mask mask = make_mask(threshold, seed, offset);
    hipStream_t s = (hipStream_t)stream;
    switch (dtype) {
        case NT_F32: launch_dropout<TF32>(x, y, count, mask, s); break;
        case NT_F16: launch_dropout<TF16>(x, y, count, mask, s); break;
        default: launch_dropout<TBF16>(x, y, count, mask, s); break;
    }
    NT_LAUNCH_CHECK("dropout_kernel launch");
    return NT_OK;
}

int32_t nt_dropout_add_layer_norm(int32_t device, const void *x, const void *residual, int32_t dtype,
                                  const void *weight, const void *bias, int32_t weight_dtype, float eps,
                                  uint32_t threshold, uint64_t seed, uint64_t offset, void *total, void *y, float *mean,
                                  float *rstd, uint64_t rows, uint64_t width, void *stream) {
    clear_error();
    const char *entry = "nt_dropout_add_layer_norm";
    int32_t rc = check_rows(entry, dtype, weight_dtype, weight != nullptr || bias != nullptr, rows, width, threshold);
    if (rc != NT_OK) return rc;
    if (rows == 0) return NT_OK;
    const uint64_t n = rows * width;
    rc = check_arrays(entry, {{x, dtype, n, false, true}, {residual, dtype, n, false, true},
                              {weight, weight_dtype, width, false, false}, {bias, weight_dtype, width, false, false},
                              {total, dtype, n, true, true}, {y, dtype, n, true, true},
                              {mean, NT_F32, rows, true, false}, {rstd, NT_F32, rows, true, false}});
    if (rc != NT_OK) return rc;
    const NormForward a{x, residual, weight, bias, total, y, mean, rstd, rows, (uint32_t)width, weight_dtype, eps,
                        make_mask(threshold, seed, offset)};
    return forward(entry, device, a, dtype, threshold == 0 ? kAdd : kDropAdd, stream);
}

int32_t nt_dropout_add_layer_norm_backward(int32_t device, const void *dy, const void *dtotal, const void *total,
                                           int32_t dtype, const float *mean, const float *rstd, const void *weight,
                                           int32_t weight_dtype, uint32_t threshold, uint64_t seed, uint64_t offset,
                                           void *dx, void *dresidual, void *dweight, void *dbias, uint64_t rows,
                                           uint64_t width, void *stream) {
    clear_error();
    const char *entry = "nt_dropout_add_layer_norm_backward";
    int32_t rc = check_rows(entry, dtype, weight_dtype, weight != nullptr || dweight != nullptr || dbias != nullptr,
                            rows, width, threshold);
    if (rc != NT_OK) return rc;
    const uint64_t n = rows * width;
    const bool any = rows > 0;
    rc = check_arrays(entry, {{dy, dtype, n, false, any}, {dtotal, dtype, n, false, false},
                              {total, dtype, n, false, any}, {mean, NT_F32, rows, false, any},
                              {rstd, NT_F32, rows, false, any}, {weight, weight_dtype, width, false, false},
                              {dx, dtype, n, true, any}, {dresidual, dtype, n, true, any},
                              {dweight, weight_dtype, width, true, false}, {dbias, weight_dtype, width, true, false}});
    if (rc != NT_OK) return rc;
    const NormBackward a{dy, dtotal, total, weight, mean, rstd, dx, dresidual, nullptr, rows, (uint32_t)width,
                         weight_dtype, make_mask(threshold, seed, offset), 0, dweight, dbias};
    return backward(entry, device, a, dtype, threshold == 0 ? kAdd : kDropAdd, stream);
}

}  // extern "C"
