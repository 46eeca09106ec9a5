// nt_row_ops.hpp — what the kernels over rows share: eight consecutive
// elements of a row in a lane's registers, parameters of any dtype, and sums
// over the lanes that hold a row.
#pragma once

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "nt_common.hpp"
#include "nt_rows.hpp"

namespace nt {

__device__ __forceinline__ float load_param(const void *base, int32_t dtype, uint64_t i, float absent) {
    if (base == nullptr) return absent;
    switch (dtype) {
        case NT_F32: return reinterpret_cast<const float *>(base)[i];
        case NT_F16: return f16_to_f32(reinterpret_cast<const uint16_t *>(base)[i]);
        default: return bf16_to_f32(reinterpret_cast<const uint16_t *>(base)[i]);
    }
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

// ---- sums over a row's lanes -------------------------------------------------------------------------
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

}  // namespace nt
