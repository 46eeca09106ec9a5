// nt_philox.hpp — the counter-based generator behind dropout, and how its
// words become drop decisions.  Plain integer arithmetic; it also builds on
// the host for its unit test.
//
// Philox4x32-10: Salmon, Moraes, Dror and Shaw, "Parallel random numbers: as
// easy as 1, 2, 3", SC 2011 (the round function and its four constants are
// the paper's).  The 128-bit counter is (group, offset), the key the seed;
// one call gives the eight 16-bit numbers of group `i / 8`, so element i of a
// flat tensor has a number of its own that depends on (seed, offset, i)
// alone: not on the tensor's shape, alignment, dtype or the launch.
//
// 16 bits per element: p is a multiple of 2^-16 (the factor of the kept
// elements is that of the rounded p, so the mean is kept exactly), and a call
// serves eight elements.  With 32 bits per element a 16-bit dropout would be
// bound by the generator's multiplies instead of by memory.
#pragma once

#include <stdint.h>

#if defined(__HIPCC__)
#define NT_PHILOX_FN __host__ __device__ __forceinline__
#else
#define NT_PHILOX_FN inline
#endif

namespace nt {

struct PhiloxWords {
    uint32_t w[4];
};

NT_PHILOX_FN PhiloxWords philox(uint64_t group, uint64_t offset, uint64_t seed) {
    uint32_t a = (uint32_t)group, b = (uint32_t)(group >> 32);
    uint32_t c = (uint32_t)offset, d = (uint32_t)(offset >> 32);
    uint32_t k0 = (uint32_t)seed, k1 = (uint32_t)(seed >> 32);
#if defined(__clang__)
#pragma unroll
#endif
    for (int round = 0; round < 10; ++round) {
        const uint64_t left = (uint64_t)0xD2511F53u * a, right = (uint64_t)0xCD9E8D57u * c;
        a = (uint32_t)(right >> 32) ^ b ^ k0;
        b = (uint32_t)right;
        c = (uint32_t)(left >> 32) ^ d ^ k1;
        d = (uint32_t)left;
        k0 += 0x9E3779B9u;
        k1 += 0xBB67AE85u;
    }
    return PhiloxWords{{a, b, c, d}};
}

// Number (0..65535) of element `k` (0..7) of the group.
NT_PHILOX_FN uint32_t philox_half(const PhiloxWords &words, int k) {
    return k & 1 ? words.w[k >> 1] >> 16 : words.w[k >> 1] & 0xffffu;
}

// An element is dropped when its number is below `threshold` (0..65536), and
// otherwise multiplied by `factor` = 65536 / (65536 - threshold).
struct Mask {
    uint64_t seed, offset;
    uint32_t threshold;
    float factor;
};

inline Mask make_mask(uint32_t threshold, uint64_t seed, uint64_t offset) {
    return Mask{seed, offset, threshold, threshold < 65536u ? (float)(65536.0 / (double)(65536u - threshold)) : 0.0f};
}

}  // namespace nt
