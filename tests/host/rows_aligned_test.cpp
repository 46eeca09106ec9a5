// Host unit test of nt_rows.hpp's aligned_rows: it holds exactly where each
// group that a lane stores, of each of a few rows and of every dtype, lies on
// 16 bytes, which stores through an aligned type need.
#include <cstdio>

#include "../../namitorch_amd/csrc/nt_rows.hpp"

using namespace nt;

static bool groups_aligned(uint32_t width, uintptr_t base) {
    for (uint32_t size : {2u, 4u})
        for (uint32_t row = 0; row < 9; ++row)
            for (uint32_t c = 0; c < width; c += kGroup) {
                const Columns at(c, width);
                if ((base + (row * (uint64_t)width + at.column) * size) % 16u != 0) return false;
            }
    return true;
}

int main() {
    int failures = 0;
    for (uint32_t width = 8; width <= 1100; ++width)
        for (uintptr_t base : {(uintptr_t)4096, (uintptr_t)4096 + 4, (uintptr_t)4096 + 8}) {
            const bool said = aligned_rows(width, {nullptr, (const void *)4096, (const void *)base});
            if (said != groups_aligned(width, base) && ++failures <= 20) std::printf("width %u base %zu\n", width, (size_t)base);
        }
    if (failures == 0) std::printf("all checks passed\n");
    return failures != 0;
}
