// Host unit test of nt_philox.hpp: the generator against the published
// answers of Philox4x32-10, the place of each element's number in its words,
// and the factor of the kept elements.
#include <cstdio>

#include "../../namitorch_amd/csrc/nt_philox.hpp"

static int failures = 0;
#define CHECK(cond)                                                       \
    do {                                                                  \
        if (!(cond)) {                                                    \
            std::printf("%s:%d: %s\n", __FILE__, __LINE__, #cond);        \
            ++failures;                                                   \
        }                                                                 \
    } while (0)

static uint64_t pair(uint32_t low, uint32_t high) { return (uint64_t)high << 32 | low; }

int main() {
    struct Known {
        uint32_t counter[4], key[2], answer[4];
    };
    const Known known[] = {
        {{0, 0, 0, 0}, {0, 0}, {0x6627e8d5u, 0xe169c58du, 0xbc57ac4cu, 0x9b00dbd8u}},
        {{~0u, ~0u, ~0u, ~0u}, {~0u, ~0u}, {0x408f276du, 0x41c83b0eu, 0xa20bc7c6u, 0x6d5451fdu}},
        {{0x243f6a88u, 0x85a308d3u, 0x13198a2eu, 0x03707344u},
         {0xa4093822u, 0x299f31d0u},
         {0xd16cfe09u, 0x94fdccebu, 0x5001e420u, 0x24126ea1u}},
    };
    for (const Known &k : known) {
        const nt::PhiloxWords words = nt::philox(pair(k.counter[0], k.counter[1]), pair(k.counter[2], k.counter[3]),
                                                 pair(k.key[0], k.key[1]));
        for (int i = 0; i < 4; ++i) {
            CHECK(words.w[i] == k.answer[i]);
            CHECK(nt::philox_half(words, 2 * i) == (k.answer[i] & 0xffffu));
            CHECK(nt::philox_half(words, 2 * i + 1) == k.answer[i] >> 16);
        }
    }
    CHECK(nt::make_mask(0, 1, 2).factor == 1.0f);
    CHECK(nt::make_mask(32768, 1, 2).factor == 2.0f);
    CHECK(nt::make_mask(6554, 1, 2).factor == (float)(65536.0 / 58982.0));
    CHECK(nt::make_mask(65535, 1, 2).factor == 65536.0f);
    CHECK(nt::make_mask(65536, 1, 2).factor == 0.0f);
    return failures != 0;
}
