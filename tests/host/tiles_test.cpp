// Host unit test of nt_tiles.hpp, and its answers for a problem.
//
// With arguments rows, classes, width, planes and whether the pass is the
// backward one: prints the plan's pieces, the logits' and the gradients' tiles
// and the splits of both products.  Without: over sizes of every magnitude the
// pieces cover the classes, keep their bytes unless they are the smallest, and
// no launch reaches 2**32 work-items.
#include <cstdio>
#include <cstdlib>

#include "../../namitorch_amd/csrc/nt_tiles.hpp"

using namespace nt;

static const char *const names[] = {"large", "middle", "tall", "few"};
static uint64_t threads_of(TileShape t) { return t == kLarge || t == kTall ? 512 : 256; }

int main(int argc, char **argv) {
    if (argc == 6) {
        const bool backward = std::atoi(argv[5]) != 0;
        const LossPlan p = loss_plan((uint32_t)std::atoll(argv[1]), (uint32_t)std::atoll(argv[2]),
                                     (uint32_t)std::atoll(argv[3]), std::atoi(argv[4]), true, backward);
        std::printf("%u %s %s %u %u\n", p.pieces, names[p.logits], names[p.grads], p.splits.input, p.splits.weight);
        return 0;
    }
    int failures = 0;
    const auto check = [&](bool good, const char *what, uint64_t rows, uint64_t classes, uint64_t width) {
        if (!good && ++failures <= 20)
            std::printf("%s: %llu x %llu x %llu\n", what, (unsigned long long)rows, (unsigned long long)classes,
                        (unsigned long long)width);
    };
    for (uint64_t rows = 1; rows < 1u << 24; rows += rows / 3 + 1)
        for (uint64_t classes = 1; classes < 1u << 30; classes += classes / 3 + 1)
            for (uint64_t width : {1u, 8u, 40u, 64u, 100u, 768u, 1001u, 4096u, 16384u, 100000u, 1u << 21}) {
                if (classes * width * 2 > 300000000000ull || rows * width * 2 > 300000000000ull) continue;
                for (int planes : {1, 3})
                    for (int pass = 0; pass < 2; ++pass) {
                        const LossPlan p = loss_plan((uint32_t)rows, (uint32_t)classes, (uint32_t)width, planes, true, pass);
                        const uint64_t last = classes - (p.pieces - 1ull) * p.piece;
                        check(p.pieces >= 1 && last >= 1 && last <= p.piece, "pieces cover the classes", rows, classes, width);
                        check(p.pieces == 1 || p.piece % 256 == 0, "pieces of whole tiles", rows, classes, width);
                        const bool least = p.piece <= 256;
                        const uint64_t packed = 2ull * planes * p.pitch * whole_steps(p.piece);
                        const uint64_t dz = 2ull * planes * whole_steps((uint32_t)rows) * whole_steps(p.piece);
                        check(least || !p.packed || packed <= kPieceBytes, "bytes of packed weights", rows, classes, width);
                        check(least || !pass || dz <= kPieceBytes, "bytes of dz", rows, classes, width);
                        const uint64_t logits = (uint64_t)tiles_of(whole_steps(p.piece), size_p(p.logits)) *
                                                tiles_of(whole_steps((uint32_t)rows), size_q(p.logits)) * threads_of(p.logits);
                        check(logits < 1ull << 32, "work-items of the logits", rows, classes, width);
                        if (!pass) continue;
                        const uint64_t across = tiles_of(p.pitch, size_p(p.grads)), q = size_q(p.grads);
                        const uint64_t both = across * (tiles_of(rows, (uint32_t)q) * (uint64_t)p.splits.input +
                                                        tiles_of(p.piece, (uint32_t)q) * (uint64_t)p.splits.weight) + 8;
                        check(both * threads_of(p.grads) < 1ull << 32, "work-items of the gradients", rows, classes, width);
                    }
            }
    if (failures == 0) std::printf("all checks passed\n");
    return failures != 0;
}
