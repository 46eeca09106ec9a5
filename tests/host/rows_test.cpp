// Host unit test of nt_rows.hpp: over every width of rows that stay in
// registers (and the numbers of rows at which the choice turns), each column
// has one owner, whole groups stay inside the row, the tiling fits its
// workgroup, and the tilings that come out are exactly those the predicates
// name, so that a launch finds its kernel and no kernel is built for none.
#include <cstdio>
#include <set>
#include <tuple>
#include <vector>

#include "../../namitorch_amd/csrc/nt_rows.hpp"

static int failures = 0;
#define CHECK(cond)                                                       \
    do {                                                                  \
        if (!(cond) && ++failures <= 20)                                  \
            std::printf("%s:%d: %s\n", __FILE__, __LINE__, #cond);        \
    } while (0)

using namespace nt;
typedef std::set<std::tuple<uint32_t, uint32_t>> Made;     // (groups a lane, lanes of a workgroup)

static void check_tiling(const RowTiling &g, uint32_t width) {
    CHECK(g.parts >= 1 && g.lanes >= 1 && (g.lanes & (g.lanes - 1)) == 0);
    CHECK(g.lanes <= g.threads && g.lanes * g.parts * kGroup >= width);
    static std::vector<int> owners;
    owners.assign(width, 0);
    for (uint32_t p = 0; p < g.parts; ++p)
        for (uint32_t lane = 0; lane < g.lanes; ++lane) {
            const Columns at((p * g.lanes + lane) * kGroup, width);
            if (at.column >= width) {
                for (uint32_t k = 0; k < kGroup; ++k) CHECK(!at.has<false>(k, width) && !at.has<true>(k, width));
                continue;
            }
            CHECK(at.column + kGroup <= width || (width < kGroup && at.column == 0));
            if (width % kGroup == 0) CHECK(at.first == 0 && at.column % kGroup == 0);
            for (uint32_t k = 0; k < kGroup; ++k)
                if (at.has<false>(k, width)) ++owners[at.column + k];
        }
    for (uint32_t c = 0; c < width; ++c) CHECK(owners[c] == 1);
}

template <int32_t DTYPE>
static Made forward_named() {
    Made named;
    if (forward_makes<DTYPE, 1, kRowThreads>()) named.emplace(1, kRowThreads);
    if (forward_makes<DTYPE, 2, kRowThreads>()) named.emplace(2, kRowThreads);
    if (DTYPE != NT_F32 && forward_makes<DTYPE, 3, kRowThreads>()) named.emplace(3, kRowThreads);
    if (forward_makes<DTYPE, 1, kWideThreads>()) named.emplace(1, kWideThreads);
    if (forward_makes<DTYPE, 2, kWideThreads>()) named.emplace(2, kWideThreads);
    if (DTYPE != NT_F32 && forward_makes<DTYPE, 3, kWideThreads>()) named.emplace(3, kWideThreads);
    return named;
}

template <int32_t DTYPE>
static Made backward_named() {
    Made named;
    if (backward_makes<DTYPE, 1, kBackwardThreads>()) named.emplace(1, kBackwardThreads);
    if (backward_makes<DTYPE, 2, kBackwardThreads>()) named.emplace(2, kBackwardThreads);
    if (backward_makes<DTYPE, 1, kWideThreads>()) named.emplace(1, kWideThreads);
    if (backward_makes<DTYPE, 2, kWideThreads>()) named.emplace(2, kWideThreads);
    return named;
}

template <int32_t DTYPE>
static void check_dtype() {
    Made forward, backward;
    for (uint32_t width = 1; width <= 16384; ++width) {
        uint32_t last = 0;
        std::vector<uint64_t> rows = {1, uint64_t(1) << 40};
        for (uint64_t lanes = 1; lanes <= kWideThreads; lanes <<= 1) {          // where one group a lane ends
            rows.push_back(kFewLanes / lanes);
            rows.push_back(kFewLanes / lanes + 1);
        }
        for (const uint64_t count : rows) {
            const RowTiling g = forward_tiling(count, width, DTYPE);
            forward.emplace(g.parts, g.threads);
            if (last != g.parts * 65536u + g.lanes) check_tiling(g, width);
            last = g.parts * 65536u + g.lanes;
        }
        const RowTiling g = backward_tiling(width, DTYPE);
        backward.emplace(g.parts, g.threads);
        check_tiling(g, width);
    }
    CHECK(forward == forward_named<DTYPE>());
    CHECK(backward == backward_named<DTYPE>());
    for (const uint32_t width : {16385u, 16392u, 32768u, 1u << 24}) {
        CHECK(forward_tiling(1, width, DTYPE).parts == 0);
        CHECK(backward_tiling(width, DTYPE).parts == 0);
    }
}

int main() {
    check_dtype<NT_F32>();
    check_dtype<NT_F16>();
    check_dtype<NT_BF16>();
    return failures != 0;
}
