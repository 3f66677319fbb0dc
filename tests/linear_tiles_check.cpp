// What the rule of csrc/q38m_linear_tiles.h runs a bf16 product on, for the tests: a host
// library of one function.
#include <iterator>

#include "q38m_linear_tiles.h"

using namespace q38m;

// result: rows and columns of a tile, parts of K and the values in each, the tiles of a part at
// most (2^32 - 1 where more), workgroups, workgroups that the card holds at once,
// waves that share K (the form for few rows; 0: tiles)
extern "C" void linear_tiles_of(uint32_t rows, uint32_t columns, uint32_t depth, uint32_t experts, uint32_t swiglu,
                                uint32_t ragged, uint32_t along, uint32_t wide, uint32_t* result) {
    const LinearSizes p{rows, columns, depth, experts, swiglu != 0u, ragged != 0u, along != 0u};
    const LinearPlan plan = linear_plan(p, wide != 0u);
    if (plan.few()) {
        with_few_shape(plan, [&](auto s) {
            using S = decltype(s);
            const uint32_t blocks = static_cast<uint32_t>(few_blocks<S>(p));
            const uint32_t values[] = {S::kRows, 16u * S::kTiles, 1u, depth, blocks, blocks, S::kResident * kMxCus, S::kWaves};
            std::copy(std::begin(values), std::end(values), result);
            return 0;
        });
        return;
    }
    with_linear_shape(plan, [&](auto s) {
        using S = decltype(s);
        const uint64_t tiles = linear_tiles<S>(p);
        const uint32_t parts = experts != 0u ? 1u : linear_parts(depth, plan.splits);
        result[0] = S::kBM;
        result[1] = S::kBN;
        result[2] = parts;
        result[3] = experts != 0u ? depth : linear_each(depth, plan.splits);
        result[4] = tiles >> 32 ? 0xffffffffu : static_cast<uint32_t>(tiles);
        result[5] = linear_grid<S>(p, parts);
        result[6] = S::kResident * kMxCus;
        result[7] = 0u;
        return 0;
    });
}
