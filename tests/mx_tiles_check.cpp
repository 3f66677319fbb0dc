// What the rule of csrc/q38m_mx_tiles.h runs a microscaled product on, for the
// tests: a host library of one function.
#include "q38m_mx_tiles.h"

using namespace q38m;

// result: rows of C and of B in a tile, whether scales come in 16-byte pieces, whether the
// weights go past the caches, the tiles at most (2^32 - 1 where more), workgroups
extern "C" void mx_tiles_of(uint32_t routes, uint32_t n, uint32_t columns, uint32_t experts, uint32_t swiglu,
                            uint32_t scales_aligned, uint32_t* result) {
    const uint32_t k128 = (columns + 127u) / 128u;
    const uint64_t scales = scales_aligned != 0u ? 16u : 4u;
    const MxSizes p{routes, n, k128, experts, swiglu != 0u, mx_wide(k128, scales, scales)};
    with_mx_tiles(p, [&](auto s) {
        using S = decltype(s);
        const uint64_t tiles = mx_tiles<S>(p);
        result[0] = S::kBM;
        result[1] = S::kBN;
        result[2] = p.wide;
        result[3] = mx_streams<S>(p);
        result[4] = tiles >> 32 ? 0xffffffffu : static_cast<uint32_t>(tiles);
        result[5] = mx_grid<S>(p);
        return 0;
    });
}
