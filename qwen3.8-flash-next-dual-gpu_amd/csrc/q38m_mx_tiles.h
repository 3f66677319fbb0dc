// The tile shapes of the microscaled products and the rule that takes one by a
// product's sizes.  Plain C++: the launches size their grids by it, and a host
// library shows the tests what a product runs on (tests/mx_tiles_check.cpp).
#pragma once

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <iterator>

namespace q38m {

constexpr uint32_t kMxXcds = 8, kMxCus = 256;
constexpr uint32_t kMxMaxExperts = 1024;

// kWM x kWN waves, each kTM x kTN matrix-instruction tiles of kMF rows: kBM rows of C by
// kBN rows of B, in a ring of kStages slots of LDS.
template <uint32_t kMF_, uint32_t kWM_, uint32_t kWN_, uint32_t kTM_, uint32_t kTN_, uint32_t kStages_>
struct MxShape {
    static constexpr uint32_t kMF = kMF_, kWM = kWM_, kWN = kWN_, kTM = kTM_, kTN = kTN_;
    static constexpr uint32_t kStages = kStages_, kWaves = kWM * kWN;
    static constexpr uint32_t kBM = kWM * kTM * kMF, kBN = kWN * kTN * kMF, kRows = kBM + kBN;
    static constexpr uint32_t kSteps = kMF / 8u;  // matrix instructions deep: 2 or 4
    // 16-byte words of LDS: the ring, the scales' and the experts' offsets.  The scales
    // of kStages stages may be under way: half as many pairs, begun and ended ones
    static constexpr uint32_t kSlot = kRows * 8u, kScaleAt = kStages * kSlot;
    static constexpr uint32_t kScaleWords = (kStages / 2u + 1u) * kRows;
    static constexpr uint32_t kOffsetsAt = kScaleAt + kScaleWords;
    static constexpr uint32_t kLds = kOffsetsAt + kMxMaxExperts / 4u;
    static constexpr uint32_t kResident = 160u * 64u / kLds;  // workgroups a CU
    static_assert(kResident != 0u, "160 KB of LDS");
};

using Mx256x256 = MxShape<32, 4, 2, 2, 4, 2>;
using Mx128x128 = MxShape<32, 2, 2, 2, 2, 2>;
using Mx64x64 = MxShape<16, 2, 2, 2, 2, 3>;
using Mx32x128 = MxShape<16, 1, 4, 2, 2, 3>;
using Mx16x128 = MxShape<16, 1, 4, 1, 2, 3>;
using Mx16x64 = MxShape<16, 1, 2, 1, 2, 4>;

// What the rule goes by.
struct MxSizes {
    uint32_t routes, n, k128;  // rows of C, rows of B (an expert's), K / 128 rounded up
    uint32_t experts;          // 0: the dense product
    bool swiglu;
    bool wide;  // a row's scales of two stages are one 16-byte piece

    constexpr uint32_t columns() const { return swiglu ? n / 2u : n; }
};

// scales of both sides at these addresses
inline bool mx_wide(uint32_t k128, uint64_t a_scales, uint64_t b_scales) {
    return k128 % 4u == 0u && a_scales % 16u == 0u && b_scales % 16u == 0u;
}

// row tiles that `routes` rows over `experts` experts need at most
constexpr uint32_t mx_max_tasks(uint32_t routes, uint32_t experts, uint32_t tile) {
    const uint32_t first = routes < experts ? routes : experts;
    return first + (routes - first) / tile;
}

// tiles: a bound where the experts' rows are known to the device alone
template <typename S>
uint64_t mx_tiles(const MxSizes& p) {
    const uint64_t across = p.swiglu ? S::kBN / 2u : S::kBN;
    const uint64_t rows = p.experts != 0u ? mx_max_tasks(p.routes, p.experts, S::kBM)
                                          : (static_cast<uint64_t>(p.routes) + S::kBM - 1u) / S::kBM;
    return rows * ((p.columns() + across - 1u) / across);
}

// workgroups of the launch: one a tile, at most as many as the card holds at once
template <typename S>
uint32_t mx_grid(const MxSizes& p) {
    const uint64_t tiles = (mx_tiles<S>(p) + kMxXcds - 1u) / kMxXcds * kMxXcds;
    return tiles < S::kResident * kMxCus ? static_cast<uint32_t>(tiles) : S::kResident * kMxCus;
}

// What a stage of all tiles takes, us: `each` for every 256 tiles.  An expert's last row
// tile is taken to be half full.
template <typename S>
float mx_stage_us(const MxSizes& p, float each) {
    const uint32_t across = p.swiglu ? S::kBN / 2u : S::kBN;
    float rows = static_cast<float>((p.routes + S::kBM - 1u) / S::kBM);
    if (p.experts != 0u) {
        const float active = static_cast<float>(p.routes < p.experts ? p.routes : p.experts);
        const float of_each = static_cast<float>(p.routes) / active / S::kBM + 0.5f;
        rows = active * (of_each > 1.0f ? of_each : 1.0f);
    }
    const float tiles = rows * static_cast<float>((p.columns() + across - 1u) / across);
    return each * std::ceil(tiles / 256.0f);
}

// Whether an expert's weights that one row tile reads alone go past the caches: where those
// of as many experts as may have a row are more than the 256 MB behind the L2s hold.
// Gate/up of 512 experts and 512 tokens, the same weights call after call, cached / past the
// caches, by bytes of codes: 201 MB 35.8 / 44.6 us, 268 MB 45.9 / 49.7, 302 MB 60 / 56, 537
// MB 106 / 94 (6.1 TB/s); 537 MB of which a skewed routing reads 300 57 / 64.  Tiles of 16
// and 32 rows alone: on 128 rows the choice between two loads costs what it gives (2,048
// tokens 130 / 129, 4,096 141 / 137, 8,192 of them 212 / 227), so many weights do not come to
// 64 rows, and in dense products the choice costs more (1 x 8,192 x 2,048 4.4 / 5.9).  And
// wide products alone: narrow scales have no such form (512 tokens, 512 experts of 1,024 x
// 1,920, 535 MB through the caches: 120 us, 4.5 TB/s).
template <typename S>
bool mx_streams(const MxSizes& p) {
    return p.experts != 0u && S::kBM <= 32u && p.wide &&
           static_cast<uint64_t>(std::min(p.routes, p.experts)) * p.n * p.k128 * 64u > (256ull << 20);
}

// Calls f with the shape that a product runs on, the one with the shortest stage.  The
// figures of `each` are fitted to these, us on 16 x 64, 16 x 128, 32 x 128, 64 x 64, 128 x
// 128 and 256 x 256 tiles:
//   1 x 8,192 x 2,048        4.5   5.1   5.2   5.2   6.8    13
//   32 x 4,096 x 4,096       6.2   7.6   7.7   7.4    10    21
//   256 x 4,096 x 4,096       14    13   9.3   8.7    12    24
//   509 x 2,048 x 8,192       25    23    16    14    20    43
//   1,024 x 4,096 x 4,096     44    42    26    21    17    28
//   4,096 x 4,096 x 4,096    158   155    96    81    49    41
//   8,192 x 8,192 x 8,192  1,409 1,108   638   531   346   280
// and gate/up (1,024 x 2,048) of 512 experts, top-10, by tokens:
//   1                        6.6   8.0   7.3   7.2   8.9    15
//   64                        65    64    64    77    80   114
//   512                       96    94    94   121   117   160
//   1,024                    138   131   106   127   122   161
//   2,048                    190   175   144   136   130   169
//   4,096                    283   266   192   199   141   176
//   8,192                    496   447   310   289   215   184
//   16,384                   885   800   518   477   313   310
//   32,768                 1,639 1,472   925   840   549   481
// 256 x 256 tiles are for wide products alone: without it they need registers that
// their waves do not have.
template <typename F>
auto with_mx_tiles(const MxSizes& p, F f) {
    const float us[] = {mx_stage_us<Mx16x64>(p, 0.2f),   mx_stage_us<Mx16x128>(p, 0.33f),
                        mx_stage_us<Mx32x128>(p, 0.45f), mx_stage_us<Mx64x64>(p, 0.38f),
                        mx_stage_us<Mx128x128>(p, 0.66f),
                        mx_stage_us<Mx256x256>(p, p.wide ? 2.0f : 1e30f)};
    switch (std::min_element(std::begin(us), std::end(us)) - us) {
        case 0: return f(Mx16x64{});
        case 1: return f(Mx16x128{});
        case 2: return f(Mx32x128{});
        case 3: return f(Mx64x64{});
        case 4: return f(Mx128x128{});
        default: return f(Mx256x256{});
    }
}

}  // namespace q38m
