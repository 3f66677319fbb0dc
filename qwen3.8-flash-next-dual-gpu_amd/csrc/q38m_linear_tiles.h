// The tile shapes of the bf16 products and the rule that takes one by a product's
// sizes.  Plain C++: the launches size their grids and scratch by it, and a host
// library shows the tests what a product runs on (tests/linear_tiles_check.cpp).
#pragma once

#include <algorithm>
#include <cmath>
#include <cstddef>
#include <cstdint>

#include "q38m_mx_tiles.h"

namespace q38m {

// kWM x kWN waves, each kTM x kTN matrix-instruction tiles of kMF rows: kBM rows of C by
// kBN columns, in a ring of kStages slots of LDS.
template <uint32_t kMF_, uint32_t kWM_, uint32_t kWN_, uint32_t kTM_, uint32_t kTN_, uint32_t kStages_>
struct LinearShape {
    static constexpr uint32_t kMF = kMF_, kWM = kWM_, kWN = kWN_, kTM = kTM_, kTN = kTN_;
    static constexpr uint32_t kStages = kStages_, kWaves = kWM * kWN;
    static constexpr uint32_t kBM = kWM * kTM * kMF, kBN = kWN * kTN * kMF, kRows = kBM + kBN;
    static constexpr uint32_t kDepth = 64;           // values of K in a stage
    static constexpr uint32_t kSteps = kMF / 8u;     // matrix instructions deep: 2 or 4
    // 16-byte words of LDS: the ring and the experts' offsets
    static constexpr uint32_t kSlot = kRows * 8u, kOffsetsAt = kStages * kSlot;
    static constexpr uint32_t kLds = kOffsetsAt + kMxMaxExperts / 4u;
    static constexpr uint32_t kResident = 160u * 64u / kLds;  // workgroups a CU
    static_assert(kResident != 0u, "160 KB of LDS");
};

using Linear256x256 = LinearShape<32, 4, 2, 2, 4, 2>;
using Linear128x128 = LinearShape<32, 2, 2, 2, 2, 2>;
using Linear64x64 = LinearShape<16, 2, 2, 2, 2, 3>;
using Linear32x128 = LinearShape<16, 1, 4, 2, 2, 3>;
using Linear16x128 = LinearShape<16, 1, 4, 1, 2, 3>;

// The form for few rows: kRows rows of C by 16 kTiles columns a workgroup, its kWaves waves a part
// of K each, in rings of kStages slots.
template <uint32_t kWaves_, uint32_t kStages_, uint32_t kTiles_>
struct FewShape {
    static constexpr uint32_t kRows = 16, kWaves = kWaves_, kStages = kStages_, kTiles = kTiles_;
    static constexpr uint32_t kLds = kWaves * kStages * (kRows + 16u * kTiles) * 8u + kMxMaxExperts / 4u;
    static constexpr uint32_t kResident = 160u * 64u / kLds;  // workgroups a CU
};

using Few8x16 = FewShape<8, 3, 1>;
using Few8x32 = FewShape<8, 2, 2>;
using Few4x32 = FewShape<4, 3, 2>;

// What the rule goes by.
struct LinearSizes {
    uint32_t rows, columns, depth;  // of C in front of a fold, and K (all experts' rows where K is ragged)
    uint32_t experts;               // 0: the dense product
    bool swiglu;
    bool ragged;  // K lies across A's stored rows; by expert: it is the expert's, and C has `rows` rows for each
    bool along;   // K lies along the stored rows of both operands

    constexpr uint32_t across() const { return swiglu ? columns / 2u : columns; }
};

// Row tiles: a bound where the experts' rows are known to the device alone.
template <typename S>
uint64_t linear_row_tiles(const LinearSizes& p) {
    const uint64_t of_rows = (static_cast<uint64_t>(p.rows) + S::kBM - 1u) / S::kBM;
    if (p.ragged && p.experts != 0u) return of_rows * std::min(p.experts, p.depth);
    return p.experts != 0u ? mx_max_tasks(p.rows, p.experts, S::kBM) : of_rows;
}

template <typename S>
uint64_t linear_tiles(const LinearSizes& p) {
    const uint64_t across = p.swiglu ? S::kBN / 2u : S::kBN;
    return linear_row_tiles<S>(p) * ((p.across() + across - 1u) / across);
}

// workgroups of the launch: one a tile (and part of K), at most as many as the card holds at once
template <typename S>
uint32_t linear_grid(const LinearSizes& p, uint32_t splits) {
    const uint64_t tiles = (linear_tiles<S>(p) * splits + kMxXcds - 1u) / kMxXcds * kMxXcds;
    return tiles < S::kResident * kMxCus ? static_cast<uint32_t>(tiles) : S::kResident * kMxCus;
}

// Values of K in each part of a dense product that is cut along K, and the parts that come of it.
constexpr uint32_t linear_each(uint32_t depth, uint32_t splits) {
    return ((depth + splits - 1u) / splits + 63u) / 64u * 64u;
}
constexpr uint32_t linear_parts(uint32_t depth, uint32_t splits) {
    const uint32_t each = linear_each(depth, splits);
    return (depth + each - 1u) / each;
}

// Workgroups of the form for few rows, a bound where the experts' rows are known to the device alone.
template <typename S>
uint64_t few_blocks(const LinearSizes& p) {
    const uint64_t across = p.swiglu ? 8u * S::kTiles : 16u * S::kTiles;
    const uint64_t rows = p.experts != 0u ? mx_max_tasks(p.rows, p.experts, S::kRows)
                                          : (static_cast<uint64_t>(p.rows) + S::kRows - 1u) / S::kRows;
    return rows * ((p.across() + across - 1u) / across);
}

// What a product is run on: the shape's number in LinearCost's order, or kFew and on of the form
// for few rows, and into how many parts its K is cut, whose sums go through the scratch.
struct LinearPlan {
    uint32_t shape, splits;
    constexpr bool few() const { return shape >= 5u; }
};

constexpr uint32_t kLinearShapes = 5, kFew = 5, kLinearMaxSplits = 32;
constexpr size_t kLinearMaxPartBytes = 256u << 20;

// What a product takes, us: a launch, and for every tile that a CU computes after another its
// stages and its end.  A stage takes `alone` at least, the answer's way from memory, and `each` for
// each of the workgroups that a CU holds.  The figures are fitted to graphs of 4,389 dense
// products of 1 to 8,192 rows (outputs and inputs 512 to 8,192, all three orders, K in 1 to 32
// parts) and of 860 experts' products (1 to 16,384 tokens, 8, 64 and 512 experts) on every shape.
// Taking the least, the rule's products are within 1.02 of the fastest shape's time in the
// geometric mean, and 1.2 at most but for weights' gradients of one or four tokens (1.65), which
// are mostly zeros written.
struct LinearCost {
    float alone, each, end;
};
constexpr LinearCost kDenseCost[kLinearShapes] = {
    {1.17f, 1.18f, 5.8f}, {0.65f, 0.45f, 1.33f}, {0.297f, 0.143f, 0.49f}, {0.295f, 0.225f, 0.61f}, {0.289f, 0.202f, 0.51f}};
constexpr LinearCost kExpertCost[kLinearShapes] = {
    {1.09f, 0.965f, 4.1f}, {0.65f, 0.395f, 0.94f}, {0.297f, 0.152f, 0.345f}, {0.19f, 0.248f, 0.43f}, {0.31f, 0.236f, 0.36f}};
constexpr LinearCost kRaggedCost[kLinearShapes] = {
    {1.34f, 1.365f, 5.8f}, {0.5f, 0.468f, 1.33f}, {0.297f, 0.106f, 0.49f}, {}, {}};
constexpr float kLaunchUs = 2.9f, kJoinUs = 2.5f, kJoinPartUs = 0.123f, kJoinMbUs = 1.26f;  // MB of a part's sums

// tiles * parts of `stages` stages each
template <typename S>
float linear_us(float tiles, float stages, const LinearCost& c) {
    const float held = std::min(static_cast<float>(S::kResident), std::ceil(tiles / 256.0f));
    return kLaunchUs + std::ceil(tiles / (256.0f * held)) * (stages * std::max(c.alone, held * c.each) + held * c.end);
}

template <typename S>
float linear_expert_us(const LinearSizes& p, uint32_t shape) {
    const uint32_t across = p.swiglu ? S::kBN / 2u : S::kBN;
    const float columns = static_cast<float>((p.across() + across - 1u) / across);
    const uint32_t routes = p.ragged ? p.depth : p.rows;
    const float active = static_cast<float>(std::min(routes, p.experts)), rows = static_cast<float>(routes) / active;
    if (p.ragged)
        return linear_us<S>(active * static_cast<float>((p.rows + S::kBM - 1u) / S::kBM) * columns, rows / 64.0f + 1.0f,
                            kRaggedCost[shape]);
    // an expert's last row tile is partly full
    const float tiles = routes <= p.experts ? 1.0f : std::max(1.0f, rows / S::kBM + 0.43f);
    return linear_us<S>(active * tiles * columns, static_cast<float>((p.depth + 63u) / 64u), kExpertCost[shape]);
}

// The plan with the least time.  wide: 256 x 256 tiles are there for it.  K that lies across A's
// rows takes tiles of 64 rows and more: fewer would not fill a load instruction.
//
// The form for few rows takes products of so few workgroups that the card holds all of them at
// once: as few waves a tile's stages in turn would leave most of it idle.  us on 8 waves by 16
// columns, 8 by 32 and 4 by 32, and on the best tiles with K cut:
//   1 x 2,048 x 2,048 (64 workgroups of 32 columns)    3.7   4.2   5.1    8.2
//   1 x 2,048 x 8,192 (64)                             7.9   9.6    13     11
//   1 x 8,192 x 2,048 (256)                            6.9   5.1   5.8    9.9
//   128 x 2,048 x 2,048 (512)                           12   7.8   6.2     11
//   61 x 8,192 x 512 (1,024)                            14   8.7   5.9    6.1
//   512 x 512 x 8,192 (512)                             29    21    20     18
//   gate/up of one token, 10 of 512 experts (320)              10.4    9.6   14.8
//   down of one token (640)                             13   9.0   6.9    6.2
inline LinearPlan linear_plan(const LinearSizes& p, bool wide) {
    if (p.along) {
        if (!p.swiglu && few_blocks<Few8x32>(p) <= 128u) return LinearPlan{kFew, 1u};
        if (few_blocks<Few8x32>(p) <= 256u) return LinearPlan{kFew + 1u, 1u};
        if (few_blocks<Few4x32>(p) <= 512u && p.depth <= 4096u) return LinearPlan{kFew + 2u, 1u};
    }
    LinearPlan best{2u, 1u};
    float least = 1e30f;
    const auto look = [&](auto s, uint32_t shape) {
        using S = decltype(s);
        if ((shape == 0u && !wide) || (p.ragged && S::kBM < 64u)) return;
        if (p.experts != 0u) {
            const float us = linear_expert_us<S>(p, shape);
            if (us < least) least = us, best = LinearPlan{shape, 1u};
            return;
        }
        const float tiles = static_cast<float>(linear_tiles<S>(p)), part_mb = static_cast<float>(p.rows) * p.columns * 4e-6f;
        for (uint32_t splits = 1; splits <= kLinearMaxSplits; splits *= 2u) {
            if (splits != 1u && (tiles * splits > 1024.0f || p.depth / splits < 128u ||
                                 part_mb * splits > kLinearMaxPartBytes * 1e-6f))
                break;
            float us = linear_us<S>(tiles * splits, static_cast<float>(linear_each(p.depth, splits) / 64u), kDenseCost[shape]);
            if (splits != 1u) us += kJoinUs + splits * (kJoinPartUs + kJoinMbUs * part_mb * 0.25f);
            if (us < least) least = us, best = LinearPlan{shape, splits};
        }
    };
    look(Linear256x256{}, 0u);
    look(Linear128x128{}, 1u);
    look(Linear64x64{}, 2u);
    look(Linear32x128{}, 3u);
    look(Linear16x128{}, 4u);
    return best;
}

// Calls f with the plan's form for few rows.
template <typename F>
auto with_few_shape(const LinearPlan& plan, F f) {
    switch (plan.shape) {
        case kFew: return f(Few8x16{});
        case kFew + 1u: return f(Few8x32{});
        default: return f(Few4x32{});
    }
}

// Calls f with the plan's tile shape.
template <typename F>
auto with_linear_shape(const LinearPlan& plan, F f) {
    switch (plan.shape) {
        case 0: return f(Linear256x256{});
        case 1: return f(Linear128x128{});
        case 2: return f(Linear64x64{});
        case 3: return f(Linear32x128{});
        default: return f(Linear16x128{});
    }
}

}  // namespace q38m
