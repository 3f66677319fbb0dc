// The tile shapes of the bf16 products and the rule that takes one by a product's
// sizes.  Plain C++: the launches size their grids and scratch by it, and a host
// library shows the tests what a product runs on (tests/linear_tiles_check.cpp).
#pragma once

#include <algorithm>
#include <cmath>
#include <cstdint>
#include <iterator>

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

// What the rule goes by.
struct LinearSizes {
    uint32_t rows, columns, depth;  // of C in front of a fold, and K (all experts' rows where K is ragged)
    uint32_t experts;               // 0: the dense product
    bool swiglu;
    bool ragged;  // K is an expert's rows, C has `rows` rows for each

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

// Values of K in each part of a dense product that is cut along K.
constexpr uint32_t linear_each(uint32_t depth, uint32_t splits) {
    return ((depth + splits - 1u) / splits + 63u) / 64u * 64u;
}

template <typename F>
auto with_linear_tiles(const LinearSizes& p, F f) {
    const uint64_t rows = p.experts != 0u && !p.ragged
                              ? p.rows / std::max(1u, std::min(p.rows, p.experts))
                              : p.rows;
    const bool few = !p.ragged;
    if (few && rows <= 16u) return f(Linear16x128{}, 1u);
    if (few && rows <= 32u) return f(Linear32x128{}, 1u);
    if (linear_tiles<Linear256x256>(p) >= 200u && rows > 128u) return f(Linear256x256{}, 1u);
    if (linear_tiles<Linear128x128>(p) >= 200u && rows > 64u) return f(Linear128x128{}, 1u);
    return f(Linear64x64{}, 1u);
}

}  // namespace q38m
