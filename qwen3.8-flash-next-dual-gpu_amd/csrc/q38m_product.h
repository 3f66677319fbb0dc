// What the products on workgroup tiles share (q38m_mx.hip, q38m_linear.hip): loads
// from memory to LDS, the row tiles of rows sorted by expert, the tiles' order over
// the eight XCDs, and the SwiGLU fold.
#pragma once

#include "q38m_device.h"
#include "q38m_internal.h"
#include "q38m_mx_tiles.h"

namespace q38m {
namespace {

typedef uint32_t v4u_any __attribute__((ext_vector_type(4), aligned(2)));  // 16 bytes at any element
typedef float v16f __attribute__((ext_vector_type(16)));
typedef uint32_t v4u __attribute__((ext_vector_type(4)));
typedef uint32_t v2u __attribute__((ext_vector_type(2)));
// at any element: rows of odd strides start anywhere
typedef uint32_t v2u_any __attribute__((ext_vector_type(2), aligned(2)));

// 1 / (1 + exp(-g)) on the base-2 exponential and reciprocal instructions (one unit in the
// last place each), and the SwiGLU fold h = g / (1 + exp(-g)) u.  The reciprocal gives zero in
// place of a result below the smallest normal, so it is taken of a quarter of the sum, whose
// reciprocal never is, and a multiplication takes the quarter back.  An exponential past 2^128
// is infinite and h a zero, as in the formula in fp32.  kExact puts the rounding of -g log2 e back (of an argument
// held to where the exponential is long infinite or zero): within 8 roundings of h; without
// it, |g| roundings more, 2^-17 of h at most, far below half a step of bf16.  (The contract's
// exp and an IEEE division take three times the instructions: an earlier form of the
// 32,768-token gate/up took 750 us with them and 640 without.)
template <bool kExact>
__device__ __forceinline__ float logistic(float g) {
    constexpr float kLog2e = 1.44269502162933349609375f;  // and what it lacks of log2 e
    constexpr float kLog2eLow = 1.92596299112661746887e-8f;
    const float x = kExact ? -__builtin_amdgcn_fmed3f(g, -128.0f, 128.0f) : -g;
    const float a = x * kLog2e;
    float e = __builtin_amdgcn_exp2f(a);
    if constexpr (kExact) {
        const float low = __builtin_fmaf(x, kLog2eLow, __builtin_fmaf(x, kLog2e, -a));
        e = __builtin_fmaf(fminf(e, 0x1p127f) * low, 0.693147180559945309f, e);  // infinite stays
    }
    return 0.25f * __builtin_amdgcn_rcpf(__builtin_fmaf(e, 0.25f, 0.25f));
}
template <bool kExact>
__device__ __forceinline__ float swiglu(float g, float u) {
    return g * logistic<kExact>(g) * u;
}

// the kernel's steps, which share its registers
#define MX_INLINE __attribute__((always_inline))

struct RowTile {
    uint32_t expert, first, count;  // rows first .. first + count of the sorted order
    bool alone;                     // all of the expert's rows
};

// The row tiles of the experts' rows, kRows at a time, found by a wave from the offsets
// (LDS, all of kMaxSortExperts, in words of 16 bytes because they are read so; those past
// the experts are the last one, `last`).  Lane l
// keeps the row tiles of the first 16 (l + 1) experts.  Offsets past `routes` count as
// routes, an end that is not behind its begin as no rows.
template <uint32_t kRows>
struct TileList {
    static constexpr uint32_t kPer = kMaxSortExperts / 64u;
    static_assert(kPer == 16u, "a row of lanes looks at a lane's experts");
    const uint32_t* offsets;
    uint32_t last, routes, sum, total;

    __device__ MX_INLINE TileList(const v4i* words, uint32_t last_, uint32_t routes_)
        : offsets(reinterpret_cast<const uint32_t*>(words)), last(last_), routes(routes_), sum(0) {
        const uint32_t lane = threadIdx.x & 63u;
        uint32_t at[kPer + 1];
#pragma unroll
        for (uint32_t i = 0; i < kPer; i += 4u) {
            const v4i w = words[(lane * kPer + i) / 4u];
            at[i] = w[0], at[i + 1u] = w[1], at[i + 2u] = w[2], at[i + 3u] = w[3];
        }
        at[kPer] = __shfl_down(at[0], 1);
        if (lane == 63u) at[kPer] = last;
#pragma unroll
        for (uint32_t i = 0; i < kPer; ++i) sum += tiles(at[i], at[i + 1u]);
#pragma unroll
        for (uint32_t d = 1; d < 64u; d <<= 1) {
            const uint32_t up = __shfl_up(sum, d);
            if (lane >= d) sum += up;
        }
        total = __builtin_amdgcn_readlane(sum, 63);
    }

    __device__ MX_INLINE uint32_t tiles(uint32_t begin, uint32_t end) const {
        begin = min(begin, routes);
        return (max(min(end, routes), begin) - begin + kRows - 1u) / kRows;
    }

    // tile < total
    __device__ MX_INLINE RowTile find(uint32_t tile) const {
        const uint32_t group = __builtin_ctzll(__ballot(sum > tile));
        const uint32_t left = tile - (group != 0u ? __builtin_amdgcn_readlane(sum, group - 1u) : 0u);
        const uint32_t e = group * kPer + threadIdx.x % kPer;
        const uint32_t begin = min(offsets[e], routes);
        const uint32_t end = min(e + 1u < kMaxSortExperts ? offsets[min(e + 1u, kMaxSortExperts - 1u)] : last, routes);
        uint32_t upto = tiles(begin, end);
        upto += __builtin_amdgcn_update_dpp(0, upto, 0x111, 0xf, 0xf, true);  // from 1, 2, 4, 8 lanes below
        upto += __builtin_amdgcn_update_dpp(0, upto, 0x112, 0xf, 0xf, true);
        upto += __builtin_amdgcn_update_dpp(0, upto, 0x114, 0xf, 0xf, true);
        upto += __builtin_amdgcn_update_dpp(0, upto, 0x118, 0xf, 0xf, true);
        const uint32_t at = __builtin_ctzll(__ballot(upto > left));
        const uint32_t before = at != 0u ? __builtin_amdgcn_readlane(upto, at - 1u) : 0u;
        const uint32_t from = __builtin_amdgcn_readlane(begin, at), to = __builtin_amdgcn_readlane(end, at);
        const uint32_t first = from + (left - before) * kRows;
        return RowTile{group * kPer + at, first, min(to - first, kRows), to - from <= kRows};
    }
};

// The order of the tiles, and each workgroup's part of it: groups of kGroup row tiles,
// column by column.  The dispatcher hands workgroups to the eight XCDs in turn, each
// with an L2 of its own: an XCD has one contiguous eighth of the order, and its
// workgroups take turns, so that those at work at the same time share rows of A and of
// B.  (Each a run of consecutive tiles, with the same rows of A, streams B at different
// places: gate/up of 512 experts, on an earlier form of the kernel, 112 us and in turns 108
// for 512 tokens, 316 and 182 for 2,048, 968 and 608 for 32,768.)
constexpr uint32_t kGroup = 4;
struct MxOrder {
    uint32_t rows, columns;   // of tiles
    uint32_t at, step, count;  // this workgroup's tiles

    __device__ MX_INLINE MxOrder(uint32_t rows_, uint32_t columns_) : rows(rows_), columns(columns_) {
        const uint64_t all = static_cast<uint64_t>(rows) * columns;
        const uint32_t xcd = blockIdx.x % kMxXcds;
        step = gridDim.x / kMxXcds;
        at = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(xcd * all / kMxXcds)) + blockIdx.x / kMxXcds;
        const uint32_t end = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>((xcd + 1u) * all / kMxXcds));
        count = at < end ? (end - at + step - 1u) / step : 0u;
    }
    __device__ MX_INLINE uint32_t height() const { return min(kGroup, rows - at / (kGroup * columns) * kGroup); }
    __device__ MX_INLINE uint32_t row() const {
        return at / (kGroup * columns) * kGroup + at % (kGroup * columns) % height();
    }
    __device__ MX_INLINE uint32_t column() const { return at % (kGroup * columns) / height(); }
};

__device__ __forceinline__ const uint8_t* mx_uniform(const uint8_t* p) {
    const uint64_t v = reinterpret_cast<uint64_t>(p);
    const uint32_t low = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v));
    const uint32_t high = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(v >> 32));
    return reinterpret_cast<const uint8_t*>(static_cast<uint64_t>(high) << 32 | low);
}

// 16 bytes (4 bytes) a lane from base + offset to consecutive LDS from byte `lds` on.  The
// compiler does not look into asm for the waits that its loads need: a scalar register that
// a vector instruction wrote (mx_uniform's lane reads) is read five wait states later at the
// earliest, m0 one after its write.  s_nop 3 is four, the move of m0 one.
#define MX_LOAD_LDS(INSTRUCTION)                                       \
    asm volatile("s_mov_b32 m0, %2\n\ts_nop 3\n\t" INSTRUCTION         \
                 :                                                     \
                 : "v"(offset), "s"(mx_uniform(base)), "s"(lds)        \
                 : "memory", "m0")
__device__ __forceinline__ void mx_load16(const uint8_t* base, uint32_t offset, uint32_t lds) {
    MX_LOAD_LDS("global_load_lds_dwordx4 %0, %1");
}
// the same past the caches
__device__ __forceinline__ void mx_load16_stream(const uint8_t* base, uint32_t offset, uint32_t lds) {
    MX_LOAD_LDS("global_load_lds_dwordx4 %0, %1 nt");
}
__device__ __forceinline__ void mx_load4(const uint8_t* base, uint32_t offset, uint32_t lds) {
    MX_LOAD_LDS("global_load_lds_dword %0, %1");
}

// until at most kOutstanding of the wave's loads are in flight and its LDS reads are
// complete, then for the workgroup's waves to get there
template <uint32_t kOutstanding>
__device__ __forceinline__ void mx_barrier() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" ::"i"(kOutstanding) : "memory");
}

}  // namespace
}  // namespace q38m
