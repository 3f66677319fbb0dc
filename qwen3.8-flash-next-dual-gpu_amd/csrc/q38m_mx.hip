// Microscaled 4-bit rows (MXFP4): quantisation, the dense product and the
// experts' products, on the block-scaled matrix instructions of gfx950.
//
// A row of K values is ceil(K / 128) * 64 bytes of codes (the even k in the
// low nibble; codes past K are zero) and one scale byte for every 32 values.
// Code c stands for (-1)^(c >> 3) * {0, .5, 1, 1.5, 2, 3, 4, 6}[c & 7], scale
// byte s for 2^(s - 127), 255 for NaN.
#include <type_traits>

#include "q38m_device.h"
#include "q38m_internal.h"
#include "q38m_mx_tiles.h"
#include "q38m_product.h"

namespace q38m {

static_assert(kMxMaxExperts == kMaxSortExperts, "the offsets that the tiles keep");

namespace {

// ---- quantisation -----------------------------------------------------------

typedef __bf16 v2bf __attribute__((ext_vector_type(2)));
typedef float v2f __attribute__((ext_vector_type(2)));
typedef unsigned short v2us __attribute__((ext_vector_type(2)));

// 2^(byte - 127) as fp32 bits; byte 0 is a subnormal
__device__ __forceinline__ float mx_scale(uint32_t byte) {
    return __uint_as_float(byte != 0u ? byte << 23 : 0x00400000u);
}

// The scale byte of a block whose largest magnitude has the exponent field f:
// 2^(floor(log2 m) - 2), the power of two that brings m into [4, 8), not below
// 2^-127; 255 where a value is not finite.
__device__ __forceinline__ uint32_t mx_scale_byte(uint32_t field) {
    return field == 255u ? 255u : (field > 2u ? field - 2u : 0u);
}

// Eight values of a row: their largest magnitude's exponent field, their codes
// under a scale (round to nearest even, above 6 to 6), and the codes' values.
template <typename T>
struct Eight;

template <>
struct Eight<uint16_t> {
    uint32_t d[4];  // bf16 pairs
    __device__ void load(const uint16_t* p) {
        const v4u_any w = *reinterpret_cast<const v4u_any*>(p);
        d[0] = w.x; d[1] = w.y; d[2] = w.z; d[3] = w.w;
    }
    __device__ void gather(const uint16_t* p, uint32_t count) {  // 1 <= count, zeros behind
        uint32_t v[8];
#pragma unroll
        for (uint32_t i = 0; i < 8u; ++i) v[i] = p[min(i, count - 1u)];
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i)
            d[i] = (2u * i < count ? v[2u * i] : 0u) | (2u * i + 1u < count ? v[2u * i + 1u] << 16 : 0u);
    }
    __device__ uint32_t field() const {
        v2us m = __builtin_bit_cast(v2us, d[0] & 0x7fff7fffu);
#pragma unroll
        for (uint32_t i = 1; i < 4u; ++i)
            m = __builtin_elementwise_max(m, __builtin_bit_cast(v2us, d[i] & 0x7fff7fffu));
        return (m.x > m.y ? m.x : m.y) >> 7;
    }
    __device__ uint32_t codes(float scale) const {
        uint32_t q = 0;
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(v2bf, d[0]), scale, 0);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(v2bf, d[1]), scale, 1);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(v2bf, d[2]), scale, 2);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(q, __builtin_bit_cast(v2bf, d[3]), scale, 3);
        return q;
    }
};

template <>
struct Eight<float> {
    float v[8];
    __device__ void load(const float* p) {
        const v4u_any a = reinterpret_cast<const v4u_any*>(p)[0], b = reinterpret_cast<const v4u_any*>(p)[1];
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) v[i] = __uint_as_float(a[i]), v[i + 4u] = __uint_as_float(b[i]);
    }
    __device__ void gather(const float* p, uint32_t count) {
#pragma unroll
        for (uint32_t i = 0; i < 8u; ++i) v[i] = p[min(i, count - 1u)];
#pragma unroll
        for (uint32_t i = 0; i < 8u; ++i) v[i] = i < count ? v[i] : 0.0f;
    }
    __device__ uint32_t field() const {
        uint32_t m = 0;
#pragma unroll
        for (uint32_t i = 0; i < 8u; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
        return m >> 23;
    }
    __device__ uint32_t codes(float scale) const {
        uint32_t q = 0;
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[0], v[1], scale, 0);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[2], v[3], scale, 1);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[4], v[5], scale, 2);
        q = __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(q, v[6], v[7], scale, 3);
        return q;
    }
};

// The eight values of a dword of codes, fp32.
__device__ __forceinline__ void mx_values(uint32_t codes, uint32_t byte, float* v) {
    const float scale = byte == 255u ? __builtin_nanf("") : mx_scale(byte);
#pragma unroll
    for (uint32_t i = 0; i < 8u; ++i) {
        const uint32_t c = codes >> (4u * i) & 15u, m = c & 7u;
        // e2m1 below 2 is m / 2; from there on exponent and mantissa bits as fp32 has them
        const float mag = m < 2u ? 0.5f * static_cast<float>(m)
                                 : __uint_as_float((126u << 23) + (m << 22));
        v[i] = (c & 8u ? -mag : mag) * scale;
    }
}

// Four lanes hold a block of 32 values, 16 lanes one scale dword.  `lanes` (a
// power of two from 16 to 256) threads walk a row, 256 / lanes rows at once.  One
// pass: each value is read once, in 16-byte pieces at any alignment, and a block's
// largest exponent found by two exchanges between lanes, so memory bounds it:
// 32,768 x 2,048 bf16 with the rounded values 51 us, 6.0 TB/s of 304 MB.  Loads or
// stores past the caches: 134 MB in and out 24.2 -> 27.3 us, 268 MB 53 -> 50, 1.1 GB
// the same.  Ten rows of 512: 2.4 us, a launch's own time.
constexpr uint32_t kQuantThreads = 256;

template <typename T>
__global__ __launch_bounds__(kQuantThreads) void mx_quantize_kernel(
    const T* __restrict__ x, uint64_t stride, uint32_t rows, uint32_t columns, uint32_t lanes_log2,
    uint32_t* __restrict__ codes, uint32_t* __restrict__ scales, T* __restrict__ rounded) {
    const uint32_t lanes = 1u << lanes_log2;
    const uint32_t row = blockIdx.x * (kQuantThreads >> lanes_log2) + (threadIdx.x >> lanes_log2);
    if (row >= rows) return;
    const uint32_t padded = (columns + 127u) / 128u * 128u;
    const T* from = x + row * stride;
    const uint64_t first_eight = static_cast<uint64_t>(row) * (padded / 8u);
    for (uint32_t c = (threadIdx.x & (lanes - 1u)) * 8u; c < padded; c += lanes * 8u) {
        Eight<T> e{};
        if (c + 8u <= columns) e.load(from + c);
        else if (c < columns) e.gather(from + c, columns - c);
        uint32_t field = e.field();
        field = max(field, static_cast<uint32_t>(__shfl_xor(static_cast<int>(field), 1)));
        field = max(field, static_cast<uint32_t>(__shfl_xor(static_cast<int>(field), 2)));
        const uint32_t byte = mx_scale_byte(field);
        const uint32_t q = byte == 255u ? 0u : e.codes(mx_scale(byte));
        codes[first_eight + c / 8u] = q;
        uint32_t four = byte;
        four |= static_cast<uint32_t>(__shfl_down(static_cast<int>(byte), 4)) << 8;
        four |= static_cast<uint32_t>(__shfl_down(static_cast<int>(byte), 8)) << 16;
        four |= static_cast<uint32_t>(__shfl_down(static_cast<int>(byte), 12)) << 24;
        if ((c & 127u) == 0u) scales[(first_eight + c / 8u) / 16u] = four;
        if (!rounded || c >= columns) continue;
        float v[8];
        mx_values(q, byte, v);
        T* to = rounded + static_cast<uint64_t>(row) * columns + c;
        constexpr uint32_t kWords = sizeof(T) * 2u;
        uint32_t d[kWords];
#pragma unroll
        for (uint32_t i = 0; i < kWords; ++i) {
            if constexpr (sizeof(T) == 4u) d[i] = __float_as_uint(v[i]);
            else d[i] = __float_as_uint(v[2 * i]) >> 16 |  // two significant bits: exact in bf16
                        (__float_as_uint(v[2 * i + 1]) & 0xffff0000u);
        }
        if (c + 8u <= columns) {
#pragma unroll
            for (uint32_t i = 0; i < kWords; i += 4u)
                reinterpret_cast<v4u_any*>(to)[i / 4u] = v4u_any{d[i], d[i + 1u], d[i + 2u], d[i + 3u]};
            continue;
        }
#pragma unroll
        for (uint32_t i = 0; i < 7u; ++i) {
            if (c + i >= columns) break;
            if constexpr (sizeof(T) == 4u) to[i] = v[i];
            else to[i] = static_cast<uint16_t>(d[i / 2u] >> i % 2u * 16u);
        }
    }
}

// ---- products -----------------------------------------------------------------

typedef int v8i __attribute__((ext_vector_type(8)));
// The block-scaled matrix instructions on 4-bit codes.  v_mfma_scale_f32_16x16x128:
// lane l holds the 32 values k = 32 (l / 16) .. + 31 of row l % 16 of A and of B and
// byte kByteA / kByteB of its scale word is that block's scale; D lane l: rows 4 (l / 16)
// + i of A, row l % 16 of B.  v_mfma_scale_f32_32x32x64: k = 32 (l / 32) .. + 31 of row
// l % 32; D lane l: rows 8 (i / 4) + 4 (l / 32) + i % 4 of A, row l % 32 of B.  Products
// and scales are exact; the sum is rounded in fp32.  In a loop over registers alone
// the 32x32 form runs at 6.6 PFLOP/s, the 16x16 form at 5.2.
template <int kByte>
__device__ __forceinline__ v4f mfma_mx(v4i a, uint32_t sa, v4i b, uint32_t sb, v4f c) {
    const v8i wa = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, wb = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wa, wb, c, 4, 4, kByte, sa, kByte, sb);
}
template <int kByte>
__device__ __forceinline__ v16f mfma_mx(v4i a, uint32_t sa, v4i b, uint32_t sb, v16f c) {
    const v8i wa = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, wb = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_32x32x64_f8f6f4(wa, wb, c, 4, 4, kByte, sa, kByte, sb);
}

// Workgroups stay and compute tile after tile of kBM rows of C by kBN rows of B (with
// the SwiGLU fold half of them gate, half up rows), kWM x kWN waves, each kTM x kTN
// matrix-instruction tiles of kMF rows.  K goes through LDS in stages of 256 values, a
// 128-byte line a row, in a ring of kStages slots, loaded straight from memory (no
// registers between, so the ring's depth costs none); the stages of a tile follow those
// of the tile before without a gap.  (Stages of 64 bytes a row, twice as many slots:
// 8,192^3 352 -> 376 us, the loads' line look-ups double.)  A slot holds kBM rows of A,
// then kBN rows of B.  Scales have a ring of their own: kWide (K a multiple of 512 and
// the scales 16-byte aligned) 16 bytes a row with every second stage, else 8 bytes a
// row and stage.
//
// The eight 16-byte pieces of row r lie at positions p ^ (r / 2 % 8): the lanes of a
// read take one piece of 16 or 32 consecutive rows, which then spread over all 64
// banks.  A load instruction fills 1 KB of consecutive LDS, eight rows; the swizzle is
// in the addresses that its lanes read.
//
// What bounds it: with few rows a launch, its first loads and how fast the L2s answer (a
// stage brings 43 to 56 KB a microsecond and CU to LDS on all five smaller shapes; 509 x 2,048
// x 8,192 14.1 us, its vector L1s held up by answers under way half the time); from tens of
// tokens on the weights' bytes (gate/up of 512 experts, 512 tokens: 94 us, 6.1 TB/s of 576
// MB); large products the clock, 1.8 GHz under their load, and the same waits, which leave the
// matrix pipes 57 % busy (8,192^3 278 us, 3.9 PFLOP/s); with few stages a tile, C's stores and
// loads that memory answers late: gate/up of 32,768 tokens 480 us, 3.4 PFLOP/s on the rows of
// its 256-row tiles, 2.9 on those that count (an earlier form of 509 us took 435 without its
// stores; with four experts' weights alone, which the L2s hold, 467 instead of 507).
template <typename S, bool kExperts, bool kSwiglu, bool kWide, bool kStream>
__global__ __launch_bounds__(64u * S::kWaves, (S::kResident * S::kWaves + 3u) / 4u) void mx_tile_kernel(MxProduct p) {
    constexpr uint32_t kMF = S::kMF, kTM = S::kTM, kTN = S::kTN, kBM = S::kBM, kBN = S::kBN;
    using Acc = std::conditional_t<kMF == 32u, v16f, v4f>;
    constexpr uint32_t kAcc = kMF == 32u ? 16u : 4u;
    __shared__ v4i ring[S::kLds];
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    __builtin_assume(wave < S::kWaves);  // settles at compile time which loads are of A and which of B
    const uint32_t n_out = kSwiglu ? p.n / 2u : p.n;
    constexpr uint32_t kColumns = kSwiglu ? kBN / 2u : kBN;
    const uint32_t columns = (n_out + kColumns - 1u) / kColumns;

    // ---- this workgroup's tiles, and what is known of those being loaded: lane t % 64
    // holds the t-th ----
    uint32_t* offsets = reinterpret_cast<uint32_t*>(ring + S::kOffsetsAt);
    const uint32_t last_offset = kExperts ? p.offsets[p.experts] : 0u;
    if constexpr (kExperts) {
        for (uint32_t e = threadIdx.x; e < kMaxSortExperts; e += 64u * S::kWaves)
            offsets[e] = e < p.experts ? p.offsets[e] : last_offset;
        __syncthreads();
#ifdef Q38M_CHECKED
        for (uint32_t e = threadIdx.x; e < p.experts; e += 64u * S::kWaves) {
            const uint32_t end = p.offsets[e + 1u];
            report(end < offsets[e] || end > p.routes, kCheckOffsets);
        }
        if (p.packed)  // each workgroup looks at a part of the sources
            for (uint32_t i = offsets[0] + blockIdx.x * 64u * S::kWaves + threadIdx.x; i < min(last_offset, p.routes);
                 i += gridDim.x * 64u * S::kWaves)
                report(p.packed[i] / p.top_k >= p.a_rows, kCheckToken);
#endif
    }
    const auto make_list = [&]() MX_INLINE {
        if constexpr (kExperts) return TileList<kBM>(ring + S::kOffsetsAt, last_offset, p.routes);
        else return 0;
    };
    const auto list = make_list();
    const auto row_tiles = [&]() MX_INLINE {
        if constexpr (kExperts) return list.total;
        else return (p.routes + kBM - 1u) / kBM;
    };
    MxOrder order(row_tiles(), columns);
    if (order.count == 0u) return;
    uint32_t known_first = 0, known_count = 0, known_column = 0;

    // ---- loads: instructions dealt to the waves, the left over ones to the first: 1 KB
    // of data each, eight rows; of scales 64 rows where they are 16-byte pieces, else 32.
    // Rows of A first, then of B, each instruction of one of them: a base of its tile for
    // all lanes and an offset below 4 GB for each ----
    constexpr uint32_t kDataA = kBM / 8u, kData = S::kRows / 8u;
    constexpr uint32_t kDataEach = kData / S::kWaves, kDataRest = kData % S::kWaves;
    constexpr uint32_t kDataLoads = kDataEach + (kDataRest != 0u ? 1u : 0u);
    constexpr uint32_t kScaleRows = kWide ? 64u : 32u;
    constexpr uint32_t kScaleA = (kBM + kScaleRows - 1u) / kScaleRows, kScale = kScaleA + (kBN + kScaleRows - 1u) / kScaleRows;
    constexpr uint32_t kScaleEach = kScale / S::kWaves, kScaleRest = kScale % S::kWaves;
    constexpr uint32_t kScaleLoads = kScaleEach + (kScaleRest != 0u ? 1u : 0u);
    const bool data_rest = kDataRest != 0u && wave < kDataRest;
    const bool scale_rest = kScaleRest != 0u && wave < kScaleRest;
    const auto data_live = [&](uint32_t t) MX_INLINE { return kDataRest == 0u || t < kDataEach || data_rest; };
    const auto scale_live = [&](uint32_t t) MX_INLINE { return kScaleRest == 0u || t < kScaleEach || scale_rest; };
    const uint32_t row_bytes = p.k128 * 64u, scale_bytes = p.k128 * 4u;
    const uint32_t stages = (p.k128 + 1u) / 2u;
    const bool odd = !kWide && (p.k128 & 1u) != 0u;  // a tile's last stage is 128 values
    const uint8_t *a_base, *b_base, *a_scale_base, *b_scale_base;
    uint32_t data[kDataLoads], scale[kScaleLoads];
    // the next tile to load, the `found`-th from one on, and the sources of its rows of A
    // where they are gathered: looked up a tile ahead, so that nobody waits for them
    uint32_t found = 0, next_column = 0;
    RowTile next{0u, 0u, 0u, false};
    uint32_t data_source[kDataLoads], scale_source[kScaleLoads];
    // On 256 x 256 tiles, which leave no registers over, what follows from the lane alone is
    // computed anew in each use outside the stages (kept from tile to tile, 12 registers went to
    // memory: 32,768-token gate/up 500 us instead of 481; where they are free keeping it is as
    // fast or faster: 509 x 2,048 x 8,192 14.1 instead of 14.4).
    const auto fresh_lane = [&]() MX_INLINE {
        uint32_t l = lane;
        if constexpr (S::kWaves == 8u) asm volatile("" : "+v"(l));
        return l;
    };
    const auto look_up = [&]() MX_INLINE {
        if (found == order.count) return;
        const uint32_t own_lane = fresh_lane();
        if (found != 0u) order.at += order.step;
        const uint32_t row = order.row();
        next_column = order.column();
        if constexpr (kExperts) next = list.find(row);
        else next = RowTile{0u, row * kBM, static_cast<uint32_t>(min(p.routes - row * kBM, kBM)), false};
        if (own_lane == found % 64u) {
            known_first = next.first;
            known_count = next.count;
            known_column = next_column;
        }
        ++found;
        if (!kExperts || !p.packed) return;
#pragma unroll
        for (uint32_t t = 0; t < kDataLoads; ++t) {
            const uint32_t i = wave + t * S::kWaves;
            if (t * S::kWaves < kDataA && data_live(t) && i < kDataA)
                data_source[t] = p.packed[next.first + min(8u * i + (own_lane >> 3), next.count - 1u)];
        }
#pragma unroll
        for (uint32_t t = 0; t < kScaleLoads; ++t) {
            const uint32_t i = wave + t * S::kWaves;
            if (t * S::kWaves < kScaleA && scale_live(t) && i < kScaleA)
                scale_source[t] = p.packed[next.first + min(kScaleRows * i + (kWide ? own_lane : own_lane >> 1), next.count - 1u)];
        }
    };
    // points the loads at the tile that was looked up, and looks up the one after it
    bool stream = false;  // of the tile being loaded: no other row tile reads this B
    const auto point = [&]() MX_INLINE {
        stream = kStream && next.alone;
        const uint32_t own_lane = fresh_lane();
        const bool gather = kExperts && p.packed;
        const uint64_t a_first = gather ? 0u : next.first;
        const uint64_t b_first = static_cast<uint64_t>(next.expert) * p.n + next_column * kColumns;
        a_base = mx_uniform(p.a_codes + a_first * row_bytes);
        a_scale_base = mx_uniform(p.a_scales + a_first * scale_bytes);
        b_base = mx_uniform(p.b_codes + b_first * row_bytes);
        b_scale_base = mx_uniform(p.b_scales + b_first * scale_bytes);
        const auto a_row = [&](uint32_t j, uint32_t source) MX_INLINE -> uint32_t {
            if (gather) return min(source / p.top_k, p.a_rows - 1u);
            return min(j, next.count - 1u);
        };
        const auto b_row = [&](uint32_t j) MX_INLINE -> uint32_t {
            uint32_t column = j, up = 0;
            if constexpr (kSwiglu) {  // a wave's tiles: half of them gate, half up
                const uint32_t t = j / kMF % kTN;
                column = j / (kTN * kMF) * (kTN / 2u * kMF) + t % (kTN / 2u) * kMF + j % kMF;
                up = t >= kTN / 2u ? n_out : 0u;
            }
            return min(column, n_out - 1u - next_column * kColumns) + up;
        };
#pragma unroll
        for (uint32_t t = 0; t < kDataLoads; ++t) {
            if (!data_live(t)) continue;
            const uint32_t i = wave + t * S::kWaves;
            const uint32_t r = 8u * i + (own_lane >> 3), piece = (own_lane & 7u) ^ (r >> 1 & 7u);
            const bool of_a = t * S::kWaves < kDataA && i < kDataA;
            data[t] = (of_a ? a_row(r, data_source[t]) : b_row(r - kBM)) * row_bytes + 16u * piece;
        }
#pragma unroll
        for (uint32_t t = 0; t < kScaleLoads; ++t) {
            if (!scale_live(t)) continue;
            const uint32_t i = wave + t * S::kWaves, r = kWide ? own_lane : own_lane >> 1;
            const bool of_a = t * S::kWaves < kScaleA && i < kScaleA;
            scale[t] = (of_a ? a_row(kScaleRows * i + r, scale_source[t])
                             : b_row(min(kScaleRows * (i - kScaleA) + r, kBN - 1u))) * scale_bytes;
        }
        look_up();
    };
    look_up();
    uint32_t tiles_left = order.count;  // with the one being loaded
    bool turn = false;
    point();
    uint32_t from = 0, to = 0, scales_to = 0;  // the stage of the tile and the slots it is loaded to
    const uint32_t ring_at = static_cast<uint32_t>(
        reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) v4i*)ring));
    constexpr uint32_t kScaleSlot = kWide ? S::kRows : S::kRows / 2u;  // words
    constexpr uint32_t kScaleSlots = S::kScaleWords / kScaleSlot;
    static_assert(kScaleSlots >= (kWide ? S::kStages / 2u + 1u : S::kStages), "scales under way");
    const auto load_scale = [&](uint32_t t) MX_INLINE {
        if (!scale_live(t)) return;
        const uint32_t i = wave + t * S::kWaves, r = kWide ? lane : lane >> 1;
        const bool of_b = t * S::kWaves >= kScaleA || i >= kScaleA;
        const uint32_t first = of_b ? kScaleRows * (i - kScaleA) : kScaleRows * i;
        // some lane of a load is within the rows: its count is the same everywhere
        if ((kBM % kScaleRows != 0u || kBN % kScaleRows != 0u) && first + r >= (of_b ? kBN : kBM)) return;
        const uint32_t at = __builtin_amdgcn_readfirstlane(
            ring_at + (S::kScaleAt + scales_to * kScaleSlot) * 16u + (first + (of_b ? kBM : 0u)) * (kWide ? 16u : 8u));
        const uint8_t* base = of_b ? b_scale_base : a_scale_base;
        if constexpr (kWide) mx_load16(base + (from & ~1u) * 8ull, scale[t], at);
        else mx_load4(base, scale[t] + 4u * min(from * 2u + (lane & 1u), p.k128 - 1u), at);
    };
    const auto load_data = [&](uint32_t t) MX_INLINE {
        if (!data_live(t)) return;
        const uint32_t i = wave + t * S::kWaves;
        uint32_t back = 0;  // a piece past the end of its row: another of the row
        if constexpr (!kWide) {
            const uint32_t piece = (lane & 7u) ^ ((4u * i + (lane >> 4)) & 7u);
            back = odd && from + 1u == stages && piece >= 4u ? 64u : 0u;
        }
        const bool of_a = t * S::kWaves < kDataA && i < kDataA;
        const uint8_t* base = (of_a ? a_base : b_base) + (from * 128ull);
        const uint32_t at = __builtin_amdgcn_readfirstlane(ring_at + to * (S::kSlot * 16u) + i * 1024u);
        if (kStream && stream && !of_a) mx_load16_stream(base, data[t] - back, at);
        else mx_load16(base, data[t] - back, at);
    };
    // to the next stage to load, at a tile's first stage with a turn to take before its loads;
    // past the last tile the last stage again, into slots that nobody reads any more, so
    // that the count of loads under way is always the same
    const auto load_next = [&](bool scales_too) MX_INLINE {
        to = to + 1u == S::kStages ? 0u : to + 1u;
        if (scales_too) scales_to = scales_to + 1u == kScaleSlots ? 0u : scales_to + 1u;
        if (from + 1u < stages) {
            ++from;
        } else if (tiles_left != 1u) {
            from = 0;
            turn = true;
        }
    };
    const auto take_turn = [&]() MX_INLINE {
        if (!turn) return;
        turn = false;
        --tiles_left;
        point();
    };

    // ---- products ----
    const uint32_t wm = wave / S::kWN, wn = wave % S::kWN;
    const uint32_t n = lane % kMF, q = lane / kMF;
    Acc acc[kTN][kTM];
#pragma unroll
    for (uint32_t j = 0; j < kTN; ++j)
#pragma unroll
        for (uint32_t i = 0; i < kTM; ++i) acc[j][i] = Acc{};
    const uint32_t a_at = wm * kTM * kMF + n, b_at = kBM + wn * kTN * kMF + n;  // rows of the slot
    const uint32_t swizzle = n >> 1 & 7u;  // as of every kMF-th row after it
    constexpr uint32_t kReads = kTM + kTN;
    v4i part[2][kReads];      // a step's fragments of A, then of B, and the next step's
    uint2 factor[2][kReads];  // a stage's scales, and the next stage's
    uint32_t slot = 0, scales = 0;  // of the stage whose fragments are read
    // a fragment of step c; those of A are zero behind a stage's end, where K ends in it
    // (and B's are others of the row)
    const auto read = [&](uint32_t c, uint32_t i, bool behind) MX_INLINE {
        const uint32_t row = i < kTM ? a_at + i * kMF : b_at + (i - kTM) * kMF;
        part[c % 2u][i] = ring[slot * S::kSlot + row * 8u + ((64u / kMF * c + q) ^ swizzle)];
        if (!kWide && 2u * c >= S::kSteps && i < kTM && behind) part[c % 2u][i] = v4i{0, 0, 0, 0};
    };
    const auto read_factor = [&](uint32_t parity, uint32_t buffer, uint32_t i) MX_INLINE {
        const uint32_t row = i < kTM ? a_at + i * kMF : b_at + (i - kTM) * kMF;
        const uint2* base = reinterpret_cast<const uint2*>(ring + S::kScaleAt + scales * kScaleSlot);
        factor[buffer][i] = kWide ? base[2u * row + parity] : base[row];
    };
    const auto shift_factor = [&](uint32_t buffer, uint32_t i) MX_INLINE {  // this lane's bytes to where the instruction takes them
        factor[buffer][i] = make_uint2(factor[buffer][i].x >> 8u * q, factor[buffer][i].y >> 8u * q);
    };
    // the matrix instructions of step c, `ops` other operations among them from the first on
    const auto multiply = [&](auto step, uint32_t buffer, auto ops, auto op) MX_INLINE {
        constexpr uint32_t kC = decltype(step)::value, kOps = decltype(ops)::value, kAll = kTM * kTN;
        constexpr uint32_t kPer = (kOps + kAll - 1u) / kAll;
        constexpr int kByte = kMF == 32u ? 2 * (kC & 1u) : 0;
        constexpr bool kSecond = 2u * kC >= S::kSteps;  // of the stage's two scale words
#pragma unroll
        for (uint32_t m = 0; m < kAll; ++m) {
            const uint32_t j = m / kTM, i = m % kTM;
            const uint2 fa = factor[buffer][i], fb = factor[buffer][kTM + j];
            acc[j][i] = mfma_mx<kByte>(part[kC % 2u][kTM + j], kSecond ? fb.y : fb.x, part[kC % 2u][i],
                                       kSecond ? fa.y : fa.x, acc[j][i]);
#pragma unroll
            for (uint32_t o = m * kPer; o < (m + 1u) * kPer && o < kOps; ++o) op(o);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    constexpr uint32_t kEarly = (kDataLoads + 1u) / 2u;  // data loads in the step behind the barrier, the rest a step later

    // A stage in kSteps steps, software pipelined: a step's fragments are read while the
    // step in front of it is multiplied.  In front of the last step the workgroup meets:
    // the next stage has come and this one is read, so its slot takes the kStages-th
    // after it.  kWide: even and odd stages take turns, their scales in two buffers.
    const auto stage = [&](auto odd_stage, bool half) MX_INLINE {
        constexpr uint32_t kParity = kWide ? decltype(odd_stage)::value : 0u;
        constexpr bool kScalesNow = !kWide || (kParity + S::kStages) % 2u == 0u;
        // loads of the kStages - 2 stages behind the next; kWide: at least half of them, rounded down, bring scales
        constexpr uint32_t kLater = S::kStages - 2u;
        constexpr uint32_t kBusy = kDataEach * kLater + (kWide ? kLater / 2u : kLater) * kScaleEach;
        const auto step = [&](auto c) MX_INLINE {
            constexpr uint32_t kC = decltype(c)::value;
            constexpr uint32_t kLoads = kC == 0u ? kDataLoads - kEarly : 0u;
            multiply(c, kParity, std::integral_constant<uint32_t, kReads + kLoads>{}, [&](uint32_t o) MX_INLINE {
                if (o < kReads) read(kC + 1u, o, half);
                else load_data(kEarly + o - kReads);
            });
            if constexpr (kC == 0u) load_next(!kWide || (kParity + S::kStages) % 2u == 0u);
        };
        step(std::integral_constant<uint32_t, 0>{});
        if constexpr (S::kSteps > 2u) {
            step(std::integral_constant<uint32_t, 1>{});
            step(std::integral_constant<uint32_t, 2>{});
        }
        if (data_rest) mx_barrier<kBusy + (kDataRest != 0u ? kLater : 0u)>();
        else mx_barrier<kBusy>();
        take_turn();
        slot = slot + 1u == S::kStages ? 0u : slot + 1u;
        if (!kWide || kParity == 1u) scales = scales + 1u == kScaleSlots ? 0u : scales + 1u;
        constexpr uint32_t kScaleOps = kScalesNow ? kScaleLoads : 0u, kLoads = kScaleOps + kEarly;
        multiply(std::integral_constant<uint32_t, S::kSteps - 1u>{}, kParity,
                 std::integral_constant<uint32_t, 3u * kReads + kLoads>{}, [&](uint32_t o) MX_INLINE {
                     if (o < kReads) read_factor(1u - kParity, 1u - kParity, o);
                     else if (o < 2u * kReads) read(0u, o - kReads, false);
                     else if (o < 2u * kReads + kScaleOps) load_scale(o - 2u * kReads);
                     else if (o < 2u * kReads + kLoads) load_data(o - 2u * kReads - kScaleOps);
                     else shift_factor(1u - kParity, o - 2u * kReads - kLoads);
                 });
        if constexpr (!kWide) {
#pragma unroll
            for (uint32_t i = 0; i < kReads; ++i) factor[0][i] = factor[1][i];
        }
    };

    // ---- C: a lane has four consecutive columns of a row, 16 bytes of fp32; in bf16 it
    // trades one of two such groups with the lane that has the columns beside the other's,
    // which gives both of them 16 bytes.  (Through strips of LDS, 64 bytes of a row at a
    // time: 8 us a 256 x 256 tile, of 26.) ----
    const auto store = [&](uint32_t t, auto* c) MX_INLINE {
        using T = std::remove_pointer_t<decltype(c)>;
        constexpr uint32_t kSize = sizeof(T), kOut = kSwiglu ? kTN / 2u : kTN;  // tiles across
        constexpr uint32_t kFours = kOut * kAcc / 4u;                           // a lane's groups of four
        const uint32_t own_lane = fresh_lane(), n = own_lane % kMF, q = own_lane / kMF;
        const uint32_t first_row = __builtin_amdgcn_readlane(known_first, t % 64u);
        const uint32_t count = __builtin_amdgcn_readlane(known_count, t % 64u);
        const uint32_t first_column = __builtin_amdgcn_readlane(known_column, t % 64u) * kColumns + wn * kOut * kMF;
#pragma unroll
        for (uint32_t i = 0; i < kTM; ++i) {
            const uint32_t m = (wm * kTM + i) * kMF + n;
            if ((wm * kTM + i) * kMF >= count) break;
            T* row = c + (static_cast<uint64_t>(first_row) + m) * p.c_stride;
            const auto put = [&](const auto& words, uint32_t column) MX_INLINE {
                constexpr uint32_t kEach = sizeof(words) / kSize;
                if (m >= count || column >= n_out) return;
                T* to = row + column;
                if (column + kEach <= n_out) {
                    using At = std::conditional_t<sizeof(words) == 16u, v4u_any, v2u_any>;
                    *reinterpret_cast<At*>(to) = words;
                    return;
                }
#pragma unroll
                for (uint32_t e = 0; e < kEach; ++e) {
                    if (column + e >= n_out) break;
                    const uint32_t word = words[e * kSize / 4u];
                    if constexpr (kSize == 4u) to[e] = __uint_as_float(word);
                    else to[e] = static_cast<uint16_t>(word >> (e % 2u * 16u));
                }
            };
            const auto four = [&](uint32_t f, float* v) MX_INLINE {
                const uint32_t j = f / (kAcc / 4u), g = f % (kAcc / 4u);
#pragma unroll
                for (uint32_t e = 0; e < 4u; ++e) {
                    v[e] = acc[j][i][4u * g + e];
                    if constexpr (kSwiglu) v[e] = swiglu<kSize == 4u>(v[e], acc[j + kOut][i][4u * g + e]);
                }
            };
            // the columns of group f start at kGap f + 4 q of the wave's
            constexpr uint32_t kGap = kMF == 32u ? 8u : 16u;
            if constexpr (kSize == 4u) {
#pragma unroll
                for (uint32_t f = 0; f < kFours; ++f) {
                    float v[4];
                    four(f, v);
                    put(v4u{__float_as_uint(v[0]), __float_as_uint(v[1]), __float_as_uint(v[2]), __float_as_uint(v[3])},
                        first_column + kGap * f + 4u * q);
                }
            } else if constexpr (kFours == 1u) {
                float v[4];
                four(0u, v);
                put(v2u{f32_to_bf16(v[0]) | f32_to_bf16(v[1]) << 16, f32_to_bf16(v[2]) | f32_to_bf16(v[3]) << 16},
                    first_column + 4u * q);
            } else {
#pragma unroll
                for (uint32_t f = 0; f < kFours; f += 2u) {
                    float v[4], w[4];
                    four(f, v);
                    four(f + 1u, w);
                    uint32_t d[4] = {f32_to_bf16(v[0]) | f32_to_bf16(v[1]) << 16, f32_to_bf16(v[2]) | f32_to_bf16(v[3]) << 16,
                                     f32_to_bf16(w[0]) | f32_to_bf16(w[1]) << 16, f32_to_bf16(w[2]) | f32_to_bf16(w[3]) << 16};
                    if constexpr (kMF == 32u) {  // q = 1 of the first group with q = 0 of the second
                        const auto low = __builtin_amdgcn_permlane32_swap(d[0], d[2], false, false);
                        const auto high = __builtin_amdgcn_permlane32_swap(d[1], d[3], false, false);
                        put(v4u{low[0], high[0], low[1], high[1]}, first_column + kGap * (f + q));
                    } else {  // odd q of the first group with the q below of the second
                        const auto low = __builtin_amdgcn_permlane16_swap(d[0], d[2], false, false);
                        const auto high = __builtin_amdgcn_permlane16_swap(d[1], d[3], false, false);
                        put(v4u{low[0], high[0], low[1], high[1]}, first_column + kGap * (f + q % 2u) + 4u * (q & 2u));
                    }
                }
            }
        }
    };

    // all stages that the ring holds under way, but for the last one's later loads
#pragma unroll
    for (uint32_t s = 0; s < S::kStages; ++s) {
        if (!kWide || s % 2u == 0u)
#pragma unroll
            for (uint32_t t = 0; t < kScaleLoads; ++t) load_scale(t);
#pragma unroll
        for (uint32_t t = 0; t < (s + 1u < S::kStages ? kDataLoads : kEarly); ++t) load_data(t);
        // the ring of pairs moves on behind a pair's second stage
        if (s + 1u < S::kStages) {
            load_next(!kWide || s % 2u == 1u);
            take_turn();
        }
    }
    constexpr uint32_t kFirst = kDataEach * (S::kStages - 2u) + (kEarly < kDataEach ? kEarly : kDataEach) +
                                (kWide ? (S::kStages - 1u) / 2u : S::kStages - 1u) * kScaleEach;
    mx_barrier<kFirst>();
#pragma unroll
    for (uint32_t i = 0; i < kReads; ++i) {
        read(0u, i, false);
        read_factor(0u, 0u, i);
    }
#pragma unroll
    for (uint32_t i = 0; i < kReads; ++i) shift_factor(0u, i);
    for (uint32_t t = 0;; ++t) {
        if constexpr (kWide) {
            for (uint32_t s = 0; s < stages; s += 2u) {
                stage(std::integral_constant<uint32_t, 0>{}, false);
                stage(std::integral_constant<uint32_t, 1>{}, false);
            }
        } else {
            for (uint32_t s = 0; s < stages; ++s)
                stage(std::integral_constant<uint32_t, 0>{}, odd && s + 1u == stages);
        }
        if (p.c_f32) store(t, p.c_f32);
        else store(t, p.c_bf16);
        if (t + 1u == order.count) break;
#pragma unroll
        for (uint32_t j = 0; j < kTN; ++j)
#pragma unroll
            for (uint32_t i = 0; i < kTM; ++i) acc[j][i] = Acc{};
    }
    mx_barrier<0>();  // no load is under way to LDS that the next workgroup gets
}

}  // namespace

hipError_t launch_mx_quantize(const void* x, uint32_t dtype, uint64_t stride, uint32_t rows,
                              uint32_t columns, void* codes, void* scales, void* rounded,
                              hipStream_t stream) {
    uint32_t lanes = 4;
    while (lanes < 8u && (8u << lanes) < columns) ++lanes;
    const uint32_t per = kQuantThreads >> lanes, grid = (rows + per - 1u) / per;
    if (dtype == Q38M_DTYPE_F32)
        mx_quantize_kernel<float><<<grid, kQuantThreads, 0, stream>>>(
            static_cast<const float*>(x), stride, rows, columns, lanes, static_cast<uint32_t*>(codes),
            static_cast<uint32_t*>(scales), static_cast<float*>(rounded));
    else
        mx_quantize_kernel<uint16_t><<<grid, kQuantThreads, 0, stream>>>(
            static_cast<const uint16_t*>(x), stride, rows, columns, lanes, static_cast<uint32_t*>(codes),
            static_cast<uint32_t*>(scales), static_cast<uint16_t*>(rounded));
    return hipGetLastError();
}

namespace {

MxSizes sizes_of(const MxProduct& p, bool swiglu) {
    return MxSizes{p.routes, p.n, p.k128, p.offsets ? p.experts : 0u, swiglu,
                   mx_wide(p.k128, reinterpret_cast<uintptr_t>(p.a_scales), reinterpret_cast<uintptr_t>(p.b_scales))};
}

template <typename S, bool kExperts, bool kSwiglu>
hipError_t launch_tiles(const MxProduct& p, const MxSizes& sizes, hipStream_t stream) {
    const auto launch = [&](auto wide, auto streamed) {
        mx_tile_kernel<S, kExperts, kSwiglu, decltype(wide)::value, decltype(streamed)::value>
            <<<mx_grid<S>(sizes), 64u * S::kWaves, 0, stream>>>(p);
    };
    if constexpr (kExperts && S::kBM <= 32u) {
        if (mx_streams<S>(sizes)) {
            launch(std::true_type{}, std::true_type{});
            return hipGetLastError();
        }
    }
    if constexpr (!std::is_same_v<S, Mx256x256>) {
        if (!sizes.wide) {
            launch(std::false_type{}, std::false_type{});
            return hipGetLastError();
        }
    }
    launch(std::true_type{}, std::false_type{});
    return hipGetLastError();
}

}  // namespace

bool mx_product_fits(const MxProduct& p, bool swiglu) {
    // tiles and their places are 32-bit numbers, and so are a tile's offsets: rows of C and
    // of an expert, a row's bytes (a tile's 256 rows of them below 2^32) and, gathered, all
    // of A's
    const uint64_t row_bytes = static_cast<uint64_t>(p.k128) * 64u;
    const uint64_t b_rows = swiglu ? p.n : 256u, a_rows = p.packed ? p.a_rows : 256u;
    return p.n <= (1u << 28) && p.routes <= (1u << 28) && b_rows * row_bytes < (1ull << 32) &&
           a_rows * row_bytes < (1ull << 32) &&
           with_mx_tiles(sizes_of(p, swiglu), [&](auto s) {
               return mx_tiles<decltype(s)>(sizes_of(p, swiglu)) < (1ull << 31);
           });
}

hipError_t launch_mx_product(const MxProduct& p, bool swiglu, hipStream_t stream) {
    const MxSizes sizes = sizes_of(p, swiglu);
    return with_mx_tiles(sizes, [&](auto s) {
        using S = decltype(s);
        if (!p.offsets) return launch_tiles<S, false, false>(p, sizes, stream);
        return swiglu ? launch_tiles<S, true, true>(p, sizes, stream)
                      : launch_tiles<S, true, false>(p, sizes, stream);
    });
}

}  // namespace q38m
