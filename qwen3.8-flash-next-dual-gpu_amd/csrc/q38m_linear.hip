// bf16 products with epilogues and their gradients, dense and by expert: bias,
// activation and residual, or the activation's derivative and residual, or the
// SwiGLU fold or its derivative, on the fp32 sums before their one rounding.
//
// Three orders of the operands (LinearOrder): a forward product has K along
// the rows of both as they are stored, the rows' gradient has it across the
// rows of B, the weights' gradient across the rows of both.
#include <type_traits>

#include "q38m_device.h"
#include "q38m_internal.h"
#include "q38m_linear_tiles.h"
#include "q38m_product.h"

namespace q38m {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// f(0) .. f(kCount - 1) with the numbers as constants of the program
template <uint32_t kCount, uint32_t kFirst = 0u, typename F>
__device__ MX_INLINE void each_of(F f) {
    if constexpr (kFirst < kCount) {
        f(std::integral_constant<uint32_t, kFirst>{});
        each_of<kCount, kFirst + 1u>(f);
    }
}

// ---- activations --------------------------------------------------------------

// Phi(-|z|), with a = |z|, t = 1 / (1 + 0.3 a): exp(-a^2 / 2) times a polynomial in t,
// fitted here by least squares over 0 <= a <= 14, weights raised where the relative error
// was largest: with the coefficients as they stand 7.8e-8, at 0, and in fp32 4.9e-7 near 0
// growing with the exponential's argument (6.6e-7 at 3, 1.9e-6 at 6).  `density` gets exp(-a^2 / 2).
__device__ __forceinline__ float normal_tail(float z, float* density) {
    const float a = fminf(__builtin_fabsf(z), 14.0f);
    const float t = __builtin_amdgcn_rcpf(__builtin_fmaf(a, 0.3f, 1.0f));
    const float e = __builtin_amdgcn_exp2f(a * a * -0.72134752044448170368f);
    float p = 0.03837830573320389f;
    p = __builtin_fmaf(p, t, -0.1691661924123764f);
    p = __builtin_fmaf(p, t, 0.2286602407693863f);
    p = __builtin_fmaf(p, t, -0.07650664448738098f);
    p = __builtin_fmaf(p, t, 0.14253564178943634f);
    p = __builtin_fmaf(p, t, 0.09468347579240799f);
    p = __builtin_fmaf(p, t, 0.12192035466432571f);
    p = __builtin_fmaf(p, t, 0.1194876879453659f);
    p = __builtin_fmaf(p, t, 7.168947831814876e-06f);
    *density = e;
    return e * p;
}

// s(t) = 1 / (1 + exp(-t)) and s(t) s(-t), both from e = exp(-|t|), which has nothing to
// cancel: s is r = 1 / (1 + e) or e r, the product e r^2.  The rounding of |t| log2 e is
// put back.
struct Sigmoid {
    float s, both;
    __device__ __forceinline__ explicit Sigmoid(float t) {
        constexpr float kLog2e = 1.44269502162933349609375f;  // and what it lacks of log2 e
        constexpr float kLog2eLow = 1.92596299112661746887e-8f;
        const float a = -fminf(__builtin_fabsf(t), 128.0f), p = a * kLog2e;
        const float low = __builtin_fmaf(a, kLog2eLow, __builtin_fmaf(a, kLog2e, -p));
        float e = __builtin_amdgcn_exp2f(p);
        e = __builtin_fmaf(e * low, 0.693147180559945309f, e);
        const float r = __builtin_amdgcn_rcpf(1.0f + e), below = e * r;
        s = t < 0.0f ? below : r;
        both = below * r;
    }
};

// z, held to where s has long been zero or one, so that nothing overflows on the way; a
// NaN stays one.
__device__ __forceinline__ float held(float z) {
    return z == z ? __builtin_amdgcn_fmed3f(z, -128.0f, 128.0f) : z;
}

// The logistic activations are z or 1 times s(z (c1 + c3 z^2)).
struct Logistic {
    float c1, c3;
    __device__ __forceinline__ explicit Logistic(uint32_t activation)
        : c1(activation == Q38M_ACT_GELU_TANH ? 1.59576912160573071176f : 1.0f),
          c3(activation == Q38M_ACT_GELU_TANH ? 0.07135481282745242f : 0.0f) {}
    __device__ __forceinline__ Sigmoid at(float z) const { return Sigmoid(z * __builtin_fmaf(c3, z * z, c1)); }
    __device__ __forceinline__ float inner(float z) const { return __builtin_fmaf(3.0f * c3, z * z, c1); }
};

// act(z) and act'(z) of kN values; `activation` is the same in all lanes
template <uint32_t kN>
__device__ __forceinline__ void activate(uint32_t activation, float (&v)[kN]) {
    if (activation == Q38M_ACT_NONE) return;
    if (activation == Q38M_ACT_RELU) {
#pragma unroll
        for (uint32_t i = 0; i < kN; ++i) v[i] = v[i] < 0.0f ? 0.0f : v[i];
    } else if (activation == Q38M_ACT_GELU) {
#pragma unroll
        for (uint32_t i = 0; i < kN; ++i) {
            float density;
            const float tail = normal_tail(v[i], &density);
            v[i] *= v[i] < 0.0f ? tail : 1.0f - tail;
        }
    } else {
        const Logistic s(activation);
#pragma unroll
        for (uint32_t i = 0; i < kN; ++i) {
            const float w = held(v[i]), y = s.at(w).s;
            v[i] = activation == Q38M_ACT_SIGMOID ? (w == w ? y : w) : v[i] * y;
        }
    }
}

template <uint32_t kN>
__device__ __forceinline__ void times_slope(uint32_t activation, const float (&z)[kN], float (&v)[kN]) {
    if (activation == Q38M_ACT_NONE) return;
    if (activation == Q38M_ACT_RELU) {
#pragma unroll
        for (uint32_t i = 0; i < kN; ++i) v[i] = z[i] > 0.0f ? v[i] : 0.0f;
    } else if (activation == Q38M_ACT_GELU) {
#pragma unroll
        for (uint32_t i = 0; i < kN; ++i) {
            float density;
            const float tail = normal_tail(z[i], &density);
            const float below = z[i] < 0.0f ? tail : 1.0f - tail;
            v[i] *= __builtin_fmaf(held(z[i]) * 0.39894228040143267794f, density, below);
        }
    } else {
        const Logistic s(activation);
#pragma unroll
        for (uint32_t i = 0; i < kN; ++i) {
            const float w = held(z[i]);
            const Sigmoid y = s.at(w);
            v[i] *= activation == Q38M_ACT_SIGMOID ? (w == w ? y.both : w) : __builtin_fmaf(w * y.both, s.inner(w), y.s);
        }
    }
}

// ---- epilogue -------------------------------------------------------------------

// kN (8, 4 or 1) consecutive elements of a matrix, as they lie there (fp32 in all words,
// bf16 in the first half of them), and as numbers
template <uint32_t kN>
struct Raw {
    uint32_t d[kN];

    __device__ __forceinline__ void load(LinearMatrix m, uint64_t at) {
        if (m.f32) {
            const float* p = static_cast<const float*>(m.data) + at;
            if constexpr (kN == 1u) {
                d[0] = __float_as_uint(*p);
            } else {
#pragma unroll
                for (uint32_t i = 0; i < kN; i += 4u) {
                    const v4u_any w = *reinterpret_cast<const v4u_any*>(p + i);
                    d[i] = w.x, d[i + 1u] = w.y, d[i + 2u] = w.z, d[i + 3u] = w.w;
                }
            }
            return;
        }
        const uint16_t* p = static_cast<const uint16_t*>(m.data) + at;
        if constexpr (kN == 1u) {
            d[0] = *p;
        } else if constexpr (kN == 4u) {
            const v2u_any w = *reinterpret_cast<const v2u_any*>(p);
            d[0] = w.x, d[1] = w.y;
        } else {
            const v4u_any w = *reinterpret_cast<const v4u_any*>(p);
            d[0] = w.x, d[1] = w.y, d[2] = w.z, d[3] = w.w;
        }
    }
    __device__ __forceinline__ void values(LinearMatrix m, float (&v)[kN]) const {
        if (m.f32) {
#pragma unroll
            for (uint32_t i = 0; i < kN; ++i) v[i] = __uint_as_float(d[i]);
            return;
        }
#pragma unroll
        for (uint32_t i = 0; i < kN; ++i)
            v[i] = __uint_as_float(i % 2u != 0u ? d[i / 2u] & 0xffff0000u : d[i / 2u] << 16);
    }
};

template <uint32_t kN>
__device__ __forceinline__ void load_row(LinearMatrix m, uint64_t at, float (&v)[kN]) {
    Raw<kN> raw;
    raw.load(m, at);
    raw.values(m, v);
}

template <uint32_t kN>
__device__ __forceinline__ void store_row(LinearMatrix m, uint64_t at, const float (&v)[kN]) {
    if (m.f32) {
        float* p = static_cast<float*>(m.data) + at;
        if constexpr (kN == 1u) {
            *p = v[0];
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kN; i += 4u)
                *reinterpret_cast<v4u_any*>(p + i) = v4u_any{__float_as_uint(v[i]), __float_as_uint(v[i + 1u]),
                                                             __float_as_uint(v[i + 2u]), __float_as_uint(v[i + 3u])};
        }
        return;
    }
    uint16_t* p = static_cast<uint16_t*>(m.data) + at;
    if constexpr (kN == 1u) {
        *p = static_cast<uint16_t>(f32_to_bf16(v[0]));
    } else {
        uint32_t d[kN / 2u];
#pragma unroll
        for (uint32_t i = 0; i < kN; i += 2u) d[i / 2u] = f32_to_bf16(v[i]) | f32_to_bf16(v[i + 1u]) << 16;
        if constexpr (kN == 8u) *reinterpret_cast<v4u_any*>(p) = v4u_any{d[0], d[1], d[2], d[3]};
        else *reinterpret_cast<v2u_any*>(p) = v2u_any{d[0], d[1]};
    }
}

// A lane's kN consecutive values of a row of C and of what lies beside it, `shift` columns
// on where a fold has two halves.
struct InRow {
    uint64_t row;
    uint32_t column;

    template <uint32_t kN>
    __device__ __forceinline__ void load(LinearMatrix m, uint32_t shift, float (&v)[kN]) const {
        load_row(m, row * m.stride + shift + column, v);
    }
    template <uint32_t kN>
    __device__ __forceinline__ void store(LinearMatrix m, uint32_t shift, const float (&v)[kN]) const {
        store_row(m, row * m.stride + shift + column, v);
    }
    template <uint32_t kN>
    __device__ __forceinline__ void load_bias(LinearMatrix m, float (&v)[kN]) const {
        load_row(m, column, v);
    }
};

// The gradients of gate, dh u (s + g s(g) s(-g)), in place of dh, and of up, dh g s, of up.
template <uint32_t kN>
__device__ __forceinline__ void swiglu_slopes(const float (&gate)[kN], float (&up)[kN], float (&dh)[kN]) {
#pragma unroll
    for (uint32_t i = 0; i < kN; ++i) {
        const Sigmoid y(gate[i]);
        const float of_up = dh[i] * (gate[i] * y.s);
        dh[i] *= __builtin_fmaf(held(gate[i]), y.both, y.s);
        dh[i] *= up[i];
        up[i] = of_up;
    }
}

// The epilogue of a lane's kN sums; n: the columns of C in front of what a fold puts beside
// them; u: the sums of up beside gate's.
template <LinearFold kFold, typename Access, uint32_t kN>
__device__ __forceinline__ void finish_all(LinearEpilogue e, Access at, uint32_t n, float (&v)[kN],
                                           const float (&u)[kN]) {
    if constexpr (kFold == LinearFold::kSwiglu) {  // pre: n columns of gate, then n of up
        if (e.pre.data) {
            at.store(e.pre, 0u, v);
            at.store(e.pre, n, u);
        }
        if (e.c.f32) {
#pragma unroll
            for (uint32_t i = 0; i < kN; ++i) v[i] = swiglu<true>(v[i], u[i]);
        } else {
#pragma unroll
            for (uint32_t i = 0; i < kN; ++i) v[i] = swiglu<false>(v[i], u[i]);
        }
    } else if constexpr (kFold == LinearFold::kSwigluGrad) {
        float gate[kN], up[kN];
        at.load(e.pre, 0u, gate);
        at.load(e.pre, n, up);
        swiglu_slopes(gate, up, v);
        at.store(e.c, n, up);
    } else if constexpr (kFold == LinearFold::kSlope) {
        if (e.activation != Q38M_ACT_NONE) {
            float z[kN];
            at.load(e.pre, 0u, z);
            times_slope(e.activation, z, v);
        }
    } else if constexpr (kFold == LinearFold::kForward) {
        if (e.bias.data) {
            float b[kN];
            at.load_bias(e.bias, b);
#pragma unroll
            for (uint32_t i = 0; i < kN; ++i) v[i] += b[i];
        }
        if (e.pre.data) at.store(e.pre, 0u, v);
        activate(e.activation, v);
    }
    if constexpr (kFold == LinearFold::kForward || kFold == LinearFold::kSlope || kFold == LinearFold::kAdd) {
        if (e.residual.data) {
            float r[kN];
            at.load(e.residual, 0u, r);
#pragma unroll
            for (uint32_t i = 0; i < kN; ++i) v[i] += r[i];
        }
    }
    at.store(e.c, 0u, v);
}

// kN sums of a row, columns from `column` on; those that are below n one by one where not all
// are: the sums move through the first place, so that one copy of the code does for all.
template <LinearFold kFold, uint32_t kN>
__device__ __forceinline__ void finish(LinearEpilogue e, uint64_t row, uint32_t column, uint32_t n,
                                       float (&v)[kN], float (&u)[kN]) {
    if (column + kN <= n) {
        finish_all<kFold>(e, InRow{row, column}, n, v, u);
        return;
    }
#pragma unroll 1
    for (; column < n; ++column) {
        float one[1] = {v[0]}, up[1] = {u[0]};
        finish_all<kFold>(e, InRow{row, column}, n, one, up);
#pragma unroll
        for (uint32_t i = 0; i + 1u < kN; ++i) v[i] = v[i + 1u], u[i] = u[i + 1u];
    }
}

// ---- products of any strides ----------------------------------------------------

// The 8 values p[0] .. p[7], zeros from `live` on.
__device__ __forceinline__ v4u load_eight(const uint16_t* p, int32_t live) {
    if (live >= 8) {
        const v4u_any w = *reinterpret_cast<const v4u_any*>(p);
        return v4u{w.x, w.y, w.z, w.w};
    }
    v4u d{0u, 0u, 0u, 0u};
#pragma unroll
    for (int32_t i = 0; i < 7; ++i)
        if (i < live) d[i / 2] |= static_cast<uint32_t>(p[i]) << i % 2 * 16;
    return d;
}

// A 64 x 64 tile of C (of B's rows 32 gate and 32 up ones with the SwiGLU fold) for each
// workgroup of four waves, 32 x 32 a wave; K through LDS 32 values at a time, by way of
// registers, so that rows may start and end at any element.  For operands whose rows do
// not start at 16 bytes.
constexpr uint32_t kAnyTile = 64, kAnyK = 32, kAnyPitch = 40;

template <LinearOrder kOrder, bool kExperts, LinearFold kFold>
__global__ __launch_bounds__(256) void linear_any_kernel(LinearProduct p) {
    constexpr bool kAcrossA = kOrder == LinearOrder::kTN, kAcrossB = kOrder != LinearOrder::kNT;
    constexpr uint32_t kAcross = kFold == LinearFold::kSwiglu ? kAnyTile / 2u : kAnyTile;
    __shared__ __align__(16) uint16_t lds[2][kAnyTile * kAnyPitch];
    __shared__ v4i offset_words[kExperts && !kAcrossA ? kMaxSortExperts / 4u : 1u];
    const uint32_t t = threadIdx.x, lane = t & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(t >> 6);
    const uint32_t n_out = kFold == LinearFold::kSwiglu ? p.columns / 2u : p.columns;
    const uint32_t columns = (n_out + kAcross - 1u) / kAcross;
    const uint32_t row_tile = blockIdx.x / columns, column0 = blockIdx.x % columns * kAcross;

    // this tile's expert, its rows of C and its part of K
    RowTile tile{0u, 0u, 0u, false};
    uint32_t k_first = 0, depth = p.depth;
    if constexpr (kExperts && kAcrossA) {
        const uint32_t tiles = (p.rows + kAnyTile - 1u) / kAnyTile;
        tile.expert = row_tile / tiles;
        tile.first = row_tile % tiles * kAnyTile;
        tile.count = min(p.rows - tile.first, kAnyTile);
        k_first = min(p.offsets[tile.expert], p.depth);
        depth = max(min(p.offsets[tile.expert + 1u], p.depth), k_first) - k_first;
    } else if constexpr (kExperts) {
        uint32_t* offsets = reinterpret_cast<uint32_t*>(offset_words);
        const uint32_t last = p.offsets[p.experts];
        for (uint32_t e = t; e < kMaxSortExperts; e += 256u) offsets[e] = e < p.experts ? p.offsets[e] : last;
        __syncthreads();
        const TileList<kAnyTile> list(offset_words, last, p.rows);
        if (row_tile >= list.total) return;
        tile = list.find(row_tile);
    } else {
        tile.first = row_tile * kAnyTile;
        tile.count = min(p.rows - tile.first, kAnyTile);
    }

    // each thread's piece of eight values: along K, row t / 4 and piece t % 4; across K,
    // stored row t / 8 and columns from 8 (t % 8) on
    const auto source = [&](uint32_t place) -> uint32_t {
        if (!p.packed) return place;
        const uint32_t row = p.packed[place] / p.top_k;
        report(row >= p.source_rows, kCheckToken);
        return min(row, p.source_rows - 1u);
    };
#ifdef Q38M_CHECKED
    if constexpr (kExperts)
        for (uint32_t e = blockIdx.x * 256u + t; e < p.experts; e += gridDim.x * 256u)
            report(p.offsets[e + 1u] < p.offsets[e] || p.offsets[e + 1u] > (kAcrossA ? p.depth : p.rows), kCheckOffsets);
#endif
    const uint32_t r = t / 4u;
    const uint16_t *a_from, *b_from;
    int32_t a_live = 0, b_live = 0;  // across K: columns there
    if constexpr (kAcrossA) {
        a_from = p.a + tile.first + 8u * (t % 8u);
        a_live = static_cast<int32_t>(tile.count) - 8 * static_cast<int32_t>(t % 8u);
    } else {
        const uint32_t place = tile.first + min(r, tile.count - 1u);
        a_from = p.a + static_cast<uint64_t>(kExperts ? source(place) : place) * p.a_stride + 8u * (t % 4u);
    }
    const uint64_t b_first = kAcrossA ? 0u : static_cast<uint64_t>(tile.expert) * (kAcrossB ? p.depth : p.columns);
    if constexpr (kAcrossB) {
        b_from = p.b + b_first * p.b_stride + column0 + 8u * (t % 8u);
        b_live = static_cast<int32_t>(min(p.columns - column0, kAnyTile)) - 8 * static_cast<int32_t>(t % 8u);
    } else {
        uint32_t column = r, up = 0;
        if constexpr (kFold == LinearFold::kSwiglu) {  // a wave's tiles: one gate, one up
            column = r / 32u * 16u + r % 16u;
            up = r / 16u % 2u * n_out;
        }
        column = min(column0 + column, n_out - 1u) + up;
        b_from = p.b + (b_first + column) * p.b_stride + 8u * (t % 4u);
    }
    const auto load = [&](uint32_t k0, v4u* d) {
        const int32_t left = static_cast<int32_t>(depth - k0) - 8 * static_cast<int32_t>(t % 4u);
        const uint32_t k = k0 + t / 8u;
        const uint64_t at = static_cast<uint64_t>(k_first) + k;
        if constexpr (kAcrossA) d[0] = load_eight(a_from + at * p.a_stride, k < depth ? a_live : 0);
        else d[0] = load_eight(a_from + k0, left);
        if constexpr (!kAcrossB) d[1] = load_eight(b_from + k0, left);
        else if constexpr (kExperts && kAcrossA)
            d[1] = k < depth ? load_eight(b_from + source(static_cast<uint32_t>(at)) * p.b_stride, b_live) : v4u{};
        else d[1] = load_eight(b_from + at * p.b_stride, k < depth ? b_live : 0);
    };
    const auto stage = [&](bool across, uint16_t* to, v4u d) {
        if (!across) {
            *reinterpret_cast<v4u*>(to + r * kAnyPitch + 8u * (t % 4u)) = d;
            return;
        }
#pragma unroll
        for (uint32_t i = 0; i < 8u; ++i)
            to[(8u * (t % 8u) + i) * kAnyPitch + t / 8u] = static_cast<uint16_t>(d[i / 2u] >> i % 2u * 16u);
    };

    v4f acc[2][2] = {};
    const uint32_t wm = wave / 2u, wn = wave % 2u, n = lane % 16u, q = lane / 16u;
    v4u d[2];
    if (depth != 0u) load(0u, d);
    for (uint32_t k0 = 0; k0 < depth; k0 += kAnyK) {
        stage(kAcrossA, lds[0], d[0]);
        stage(kAcrossB, lds[1], d[1]);
        __syncthreads();
        if (k0 + kAnyK < depth) load(k0 + kAnyK, d);
        bf16x8 a[2], b[2];
#pragma unroll
        for (uint32_t i = 0; i < 2u; ++i) {
            a[i] = *reinterpret_cast<const bf16x8*>(lds[0] + (wm * 32u + i * 16u + n) * kAnyPitch + 8u * q);
            b[i] = *reinterpret_cast<const bf16x8*>(lds[1] + (wn * 32u + i * 16u + n) * kAnyPitch + 8u * q);
        }
#pragma unroll
        for (uint32_t j = 0; j < 2u; ++j)
#pragma unroll
            for (uint32_t i = 0; i < 2u; ++i)
                acc[j][i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(b[j], a[i], acc[j][i], 0, 0, 0);
        __syncthreads();
    }

    // a lane has four consecutive columns of a row
#pragma unroll
    for (uint32_t i = 0; i < 2u; ++i) {
        const uint32_t m = wm * 32u + i * 16u + n;
        if (m >= tile.count) continue;
        const uint64_t row = (kExperts && kAcrossA ? static_cast<uint64_t>(tile.expert) * p.rows : 0u) + tile.first + m;
#pragma unroll
        for (uint32_t j = 0; j < (kFold == LinearFold::kSwiglu ? 1u : 2u); ++j) {
            const uint32_t column = column0 + (kFold == LinearFold::kSwiglu ? wn * 16u : wn * 32u + j * 16u) + 4u * q;
            if (column >= n_out) continue;
            float v[4] = {acc[j][i][0], acc[j][i][1], acc[j][i][2], acc[j][i][3]};
            float u[4] = {acc[1][i][0], acc[1][i][1], acc[1][i][2], acc[1][i][3]};
            finish<kFold>(p.e, row, column, n_out, v, u);
        }
    }
}

// ---- products of rows at 16 bytes -------------------------------------------------

typedef short v4s __attribute__((ext_vector_type(4)));
constexpr int kVmcnt0 = 0x0f70;  // a wait for all of a wave's loads and stores

// v_mfma_f32_32x32x16_bf16: lane l holds k = 8 (l / 32) .. + 7 of row l % 32 of A and of B;
// D lane l: rows 8 (i / 4) + 4 (l / 32) + i % 4 of A, row l % 32 of B.
// v_mfma_f32_16x16x32_bf16: k = 8 (l / 16) .. + 7 of row l % 16; D lane l: rows 4 (l / 16)
// + i of A, row l % 16 of B.
__device__ __forceinline__ v4f mfma_bf16(v4i a, v4i b, v4f c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ v16f mfma_bf16(v4i a, v4i b, v16f c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// The block of LDS that holds an operand's 64 values of K for kWidth rows of C (columns of
// C): 128 bytes for each of them.
//
// Along K (as stored): a row's 64 values are eight 16-byte pieces, at positions p ^ (r / 2
// % 8), so that the lanes of a read, one piece of 16 or 32 consecutive rows, spread over
// all 64 banks.
//
// Across K: a stored row has kWidth values of one k, in units of 32 bytes.  A transposing
// read (ds_read_b64_tr_b16) takes for 16 lanes four k by 16 columns, one unit of each k:
// lane i gives the address of a quarter (i % 4) of k i / 4's unit and gets column i's four
// values.  The units of k lie at positions u ^ x(k), where x differs between the eight k
// whose units 32 lanes read together.
template <bool kAcross, uint32_t kWidth>
struct Block {
    static constexpr uint32_t kUnits = kWidth / 16u;
    static constexpr uint32_t kRowLanes = kWidth / 8u;  // 16-byte pieces of a stored row across K
    static_assert(!kAcross || kWidth >= 64u, "a load instruction brings whole stored rows");

    // the stored row (across K: the k) and 16-byte piece of it of load instruction i's lane
    __device__ MX_INLINE static uint32_t row(uint32_t i, uint32_t lane) {
        if constexpr (kAcross) return i * (64u / kRowLanes) + lane / kRowLanes;
        else return 8u * i + (lane >> 3);
    }
    __device__ MX_INLINE static uint32_t piece(uint32_t i, uint32_t lane) {
        if constexpr (kAcross) return (lane % kRowLanes) ^ (flip(row(i, lane)) << 1);
        else return (lane & 7u) ^ (row(i, lane) >> 1 & 7u);
    }
    __device__ MX_INLINE static uint32_t flip(uint32_t k) {
        if constexpr (kUnits >= 8u) return (k & 3u) << 1 | (k >> 3 & 1u);
        else return k & 2u | (k >> 3 & 1u);
    }
};

// Transposes four registers over four lanes: lane i's register k becomes lane k's register i.
__device__ MX_INLINE v4u transpose_quad(v4u r, uint32_t lane) {
    const bool odd = (lane & 1u) != 0u, high = (lane & 2u) != 0u;
    const uint32_t a = __builtin_amdgcn_mov_dpp(odd ? r.x : r.y, 0xb1, 0xf, 0xf, true);  // of lane ^ 1
    const uint32_t b = __builtin_amdgcn_mov_dpp(odd ? r.z : r.w, 0xb1, 0xf, 0xf, true);
    r = odd ? v4u{a, r.y, b, r.w} : v4u{r.x, a, r.z, b};
    const uint32_t c = __builtin_amdgcn_mov_dpp(high ? r.x : r.z, 0x4e, 0xf, 0xf, true);  // of lane ^ 2
    const uint32_t d = __builtin_amdgcn_mov_dpp(high ? r.y : r.w, 0x4e, 0xf, 0xf, true);
    return high ? v4u{c, d, r.z, r.w} : v4u{r.x, r.y, c, d};
}

// 64 columns of the 32 rows that two of a wave's 32 x 32 tiles side by side have: lane l has of row
// n = l % 32 the columns 16 k + 8 q .. + 7, q = l / 32, k = 0 .. 3.  Memory is read and written in
// whole lines: four lanes' pieces of 16 bytes change places, so that a lane has its neighbours'
// rows in turn and a piece of each, and eight lanes a line.  Each lane its own row's pieces, 32
// bytes of a line at a time, past the caches or not: 16,384 tokens' gate/up weight gradient in
// fp32 2,650 us, in whole lines 2,270, past the caches too 2,090 (1,959 with what came later);
// part lines past the caches cost the rows' products more than a fifth.
//
// kPast: past the caches (linear_past).
template <bool kPast>
struct Span {
    uint64_t row;           // of C: the tile's first
    uint32_t first, count;  // the lane's row of the tile, the tile's rows
    uint32_t column;        // the span's first
    uint32_t lane;

    __device__ MX_INLINE uint64_t place(LinearMatrix m, uint32_t r) const {
        return (row + min(r, count - 1u)) * m.stride + column;
    }
    // the pieces of row first / 4 * 4 + k: bf16 columns 16 (n % 4) + 8 q, fp32 columns 32 half + 8 (n % 4) + 4 q
    __device__ MX_INLINE uint32_t row_of(uint32_t k) const { return (first & ~3u) + k; }
    __device__ MX_INLINE uint32_t column_of() const { return 16u * (lane & 3u) + lane / 32u * 8u; }
    __device__ MX_INLINE uint32_t wide_column_of() const { return 8u * (lane & 3u) + lane / 32u * 4u; }

    __device__ MX_INLINE float* wide_piece(LinearMatrix m, uint32_t half, uint32_t k) const {
        return static_cast<float*>(m.data) + place(m, row_of(k)) + 32u * half + wide_column_of();
    }
    __device__ MX_INLINE uint16_t* piece(LinearMatrix m, uint32_t k) const {
        return static_cast<uint16_t*>(m.data) + place(m, row_of(k)) + column_of();
    }
    static __device__ MX_INLINE void put(v4u_any v, void* to) {
        if constexpr (kPast) __builtin_nontemporal_store(v, static_cast<v4u_any*>(to));
        else *static_cast<v4u_any*>(to) = v;
    }
    static __device__ MX_INLINE v4u_any get(const void* from) {
        if constexpr (kPast) return __builtin_nontemporal_load(static_cast<const v4u_any*>(from));
        else return *static_cast<const v4u_any*>(from);
    }

    __device__ MX_INLINE void store(LinearMatrix m, const float (&v)[32]) const {
        v4u d[4];
        if (m.f32) {
            each_of<2>([&](auto hc) MX_INLINE {
                constexpr uint32_t half = decltype(hc)::value;
                each_of<8>([&](auto c) MX_INLINE {
                    constexpr uint32_t k = decltype(c)::value / 4u, e = decltype(c)::value % 4u;
                    const auto both = __builtin_amdgcn_permlane32_swap(__float_as_uint(v[16u * half + 8u * k + e]),
                                                                       __float_as_uint(v[16u * half + 8u * k + 4u + e]), false, false);
                    d[e][2u * k] = both[0];
                    d[e][2u * k + 1u] = both[1];
                });
                each_of<4>([&](auto e) MX_INLINE { d[decltype(e)::value] = transpose_quad(d[decltype(e)::value], lane); });
                each_of<4>([&](auto kc) MX_INLINE {
                    constexpr uint32_t k = decltype(kc)::value;
                    if (row_of(k) >= count) return;
                    put(v4u_any{d[0][k], d[1][k], d[2][k], d[3][k]}, wide_piece(m, half, k));
                });
            });
            return;
        }
        each_of<16>([&](auto c) MX_INLINE {
            constexpr uint32_t k = decltype(c)::value / 4u, e = decltype(c)::value % 4u;
            d[e][k] = f32_to_bf16(v[8u * k + 2u * e]) | f32_to_bf16(v[8u * k + 2u * e + 1u]) << 16;
        });
        each_of<4>([&](auto e) MX_INLINE { d[decltype(e)::value] = transpose_quad(d[decltype(e)::value], lane); });
        each_of<4>([&](auto kc) MX_INLINE {
            constexpr uint32_t k = decltype(kc)::value;
            if (row_of(k) >= count) return;
            put(v4u_any{d[0][k], d[1][k], d[2][k], d[3][k]}, piece(m, k));
        });
    }

    // m's values, added to the lane's groups of four that the sums are stored from: group 2 k + c has
    // columns 16 k + 8 c + 4 q of its row.
    template <typename F>
    __device__ MX_INLINE void read(LinearMatrix m, F add) const {
        v4u d[4];  // [e][k]: dword e of piece k
        const auto load = [&](auto piece_of) MX_INLINE {
            each_of<4>([&](auto kc) MX_INLINE {
                constexpr uint32_t k = decltype(kc)::value;
                const v4u_any w = get(piece_of(k));
                d[0][k] = w.x, d[1][k] = w.y, d[2][k] = w.z, d[3][k] = w.w;
            });
            each_of<4>([&](auto e) MX_INLINE { d[decltype(e)::value] = transpose_quad(d[decltype(e)::value], lane); });
        };
        if (m.f32) {
            each_of<2>([&](auto hc) MX_INLINE {
                constexpr uint32_t half = decltype(hc)::value;
                load([&](uint32_t k) MX_INLINE { return wide_piece(m, half, k); });
                each_of<16>([&](auto c) MX_INLINE {
                    constexpr uint32_t k = decltype(c)::value / 4u, e = decltype(c)::value % 4u;
                    add(std::integral_constant<uint32_t, 4u * half + k>{}, std::integral_constant<uint32_t, e>{},
                        __uint_as_float(d[e][k]));
                });
            });
            return;
        }
        load([&](uint32_t k) MX_INLINE { return piece(m, k); });
        each_of<8>([&](auto c) MX_INLINE {  // eight columns of a row a lane to four of both of its groups
            constexpr uint32_t k = decltype(c)::value / 2u, e = decltype(c)::value % 2u;
            const auto both = __builtin_amdgcn_permlane32_swap(d[e][k], d[2u + e][k], false, false);
            each_of<2>([&](auto gc) MX_INLINE {
                const std::integral_constant<uint32_t, 2u * k + decltype(gc)::value> group;
                add(group, std::integral_constant<uint32_t, 2u * e>{}, __uint_as_float(both[decltype(gc)::value] << 16));
                add(group, std::integral_constant<uint32_t, 2u * e + 1u>{}, __uint_as_float(both[decltype(gc)::value] & 0xffff0000u));
            });
        });
    }
};

// Workgroups stay and compute tile after tile of kBM x kBN values of C (with the SwiGLU fold
// half of the columns gate, half up), kWM x kWN waves, each kTM x kTN matrix-instruction
// tiles of kMF rows.  K goes through LDS in stages of 64 values, in a ring of kStages slots,
// loaded straight from memory; the stages of a tile follow those of the tile before without
// a gap.
//
// What bounds it, by counters:
// - large products (8,192^3 819 us without an epilogue, 1,343 TFLOP/s; across K of one or both
//   operands 818 and 798): the card's clock, 1.7 GHz of 2.4 under this load, and matrix pipes busy
//   for 59 to 68 % of it, the L1s' answers under way for 25 to 45 %; no LDS conflicts.
//   128 x 128 tiles move twice as much through LDS for the same products (with GELU 1,159 us, 942).
// - many experts' products with much to store (gate/up of 32,768 tokens 1,600 us, 859 TFLOP/s of
//   rows that are there): row tiles that an expert's last rows fill partly, a sixth of the products,
//   and the stores, during which this workgroup multiplies nothing: a second set of sums does not fit
//   the registers.
// - experts of few rows (512 tokens 355 us, 6.1 TB/s) and weights' gradients in fp32 (16,384 tokens'
//   gate/up 1,960 to 2,120 us, 4.5 to 4.9 TB/s read and written): memory.
// - few tiles (509 x 2,048 x 8,192 31 us and a join of 4): one stage's latency after another, so K
//   is cut until the card is full, and the parts' sums are joined by a second launch in their order.
template <typename S, LinearOrder kOrder, bool kExperts, LinearFold kFold, bool kPast>
__global__ __launch_bounds__(64u * S::kWaves, (S::kResident * S::kWaves + 3u) / 4u) void linear_tile_kernel(
    LinearProduct p, uint32_t each) {
    constexpr uint32_t kMF = S::kMF, kTM = S::kTM, kTN = S::kTN, kBM = S::kBM, kBN = S::kBN;
    constexpr bool kAcrossA = kOrder == LinearOrder::kTN, kAcrossB = kOrder != LinearOrder::kNT;
    constexpr bool kSwiglu = kFold == LinearFold::kSwiglu;
    constexpr bool kRagged = kExperts && kAcrossA;   // K is the expert's rows
    constexpr bool kListed = kExperts && !kAcrossA;  // rows of C are
    static_assert(!kSwiglu || kTN % 2u == 0u, "a wave's tiles: half of them gate, half up");
    using A = Block<kAcrossA, kBM>;
    using B = Block<kAcrossB, kBN>;
    using Acc = std::conditional_t<kMF == 32u, v16f, v4f>;
    constexpr uint32_t kAcc = kMF == 32u ? 16u : 4u;
    __shared__ v4i ring[kExperts ? S::kLds : S::kOffsetsAt];
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    __builtin_assume(wave < S::kWaves);  // settles at compile time which loads are of A and which of B
    const uint32_t n_out = kSwiglu ? p.columns / 2u : p.columns;
    constexpr uint32_t kColumns = kSwiglu ? kBN / 2u : kBN;
    const uint32_t columns = (n_out + kColumns - 1u) / kColumns;

    // ---- this workgroup's tiles ----
    uint32_t* offsets = reinterpret_cast<uint32_t*>(ring + S::kOffsetsAt);
    const uint32_t last_offset = kExperts ? p.offsets[p.experts] : 0u;
    const uint32_t routes = kRagged ? p.depth : p.rows;
    if constexpr (kExperts) {
        for (uint32_t e = threadIdx.x; e < kMaxSortExperts; e += 64u * S::kWaves)
            offsets[e] = e < p.experts ? p.offsets[e] : last_offset;
        __syncthreads();
#ifdef Q38M_CHECKED
        for (uint32_t e = threadIdx.x; e < p.experts; e += 64u * S::kWaves) {
            const uint32_t end = p.offsets[e + 1u];
            report(end < offsets[e] || end > routes, kCheckOffsets);
        }
        if (p.packed)  // each workgroup looks at a part of the sources
            for (uint32_t i = offsets[0] + blockIdx.x * 64u * S::kWaves + threadIdx.x; i < min(last_offset, routes);
                 i += gridDim.x * 64u * S::kWaves)
                report(p.packed[i] / p.top_k >= p.source_rows, kCheckToken);
#endif
    }
    // K that is ragged: an expert's rows are one "row tile" of the list
    const auto make_list = [&]() MX_INLINE {
        if constexpr (kExperts) return TileList<kRagged ? 1u << 24 : kBM>(ring + S::kOffsetsAt, last_offset, routes);
        else return 0;
    };
    const auto list = make_list();
    const uint32_t of_rows = (p.rows + kBM - 1u) / kBM;  // row tiles of a matrix C
    const auto row_tiles = [&]() MX_INLINE {
        if constexpr (kRagged) return list.total * of_rows;
        else if constexpr (kExperts) return list.total;
        else return of_rows * ((p.depth + each - 1u) / each);
    };
    if constexpr (kRagged) {
        // experts without rows: zeros, and what they are added to, unless that is there already
        if (p.e.residual.data != p.e.c.data) {
            // The threads of all workgroups go round these experts' pieces of eight values; 64 experts are
            // looked at in one, and no piece's place is divided out (bf16 gradients of 512 experts, 61
            // tokens: 221 us, 168 of them for the experts that have rows; one expert after another, with
            // a division a piece, 300).
            const uint32_t pieces = (n_out + 7u) / 8u, threads = gridDim.x * 64u * S::kWaves;
            const uint32_t start = blockIdx.x * 64u * S::kWaves + threadIdx.x;
            const uint32_t step_rows = threads / pieces, step_pieces = threads % pieces;
            uint32_t row = start / pieces, piece = start % pieces;
            for (uint32_t e0 = 0; e0 < p.experts; e0 += 64u) {
                const uint32_t own = e0 + lane;  // offsets has kMaxSortExperts, a multiple of 64
                const uint32_t begin = offsets[own], end = own + 1u < kMaxSortExperts ? offsets[own + 1u] : last_offset;
                uint64_t empty = __ballot(own < p.experts && min(end, routes) <= min(begin, routes));
                for (; empty != 0u; empty &= empty - 1u) {
                    const uint64_t first = static_cast<uint64_t>(e0 + __builtin_ctzll(empty)) * p.rows;
                    while (row < p.rows) {
                        float v[8] = {}, u[8] = {};
                        finish<kFold>(p.e, first + row, piece * 8u, n_out, v, u);
                        row += step_rows;
                        piece += step_pieces;
                        if (piece >= pieces) piece -= pieces, ++row;
                    }
                    row -= p.rows;
                }
            }
        }
    }
    MxOrder order(row_tiles(), columns);
    if (order.count == 0u) return;
    // what is known of the tiles being loaded: lane t % 64 holds the t-th
    uint32_t known_first = 0, known_column = 0, known_depth = 0;
    [[maybe_unused]] uint32_t known_count = 0, known_matrix = 0;

    // ---- loads: instructions dealt to the waves, the left over ones to the first: 1 KB of
    // data each.  Those of A first, then of B, each instruction of one of them: a base of its
    // tile and stage for all lanes and an offset below 4 GB for each ----
    constexpr uint32_t kDataA = kBM / 8u, kData = S::kRows / 8u;
    constexpr uint32_t kDataEach = kData / S::kWaves, kDataRest = kData % S::kWaves;
    constexpr uint32_t kDataLoads = kDataEach + (kDataRest != 0u ? 1u : 0u);
    const bool data_rest = kDataRest != 0u && wave < kDataRest;
    const auto data_live = [&](uint32_t t) MX_INLINE { return kDataRest == 0u || t < kDataEach || data_rest; };
    const auto of_a = [&](uint32_t t) MX_INLINE { return t * S::kWaves < kDataA && wave + t * S::kWaves < kDataA; };
    const uint32_t a_bytes = static_cast<uint32_t>(p.a_stride) * 2u, b_bytes = static_cast<uint32_t>(p.b_stride) * 2u;
    const uint64_t a_step = kAcrossA ? 64ull * a_bytes : 128u, b_step = kAcrossB ? 64ull * b_bytes : 128u;
    const uint8_t* a_all = reinterpret_cast<const uint8_t*>(p.a);
    const uint8_t* b_all = reinterpret_cast<const uint8_t*>(p.b);
    const bool gather = kExperts && kOrder != LinearOrder::kNN && p.packed;
    const uint8_t *a_base, *b_base;  // of the stage being loaded
    uint32_t data[kDataLoads];
    // the next tile to load, the `found`-th from one on, looked up a tile ahead, so that nobody
    // waits; with the sources of its rows of A where they are gathered
    uint32_t found = 0, next_column = 0, next_from = 0, next_depth = 0;
    RowTile next{0u, 0u, 0u, false};
    uint32_t source[kDataLoads];
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
        next_from = 0u;
        next_depth = p.depth;
        uint32_t matrix = 0;
        if constexpr (kRagged) {
            const RowTile all = list.find(row / of_rows);
            next = RowTile{all.expert, row % of_rows * kBM, 0u, false};
            next.count = min(p.rows - next.first, kBM);
            next_from = all.first;
            next_depth = all.count;
            matrix = all.expert;
        } else if constexpr (kExperts) {
            next = list.find(row);
        } else {
            matrix = row / of_rows;  // the part of K, whose sums are a matrix of their own
            next = RowTile{0u, row % of_rows * kBM, 0u, false};
            next.count = min(p.rows - next.first, kBM);
            next_from = matrix * each;
            next_depth = min(p.depth - next_from, each);
        }
        if (own_lane == found % 64u) {
            known_first = next.first;
            if constexpr (kListed) known_count = next.count;
            else known_matrix = matrix;
            known_column = next_column;
            known_depth = next_depth;
        }
        ++found;
        if constexpr (kExperts && !kAcrossB) {
            if (!p.packed) return;
#pragma unroll
            for (uint32_t t = 0; t < kDataLoads; ++t)
                if (data_live(t) && of_a(t))
                    source[t] = p.packed[next.first + min(A::row(wave + t * S::kWaves, own_lane), next.count - 1u)];
        }
    };
    uint32_t from = 0, stages = 0, depth = 0, k_from = 0;  // of the tile being loaded: the stage, and its K
    // points the loads at the tile that was looked up, and looks up the one after it
    uint32_t a_last = 0, b_last = 0;  // across K: the last piece that is there of a stored row
    const auto point = [&]() MX_INLINE {
        const uint32_t own_lane = fresh_lane();
        depth = next_depth;
        stages = (depth + 63u) / 64u;
        k_from = next_from;
        if constexpr (kAcrossA) {
            a_base = a_all + static_cast<uint64_t>(next_from) * a_bytes + 2ull * next.first;
        } else {
            a_base = a_all + (gather ? 0ull : static_cast<uint64_t>(next.first) * a_bytes) + 2ull * next_from;
        }
        const uint64_t b_first = kRagged ? (gather ? 0u : next_from)
                                 : kExperts ? static_cast<uint64_t>(next.expert) * (kAcrossB ? p.depth : p.columns)
                                            : (kAcrossB ? next_from : 0u);
        b_base = b_all + (b_first + (kAcrossB ? 0u : next_column * kColumns)) * b_bytes +
                 2ull * (kAcrossB ? next_column * kColumns : next_from);
        a_base = mx_uniform(a_base);
        b_base = mx_uniform(b_base);
        a_last = (next.count - 1u) / 8u;
        b_last = (min(p.columns - next_column * kColumns, kBN) - 1u) / 8u;
#pragma unroll
        for (uint32_t t = 0; t < kDataLoads; ++t) {
            if (!data_live(t)) continue;
            const uint32_t i = wave + t * S::kWaves;
            if (of_a(t)) {
                const uint32_t r = A::row(i, own_lane), piece = A::piece(i, own_lane);
                if constexpr (kAcrossA) data[t] = r * a_bytes + 16u * min(piece, a_last);
                else data[t] = (gather ? min(source[t] / p.top_k, p.source_rows - 1u) : min(r, next.count - 1u)) * a_bytes + 16u * piece;
            } else {
                const uint32_t r = B::row(i - kDataA, own_lane), piece = B::piece(i - kDataA, own_lane);
                if constexpr (kAcrossB) {
                    data[t] = r * b_bytes + 16u * min(piece, b_last);
                } else {
                    uint32_t column = r, up = 0;
                    if constexpr (kSwiglu) {  // a wave's tiles: half of them gate, half up
                        const uint32_t tile = r / kMF % kTN;
                        column = r / (kTN * kMF) * (kTN / 2u * kMF) + tile % (kTN / 2u) * kMF + r % kMF;
                        up = tile >= kTN / 2u ? n_out : 0u;
                    }
                    data[t] = (min(column, n_out - 1u - next_column * kColumns) + up) * b_bytes + 16u * piece;
                }
            }
        }
        look_up();
    };
    // gathered stored rows along K: the stage's sources, looked up a stage ahead
    const auto look_ahead = [&](uint32_t first, uint32_t stage, uint32_t count) MX_INLINE {
        const uint32_t own_lane = fresh_lane();
#pragma unroll
        for (uint32_t t = 0; t < kDataLoads; ++t) {
            const uint32_t i = wave + t * S::kWaves;
            if (data_live(t) && !of_a(t))
                source[t] = p.packed[first + min(stage * 64u + B::row(i - kDataA, own_lane), count - 1u)];
        }
    };
    const auto take_sources = [&]() MX_INLINE {
        const uint32_t own_lane = fresh_lane();
#pragma unroll
        for (uint32_t t = 0; t < kDataLoads; ++t) {
            const uint32_t i = wave + t * S::kWaves;
            if (data_live(t) && !of_a(t))
                data[t] = min(source[t] / p.top_k, p.source_rows - 1u) * b_bytes + 16u * min(B::piece(i - kDataA, own_lane), b_last);
        }
        if (from + 1u < stages) look_ahead(k_from, from + 1u, depth);
        else look_ahead(next_from, 0u, next_depth);
    };
    // a tile's last stage where K ends inside it: what lies behind is another piece, or row, of it
    const auto hold_back = [&]() MX_INLINE {
        const uint32_t valid = depth - from * 64u;
        if (valid >= 64u) return;
        const uint32_t own_lane = fresh_lane();
#pragma unroll
        for (uint32_t t = 0; t < kDataLoads; ++t) {
            if (!data_live(t)) continue;
            const uint32_t i = wave + t * S::kWaves;
            const auto behind = [&](uint32_t at, uint32_t last) MX_INLINE { return at > last ? at - last : 0u; };
            if (of_a(t)) {
                if constexpr (kAcrossA) data[t] -= behind(A::row(i, own_lane), valid - 1u) * a_bytes;
                else data[t] -= behind(A::piece(i, own_lane), (valid - 1u) / 8u) * 16u;
            } else if constexpr (kAcrossB) {
                if (!(kRagged && gather)) data[t] -= behind(B::row(i - kDataA, own_lane), valid - 1u) * b_bytes;
            } else {
                data[t] -= behind(B::piece(i - kDataA, own_lane), (valid - 1u) / 8u) * 16u;
            }
        }
    };
    look_up();
    uint32_t tiles_left = order.count;  // with the one being loaded
    uint32_t moved = 0u;  // what the next loads are for: 1, the next stage; 2, the next tile; 0, the same stage
    point();
    if constexpr (kRagged) {
        if (gather) {
            look_ahead(k_from, 0u, depth);
            take_sources();
        }
    }
    if (stages == 1u) hold_back();
    uint32_t to = 0;  // the slot that is loaded
    const uint32_t ring_at = static_cast<uint32_t>(
        reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) v4i*)ring));
    const auto load_data = [&](uint32_t t) MX_INLINE {
        if (!data_live(t)) return;
        const uint32_t i = wave + t * S::kWaves;
        const uint32_t at = __builtin_amdgcn_readfirstlane(ring_at + to * (S::kSlot * 16u) + i * 1024u);
        mx_load16(of_a(t) ? a_base : b_base, data[t], at);
    };
    // to the next stage to load; past the last tile the last stage again, into slots that nobody
    // reads any more, so that the count of loads under way is always the same
    const auto load_next = [&]() MX_INLINE {
        to = to + 1u == S::kStages ? 0u : to + 1u;
        const bool within = from + 1u < stages;
        moved = within ? 1u : tiles_left != 1u ? 2u : 0u;
        if (!within) return;
        ++from;
        a_base += a_step;
        if (!(kRagged && gather)) b_base += b_step;
    };
    // what the next stage's loads need, behind the barrier in front of them
    const auto take_turn = [&]() MX_INLINE {
        if (moved == 2u) {
            --tiles_left;
            from = 0;
            point();
        }
        if constexpr (kRagged) {
            if (gather) take_sources();
        }
        if (moved != 0u && from + 1u == stages) hold_back();
    };

    // ---- products ----
    const uint32_t wm = wave / S::kWN, wn = wave % S::kWN;
    const uint32_t n = lane % kMF, q = lane / kMF;
    Acc acc[kTN][kTM];
    constexpr uint32_t kOut = kSwiglu ? kTN / 2u : kTN;  // column tiles of C
    constexpr uint32_t kGap = kMF == 32u ? 8u : 16u;     // the columns of a lane's group f of four: from kGap f + 4 q on
    const auto first_row = [&](uint32_t t) MX_INLINE {
        const uint32_t first = __builtin_amdgcn_readlane(known_first, t % 64u);
        if constexpr (kListed) return static_cast<uint64_t>(first);
        else return static_cast<uint64_t>(__builtin_amdgcn_readlane(known_matrix, t % 64u)) * p.rows + first;
    };
    const auto count_of = [&](uint32_t t) MX_INLINE -> uint32_t {
        if constexpr (kListed) return __builtin_amdgcn_readlane(known_count, t % 64u);
        else return min(p.rows - __builtin_amdgcn_readlane(known_first, t % 64u), kBM);
    };
    const auto first_column = [&](uint32_t t) MX_INLINE {
        return __builtin_amdgcn_readlane(known_column, t % 64u) * kColumns + wn * kOut * kMF;
    };
    // Sums that are stored as they are go to memory in whole lines.  With the other folds the
    // exchange between lanes costs what it gives (in half lines, for want of registers: gate/up of
    // 32,768 tokens 1,594 us and so 1,647, down's row gradient of 16,384 763 and 884).
    constexpr bool kSpans = kMF == 32u && kOut % 2u == 0u && (kFold == LinearFold::kStore || kFold == LinearFold::kAdd);
    [[maybe_unused]] const auto span = [&](uint32_t t, uint32_t i, uint32_t place) MX_INLINE {
        const uint32_t own_lane = fresh_lane();
        return Span<kPast>{first_row(t), (wm * kTM + i) * kMF + (own_lane & 31u), count_of(t), first_column(t) + 64u * place, own_lane};
    };
    const auto begin = [&]() MX_INLINE {
#pragma unroll
        for (uint32_t j = 0; j < kTN; ++j)
#pragma unroll
            for (uint32_t i = 0; i < kTM; ++i) acc[j][i] = Acc{};
    };
    constexpr uint32_t kReads = kTM + kTN;
    // where a lane's fragments start in a slot, bytes
    uint32_t part_at[kReads];
#pragma unroll
    for (uint32_t i = 0; i < kReads; ++i) {
        const uint32_t tile = i < kTM ? wm * kTM + i : wn * kTN + i - kTM;
        const uint32_t block = i < kTM ? 0u : kBM * 128u;
        const bool across = i < kTM ? kAcrossA : kAcrossB;
        const uint32_t width = i < kTM ? kBM : kBN;
        if (across) {
            const uint32_t k = 8u * q + lane % 16u / 4u, unit = tile * (kMF / 16u) + lane % kMF / 16u;
            const uint32_t flip = i < kTM ? A::flip(k) : B::flip(k);
            part_at[i] = block + k * 2u * width + (unit ^ flip) * 32u + lane % 4u * 8u;
        } else {
            part_at[i] = block + (tile * kMF + n) * 128u;
        }
    }
    const uint32_t swizzle = n >> 1 & 7u;  // along K, as of every kMF-th row after it
    v4i part[2][kReads];  // a step's fragments of A, then of B, and the next step's
    uint32_t slot = 0;    // of the stage whose fragments are read
    auto* lds = (__attribute__((address_space(3))) char*)ring;
    const auto read = [&](uint32_t c, uint32_t i) MX_INLINE {
        const uint32_t at = slot * (S::kSlot * 16u) + part_at[i];
        if (i < kTM ? kAcrossA : kAcrossB) {
            const uint32_t row = (i < kTM ? kBM : kBN) * 2u;
            const v4s low = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) v4s*)(lds + at + 512u / kMF * c * row));
            const v4s high = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
                (__attribute__((address_space(3))) v4s*)(lds + at + (512u / kMF * c + 4u) * row));
            const v2u a = __builtin_bit_cast(v2u, low), b = __builtin_bit_cast(v2u, high);
            part[c % 2u][i] = v4i{static_cast<int>(a.x), static_cast<int>(a.y), static_cast<int>(b.x), static_cast<int>(b.y)};
        } else {
            part[c % 2u][i] = *(__attribute__((address_space(3))) v4i*)(lds + at + ((64u / kMF * c + q) ^ swizzle) * 16u);
        }
    };
    // zeros behind the `valid` values of K of the stage in this slot, of both operands: what
    // was loaded there may be anything, NaN too
    const auto clear = [&](uint32_t valid) MX_INLINE {
        const uint32_t first = slot * S::kSlot;
        const auto part_of = [&](uint32_t w, bool across, uint32_t width, uint32_t block) MX_INLINE {
            const uint32_t at = first + block + w;
            if (across) {
                if (w / (width / 8u) >= valid) ring[at] = v4i{0, 0, 0, 0};
                return;
            }
            const uint32_t row = w / 8u, k = 8u * ((w & 7u) ^ (row >> 1 & 7u));
            if (k >= valid) {
                ring[at] = v4i{0, 0, 0, 0};
            } else if (k + 8u > valid) {
                v4i v = ring[at];
#pragma unroll
                for (uint32_t e = 0; e < 4u; ++e) {
                    if (k + 2u * e >= valid) v[e] = 0;
                    else if (k + 2u * e + 1u >= valid) v[e] &= 0xffff;
                }
                ring[at] = v;
            }
        };
#pragma unroll 1
        for (uint32_t w = threadIdx.x; w < kBM * 8u; w += 64u * S::kWaves) part_of(w, kAcrossA, kBM, 0u);
#pragma unroll 1
        for (uint32_t w = threadIdx.x; w < kBN * 8u; w += 64u * S::kWaves) part_of(w, kAcrossB, kBN, kBM * 8u);
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
    };
    // the matrix instructions of step c, `ops` other operations among them from the first on
    const auto multiply = [&](auto step, auto ops, auto op) MX_INLINE {
        constexpr uint32_t kC = decltype(step)::value, kOps = decltype(ops)::value, kAll = kTM * kTN;
        constexpr uint32_t kPer = (kOps + kAll - 1u) / kAll;
#pragma unroll
        for (uint32_t m = 0; m < kAll; ++m) {
            const uint32_t j = m / kTM, i = m % kTM;
            acc[j][i] = mfma_bf16(part[kC % 2u][kTM + j], part[kC % 2u][i], acc[j][i]);
#pragma unroll
            for (uint32_t o = m * kPer; o < (m + 1u) * kPer && o < kOps; ++o) op(o);
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    constexpr uint32_t kEarly = (kDataLoads + 1u) / 2u;  // data loads in the step behind the barrier, the rest a step later

    // A stage in kSteps steps, software pipelined: a step's fragments are read while the step in
    // front of it is multiplied.  In front of the last step the workgroup meets: the next stage
    // (`valid` values of K) has come and this one is read, so its slot takes the kStages-th after it.
    const auto stage = [&](uint32_t valid) MX_INLINE {
        constexpr uint32_t kLater = S::kStages - 2u;  // loads of the stages behind the next may be under way
        const auto step = [&](auto c) MX_INLINE {
            constexpr uint32_t kC = decltype(c)::value;
            constexpr uint32_t kLoads = kC == 0u ? kDataLoads - kEarly : 0u;
            multiply(c, std::integral_constant<uint32_t, kReads + kLoads>{}, [&](uint32_t o) MX_INLINE {
                if (o < kReads) read(kC + 1u, o);
                else load_data(kEarly + o - kReads);
            });
            if constexpr (kC == 0u) load_next();
        };
        step(std::integral_constant<uint32_t, 0>{});
        if constexpr (S::kSteps > 2u) {
            step(std::integral_constant<uint32_t, 1>{});
            step(std::integral_constant<uint32_t, 2>{});
        }
        if (data_rest) mx_barrier<(kDataEach + (kDataRest != 0u ? 1u : 0u)) * kLater>();
        else mx_barrier<kDataEach * kLater>();
        take_turn();
        slot = slot + 1u == S::kStages ? 0u : slot + 1u;
        if (valid < 64u) clear(valid);
        multiply(std::integral_constant<uint32_t, S::kSteps - 1u>{}, std::integral_constant<uint32_t, kReads + kEarly>{},
                 [&](uint32_t o) MX_INLINE {
                     if (o < kReads) read(0u, o);
                     else load_data(o - kReads);
                 });
    };

    // ---- C: a lane has four consecutive columns of a row and trades one of two such groups with
    // the lane that has the columns beside the other's, which gives both of them eight ----
    const auto store = [&](uint32_t t) MX_INLINE {
        using None = std::integral_constant<uint32_t, 0u>;
        constexpr uint32_t kFours = kOut * kAcc / 4u;  // a lane's groups of four
        constexpr uint32_t kN = kFours == 1u ? 4u : 8u;
        const uint32_t own_lane = fresh_lane(), n = own_lane % kMF, q = own_lane / kMF;
        const uint32_t count = count_of(t);
        const uint64_t row0 = first_row(t);
        const uint32_t column0 = first_column(t);
        // A residual is added to all of a wave's sums in front of their stores.  (A span's values where its
        // stores have them, a kernel for each pair of types, which kept none or 5 to 20 registers in memory:
        // gate/up weights of 16,384 tokens added up in fp32 1,930 us, so 1,959, but memory that is read and
        // written by turns costs a short batch's: 61 x 8,192 x 2,048 29.4, so 26.2.)
        constexpr uint32_t kPlaces = kOut / 2u;
        if constexpr (kSpans && kFold == LinearFold::kAdd) {
            if (column0 + 32u * kOut <= n_out && p.e.residual.data)
                each_of<kTM * kPlaces>([&](auto sc) MX_INLINE {
                    constexpr uint32_t i = decltype(sc)::value / kPlaces, place = decltype(sc)::value % kPlaces;
                    if ((wm * kTM + i) * kMF >= count) return;
                    span(t, i, place).read(p.e.residual, [&](auto fc, auto ec, float v) MX_INLINE {
                        constexpr uint32_t f = 8u * place + decltype(fc)::value;
                        acc[f / 4u][i][4u * (f % 4u) + decltype(ec)::value] += v;
                    });
                    if constexpr (S::kWaves == 8u) __builtin_amdgcn_sched_barrier(0);
                });
        }
        each_of<kTM>([&](auto ic) MX_INLINE {
            constexpr uint32_t i = decltype(ic)::value;
            const uint32_t m = (wm * kTM + i) * kMF + n;
            if ((wm * kTM + i) * kMF >= count) return;
            asm volatile("" ::: "memory");  // a row's bias is not kept for the next one
            const auto values = [&](auto fc, auto shift, auto& v, auto at) MX_INLINE {
                constexpr uint32_t f = decltype(fc)::value, kShift = decltype(shift)::value, kAt = decltype(at)::value;
                constexpr uint32_t kEach = kAcc / 4u;
                each_of<4>([&](auto ec) MX_INLINE {
                    constexpr uint32_t e = decltype(ec)::value;
                    if constexpr (kN == 4u) {
                        v[kAt + e] = acc[f / kEach + kShift][i][4u * (f % kEach) + e];
                    } else {
                        const uint32_t a = __float_as_uint(acc[f / kEach + kShift][i][4u * (f % kEach) + e]);
                        const uint32_t b = __float_as_uint(acc[(f + 1u) / kEach + kShift][i][4u * ((f + 1u) % kEach) + e]);
                        const auto both = [&]() MX_INLINE {
                            if constexpr (kMF == 32u) return __builtin_amdgcn_permlane32_swap(a, b, false, false);
                            else return __builtin_amdgcn_permlane16_swap(a, b, false, false);
                        }();
                        v[kAt + e] = __uint_as_float(both[0]);
                        v[kAt + 4u + e] = __uint_as_float(both[1]);
                    }
                });
            };
            using Up = std::integral_constant<uint32_t, kSwiglu ? kOut : 0u>;
            if constexpr (kSpans) {
                if (column0 + 32u * kOut <= n_out) {
                    each_of<kPlaces>([&](auto pc) MX_INLINE {
                        constexpr uint32_t place = decltype(pc)::value;
                        float v[32];
                        each_of<4>([&](auto kc) MX_INLINE {
                            constexpr uint32_t k = decltype(kc)::value;
                            using Group = std::integral_constant<uint32_t, 2u * (4u * place + k)>;
                            using At = std::integral_constant<uint32_t, 8u * k>;
                            values(Group{}, None{}, v, At{});
                        });
                        span(t, i, place).store(p.e.c, v);
                        if constexpr (S::kWaves == 8u) __builtin_amdgcn_sched_barrier(0);
                    });
                    return;
                }
            }
            const auto column_of = [&](uint32_t f) MX_INLINE {
                return column0 + (kN == 4u ? 4u * q : kMF == 32u ? kGap * (f + q) : kGap * (f + q % 2u) + 4u * (q & 2u));
            };
            // what the SwiGLU's derivative reads of a row, under way together: gate's, then up's
            constexpr uint32_t kGroups = kFours * 4u / kN;
            constexpr bool kBeside = kFold == LinearFold::kSwigluGrad && kN == 8u;
            [[maybe_unused]] Raw<kN> beside[kBeside ? 2u * kGroups : 1u];
            if constexpr (kBeside) {
                if (n_out >= kN) {
                    const uint64_t at = (row0 + min(m, count - 1u)) * p.e.pre.stride;
                    each_of<kGroups>([&](auto gc) MX_INLINE {
                        constexpr uint32_t g = decltype(gc)::value;
                        const uint32_t column = min(column_of(g * (kN / 4u)), n_out - kN);
                        beside[g].load(p.e.pre, at + column);
                        beside[kGroups + g].load(p.e.pre, at + n_out + column);
                    });
                }
            }
            each_of<kGroups>([&](auto gc) MX_INLINE {
                constexpr uint32_t f = decltype(gc)::value * (kN / 4u);
                const uint32_t column = column_of(f);
                float v[kN], u[kN] = {};
                values(std::integral_constant<uint32_t, f>{}, None{}, v, None{});
                if constexpr (kSwiglu) values(std::integral_constant<uint32_t, f>{}, Up{}, u, None{});
                if constexpr (kBeside) {
                    if (column + kN <= n_out) {
                        float gate[kN];
                        beside[decltype(gc)::value].values(p.e.pre, gate);
                        beside[kGroups + decltype(gc)::value].values(p.e.pre, u);
                        swiglu_slopes(gate, u, v);
                        if (m < count) {
                            const InRow at{row0 + m, column};
                            at.store(p.e.c, n_out, u);
                            at.store(p.e.c, 0u, v);
                        }
                        return;
                    }
                }
                if (m < count && column < n_out) finish<kFold>(p.e, row0 + m, column, n_out, v, u);
                if constexpr (S::kWaves == 8u) __builtin_amdgcn_sched_barrier(0);
            });
        });
        // The compiler cannot tell that a load under a condition is used under the same one, and
        // would wait for it in the next tile's stages: it is told here that none is under way.
        if constexpr (kFold != LinearFold::kStore && kFold != LinearFold::kSwiglu) __builtin_amdgcn_s_waitcnt(kVmcnt0);
    };

    // all stages that the ring holds under way, but for the last one's later loads
#pragma unroll
    for (uint32_t s = 0; s < S::kStages; ++s) {
#pragma unroll
        for (uint32_t t = 0; t < (s + 1u < S::kStages ? kDataLoads : kEarly); ++t) load_data(t);
        if (s + 1u < S::kStages) {
            load_next();
            take_turn();
        }
    }
    // the first stage has come when no more than the others' loads are under way
    constexpr uint32_t kFirst = kDataEach * (S::kStages - 2u) + (kEarly < kDataEach ? kEarly : kDataEach);
    mx_barrier<kFirst>();
    const auto depth_of = [&](uint32_t t) MX_INLINE -> uint32_t {
        return __builtin_amdgcn_readlane(known_depth, t % 64u);
    };
    uint32_t left = depth_of(0u);  // values of K of the tile that are not multiplied yet
    if (left < 64u) clear(left);
#pragma unroll
    for (uint32_t i = 0; i < kReads; ++i) read(0u, i);
    begin();
    for (uint32_t t = 0;; ++t) {
        const uint32_t after = t + 1u == order.count ? 64u : depth_of(t + 1u);
        for (; left > 64u; left -= 64u) stage(left - 64u);
        stage(after);
        store(t);
        if (t + 1u == order.count) break;
        left = after;
        begin();
    }
    mx_barrier<0>();  // no load is under way to LDS that the next workgroup gets
}

// Few rows (generated tokens, experts of a few rows): a workgroup has 16 rows of C by 16 or 32
// columns (with the SwiGLU fold 16 of gate and 16 of up), and its waves a part of K each, whose
// sums meet in LDS in the waves' order.  A wave streams its part through a ring of its own, 64
// values of K of all rows at a time, and waits for no other, so a CU has the bytes of many stages
// under way from its first clocks on; what bounds it is a launch, the first answers from memory
// and, of larger matrices, memory's rate (1 x 8,192 x 2,048 5.1 us, 6.6 TB/s of weights that the
// caches behind the L2s hold; on 16 x 128 tiles with K in four parts and their join 9.9).
template <typename S, bool kExperts, LinearFold kFold>
__global__ __launch_bounds__(64u * S::kWaves) void linear_few_kernel(LinearProduct p) {
    constexpr bool kSwiglu = kFold == LinearFold::kSwiglu;
    constexpr uint32_t kFewRows = S::kRows, kFewWaves = S::kWaves, kFewStages = S::kStages, kTiles = S::kTiles;
    static_assert(!kSwiglu || kTiles == 2u, "a tile of gate, one of up");
    constexpr uint32_t kRowsB = 16u * kTiles, kRows = kFewRows + kRowsB, kSlot = kRows * 8u;  // 16-byte words
    constexpr uint32_t kAcross = kSwiglu ? kRowsB / 2u : kRowsB;
    __shared__ v4i ring[kFewWaves * kFewStages * kSlot];
    __shared__ v4i offset_words[kExperts ? kMaxSortExperts / 4u : 1u];
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t n_out = kSwiglu ? p.columns / 2u : p.columns;
    const uint32_t columns = (n_out + kAcross - 1u) / kAcross;
    const uint32_t row_tile = blockIdx.x / columns, column0 = blockIdx.x % columns * kAcross;
    RowTile tile{0u, row_tile * kFewRows, 0u, false};
    if constexpr (kExperts) {
        uint32_t* offsets = reinterpret_cast<uint32_t*>(offset_words);
        const uint32_t last = p.offsets[p.experts];
        for (uint32_t e = threadIdx.x; e < kMaxSortExperts; e += 64u * kFewWaves) offsets[e] = e < p.experts ? p.offsets[e] : last;
        __syncthreads();
#ifdef Q38M_CHECKED
        for (uint32_t e = threadIdx.x; e < p.experts; e += 64u * kFewWaves)
            report(p.offsets[e + 1u] < offsets[e] || p.offsets[e + 1u] > p.rows, kCheckOffsets);
#endif
        const TileList<kFewRows> list(offset_words, last, p.rows);
        if (row_tile >= list.total) return;
        tile = list.find(row_tile);
    } else {
        tile.count = min(p.rows - tile.first, kFewRows);
    }
    const bool all_rows = tile.count > 8u;  // else the second eight rows of A are not loaded, and their sums not stored

    // this wave's stages, and its loads: two of A (one), four of B, eight rows each
    const uint32_t stages = (p.depth + 63u) / 64u;
    const uint32_t first = wave * stages / kFewWaves, end = (wave + 1u) * stages / kFewWaves;
    const uint32_t a_bytes = static_cast<uint32_t>(p.a_stride) * 2u, b_bytes = static_cast<uint32_t>(p.b_stride) * 2u;
    const bool gather = kExperts && p.packed;
    const uint8_t* a_base = reinterpret_cast<const uint8_t*>(p.a) + (gather ? 0ull : static_cast<uint64_t>(tile.first) * a_bytes);
    const uint8_t* b_base = reinterpret_cast<const uint8_t*>(p.b) +
                            (static_cast<uint64_t>(tile.expert) * p.columns + column0) * b_bytes;
    a_base = mx_uniform(a_base);
    b_base = mx_uniform(b_base);
    constexpr uint32_t kLoads = kRows / 8u;
    uint32_t data[kLoads];
    each_of<kLoads>([&](auto tc) MX_INLINE {
        constexpr uint32_t t = decltype(tc)::value;
        const uint32_t r = 8u * t + (lane >> 3), piece = (lane & 7u) ^ (r >> 1 & 7u);
        if constexpr (t < kFewRows / 8u) {
            uint32_t row = min(r, tile.count - 1u);
            if (gather) {
                row = p.packed[tile.first + row] / p.top_k;
                report(row >= p.source_rows, kCheckToken);
                row = min(row, p.source_rows - 1u);
            }
            data[t] = row * a_bytes + 16u * piece;
        } else {
            uint32_t column = r - kFewRows, up = 0;
            if constexpr (kSwiglu) {  // 16 of gate, 16 of up
                up = column / 16u * n_out;
                column %= 16u;
            }
            data[t] = (min(column, n_out - 1u - column0) + up) * b_bytes + 16u * piece;
        }
    });
    const uint32_t ring_at = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(
        reinterpret_cast<uintptr_t>((__attribute__((address_space(3))) v4i*)ring)) + wave * (kFewStages * kSlot * 16u));
    const auto load = [&](uint32_t s, uint32_t slot) MX_INLINE {
        const uint32_t valid = p.depth - s * 64u;
        const uint64_t shift = s * 128ull;
        each_of<kLoads>([&](auto tc) MX_INLINE {
            constexpr uint32_t t = decltype(tc)::value;
            if (t == 1u && !all_rows) return;
            uint32_t at = data[t];
            if (valid < 64u) {  // a piece behind K is another of the row
                const uint32_t piece = (lane & 7u) ^ ((8u * t + (lane >> 3)) >> 1 & 7u), last = (valid - 1u) / 8u;
                at -= piece > last ? (piece - last) * 16u : 0u;
            }
            mx_load16((t < kFewRows / 8u ? a_base : b_base) + shift, at, ring_at + slot * (kSlot * 16u) + t * 1024u);
        });
    };
    v4f acc[kTiles] = {};
    const uint32_t n = lane % 16u, q = lane / 16u, swizzle = n >> 1 & 7u;
    const uint32_t count = end - first;
    each_of<kFewStages - 1u>([&](auto s) MX_INLINE {
        if (decltype(s)::value < count) load(first + decltype(s)::value, decltype(s)::value);
    });
    uint32_t slot = 0;
    for (uint32_t s = 0; s < count; ++s) {
        // The stages behind this one may be under way.  The slot that is loaded held the stage in front of
        // this one, whose fragments have been read: the wait at the end of its turn says so.
        if (s + kFewStages - 1u < count) {
            load(first + s + kFewStages - 1u, slot == 0u ? kFewStages - 1u : slot - 1u);
            if (all_rows) asm volatile("s_waitcnt vmcnt(%0)" ::"i"((kFewStages - 1u) * kLoads) : "memory");
            else asm volatile("s_waitcnt vmcnt(%0)" ::"i"((kFewStages - 1u) * (kLoads - 1u)) : "memory");
        } else {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        }
        v4i* at = ring + (wave * kFewStages + slot) * kSlot;
        const uint32_t valid = p.depth - (first + s) * 64u;
        if (valid < 64u) {  // zeros behind K, of both operands
            for (uint32_t w = lane; w < kSlot; w += 64u) {
                const uint32_t k = 8u * ((w & 7u) ^ (w >> 4 & 7u));
                if (k + 8u <= valid) continue;
                v4i v = k >= valid ? v4i{0, 0, 0, 0} : at[w];
#pragma unroll
                for (uint32_t e = 0; e < 4u; ++e) {
                    if (k + 2u * e >= valid) v[e] = 0;
                    else if (k + 2u * e + 1u >= valid) v[e] &= 0xffff;
                }
                at[w] = v;
            }
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
        }
#pragma unroll
        for (uint32_t c = 0; c < 2u; ++c) {
            const uint32_t piece = (4u * c + q) ^ swizzle;
            const v4i a = at[n * 8u + piece];
            each_of<kTiles>([&](auto jc) MX_INLINE {
                constexpr uint32_t j = decltype(jc)::value;
                acc[j] = mfma_bf16(at[(kFewRows + 16u * j + n) * 8u + piece], a, acc[j]);
            });
        }
        asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");  // the next turn loads its slot anew
        slot = slot + 1u == kFewStages ? 0u : slot + 1u;
    }
    __syncthreads();
    v4f* sums = reinterpret_cast<v4f*>(ring);
    each_of<kTiles>([&](auto j) MX_INLINE { sums[(wave * kTiles + decltype(j)::value) * 64u + lane] = acc[decltype(j)::value]; });
    __syncthreads();
    if (wave >= (kSwiglu ? 1u : kTiles)) return;
    const auto joined = [&](uint32_t half) MX_INLINE {
        v4f sum = sums[half * 64u + lane];
#pragma unroll
        for (uint32_t w = 1; w < kFewWaves; ++w) sum += sums[(w * kTiles + half) * 64u + lane];
        return sum;
    };
    const uint32_t column = column0 + (kSwiglu ? 0u : wave * 16u) + 4u * q;
    const v4f sum = joined(kSwiglu ? 0u : wave);
    float v[4] = {sum[0], sum[1], sum[2], sum[3]}, u[4] = {};
    if constexpr (kSwiglu) {
        const v4f up = joined(1u);
        u[0] = up[0], u[1] = up[1], u[2] = up[2], u[3] = up[3];
    }
    if (n < tile.count && column < n_out)
        finish<kFold>(p.e, static_cast<uint64_t>(tile.first) + n, column, n_out, v, u);
}

// Sums of the parts of K, in their order, and the epilogue: eight columns of a row a thread,
// one where a row's end comes before.
template <LinearFold kFold, uint32_t kN>
__device__ __forceinline__ void join_columns(const float* parts, uint32_t count, uint32_t rows, uint64_t row,
                                             uint32_t column, uint32_t columns, LinearEpilogue e) {
    const LinearMatrix m{const_cast<float*>(parts), columns, true};
    float v[kN], u[kN] = {};
    load_row(m, row * columns + column, v);
#pragma unroll 4
    for (uint32_t s = 1; s < count; ++s) {
        float w[kN];
        load_row(m, (static_cast<uint64_t>(s) * rows + row) * columns + column, w);
#pragma unroll
        for (uint32_t k = 0; k < kN; ++k) v[k] += w[k];
    }
    finish_all<kFold>(e, InRow{row, column}, columns, v, u);
}

template <LinearFold kFold>
__global__ __launch_bounds__(256) void linear_join_kernel(const float* __restrict__ parts, uint32_t count, uint32_t rows,
                                                          uint32_t columns, LinearEpilogue e) {
    const uint32_t pieces = (columns + 7u) / 8u;
    const uint64_t all = static_cast<uint64_t>(rows) * pieces;
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < all; i += gridDim.x * 256ull) {
        const uint64_t row = i / pieces;
        uint32_t column = static_cast<uint32_t>(i % pieces) * 8u;
        if (column + 8u <= columns) {
            join_columns<kFold, 8>(parts, count, rows, row, column, columns, e);
            continue;
        }
        for (; column < columns; ++column) join_columns<kFold, 1>(parts, count, rows, row, column, columns, e);
    }
}

// Rows of any stride and alignment to rows at 16 bytes: a piece of eight values a thread, zeros behind
// a row's end.  Memory bounds it: read once, written once, and read again by the product.
__global__ __launch_bounds__(256) void linear_rows_kernel(const uint16_t* __restrict__ from, uint64_t stride,
                                                          uint64_t pieces, uint32_t row_pieces, uint32_t columns,
                                                          v4u* __restrict__ to) {
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < pieces; i += gridDim.x * 256ull) {
        const uint64_t row = i / row_pieces;
        const uint32_t column = static_cast<uint32_t>(i % row_pieces) * 8u;
        to[i] = load_eight(from + row * stride + column, static_cast<int32_t>(columns - column));
    }
}

// ---- activation and bias gradients ------------------------------------------------

// Eight columns of a row for each thread; memory bounds it (16,384 x 8,192 bf16 with GELU 160 us,
// 5.1 TB/s; fp32 305, 5.3).
__global__ __launch_bounds__(256) void activation_backward_kernel(LinearMatrix dy, LinearMatrix pre,
                                                                  uint32_t activation, LinearMatrix dz, uint64_t pieces,
                                                                  uint32_t row_pieces, uint32_t columns) {
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < pieces; i += gridDim.x * 256ull) {
        const uint64_t row = i / row_pieces;
        uint32_t column = static_cast<uint32_t>(i % row_pieces) * 8u;
        const auto part = [&](auto count) {
            float v[decltype(count)::value], z[decltype(count)::value];
            load_row(dy, row * dy.stride + column, v);
            load_row(pre, row * pre.stride + column, z);
            times_slope(activation, z, v);
            store_row(dz, row * dz.stride + column, v);
        };
        if (column + 8u <= columns) {
            part(std::integral_constant<uint32_t, 8>{});
            continue;
        }
        for (; column < columns; ++column) part(std::integral_constant<uint32_t, 1>{});
    }
}

// Sums of 64 columns over `each` rows for each workgroup: 8 columns and every 32nd row for
// a thread, its sum then joined with the other rows' in their order.  One part of the rows
// writes d_bias, several their partial sums [part][columns], which a second launch joins: no
// atomics, so that the order is always the same.  Memory bounds it where there is much of it
// (131,072 x 8,192 388 us, 5.5 TB/s; 4,096 x 8,192 16 us, 5 of them the second launch).
constexpr uint32_t kBiasColumns = 64, kBiasRows = 256, kBiasParts = 64;

__global__ __launch_bounds__(256) void bias_sum_kernel(const uint16_t* __restrict__ dz, uint64_t stride, uint32_t rows,
                                                       uint32_t columns, uint32_t each, LinearMatrix out) {
    __shared__ float sums[32][kBiasColumns];
    const uint32_t column = blockIdx.x * kBiasColumns + threadIdx.x % 8u * 8u;
    const uint32_t from = blockIdx.y * each, to = min(rows - from, each) + from;
    float sum[8] = {};
    const LinearMatrix m{const_cast<uint16_t*>(dz), stride, false};
    if (column + 8u <= columns) {
#pragma unroll 4
        for (uint32_t r = from + threadIdx.x / 8u; r < to; r += 32u) {
            float v[8];
            load_row(m, r * stride + column, v);
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i) sum[i] += v[i];
        }
    } else if (column < columns) {
        for (uint32_t r = from + threadIdx.x / 8u; r < to; r += 32u)
#pragma unroll
            for (uint32_t i = 0; i < 7u; ++i)
                if (column + i < columns) sum[i] += bf16_to_f32(dz[r * stride + column + i]);
    }
#pragma unroll
    for (uint32_t i = 0; i < 8u; ++i) sums[threadIdx.x / 8u][threadIdx.x % 8u * 8u + i] = sum[i];
    __syncthreads();
    const uint32_t c = blockIdx.x * kBiasColumns + threadIdx.x;
    if (threadIdx.x >= kBiasColumns || c >= columns) return;
    float total = 0.0f;
#pragma unroll
    for (uint32_t i = 0; i < 32u; ++i) total += sums[i][threadIdx.x];
    const uint64_t at = static_cast<uint64_t>(blockIdx.y) * columns + c;
    if (out.f32) static_cast<float*>(out.data)[at] = total;
    else static_cast<uint16_t*>(out.data)[at] = static_cast<uint16_t>(f32_to_bf16(total));
}

__global__ __launch_bounds__(256) void bias_join_kernel(const float* __restrict__ parts, uint32_t count,
                                                        uint32_t columns, LinearMatrix out) {
    const uint32_t c = blockIdx.x * 256u + threadIdx.x;
    if (c >= columns) return;
    float total = 0.0f;
#pragma unroll 8
    for (uint32_t i = 0; i < count; ++i) total += parts[static_cast<uint64_t>(i) * columns + c];
    if (out.f32) static_cast<float*>(out.data)[c] = total;
    else static_cast<uint16_t*>(out.data)[c] = static_cast<uint16_t>(f32_to_bf16(total));
}

// parts of the rows: enough workgroups for the CUs, kBiasRows rows each at least
uint32_t bias_parts(uint32_t rows, uint32_t columns) {
    const uint32_t across = (columns + kBiasColumns - 1u) / kBiasColumns;
    const uint32_t wanted = (2u * kMxCus + across - 1u) / across;
    return std::max(1u, std::min(std::min(wanted, kBiasParts), rows / kBiasRows));
}

uint64_t any_tiles(const LinearProduct& p, LinearOrder order, LinearFold fold) {
    const uint64_t across = fold == LinearFold::kSwiglu ? kAnyTile / 2u : kAnyTile;
    const uint64_t columns = fold == LinearFold::kSwiglu ? p.columns / 2u : p.columns;
    uint64_t rows = (p.rows + kAnyTile - 1ull) / kAnyTile;
    if (p.offsets) rows = order == LinearOrder::kTN ? rows * p.experts : mx_max_tasks(p.rows, p.experts, kAnyTile);
    return rows * ((columns + across - 1u) / across);
}

LinearSizes linear_sizes(const LinearProduct& p, LinearOrder order, LinearFold fold) {
    return LinearSizes{p.rows, p.columns, p.depth, p.offsets ? p.experts : 0u, fold == LinearFold::kSwiglu,
                       order == LinearOrder::kTN, order == LinearOrder::kNT};
}

// Whether every operand row starts at 16 bytes, and a lane's offsets from its tile's base are
// 32-bit numbers: 256 rows along K, 64 across it, all those that are gathered, and the distance
// from gate to up.
bool linear_on_tiles(const LinearProduct& p, LinearOrder order, LinearFold fold) {
    if ((reinterpret_cast<uintptr_t>(p.a) | reinterpret_cast<uintptr_t>(p.b)) % 16u != 0u ||
        (p.a_stride | p.b_stride) % 8u != 0u)
        return false;
    const uint64_t limit = 1ull << 31;  // of elements
    const uint64_t a_rows = order == LinearOrder::kNT && p.packed ? p.source_rows : 256u;
    const uint64_t b_rows = order == LinearOrder::kTN && p.packed ? p.source_rows
                            : fold == LinearFold::kSwiglu        ? p.columns + 256ull
                                                                 : 256u;
    return p.a_stride < limit && p.b_stride < limit && std::max<uint64_t>(a_rows, 256u) * p.a_stride < limit &&
           std::max<uint64_t>(b_rows, 256u) * p.b_stride < limit;
}

constexpr uint64_t kLinearStayBytes = 1u << 27;

// 256 x 256 tiles leave the SwiGLU's gradient too few registers.
bool linear_wide(LinearFold fold) { return fold != LinearFold::kSwigluGrad; }

size_t part_bytes(const LinearSizes& p, const LinearPlan& plan) {
    const uint32_t parts = p.experts != 0u ? 1u : linear_parts(p.depth, plan.splits);
    return parts > 1u ? static_cast<size_t>(parts) * p.rows * p.columns * sizeof(float) : 0u;
}

// Whether whole lines of C go past the caches, and the residual's come so: weights' gradients and
// experts' rows always, dense rows, which the next layer reads, where they are more than stays in
// the memory-side cache beside the operands until then.  us past the caches and through them: four layers
// of 2,048 x 2,048 over 2,048 rows 131 and 115, the same with residuals 139 and 122, of 512 and 8,192
// by turns over 8,192 rows 366 and 340; forward 8,192 x 8,192 x 512 into 268 MB of fp32 94 and 88, with an
// fp32 residual 143 and 170, 16,384 x 8,192 x 2,048 in bf16 with a residual 485 and 528.  Smaller ones by
// themselves, their rows read by nobody: 4,096 x 8,192 x 512 into fp32 55 and 48, 1,024 x 8,192 x 2,048 36 and 38.
bool linear_past(const LinearProduct& p, uint32_t parts) {
    const uint64_t values = static_cast<uint64_t>(p.rows) * p.columns;
    const uint64_t residual = !p.e.residual.data ? 0u : p.e.residual.f32 ? 4u : 2u;
    return values * (parts * (p.e.c.f32 ? 4u : 2u) + residual) > kLinearStayBytes;
}

template <typename S, LinearOrder kOrder, bool kExperts, LinearFold kFold>
hipError_t launch_tiles(const LinearProduct& p, const LinearSizes& sizes, uint32_t splits, void* scratch,
                        hipStream_t stream) {
    if constexpr ((kOrder == LinearOrder::kTN && S::kBM < 64u) ||
                  (kFold == LinearFold::kSwigluGrad && S::kBM == 256u)) {
        return hipErrorInvalidValue;  // the rule takes none
    } else {
        const uint32_t each = kExperts ? 0u : linear_each(p.depth, splits);
        const uint32_t parts = kExperts ? 1u : linear_parts(p.depth, splits);
        LinearProduct q = p;
        if (parts > 1u) {
            q.e = LinearEpilogue{};
            q.e.c = LinearMatrix{scratch, p.columns, true};
        }
        const auto start = [&](auto past) {
            linear_tile_kernel<S, kOrder, kExperts, kFold, decltype(past)::value>
                <<<linear_grid<S>(sizes, parts), 64u * S::kWaves, 0, stream>>>(q, each);
        };
        // other tiles have stores of one kind
        constexpr bool kEither = !kExperts && kOrder != LinearOrder::kTN && S::kMF == 32u &&
                                 (kFold == LinearFold::kStore || kFold == LinearFold::kAdd);
        if constexpr (!kEither) start(std::true_type{});
        else if (linear_past(q, parts)) start(std::true_type{});
        else start(std::false_type{});
        if constexpr (!kExperts) {
            if (parts > 1u) {
                if (hipError_t rc = hipGetLastError(); rc != hipSuccess) return rc;
                const uint64_t pieces = static_cast<uint64_t>(p.rows) * ((p.columns + 7u) / 8u);
                const uint32_t grid = static_cast<uint32_t>(std::min<uint64_t>((pieces + 255u) / 256u, 16u * kMxCus));
                linear_join_kernel<kFold><<<grid, 256, 0, stream>>>(static_cast<const float*>(scratch), parts, p.rows,
                                                                   p.columns, p.e);
            }
        }
        return hipGetLastError();
    }
}

struct Operand {  // as it is stored
    const uint16_t* data;
    uint64_t stride;
    uint32_t rows, columns;
    bool at_16() const { return reinterpret_cast<uintptr_t>(data) % 16u == 0u && stride % 8u == 0u; }
    uint64_t row_pieces() const { return (columns + 7ull) / 8u; }
    size_t copy_bytes() const { return rows * row_pieces() * 16u; }
};

Operand operand_a(const LinearProduct& p, LinearOrder order) {
    return order == LinearOrder::kTN ? Operand{p.a, p.a_stride, p.depth, p.rows} : Operand{p.a, p.a_stride, p.rows, p.depth};
}
Operand operand_b(const LinearProduct& p, LinearOrder order) {
    return order == LinearOrder::kNT ? Operand{p.b, p.b_stride, p.columns, p.depth} : Operand{p.b, p.b_stride, p.depth, p.columns};
}

size_t up_to_16(size_t bytes) { return (bytes + 15u) / 16u * 16u; }

// The parts of K, and in front of them copies of operands whose rows do not start at 16 bytes.
LinearRun run_with_copies(const LinearProduct& p, LinearOrder order, LinearFold fold) {
    LinearProduct q = p;
    const Operand a = operand_a(p, order), b = operand_b(p, order);
    LinearRun run{};
    run.copy_a = !a.at_16();
    run.copy_b = !b.at_16();
    if (run.copy_a) q.a = nullptr, q.a_stride = a.row_pieces() * 8u;
    if (run.copy_b) q.b = nullptr, q.b_stride = b.row_pieces() * 8u;
    const LinearSizes sizes = linear_sizes(p, order, fold);
    run.plan = linear_plan(sizes, linear_wide(fold));
    run.on_tiles = linear_on_tiles(q, order, fold);
    run.fits = run.plan.few() || with_linear_shape(run.plan, [&](auto s) {
        return linear_tiles<decltype(s)>(sizes) * run.plan.splits < (1ull << 31);
    });
    run.scratch_bytes = run.plan.few() ? 0u : part_bytes(sizes, run.plan);
    if (run.copy_a) run.scratch_bytes = up_to_16(run.scratch_bytes) + a.copy_bytes();
    if (run.copy_b) run.scratch_bytes = up_to_16(run.scratch_bytes) + b.copy_bytes();
    return run;
}

// Whether copies pay: the kernel for any strides goes through K 32 values at a time, 8.9 us for 1,000
// of them where its tiles are at work at the same time, the copies are a launch each and their bytes.
// us without and with copies, rows x outputs x inputs, all odd: 61 x 2,001 x 501 10 and 13, 1 x 8,191 x
// 2,001 34 and 22, 512 x 8,191 x 501 21 and 33, 4,001 x 8,191 x 501 142 and 93, x 8,001 1,899 and 563;
// the input's gradient of 61 x 333 x 501 15 and 11, of 4,001 x 8,191 x 2,001 703 and 191; the weight's of
// 61 x 2,001 x 2,001 10 and 12, of 512 x 2,001 x 2,001 42 and 20.
bool copies_pay(const LinearProduct& p) {
    const double products = static_cast<double>(p.rows) * p.columns * p.depth;
    return p.depth >= 320u || (p.depth >= 96u && products >= 3e9);
}

// Contiguous matrices of a layer: null data has the alignment that a copy would have.
LinearProduct layer_product(uint32_t rows, uint32_t columns, uint32_t depth, uint64_t a_stride, uint64_t b_stride) {
    return LinearProduct{nullptr, nullptr, a_stride, b_stride, nullptr, nullptr, rows, columns, depth, 0u, 1u, 1u, {}};
}

}  // namespace

size_t linear_scratch_bytes(uint32_t rows, uint32_t outputs, uint32_t inputs) {
    const auto stride = [&](uint32_t of, uint64_t columns) { return of == 1u ? (columns + 7u) / 8u * 8u : columns; };
    const uint64_t x = stride(rows, inputs), w = stride(outputs, inputs), dz = stride(rows, outputs);
    size_t most = bias_scratch_bytes(rows, outputs);
    const auto with = [&](const LinearProduct& p, LinearOrder order, LinearFold fold) {
        const LinearRun run = run_with_copies(p, order, fold);
        if (run.on_tiles && run.fits && ((!run.copy_a && !run.copy_b) || copies_pay(p)))
            most = std::max(most, run.scratch_bytes);
    };
    with(layer_product(rows, outputs, inputs, x, w), LinearOrder::kNT, LinearFold::kForward);
    with(layer_product(rows, inputs, outputs, dz, w), LinearOrder::kNN, LinearFold::kSlope);
    with(layer_product(outputs, inputs, rows, dz, x), LinearOrder::kTN, LinearFold::kAdd);
    return most;
}

size_t bias_scratch_bytes(uint32_t rows, uint32_t columns) {
    const uint32_t parts = bias_parts(rows, columns);
    return parts > 1u ? static_cast<size_t>(parts) * columns * sizeof(float) : 0u;
}

LinearRun linear_run(const LinearProduct& p, LinearOrder order, LinearFold fold, size_t scratch_bytes) {
    LinearRun run = run_with_copies(p, order, fold);
    const bool copies = run.copy_a || run.copy_b;
    // experts' rows are not copied: their calls have no scratch
    if (run.on_tiles && (!copies || (!p.offsets && copies_pay(p) && scratch_bytes >= run.scratch_bytes)))
        return run;
    return LinearRun{{2u, 1u}, false, any_tiles(p, order, fold) < (1ull << 24), false, false, 0u};  // threads of a launch
}

hipError_t launch_linear(const LinearProduct& given, LinearOrder order, LinearFold fold, const LinearRun& run, void* scratch,
                         hipStream_t stream) {
    LinearProduct p = given;
    const LinearSizes sizes = linear_sizes(p, order, fold);
    size_t used = !run.on_tiles || run.plan.few() ? 0u : part_bytes(sizes, run.plan);
    const auto copy = [&](const Operand& o) -> const uint16_t* {
        used = up_to_16(used);
        v4u* to = reinterpret_cast<v4u*>(static_cast<uint8_t*>(scratch) + used);
        used += o.copy_bytes();
        const uint64_t pieces = o.rows * o.row_pieces();
        const uint32_t grid = static_cast<uint32_t>(std::min<uint64_t>((pieces + 255u) / 256u, 16u * kMxCus));
        linear_rows_kernel<<<grid, 256, 0, stream>>>(o.data, o.stride, pieces, static_cast<uint32_t>(o.row_pieces()), o.columns, to);
        return reinterpret_cast<const uint16_t*>(to);
    };
    if (run.copy_a) {
        const Operand a = operand_a(p, order);
        p.a = copy(a);
        p.a_stride = a.row_pieces() * 8u;
    }
    if (run.copy_b) {
        const Operand b = operand_b(p, order);
        p.b = copy(b);
        p.b_stride = b.row_pieces() * 8u;
    }
    if (run.copy_a || run.copy_b)
        if (hipError_t rc = hipGetLastError(); rc != hipSuccess) return rc;
    const auto launch = [&](auto o, auto experts, auto f) -> hipError_t {
        constexpr LinearOrder kOrder = decltype(o)::value;
        constexpr bool kExperts = decltype(experts)::value;
        constexpr LinearFold kFold = decltype(f)::value;
        if (!run.on_tiles) {
            linear_any_kernel<kOrder, kExperts, kFold>
                <<<static_cast<uint32_t>(any_tiles(p, order, fold)), 256, 0, stream>>>(p);
            return hipGetLastError();
        }
        if constexpr (kOrder == LinearOrder::kNT) {
            if (run.plan.few())
                return with_few_shape(run.plan, [&](auto s) -> hipError_t {
                    using S = decltype(s);
                    if constexpr (kFold == LinearFold::kSwiglu && S::kTiles != 2u) {
                        return hipErrorInvalidValue;  // the rule takes none
                    } else {
                        linear_few_kernel<S, kExperts, kFold>
                            <<<static_cast<uint32_t>(few_blocks<S>(sizes)), 64u * S::kWaves, 0, stream>>>(p);
                        return hipGetLastError();
                    }
                });
        }
        return with_linear_shape(run.plan, [&](auto s) -> hipError_t {
            return launch_tiles<decltype(s), kOrder, kExperts, kFold>(p, sizes, run.plan.splits, scratch, stream);
        });
    };
    using NT = std::integral_constant<LinearOrder, LinearOrder::kNT>;
    using NN = std::integral_constant<LinearOrder, LinearOrder::kNN>;
    using TN = std::integral_constant<LinearOrder, LinearOrder::kTN>;
    using Store = std::integral_constant<LinearFold, LinearFold::kStore>;
    using Add = std::integral_constant<LinearFold, LinearFold::kAdd>;
    using Forward = std::integral_constant<LinearFold, LinearFold::kForward>;
    using Slope = std::integral_constant<LinearFold, LinearFold::kSlope>;
    using Swiglu = std::integral_constant<LinearFold, LinearFold::kSwiglu>;
    using SwigluGrad = std::integral_constant<LinearFold, LinearFold::kSwigluGrad>;
    const auto added = [&](auto o, auto experts) {
        return p.e.residual.data ? launch(o, experts, Add{}) : launch(o, experts, Store{});
    };
    if (!p.offsets) {
        // Where nothing is done to the sums but a residual's addition they go to memory in whole lines: the
        // input's gradient 8,192 x 512 x 8,192 (rows x outputs x inputs) with a residual 128 us and so 103,
        // without one 81 and 74; forward 8,192 x 8,192 x 2,048 276 and 246, 240 and 226.
        const bool as_they_are = p.e.activation == Q38M_ACT_NONE && !p.e.bias.data;
        if (order == LinearOrder::kNT && as_they_are && !p.e.pre.data) return added(NT{}, std::false_type{});
        if (order == LinearOrder::kNT) return launch(NT{}, std::false_type{}, Forward{});
        if (order == LinearOrder::kNN && as_they_are) return added(NN{}, std::false_type{});
        if (order == LinearOrder::kNN) return launch(NN{}, std::false_type{}, Slope{});
        return added(TN{}, std::false_type{});
    }
    if (fold == LinearFold::kSwiglu) return launch(NT{}, std::true_type{}, Swiglu{});
    if (fold == LinearFold::kSwigluGrad) return launch(NN{}, std::true_type{}, SwigluGrad{});
    if (order == LinearOrder::kNT) return launch(NT{}, std::true_type{}, Store{});
    if (order == LinearOrder::kNN) return launch(NN{}, std::true_type{}, Store{});
    return added(TN{}, std::true_type{});
}

hipError_t launch_activation_backward(const LinearMatrix& dy, const LinearMatrix& pre,
                                      uint32_t activation, const LinearMatrix& dz, uint32_t rows,
                                      uint32_t columns, hipStream_t stream) {
    const uint32_t row_pieces = (columns + 7u) / 8u;
    const uint64_t pieces = static_cast<uint64_t>(rows) * row_pieces;
    const uint32_t grid = static_cast<uint32_t>(std::min<uint64_t>((pieces + 255u) / 256u, 16u * kMxCus));
    activation_backward_kernel<<<grid, 256, 0, stream>>>(dy, pre, activation, dz, pieces, row_pieces, columns);
    return hipGetLastError();
}

hipError_t launch_bias_backward(const uint16_t* dz, uint64_t stride, uint32_t rows,
                                uint32_t columns, const LinearMatrix& d_bias, void* scratch,
                                hipStream_t stream) {
    const uint32_t parts = bias_parts(rows, columns), each = (rows + parts - 1u) / parts;
    const uint32_t used = (rows + each - 1u) / each;
    const uint32_t across = (columns + kBiasColumns - 1u) / kBiasColumns;
    if (used == 1u) {
        bias_sum_kernel<<<across, 256, 0, stream>>>(dz, stride, rows, columns, each, d_bias);
        return hipGetLastError();
    }
    const LinearMatrix partial{scratch, columns, true};
    bias_sum_kernel<<<dim3(across, used), 256, 0, stream>>>(dz, stride, rows, columns, each, partial);
    if (hipError_t rc = hipGetLastError(); rc != hipSuccess) return rc;
    bias_join_kernel<<<(columns + 255u) / 256u, 256, 0, stream>>>(static_cast<const float*>(scratch), used, columns,
                                                                 d_bias);
    return hipGetLastError();
}

}  // namespace q38m
