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
#include "q38m_product.h"

namespace q38m {
namespace {

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

// ---- activations --------------------------------------------------------------

// Phi(-|z|), with a = |z|, t = 1 / (1 + 0.3 a): exp(-a^2 / 2) times a polynomial in t,
// fitted here by least squares over 0 <= a <= 14, weights raised where the relative error
// was largest: 5.8e-8, and in fp32 4.9e-7 near 0 growing with the exponential's argument
// (6.6e-7 at 3, 1.9e-6 at 6).  `density` gets exp(-a^2 / 2).
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

// kN (4 or 8) consecutive elements of a matrix, `live` of them there
template <uint32_t kN>
__device__ __forceinline__ void load_row(const LinearMatrix& m, uint64_t at, uint32_t live, float (&v)[kN]) {
    if (m.f32) {
        const float* p = static_cast<const float*>(m.data) + at;
        if (live >= kN) {
#pragma unroll
            for (uint32_t i = 0; i < kN; i += 4u) {
                const v4u_any w = *reinterpret_cast<const v4u_any*>(p + i);
                v[i] = __uint_as_float(w.x), v[i + 1u] = __uint_as_float(w.y);
                v[i + 2u] = __uint_as_float(w.z), v[i + 3u] = __uint_as_float(w.w);
            }
            return;
        }
#pragma unroll
        for (uint32_t i = 0; i < kN; ++i) v[i] = i < live ? p[i] : 0.0f;
        return;
    }
    const uint16_t* p = static_cast<const uint16_t*>(m.data) + at;
    if (live >= kN) {
        uint32_t d[kN / 2u];
        if constexpr (kN == 8u) {
            const v4u_any w = *reinterpret_cast<const v4u_any*>(p);
            d[0] = w.x, d[1] = w.y, d[2] = w.z, d[3] = w.w;
        } else {
            const v2u_any w = *reinterpret_cast<const v2u_any*>(p);
            d[0] = w.x, d[1] = w.y;
        }
#pragma unroll
        for (uint32_t i = 0; i < kN; i += 2u) {
            v[i] = __uint_as_float(d[i / 2u] << 16);
            v[i + 1u] = __uint_as_float(d[i / 2u] & 0xffff0000u);
        }
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < kN; ++i) v[i] = i < live ? bf16_to_f32(p[i]) : 0.0f;
}

template <uint32_t kN>
__device__ __forceinline__ void store_row(const LinearMatrix& m, uint64_t at, uint32_t live, const float (&v)[kN]) {
    if (m.f32) {
        float* p = static_cast<float*>(m.data) + at;
        if (live >= kN) {
#pragma unroll
            for (uint32_t i = 0; i < kN; i += 4u)
                *reinterpret_cast<v4u_any*>(p + i) = v4u_any{__float_as_uint(v[i]), __float_as_uint(v[i + 1u]),
                                                             __float_as_uint(v[i + 2u]), __float_as_uint(v[i + 3u])};
            return;
        }
#pragma unroll
        for (uint32_t i = 0; i < kN - 1u; ++i)
            if (i < live) p[i] = v[i];
        return;
    }
    uint16_t* p = static_cast<uint16_t*>(m.data) + at;
    uint32_t d[kN / 2u];
#pragma unroll
    for (uint32_t i = 0; i < kN; i += 2u) d[i / 2u] = f32_to_bf16(v[i]) | f32_to_bf16(v[i + 1u]) << 16;
    if (live >= kN) {
        if constexpr (kN == 8u) *reinterpret_cast<v4u_any*>(p) = v4u_any{d[0], d[1], d[2], d[3]};
        else *reinterpret_cast<v2u_any*>(p) = v2u_any{d[0], d[1]};
        return;
    }
#pragma unroll
    for (uint32_t i = 0; i < kN - 1u; ++i)
        if (i < live) p[i] = static_cast<uint16_t>(d[i / 2u] >> i % 2u * 16u);
}

// The epilogue of kN sums of row `row`, columns from `column` on (below n of them).
template <uint32_t kN>
__device__ __forceinline__ void finish_plain(const LinearEpilogue& e, uint64_t row, uint32_t column, uint32_t n,
                                             float (&v)[kN]) {
    const uint32_t live = n - column;
    if (e.slope) {
        if (e.activation != Q38M_ACT_NONE) {
            float z[kN];
            load_row(e.pre, row * e.pre.stride + column, live, z);
            times_slope(e.activation, z, v);
        }
    } else {
        if (e.bias.data) {
            float b[kN];
            load_row(e.bias, column, live, b);
#pragma unroll
            for (uint32_t i = 0; i < kN; ++i) v[i] += b[i];
        }
        if (e.pre.data) store_row(e.pre, row * e.pre.stride + column, live, v);
        activate(e.activation, v);
    }
    if (e.residual.data) {
        float r[kN];
        load_row(e.residual, row * e.residual.stride + column, live, r);
#pragma unroll
        for (uint32_t i = 0; i < kN; ++i) v[i] += r[i];
    }
    store_row(e.c, row * e.c.stride + column, live, v);
}

// Gate and up sums of the same columns; pre has n columns of gate, then n of up.
template <uint32_t kN>
__device__ __forceinline__ void finish_swiglu(const LinearEpilogue& e, uint64_t row, uint32_t column, uint32_t n,
                                              const float (&gate)[kN], const float (&up)[kN]) {
    const uint32_t live = n - column;
    if (e.pre.data) {
        store_row(e.pre, row * e.pre.stride + column, live, gate);
        store_row(e.pre, row * e.pre.stride + n + column, live, up);
    }
    float h[kN];
    if (e.c.f32) {
#pragma unroll
        for (uint32_t i = 0; i < kN; ++i) h[i] = swiglu<true>(gate[i], up[i]);
    } else {
#pragma unroll
        for (uint32_t i = 0; i < kN; ++i) h[i] = swiglu<false>(gate[i], up[i]);
    }
    store_row(e.c, row * e.c.stride + column, live, h);
}

// The gradients of gate and up of h's: dh u (s + g s(g) s(-g)) and dh g s.
template <uint32_t kN>
__device__ __forceinline__ void finish_swiglu_grad(const LinearEpilogue& e, uint64_t row, uint32_t column, uint32_t n,
                                                   const float (&dh)[kN]) {
    const uint32_t live = n - column;
    float g[kN], u[kN];
    load_row(e.pre, row * e.pre.stride + column, live, g);
    load_row(e.pre, row * e.pre.stride + n + column, live, u);
    float dg[kN], du[kN];
#pragma unroll
    for (uint32_t i = 0; i < kN; ++i) {
        const Sigmoid y(g[i]);
        dg[i] = dh[i] * u[i] * __builtin_fmaf(held(g[i]), y.both, y.s);
        du[i] = dh[i] * (g[i] * y.s);
    }
    store_row(e.c, row * e.c.stride + column, live, dg);
    store_row(e.c, row * e.c.stride + n + column, live, du);
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
    __shared__ uint32_t offsets[kExperts && !kAcrossA ? kMaxSortExperts : 1u];
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
        const uint32_t last = p.offsets[p.experts];
        for (uint32_t e = t; e < kMaxSortExperts; e += 256u) offsets[e] = e < p.experts ? p.offsets[e] : last;
        __syncthreads();
        const TileList<kAnyTile> list(offsets, last, p.rows);
        if (row_tile >= list.total) return;
        tile = list.find(row_tile);
    } else {
        tile.first = row_tile * kAnyTile;
        tile.count = min(p.rows - tile.first, kAnyTile);
    }

    // each thread's piece of eight values: along K, row t / 4 and piece t % 4; across K,
    // stored row t / 8 and columns from 8 (t % 8) on
    const auto source = [&](uint32_t place) {
        return p.packed ? min(p.packed[place] / p.top_k, p.source_rows - 1u) : place;
    };
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
            if constexpr (kFold == LinearFold::kSwiglu) {
                const float u[4] = {acc[1][i][0], acc[1][i][1], acc[1][i][2], acc[1][i][3]};
                finish_swiglu(p.e, row, column, n_out, v, u);
            } else if constexpr (kFold == LinearFold::kSwigluGrad) {
                finish_swiglu_grad(p.e, row, column, n_out, v);
            } else {
                finish_plain(p.e, row, column, n_out, v);
            }
        }
    }
}

// ---- activation and bias gradients ------------------------------------------------

// Eight columns of a row for each thread; memory bounds it.
__global__ __launch_bounds__(256) void activation_backward_kernel(LinearMatrix dy, LinearMatrix pre,
                                                                  uint32_t activation, LinearMatrix dz, uint64_t pieces,
                                                                  uint32_t row_pieces, uint32_t columns) {
    for (uint64_t i = blockIdx.x * 256ull + threadIdx.x; i < pieces; i += gridDim.x * 256ull) {
        const uint64_t row = i / row_pieces;
        const uint32_t column = static_cast<uint32_t>(i % row_pieces) * 8u, live = columns - column;
        float v[8], z[8];
        load_row(dy, row * dy.stride + column, live, v);
        load_row(pre, row * pre.stride + column, live, z);
        times_slope(activation, z, v);
        store_row(dz, row * dz.stride + column, live, v);
    }
}

// Sums of 64 columns over `each` rows for each workgroup: 8 columns and every 32nd row for
// a thread, its sum then joined with the other rows' in their order.  One part of the rows
// writes d_bias, several their partial sums [part][columns], which a second launch joins.
constexpr uint32_t kBiasColumns = 64, kBiasRows = 256, kBiasParts = 64;

__global__ __launch_bounds__(256) void bias_sum_kernel(const uint16_t* __restrict__ dz, uint64_t stride, uint32_t rows,
                                                       uint32_t columns, uint32_t each, LinearMatrix out) {
    __shared__ float sums[32][kBiasColumns];
    const uint32_t column = blockIdx.x * kBiasColumns + threadIdx.x % 8u * 8u;
    const uint32_t from = blockIdx.y * each, to = min(rows - from, each) + from;
    float sum[8] = {};
    if (column < columns) {
        const LinearMatrix m{const_cast<uint16_t*>(dz), stride, false};
#pragma unroll 4
        for (uint32_t r = from + threadIdx.x / 8u; r < to; r += 32u) {
            float v[8];
            load_row(m, r * stride + column, columns - column, v);
#pragma unroll
            for (uint32_t i = 0; i < 8u; ++i) sum[i] += v[i];
        }
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

}  // namespace

size_t linear_scratch_bytes(uint32_t rows, uint32_t outputs, uint32_t) {
    const uint32_t parts = bias_parts(rows, outputs);
    return parts > 1u ? static_cast<size_t>(parts) * outputs * sizeof(float) : 0u;
}

bool linear_fits(const LinearProduct& p, LinearOrder order, LinearFold fold) {
    return any_tiles(p, order, fold) < (1ull << 31);
}

hipError_t launch_linear(const LinearProduct& p, LinearOrder order, LinearFold fold, void*, hipStream_t stream) {
    const uint32_t grid = static_cast<uint32_t>(any_tiles(p, order, fold));
    const auto launch = [&](auto o, auto experts, auto f) {
        linear_any_kernel<decltype(o)::value, decltype(experts)::value, decltype(f)::value>
            <<<grid, 256, 0, stream>>>(p);
    };
    using NT = std::integral_constant<LinearOrder, LinearOrder::kNT>;
    using NN = std::integral_constant<LinearOrder, LinearOrder::kNN>;
    using TN = std::integral_constant<LinearOrder, LinearOrder::kTN>;
    using Plain = std::integral_constant<LinearFold, LinearFold::kPlain>;
    using Swiglu = std::integral_constant<LinearFold, LinearFold::kSwiglu>;
    using SwigluGrad = std::integral_constant<LinearFold, LinearFold::kSwigluGrad>;
    if (!p.offsets) {
        if (order == LinearOrder::kNT) launch(NT{}, std::false_type{}, Plain{});
        else if (order == LinearOrder::kNN) launch(NN{}, std::false_type{}, Plain{});
        else launch(TN{}, std::false_type{}, Plain{});
    } else if (fold == LinearFold::kSwiglu) {
        launch(NT{}, std::true_type{}, Swiglu{});
    } else if (fold == LinearFold::kSwigluGrad) {
        launch(NN{}, std::true_type{}, SwigluGrad{});
    } else {
        if (order == LinearOrder::kNT) launch(NT{}, std::true_type{}, Plain{});
        else if (order == LinearOrder::kNN) launch(NN{}, std::true_type{}, Plain{});
        else launch(TN{}, std::true_type{}, Plain{});
    }
    return hipGetLastError();
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
