// Microscaled 4-bit rows (MXFP4): quantisation, the dense product and the
// experts' products, on the block-scaled matrix instructions of gfx950.
//
// A row of K values is ceil(K / 128) * 64 bytes of codes (the even k in the
// low nibble; codes past K are zero) and one scale byte for every 32 values.
// Code c stands for (-1)^(c >> 3) * {0, .5, 1, 1.5, 2, 3, 4, 6}[c & 7], scale
// byte s for 2^(s - 127), 255 for NaN.
#include "q38m_device.h"
#include "q38m_internal.h"

namespace q38m {

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
        const uint4 w = *reinterpret_cast<const uint4*>(p);
        d[0] = w.x; d[1] = w.y; d[2] = w.z; d[3] = w.w;
    }
    __device__ void gather(const uint16_t* p, uint32_t count) {
#pragma unroll
        for (uint32_t i = 0; i < 4u; ++i) {
            const uint32_t lo = 2u * i < count ? p[2u * i] : 0u;
            const uint32_t hi = 2u * i + 1u < count ? p[2u * i + 1u] : 0u;
            d[i] = lo | hi << 16;
        }
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
        const float4 a = reinterpret_cast<const float4*>(p)[0];
        const float4 b = reinterpret_cast<const float4*>(p)[1];
        v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
        v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    }
    __device__ void gather(const float* p, uint32_t count) {
#pragma unroll
        for (uint32_t i = 0; i < 8u; ++i) v[i] = i < count ? p[i] : 0.0f;
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
// power of two from 16 to 256) threads walk a row, 256 / lanes rows at once.
constexpr uint32_t kQuantThreads = 256;

template <typename T>
__global__ __launch_bounds__(kQuantThreads) void mx_quantize_kernel(
    const T* __restrict__ x, uint64_t stride, uint32_t rows, uint32_t columns, bool whole,
    uint32_t lanes_log2, uint32_t* __restrict__ codes, uint32_t* __restrict__ scales,
    T* __restrict__ rounded, bool rounded_whole) {
    const uint32_t lanes = 1u << lanes_log2;
    const uint32_t row = blockIdx.x * (kQuantThreads >> lanes_log2) + (threadIdx.x >> lanes_log2);
    if (row >= rows) return;
    const uint32_t padded = (columns + 127u) / 128u * 128u;
    const T* from = x + row * stride;
    const uint64_t first_eight = static_cast<uint64_t>(row) * (padded / 8u);
    for (uint32_t c = (threadIdx.x & (lanes - 1u)) * 8u; c < padded; c += lanes * 8u) {
        Eight<T> e;
        if (whole && c + 8u <= columns) e.load(from + c);
        else e.gather(from + c, c < columns ? columns - c : 0u);
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
        if (!rounded) continue;
        float v[8];
        mx_values(q, byte, v);
        T* to = rounded + static_cast<uint64_t>(row) * columns + c;
        if constexpr (sizeof(T) == 4u) {
            if (rounded_whole && c + 8u <= columns) {
                reinterpret_cast<float4*>(to)[0] = make_float4(v[0], v[1], v[2], v[3]);
                reinterpret_cast<float4*>(to)[1] = make_float4(v[4], v[5], v[6], v[7]);
            } else {
                for (uint32_t i = 0; i < 8u && c + i < columns; ++i) to[i] = v[i];
            }
        } else {
            if (rounded_whole && c + 8u <= columns) {
                uint32_t d[4];
#pragma unroll
                for (uint32_t i = 0; i < 4u; ++i)  // two significant bits: exact in bf16
                    d[i] = __float_as_uint(v[2 * i]) >> 16 |
                           (__float_as_uint(v[2 * i + 1]) & 0xffff0000u);
                *reinterpret_cast<uint4*>(to) = make_uint4(d[0], d[1], d[2], d[3]);
            } else {
                for (uint32_t i = 0; i < 8u && c + i < columns; ++i)
                    to[i] = static_cast<uint16_t>(__float_as_uint(v[i]) >> 16);
            }
        }
    }
}

// ---- products -----------------------------------------------------------------

typedef int v8i __attribute__((ext_vector_type(8)));

// v_mfma_scale_f32_16x16x128_f8f6f4 on 4-bit codes: lane l holds the 32 values
// k = 32 (l / 16) .. + 31 of row l % 16 of A and of B and their scale byte (the
// low one); D lane l: rows 4 (l / 16) + i of A, row l % 16 of B.  Products and
// scales are exact; the sum is rounded in fp32.
__device__ __forceinline__ v4f mfma_mx_16x16x128(v4i a, uint32_t sa, v4i b, uint32_t sb, v4f c) {
    const v8i wa = {a[0], a[1], a[2], a[3], 0, 0, 0, 0}, wb = {b[0], b[1], b[2], b[3], 0, 0, 0, 0};
    return __builtin_amdgcn_mfma_scale_f32_16x16x128_f8f6f4(wa, wb, c, 4, 4, 0, sa, 0, sb);
}

struct MxTask {
    uint32_t expert, first, count;  // rows first .. first + count of the sorted order
};

// Row tile `task` of the experts' rows, kRows at a time, found by every wave
// for itself: lanes hold consecutive experts, a sum over the lanes of their
// tiles gives the lane that holds the tile.  Offsets past `routes` or falling
// ones count as no rows.  count = 0: there is no such tile.
template <uint32_t kRows>
__device__ MxTask find_task(const uint32_t* __restrict__ offsets, uint32_t experts,
                            uint32_t routes, uint32_t task) {
    const uint32_t lane = threadIdx.x & 63u;
    const uint32_t per = (experts + 63u) / 64u, e0 = lane * per;
    const uint32_t e1 = min(e0 + per, experts);
    uint32_t tiles = 0, begin = e0 < experts ? min(offsets[e0], routes) : 0u, next = begin;
    for (uint32_t e = e0; e < e1; ++e) {
        const uint32_t end = min(offsets[e + 1u], routes);
        if (end > next) {
            tiles += (end - next + kRows - 1u) / kRows;
        }
        next = end;
    }
    uint32_t sum = tiles;
#pragma unroll
    for (uint32_t d = 1; d < 64u; d <<= 1) {
        const uint32_t up = __shfl_up(sum, d);
        if (lane >= d) sum += up;
    }
    const uint64_t past = __ballot(sum > task);
    MxTask found{0u, 0u, 0u};
    if (past == 0u) return found;
    const uint32_t owner = __builtin_ctzll(past);
    uint32_t left = task - (sum - tiles), expert = e0;
    if (lane == owner) {
        next = begin;
        for (uint32_t e = e0; e < e1; ++e) {
            const uint32_t end = min(offsets[e + 1u], routes);
            const uint32_t n = end > next ? (end - next + kRows - 1u) / kRows : 0u;
            if (left < n) {
                expert = e;
                found.first = next + left * kRows;
                found.count = min(end - found.first, kRows);
                break;
            }
            left -= n;
            next = end;
        }
    }
    found.expert = __builtin_amdgcn_readlane(expert, owner);
    found.first = __builtin_amdgcn_readlane(found.first, owner);
    found.count = __builtin_amdgcn_readlane(found.count, owner);
    return found;
}

// h = silu(g) u
__device__ __forceinline__ float swiglu(float g, float u) { return g / (1.0f + exp_q(-g)) * u; }

// One wave per 16 x 16 tile of C (with the SwiGLU fold, of its gate half and
// its up half), operands straight from memory.
template <bool kSwiglu>
__global__ __launch_bounds__(64) void mx_product_kernel(MxProduct p) {
    const uint32_t lane = threadIdx.x, r = lane & 15u, q = lane >> 4;
    MxTask t;
    if (p.offsets) {
        t = find_task<16>(p.offsets, p.experts, p.routes, blockIdx.y);
        if (t.count == 0u) return;
    } else {
        t = MxTask{0u, blockIdx.y * 16u, min(p.routes - blockIdx.y * 16u, 16u)};
    }
    const uint32_t n_out = kSwiglu ? p.n / 2u : p.n;
    const uint32_t n0 = blockIdx.x * 16u;
    const uint32_t row_bytes = p.k128 * 64u, scale_bytes = p.k128 * 4u;
    uint32_t source = t.first + min(r, t.count - 1u);
    if (p.packed) source = p.packed[source] / p.top_k;
    const bool real = r < t.count && source < p.a_rows;
    source = min(source, p.a_rows - 1u);
    const uint8_t* a = p.a_codes + static_cast<uint64_t>(source) * row_bytes + 16u * q;
    const uint8_t* as = p.a_scales + static_cast<uint64_t>(source) * scale_bytes + q;
    const uint32_t column = min(n0 + r, n_out - 1u);
    const uint64_t w_row = static_cast<uint64_t>(t.expert) * p.n + column;
    const uint8_t* b = p.b_codes + w_row * row_bytes + 16u * q;
    const uint8_t* bs = p.b_scales + w_row * scale_bytes + q;
    const uint64_t up = static_cast<uint64_t>(n_out) * row_bytes;
    const uint64_t up_scale = static_cast<uint64_t>(n_out) * scale_bytes;
    v4f acc = {0, 0, 0, 0}, acc_up = {0, 0, 0, 0};
    for (uint32_t k = 0; k < p.k128; ++k) {
        v4i av = *reinterpret_cast<const v4i*>(a + 64u * k);
        if (!real) av = v4i{0, 0, 0, 0};
        const uint32_t sa = real ? as[4u * k] : 127u;
        acc = mfma_mx_16x16x128(av, sa, *reinterpret_cast<const v4i*>(b + 64u * k), bs[4u * k], acc);
        if constexpr (kSwiglu)
            acc_up = mfma_mx_16x16x128(av, sa, *reinterpret_cast<const v4i*>(b + up + 64u * k),
                                       bs[up_scale + 4u * k], acc_up);
    }
    if (n0 + r >= n_out) return;
#pragma unroll
    for (uint32_t i = 0; i < 4u; ++i) {
        const uint32_t m = 4u * q + i;
        if (m >= t.count) break;
        const float v = kSwiglu ? swiglu(acc[i], acc_up[i]) : acc[i];
        const uint64_t at = static_cast<uint64_t>(t.first + m) * p.c_stride + n0 + r;
        if (p.c_f32) p.c_f32[at] = v;
        else p.c_bf16[at] = static_cast<uint16_t>(f32_to_bf16(v));
    }
}

}  // namespace

hipError_t launch_mx_quantize(const void* x, uint32_t dtype, uint64_t stride, uint32_t rows,
                              uint32_t columns, void* codes, void* scales, void* rounded,
                              hipStream_t stream) {
    uint32_t lanes = 4;
    while (lanes < 8u && (8u << lanes) < columns) ++lanes;
    const uint32_t per = kQuantThreads >> lanes, grid = (rows + per - 1u) / per;
    const uint32_t size = dtype == Q38M_DTYPE_F32 ? 4u : 2u;
    const bool whole = reinterpret_cast<uintptr_t>(x) % 16u == 0u && stride * size % 16u == 0u;
    const bool rounded_whole = reinterpret_cast<uintptr_t>(rounded) % 16u == 0u &&
                               static_cast<uint64_t>(columns) * size % 16u == 0u;
    if (dtype == Q38M_DTYPE_F32)
        mx_quantize_kernel<float><<<grid, kQuantThreads, 0, stream>>>(
            static_cast<const float*>(x), stride, rows, columns, whole, lanes,
            static_cast<uint32_t*>(codes), static_cast<uint32_t*>(scales),
            static_cast<float*>(rounded), rounded_whole);
    else
        mx_quantize_kernel<uint16_t><<<grid, kQuantThreads, 0, stream>>>(
            static_cast<const uint16_t*>(x), stride, rows, columns, whole, lanes,
            static_cast<uint32_t*>(codes), static_cast<uint32_t*>(scales),
            static_cast<uint16_t*>(rounded), rounded_whole);
    return hipGetLastError();
}

namespace {
dim3 product_grid(const MxProduct& p, bool swiglu) {
    const uint32_t n_out = swiglu ? p.n / 2u : p.n;
    const uint32_t tasks = p.offsets ? mx_max_tasks(p.routes, p.experts, 16u)
                                     : (p.routes + 15u) / 16u;
    return dim3((n_out + 15u) / 16u, tasks);
}
}  // namespace

bool mx_product_fits(const MxProduct& p, bool swiglu) {
    if (p.n > (1u << 28) || p.routes > (1u << 28)) return false;
    const dim3 grid = product_grid(p, swiglu);
    return grid.x < (1u << 25) && grid.y < (1u << 16);
}

hipError_t launch_mx_product(const MxProduct& p, bool swiglu, hipStream_t stream) {
    const dim3 grid = product_grid(p, swiglu);
    if (swiglu) mx_product_kernel<true><<<grid, 64, 0, stream>>>(p);
    else mx_product_kernel<false><<<grid, 64, 0, stream>>>(p);
    return hipGetLastError();
}

}  // namespace q38m
