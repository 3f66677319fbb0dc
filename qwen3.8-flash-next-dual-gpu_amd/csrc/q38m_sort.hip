// Tokens sorted by expert and back: the stable sort of routes by expert, the
// token rows brought into that order, the experts' rows summed back with the
// router's weights, and the gradients of both directions.
//
// A route is a (token, rank) pair, numbered token * top_k + rank.  Sorted by
// (expert, route number) the kept routes get the packed places 0, 1, ...; a
// route whose id names no expert is dropped: its order entry lies behind the
// last expert's and its inverse is Q38M_ROUTE_DROPPED.
#include <initializer_list>

#include "q38m_device.h"
#include "q38m_internal.h"

namespace q38m {

namespace {

// Lanes of this wave whose key equals this lane's: one ballot per key bit.
template <uint32_t kBits>
__device__ __forceinline__ uint64_t equal_lanes(uint32_t key, bool live) {
    uint64_t mask = __ballot(live);
#pragma unroll
    for (uint32_t b = 0; b < kBits; ++b) {
        const bool set = (key >> b) & 1u;
        const uint64_t with = __ballot(set);
        mask &= set ? with : ~with;
    }
    return mask;
}

// the ids' sort key: the expert, or `experts` for a dropped route
__device__ __forceinline__ uint32_t route_key(int32_t id, uint32_t experts) {
    return static_cast<uint32_t>(id) < experts ? static_cast<uint32_t>(id) : experts;
}

constexpr uint32_t kKeyBits = 11;  // keys 0 .. kMaxSortExperts
constexpr uint32_t kKeys = kMaxSortExperts + 1u;
static_assert(kKeys <= (1u << kKeyBits), "key bits");

// Exclusive sum of `v` over a workgroup of kWaves waves.
template <uint32_t kWaves>
__device__ uint32_t group_exclusive_sum(uint32_t v, uint32_t* wave_sums) {
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    uint32_t sum = v;
#pragma unroll
    for (uint32_t d = 1; d < 64u; d <<= 1) {
        const uint32_t up = __shfl_up(sum, d);
        if (lane >= d) sum += up;
    }
    if (lane == 63u) wave_sums[wave] = sum;
    __syncthreads();
    uint32_t base = 0;
    for (uint32_t w = 0; w < wave; ++w) base += wave_sums[w];
    return base + sum - v;
}

// Scatters one wave's routes [first, last), in order: a route's place is its
// key's next one in `place` (this wave's row), advanced as the wave goes.
__device__ __forceinline__ void scatter_routes(const int32_t* __restrict__ ids, uint32_t first,
                                               uint32_t last, uint32_t experts, uint32_t* place,
                                               uint32_t* __restrict__ packed,
                                               uint32_t* __restrict__ inverse) {
    const uint32_t lane = threadIdx.x & 63u;
    for (uint32_t r0 = first; r0 < last; r0 += 64u) {
        const uint32_t r = r0 + lane;
        const bool live = r < last;
        const uint32_t key = live ? route_key(ids[r], experts) : experts;
        const uint64_t same = equal_lanes<kKeyBits>(key, live);
        const uint32_t below = __popcll(same & ((1ull << lane) - 1u));
        if (live) {
            const uint32_t at = place[key] + below;
            packed[at] = r;
            inverse[r] = key < experts ? at : Q38M_ROUTE_DROPPED;
        }
        // every lane has read its place before the last of each key moves it on
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        if (live && (same >> lane) == 1u) place[key] += below + 1u;
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    }
}

// One workgroup sorts everything: each wave counts its own contiguous routes,
// the counts become places by a sum over the waves of a key and over the keys.
constexpr uint32_t kSmallWaves = 16;
__global__ __launch_bounds__(kSmallWaves * 64) void sort_small_kernel(
    const int32_t* __restrict__ ids, uint32_t routes, uint32_t experts,
    uint32_t* __restrict__ offsets, uint32_t* __restrict__ packed,
    uint32_t* __restrict__ inverse) {
    __shared__ uint32_t place[kSmallWaves][kKeys];
    __shared__ uint32_t sums[kSmallWaves];
    const uint32_t t = threadIdx.x, lane = t & 63u, wave = t >> 6;
    const uint32_t per = (routes + kSmallWaves * 64u - 1u) / (kSmallWaves * 64u) * 64u;
    const uint32_t first = min(wave * per, routes), last = min(first + per, routes);
    for (uint32_t k = lane; k <= experts; k += 64u) place[wave][k] = 0u;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (uint32_t r = first + lane; r < last; r += 64u)
        atomicAdd(&place[wave][route_key(ids[r], experts)], 1u);
    __syncthreads();
    // thread t owns key t; key kMaxSortExperts (dropped, all experts in use)
    // is placed behind the rest by thread 0 below
    uint32_t total = 0;
    if (t <= experts)
        for (uint32_t w = 0; w < kSmallWaves; ++w) total += place[w][t];
    uint32_t base = group_exclusive_sum<kSmallWaves>(total, sums);
    if (t <= experts) {
        offsets[t] = base;
        for (uint32_t w = 0; w < kSmallWaves; ++w) {
            const uint32_t n = place[w][t];
            place[w][t] = base;
            base += n;
        }
    }
    if (t == kMaxSortExperts - 1u && experts == kMaxSortExperts) {
        offsets[experts] = base;  // the last expert's end
        for (uint32_t w = 0; w < kSmallWaves; ++w) {
            const uint32_t n = place[w][experts];
            place[w][experts] = base;
            base += n;
        }
    }
    __syncthreads();
    scatter_routes(ids, first, last, experts, place[wave], packed, inverse);
}

// The same in three launches over chunks of routes.
constexpr uint32_t kChunkWaves = 4;
__global__ __launch_bounds__(kChunkWaves * 64) void sort_count_kernel(
    const int32_t* __restrict__ ids, uint32_t routes, uint32_t experts,
    uint32_t* __restrict__ counts) {
    __shared__ uint32_t count[kKeys];
    for (uint32_t k = threadIdx.x; k <= experts; k += kChunkWaves * 64u) count[k] = 0u;
    __syncthreads();
    const uint32_t first = blockIdx.x * kSortChunk, last = min(first + kSortChunk, routes);
    for (uint32_t r = first + threadIdx.x; r < last; r += kChunkWaves * 64u)
        atomicAdd(&count[route_key(ids[r], experts)], 1u);
    __syncthreads();
    uint32_t* out = counts + static_cast<size_t>(blockIdx.x) * (experts + 1u);
    for (uint32_t k = threadIdx.x; k <= experts; k += kChunkWaves * 64u) out[k] = count[k];
}

// counts[chunk][key] -> the place of the chunk's first route of the key
__global__ __launch_bounds__(1024) void sort_place_kernel(uint32_t* __restrict__ counts,
                                                          uint32_t chunks, uint32_t experts,
                                                          uint32_t* __restrict__ offsets) {
    __shared__ uint32_t sums[16];
    const uint32_t t = threadIdx.x, stride = experts + 1u;
    const bool mine = t <= experts;
    uint32_t total = 0;
    if (mine)
        for (uint32_t c = 0; c < chunks; ++c) total += counts[static_cast<size_t>(c) * stride + t];
    uint32_t base = group_exclusive_sum<16>(total, sums);
    // with all 1,024 experts in use the last thread places the dropped ones too
    const uint32_t keys = t == kMaxSortExperts - 1u && experts == kMaxSortExperts ? 2u : 1u;
    if (!mine) return;
    for (uint32_t k = t; k < t + keys; ++k) {
        offsets[k] = base;
        for (uint32_t c = 0; c < chunks; ++c) {
            uint32_t* at = &counts[static_cast<size_t>(c) * stride + k];
            const uint32_t n = *at;
            *at = base;
            base += n;
        }
    }
}

__global__ __launch_bounds__(kChunkWaves * 64) void sort_scatter_kernel(
    const int32_t* __restrict__ ids, uint32_t routes, uint32_t experts,
    const uint32_t* __restrict__ places, uint32_t* __restrict__ packed,
    uint32_t* __restrict__ inverse) {
    __shared__ uint32_t place[kChunkWaves][kKeys];
    const uint32_t t = threadIdx.x, lane = t & 63u, wave = t >> 6;
    constexpr uint32_t per = kSortChunk / kChunkWaves;
    const uint32_t begin = blockIdx.x * kSortChunk;
    const uint32_t first = min(begin + wave * per, routes), last = min(first + per, routes);
    for (uint32_t k = lane; k <= experts; k += 64u) place[wave][k] = 0u;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    for (uint32_t r = first + lane; r < last; r += 64u)
        atomicAdd(&place[wave][route_key(ids[r], experts)], 1u);
    __syncthreads();
    const uint32_t* from = places + static_cast<size_t>(blockIdx.x) * (experts + 1u);
    for (uint32_t k = t; k <= experts; k += kChunkWaves * 64u) {
        uint32_t base = from[k];
        for (uint32_t w = 0; w < kChunkWaves; ++w) {
            const uint32_t n = place[w][k];
            place[w][k] = base;
            base += n;
        }
    }
    __syncthreads();
    scatter_routes(ids, first, last, experts, place[wave], packed, inverse);
}

// ---- rows -------------------------------------------------------------------

// kN consecutive values of a row as fp32, and back (one rounding).  kN = 8 is
// 16-byte aligned; kN = 1 takes any row.
template <typename T, uint32_t kN>
struct Piece;

template <uint32_t kN>
struct Piece<float, kN> {
    __device__ static void load(const float* p, float* v) {
        if constexpr (kN == 8u) {
            const float4 a = reinterpret_cast<const float4*>(p)[0];
            const float4 b = reinterpret_cast<const float4*>(p)[1];
            v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w;
            v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
        } else {
            v[0] = *p;
        }
    }
    __device__ static void store(float* p, const float* v) {
        if constexpr (kN == 8u) {
            reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
            reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
        } else {
            *p = v[0];
        }
    }
};

template <uint32_t kN>
struct Piece<uint16_t, kN> {
    __device__ static void load(const uint16_t* p, float* v) {
        if constexpr (kN == 8u) {
            const uint4 w = *reinterpret_cast<const uint4*>(p);
            const uint32_t d[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i) {
                v[2 * i] = __uint_as_float(d[i] << 16);
                v[2 * i + 1] = __uint_as_float(d[i] & 0xffff0000u);
            }
        } else {
            v[0] = bf16_to_f32(*p);
        }
    }
    __device__ static void store(uint16_t* p, const float* v) {
        if constexpr (kN == 8u) {
            uint32_t d[4];
#pragma unroll
            for (uint32_t i = 0; i < 4u; ++i)
                d[i] = f32_to_bf16(v[2 * i]) | f32_to_bf16(v[2 * i + 1]) << 16;
            *reinterpret_cast<uint4*>(p) = make_uint4(d[0], d[1], d[2], d[3]);
        } else {
            *p = static_cast<uint16_t>(f32_to_bf16(v[0]));
        }
    }
};

constexpr uint32_t kRowThreads = 256;

// A workgroup takes kRowThreads / lanes tokens, `lanes` (a power of two)
// threads each, which walk the row kN values a thread.
struct RowPlace {
    uint32_t token, column, step;
};
template <uint32_t kN>
__device__ __forceinline__ RowPlace row_place(uint32_t lanes_log2) {
    const uint32_t lanes = 1u << lanes_log2;
    return RowPlace{blockIdx.x * (kRowThreads >> lanes_log2) + (threadIdx.x >> lanes_log2),
                    (threadIdx.x & (lanes - 1u)) * kN, lanes * kN};
}

// rows[inverse[t k + r]] = x[t] for every kept route
template <typename T, uint32_t kN>
__global__ __launch_bounds__(kRowThreads) void permute_kernel(
    const T* __restrict__ x, const uint32_t* __restrict__ inverse, uint32_t tokens,
    uint32_t top_k, uint32_t width, uint32_t lanes_log2, T* __restrict__ rows) {
    const RowPlace p = row_place<kN>(lanes_log2);
    if (p.token >= tokens) return;
    const uint32_t routes = tokens * top_k;
    const uint32_t* at = inverse + static_cast<size_t>(p.token) * top_k;
    for (uint32_t c = p.column; c < width; c += p.step) {
        float v[kN];
        Piece<T, kN>::load(x + static_cast<size_t>(p.token) * width + c, v);
        for (uint32_t r = 0; r < top_k; ++r)
            if (at[r] < routes)
                Piece<T, kN>::store(rows + static_cast<size_t>(at[r]) * width + c, v);
    }
}

// y[t] = sum over t's kept routes, in rank order, of weight * row
template <typename T, uint32_t kN>
__global__ __launch_bounds__(kRowThreads) void unpermute_kernel(
    const T* __restrict__ rows, const uint32_t* __restrict__ inverse,
    const float* __restrict__ weights, uint32_t tokens, uint32_t top_k, uint32_t width,
    uint32_t lanes_log2, T* __restrict__ y) {
    const RowPlace p = row_place<kN>(lanes_log2);
    if (p.token >= tokens) return;
    const uint32_t routes = tokens * top_k;
    const size_t first = static_cast<size_t>(p.token) * top_k;
    for (uint32_t c = p.column; c < width; c += p.step) {
        float sum[kN] = {};
        for (uint32_t r = 0; r < top_k; ++r) {
            const uint32_t at = inverse[first + r];
            if (at >= routes) continue;
            const float w = weights ? weights[first + r] : 1.0f;
            float v[kN];
            Piece<T, kN>::load(rows + static_cast<size_t>(at) * width + c, v);
#pragma unroll
            for (uint32_t i = 0; i < kN; ++i) sum[i] = __builtin_fmaf(w, v[i], sum[i]);
        }
        Piece<T, kN>::store(y + static_cast<size_t>(p.token) * width + c, sum);
    }
}

// One wave per route: d_rows[at] = w dy[t], d_weights[route] = <dy[t], rows[at]>
template <typename T, uint32_t kN>
__global__ __launch_bounds__(kRowThreads) void unpermute_backward_kernel(
    const T* __restrict__ dy, const T* __restrict__ rows, const uint32_t* __restrict__ inverse,
    const float* __restrict__ weights, uint32_t routes, uint32_t top_k, uint32_t width,
    T* __restrict__ d_rows, float* __restrict__ d_weights) {
    const uint32_t route = blockIdx.x * (kRowThreads / 64u) + (threadIdx.x >> 6);
    const uint32_t lane = threadIdx.x & 63u;
    if (route >= routes) return;
    const uint32_t at = inverse[route];
    float dot = 0.0f;
    if (at < routes) {
        const float w = weights[route];
        const T* from = dy + static_cast<size_t>(route / top_k) * width;
        const size_t row = static_cast<size_t>(at) * width;
        for (uint32_t c = lane * kN; c < width; c += 64u * kN) {
            float g[kN], v[kN];
            Piece<T, kN>::load(from + c, g);
            if (d_weights) {
                Piece<T, kN>::load(rows + row + c, v);
#pragma unroll
                for (uint32_t i = 0; i < kN; ++i) dot = __builtin_fmaf(g[i], v[i], dot);
            }
            if (d_rows) {
#pragma unroll
                for (uint32_t i = 0; i < kN; ++i) g[i] *= w;
                Piece<T, kN>::store(d_rows + row + c, g);
            }
        }
    }
    if (!d_weights) return;
#pragma unroll
    for (uint32_t d = 32u; d != 0u; d >>= 1) dot += __shfl_xor(dot, d);
    if (lane == 0u) d_weights[route] = dot;
}

// 16-byte pieces where every row starts on one
bool whole_pieces(uint32_t width, std::initializer_list<const void*> ptrs) {
    if (width % 8u != 0u) return false;
    for (const void* p : ptrs)
        if (reinterpret_cast<uintptr_t>(p) % 16u != 0u) return false;
    return true;
}

uint32_t row_lanes_log2(uint32_t width, uint32_t piece) {
    uint32_t log2 = 0;
    while (log2 < 8u && (piece << log2) < width) ++log2;
    return log2;
}

uint32_t row_grid(uint32_t tokens, uint32_t lanes_log2) {
    const uint32_t per = kRowThreads >> lanes_log2;
    return (tokens + per - 1u) / per;
}

template <typename T>
hipError_t permute(const T* x, const uint32_t* inverse, uint32_t tokens, uint32_t top_k,
                   uint32_t width, T* rows, hipStream_t stream) {
    if (whole_pieces(width, {x, rows})) {
        const uint32_t lanes = row_lanes_log2(width, 8u);
        permute_kernel<T, 8><<<row_grid(tokens, lanes), kRowThreads, 0, stream>>>(
            x, inverse, tokens, top_k, width, lanes, rows);
    } else {
        const uint32_t lanes = row_lanes_log2(width, 1u);
        permute_kernel<T, 1><<<row_grid(tokens, lanes), kRowThreads, 0, stream>>>(
            x, inverse, tokens, top_k, width, lanes, rows);
    }
    return hipGetLastError();
}

template <typename T>
hipError_t unpermute(const T* rows, const uint32_t* inverse, const float* weights,
                     uint32_t tokens, uint32_t top_k, uint32_t width, T* y, hipStream_t stream) {
    if (whole_pieces(width, {rows, y})) {
        const uint32_t lanes = row_lanes_log2(width, 8u);
        unpermute_kernel<T, 8><<<row_grid(tokens, lanes), kRowThreads, 0, stream>>>(
            rows, inverse, weights, tokens, top_k, width, lanes, y);
    } else {
        const uint32_t lanes = row_lanes_log2(width, 1u);
        unpermute_kernel<T, 1><<<row_grid(tokens, lanes), kRowThreads, 0, stream>>>(
            rows, inverse, weights, tokens, top_k, width, lanes, y);
    }
    return hipGetLastError();
}

template <typename T>
hipError_t unpermute_backward(const T* dy, const T* rows, const uint32_t* inverse,
                              const float* weights, uint32_t tokens, uint32_t top_k,
                              uint32_t width, T* d_rows, float* d_weights, hipStream_t stream) {
    const uint32_t routes = tokens * top_k;
    const uint32_t grid = (routes + kRowThreads / 64u - 1u) / (kRowThreads / 64u);
    if (whole_pieces(width, {dy, rows, d_rows}))
        unpermute_backward_kernel<T, 8><<<grid, kRowThreads, 0, stream>>>(
            dy, rows, inverse, weights, routes, top_k, width, d_rows, d_weights);
    else
        unpermute_backward_kernel<T, 1><<<grid, kRowThreads, 0, stream>>>(
            dy, rows, inverse, weights, routes, top_k, width, d_rows, d_weights);
    return hipGetLastError();
}

}  // namespace

hipError_t launch_sort_routes(const int32_t* ids, uint32_t routes, uint32_t experts,
                              uint32_t* offsets, uint32_t* packed, uint32_t* inverse,
                              uint32_t* scratch, hipStream_t stream) {
    if (routes <= kSortSmallRoutes) {
        sort_small_kernel<<<1, kSmallWaves * 64u, 0, stream>>>(ids, routes, experts, offsets,
                                                               packed, inverse);
        return hipGetLastError();
    }
    const uint32_t chunks = sort_chunks(routes);
    sort_count_kernel<<<chunks, kChunkWaves * 64u, 0, stream>>>(ids, routes, experts, scratch);
    sort_place_kernel<<<1, 1024, 0, stream>>>(scratch, chunks, experts, offsets);
    sort_scatter_kernel<<<chunks, kChunkWaves * 64u, 0, stream>>>(ids, routes, experts, scratch,
                                                                  packed, inverse);
    return hipGetLastError();
}

hipError_t launch_permute_rows(const void* x, uint32_t dtype, const uint32_t* inverse,
                               uint32_t tokens, uint32_t top_k, uint32_t width, void* rows,
                               hipStream_t stream) {
    if (dtype == Q38M_DTYPE_F32)
        return permute(static_cast<const float*>(x), inverse, tokens, top_k, width,
                       static_cast<float*>(rows), stream);
    return permute(static_cast<const uint16_t*>(x), inverse, tokens, top_k, width,
                   static_cast<uint16_t*>(rows), stream);
}

hipError_t launch_unpermute_rows(const void* rows, uint32_t dtype, const uint32_t* inverse,
                                 const float* weights, uint32_t tokens, uint32_t top_k,
                                 uint32_t width, void* y, hipStream_t stream) {
    if (dtype == Q38M_DTYPE_F32)
        return unpermute(static_cast<const float*>(rows), inverse, weights, tokens, top_k, width,
                         static_cast<float*>(y), stream);
    return unpermute(static_cast<const uint16_t*>(rows), inverse, weights, tokens, top_k, width,
                     static_cast<uint16_t*>(y), stream);
}

hipError_t launch_unpermute_backward(const void* dy, const void* rows, uint32_t dtype,
                                     const uint32_t* inverse, const float* weights,
                                     uint32_t tokens, uint32_t top_k, uint32_t width,
                                     void* d_rows, float* d_weights, hipStream_t stream) {
    if (dtype == Q38M_DTYPE_F32)
        return unpermute_backward(static_cast<const float*>(dy), static_cast<const float*>(rows),
                                  inverse, weights, tokens, top_k, width,
                                  static_cast<float*>(d_rows), d_weights, stream);
    return unpermute_backward(static_cast<const uint16_t*>(dy),
                              static_cast<const uint16_t*>(rows), inverse, weights, tokens, top_k,
                              width, static_cast<uint16_t*>(d_rows), d_weights, stream);
}

}  // namespace q38m
