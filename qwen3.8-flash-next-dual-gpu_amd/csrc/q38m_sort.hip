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

// One wave's routes, kSteps times 64 from `first` up to `last`, in registers.
template <uint32_t kSteps>
struct WaveRoutes {
    uint32_t key[kSteps], first, last;

    __device__ WaveRoutes(const int32_t* __restrict__ ids, uint32_t first_, uint32_t last_,
                          uint32_t experts)
        : first(first_), last(last_) {
        int32_t id[kSteps];  // all loads under way at once
#pragma unroll
        for (uint32_t s = 0; s < kSteps; ++s) id[s] = live(s) ? ids[route(s)] : -1;
#pragma unroll
        for (uint32_t s = 0; s < kSteps; ++s) key[s] = route_key(id[s], experts);
    }
    __device__ uint32_t route(uint32_t s) const { return first + 64u * s + (threadIdx.x & 63u); }
    __device__ bool live(uint32_t s) const { return route(s) < last; }

    __device__ void count(uint32_t* counts) const {
#pragma unroll
        for (uint32_t s = 0; s < kSteps; ++s)
            if (live(s)) atomicAdd(&counts[key[s]], 1u);
    }
    // a route's place is its key's next one in `place` (this wave's), advanced as the wave goes
    __device__ void scatter(uint32_t experts, uint32_t* place, uint32_t* __restrict__ packed,
                            uint32_t* __restrict__ inverse) const {
        const uint32_t lane = threadIdx.x & 63u;
#pragma unroll
        for (uint32_t s = 0; s < kSteps; ++s) {
            if (first + 64u * s >= last) break;
            const uint64_t same = equal_lanes<kKeyBits>(key[s], live(s));
            const uint32_t below = __popcll(same & ((1ull << lane) - 1u));
            if (live(s)) {
                const uint32_t at = place[key[s]] + below;
                packed[at] = route(s);
                inverse[route(s)] = key[s] < experts ? at : Q38M_ROUTE_DROPPED;
            }
            // every lane has read its place before the last of each key moves it on
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            if (live(s) && (same >> lane) == 1u) place[key[s]] += below + 1u;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        }
    }
};

// One workgroup sorts everything: each wave counts its own contiguous routes, the counts
// become places by a sum over the waves of a key and over the keys.  What takes its time
// is latency: ids read, LDS counters, the sums, writes (512 tokens, top-10: 9.9 us with
// the ids read again for every step; see the table of cases).
constexpr uint32_t kSmallWaves = 16;
__global__ __launch_bounds__(kSmallWaves * 64) void sort_small_kernel(
    const int32_t* __restrict__ ids, uint32_t routes, uint32_t experts,
    uint32_t* __restrict__ offsets, uint32_t* __restrict__ packed,
    uint32_t* __restrict__ inverse) {
    __shared__ uint32_t place[kSmallWaves][kKeys];
    __shared__ uint32_t sums[kSmallWaves];
    const uint32_t t = threadIdx.x, lane = t & 63u, wave = t >> 6;
    const uint32_t per = (routes + kSmallWaves * 64u - 1u) / (kSmallWaves * 64u) * 64u;
    const uint32_t first = min(wave * per, routes);
    const WaveRoutes<kSortSmallRoutes / (kSmallWaves * 64u)> mine(ids, first, min(first + per, routes), experts);
    for (uint32_t k = lane; k <= experts; k += 64u) place[wave][k] = 0u;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    mine.count(place[wave]);
    __syncthreads();
    // thread t owns key t; where all 1,024 experts are in use the last thread also owns
    // the key of the dropped routes
    uint32_t count[kSmallWaves], total = 0;
#pragma unroll
    for (uint32_t w = 0; w < kSmallWaves; ++w) {
        count[w] = t <= experts ? place[w][t] : 0u;
        total += count[w];
    }
    uint32_t base = group_exclusive_sum<kSmallWaves>(total, sums);
    if (t <= experts) {
        offsets[t] = base;
#pragma unroll
        for (uint32_t w = 0; w < kSmallWaves; ++w) {
            place[w][t] = base;
            base += count[w];
        }
    }
    if (t == kMaxSortExperts - 1u && experts == kMaxSortExperts) {
        offsets[experts] = base;
        for (uint32_t w = 0; w < kSmallWaves; ++w) {
            const uint32_t n = place[w][experts];
            place[w][experts] = base;
            base += n;
        }
    }
    __syncthreads();
    mine.scatter(experts, place[wave], packed, inverse);
}

// The same in three launches over chunks of routes: the chunks' counts; each key's
// counts summed over the chunks in front; the scatter, which sums the keys' totals.
constexpr uint32_t kChunkWaves = 4, kChunkSteps = kSortChunk / (kChunkWaves * 64u);
__global__ __launch_bounds__(kChunkWaves * 64) void sort_count_kernel(
    const int32_t* __restrict__ ids, uint32_t routes, uint32_t experts,
    uint32_t* __restrict__ counts) {
    __shared__ uint32_t count[kKeys];
    const uint32_t first = blockIdx.x * kSortChunk + (threadIdx.x >> 6) * (kChunkSteps * 64u);
    const WaveRoutes<kChunkSteps> mine(ids, first, min(first + kChunkSteps * 64u, routes), experts);
    for (uint32_t k = threadIdx.x; k <= experts; k += kChunkWaves * 64u) count[k] = 0u;
    __syncthreads();
    mine.count(count);
    __syncthreads();
    uint32_t* out = counts + static_cast<size_t>(blockIdx.x) * (experts + 1u);
    for (uint32_t k = threadIdx.x; k <= experts; k += kChunkWaves * 64u) out[k] = count[k];
}

// counts[chunk][key] -> how many of the key lie in the chunks in front; totals[key].  A
// workgroup has 64 keys, a lane each, and its waves a run of chunks each.  (All keys in one
// workgroup, one chunk after the other: 110 us for 327,680 routes.)
constexpr uint32_t kPlaceWaves = 16;
__global__ __launch_bounds__(kPlaceWaves * 64) void sort_place_kernel(
    uint32_t* __restrict__ counts, uint32_t chunks, uint32_t experts, uint32_t* __restrict__ totals) {
    __shared__ uint32_t sums[kPlaceWaves][64];
    const uint32_t lane = threadIdx.x & 63u, wave = threadIdx.x >> 6;
    const uint32_t key = blockIdx.x * 64u + lane, stride = experts + 1u;
    const bool mine = key <= experts;
    const uint32_t per = (chunks + kPlaceWaves - 1u) / kPlaceWaves;
    const uint32_t first = min(wave * per, chunks), last = min(first + per, chunks);
    uint32_t total = 0;
#pragma unroll 8
    for (uint32_t c = first; c < last; ++c) total += mine ? counts[static_cast<size_t>(c) * stride + key] : 0u;
    sums[wave][lane] = total;
    __syncthreads();
    uint32_t base = 0;
    for (uint32_t w = 0; w < wave; ++w) base += sums[w][lane];
    if (!mine) return;
    if (wave == kPlaceWaves - 1u) totals[key] = base + total;
    for (uint32_t c0 = first; c0 < last; c0 += 8u) {  // eight loads under way at once
        uint32_t n[8];
#pragma unroll
        for (uint32_t i = 0; i < 8u; ++i)
            n[i] = c0 + i < last ? counts[static_cast<size_t>(c0 + i) * stride + key] : 0u;
#pragma unroll
        for (uint32_t i = 0; i < 8u; ++i) {
            if (c0 + i < last) counts[static_cast<size_t>(c0 + i) * stride + key] = base;
            base += n[i];
        }
    }
}

__global__ __launch_bounds__(kChunkWaves * 64) void sort_scatter_kernel(
    const int32_t* __restrict__ ids, uint32_t routes, uint32_t experts,
    const uint32_t* __restrict__ counts, const uint32_t* __restrict__ totals,
    uint32_t* __restrict__ offsets, uint32_t* __restrict__ packed, uint32_t* __restrict__ inverse) {
    __shared__ uint32_t place[kChunkWaves][kKeys];
    __shared__ uint32_t sums[kChunkWaves];
    const uint32_t t = threadIdx.x, lane = t & 63u, wave = t >> 6;
    const uint32_t first = blockIdx.x * kSortChunk + wave * (kChunkSteps * 64u);
    const WaveRoutes<kChunkSteps> mine(ids, first, min(first + kChunkSteps * 64u, routes), experts);
    for (uint32_t k = lane; k <= experts; k += 64u) place[wave][k] = 0u;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    mine.count(place[wave]);
    // thread t owns kOwn consecutive keys, which covers all
    constexpr uint32_t kThreads = kChunkWaves * 64u, kOwn = (kKeys + kThreads - 1u) / kThreads;
    const uint32_t* in_front = counts + static_cast<size_t>(blockIdx.x) * (experts + 1u);
    uint32_t total[kOwn], front[kOwn], all = 0;
#pragma unroll
    for (uint32_t i = 0; i < kOwn; ++i) {
        const uint32_t k = t * kOwn + i;
        total[i] = k <= experts ? totals[k] : 0u;
        front[i] = k <= experts ? in_front[k] : 0u;
        all += total[i];
    }
    uint32_t base = group_exclusive_sum<kChunkWaves>(all, sums);  // and the waves' counts are there
#pragma unroll
    for (uint32_t i = 0; i < kOwn; ++i) {
        const uint32_t k = t * kOwn + i;
        if (k > experts) break;
        if (blockIdx.x == 0u) offsets[k] = base;
        uint32_t at = base + front[i];
#pragma unroll
        for (uint32_t w = 0; w < kChunkWaves; ++w) {
            const uint32_t n = place[w][k];
            place[w][k] = at;
            at += n;
        }
        base += total[i];
    }
    __syncthreads();
    mine.scatter(experts, place[wave], packed, inverse);
}

// ---- rows -------------------------------------------------------------------

// kN consecutive values of a row as fp32, and back (one rounding).  kN = 8 is
// 16-byte aligned; kN = 1 takes any row.
template <typename T, uint32_t kN>
struct Piece;

template <uint32_t kN>
struct Piece<float, kN> {
    struct Raw {
        float v[kN];
    };
    __device__ static Raw get(const float* p) {
        Raw r;
        if constexpr (kN == 8u) {
            const float4 a = reinterpret_cast<const float4*>(p)[0];
            const float4 b = reinterpret_cast<const float4*>(p)[1];
            r.v[0] = a.x; r.v[1] = a.y; r.v[2] = a.z; r.v[3] = a.w;
            r.v[4] = b.x; r.v[5] = b.y; r.v[6] = b.z; r.v[7] = b.w;
        } else {
            r.v[0] = *p;
        }
        return r;
    }
    __device__ static void widen(const Raw& r, float* v) {
#pragma unroll
        for (uint32_t i = 0; i < kN; ++i) v[i] = r.v[i];
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
    struct Raw {
        uint32_t d[(kN + 1u) / 2u];
    };
    __device__ static Raw get(const uint16_t* p) {
        Raw r;
        if constexpr (kN == 8u) {
            const uint4 w = *reinterpret_cast<const uint4*>(p);
            r.d[0] = w.x; r.d[1] = w.y; r.d[2] = w.z; r.d[3] = w.w;
        } else {
            r.d[0] = *p;
        }
        return r;
    }
    __device__ static void widen(const Raw& r, float* v) {
#pragma unroll
        for (uint32_t i = 0; i < kN; ++i)
            v[i] = __uint_as_float(i % 2u ? r.d[i / 2u] & 0xffff0000u : r.d[i / 2u] << 16);
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

template <typename T, uint32_t kN>
__device__ __forceinline__ void load_piece(const T* p, float* v) {
    Piece<T, kN>::widen(Piece<T, kN>::get(p), v);
}

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
        load_piece<T, kN>(x + static_cast<size_t>(p.token) * width + c, v);
        for (uint32_t r = 0; r < top_k; ++r)
            if (at[r] < routes)
                Piece<T, kN>::store(rows + static_cast<size_t>(at[r]) * width + c, v);
    }
}

// y[t] = sum over t's kept routes, in rank order, of weight * row.  The rows of kRanks
// routes are under way at once.
template <typename T, uint32_t kN>
__global__ __launch_bounds__(kRowThreads) void unpermute_kernel(
    const T* __restrict__ rows, const uint32_t* __restrict__ inverse,
    const float* __restrict__ weights, uint32_t tokens, uint32_t top_k, uint32_t width,
    uint32_t lanes_log2, T* __restrict__ y) {
    constexpr uint32_t kRanks = sizeof(T) == 2u ? 16u : 8u;
    const RowPlace p = row_place<kN>(lanes_log2);
    if (p.token >= tokens) return;
    const uint32_t routes = tokens * top_k;
    const size_t first = static_cast<size_t>(p.token) * top_k;
    for (uint32_t c = p.column; c < width; c += p.step) {
        float sum[kN] = {};
        for (uint32_t r0 = 0; r0 < top_k; r0 += kRanks) {
            uint32_t at[kRanks];
            float w[kRanks];
#pragma unroll
            for (uint32_t i = 0; i < kRanks; ++i) {
                at[i] = Q38M_ROUTE_DROPPED;
                w[i] = 1.0f;
                if (r0 + i < top_k) {
                    at[i] = inverse[first + r0 + i];
                    if (weights) w[i] = weights[first + r0 + i];
                }
            }
            typename Piece<T, kN>::Raw raw[kRanks];
#pragma unroll
            for (uint32_t i = 0; i < kRanks; ++i) {
                raw[i] = typename Piece<T, kN>::Raw{};
                if (at[i] < routes) raw[i] = Piece<T, kN>::get(rows + static_cast<size_t>(at[i]) * width + c);
            }
#pragma unroll
            for (uint32_t i = 0; i < kRanks; ++i) {
                if (at[i] >= routes) w[i] = 0.0f;  // of a row of zeros
                float v[kN];
                Piece<T, kN>::widen(raw[i], v);
#pragma unroll
                for (uint32_t j = 0; j < kN; ++j) sum[j] = __builtin_fmaf(w[i], v[j], sum[j]);
            }
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
            load_piece<T, kN>(from + c, g);
            if (d_weights) {
                load_piece<T, kN>(rows + row + c, v);
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
    uint32_t* totals = scratch + static_cast<size_t>(chunks) * (experts + 1u);
    sort_count_kernel<<<chunks, kChunkWaves * 64u, 0, stream>>>(ids, routes, experts, scratch);
    sort_place_kernel<<<(experts + 64u) / 64u, kPlaceWaves * 64u, 0, stream>>>(scratch, chunks, experts, totals);
    sort_scatter_kernel<<<chunks, kChunkWaves * 64u, 0, stream>>>(ids, routes, experts, scratch, totals,
                                                                  offsets, packed, inverse);
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
