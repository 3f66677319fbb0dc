// Tokens sorted by expert and back: the stable sort of routes by expert, the
// token rows brought into that order, the experts' rows summed back with the
// router's weights, and the gradients of both directions.
//
// A route is a (token, rank) pair, numbered token * top_k + rank.  Sorted by
// (expert, route number) the kept routes get the packed places 0, 1, ...; a
// route whose id names no expert is dropped: its order entry lies behind the
// last expert's and its inverse is Q38M_ROUTE_DROPPED.
#include <algorithm>
#include <type_traits>

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
// is latency: ids read, LDS counters, the sums, writes (512 tokens, top-10, whose bytes
// would take 0.01 us: 8.2 us; with the ids read again for every step 9.9).
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
// counts summed over the chunks in front; the scatter, which sums the keys' totals.  327,680
// routes of 512 experts: 4.7, 6.3 and 6.0 us, all latency (their 5 MB would take 1 us).
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

// 16 bytes at any element (a row of odd width starts anywhere)
typedef uint32_t v4u_any __attribute__((ext_vector_type(4), aligned(2)));

// kN consecutive values of a row, and as fp32 (back: one rounding): 16 bytes, or one value
// of a row that is narrower.  kStream: past the caches.  (Eight values of fp32, two
// instructions that touch every second 16 bytes each: 2,929 x 10 rows of 2,048 sorted, there
// and back 142 us instead of 138.  Rows of odd widths a value a lane: 9,983 x 10 rows of 601
// bf16 126 us instead of 60.)
template <typename T, uint32_t kN>
struct Piece {
    static constexpr uint32_t kWords = (kN * sizeof(T) + 3u) / 4u;
    static_assert(kN == 1u || kWords == 4u, "a value or 16 bytes");
    uint32_t d[kWords];

    template <bool kStream>
    __device__ static Piece get(const T* p) {
        Piece r;
        if constexpr (kN != 1u) {
            v4u_any w;
            if constexpr (kStream) w = __builtin_nontemporal_load(reinterpret_cast<const v4u_any*>(p));
            else w = *reinterpret_cast<const v4u_any*>(p);
            r.d[0] = w.x, r.d[1] = w.y, r.d[2] = w.z, r.d[3] = w.w;
        } else if constexpr (sizeof(T) == 4u) {
            r.d[0] = __float_as_uint(*p);
        } else {
            r.d[0] = *p;
        }
        return r;
    }
    template <bool kStream>
    __device__ void put(T* p) const {
        if constexpr (kN != 1u) {
            const v4u_any w = {d[0], d[1], d[2], d[3]};
            if constexpr (kStream) __builtin_nontemporal_store(w, reinterpret_cast<v4u_any*>(p));
            else *reinterpret_cast<v4u_any*>(p) = w;
        } else if constexpr (sizeof(T) == 4u) {
            *p = __uint_as_float(d[0]);
        } else {
            *p = static_cast<T>(d[0]);
        }
    }
    __device__ void widen(float* v) const {
#pragma unroll
        for (uint32_t i = 0; i < kN; ++i) {
            if constexpr (sizeof(T) == 4u) v[i] = __uint_as_float(d[i]);
            else v[i] = __uint_as_float(i % 2u ? d[i / 2u] & 0xffff0000u : d[i / 2u] << 16);
        }
    }
    __device__ static Piece round(const float* v) {
        Piece r;
#pragma unroll
        for (uint32_t i = 0; i < kN; ++i) {
            if constexpr (sizeof(T) == 4u) r.d[i] = __float_as_uint(v[i]);
            else if (i % 2u) r.d[i / 2u] |= f32_to_bf16(v[i]) << 16;
            else r.d[i / 2u] = f32_to_bf16(v[i]);
        }
        return r;
    }
};

constexpr uint32_t kRowThreads = 256;

// whether an inverse entry is a place
__device__ __forceinline__ bool in_range(uint32_t at, uint32_t routes) {
    report(at >= routes && at != Q38M_ROUTE_DROPPED, kCheckRoute);
    return at < routes;
}

// A workgroup takes kRowThreads / lanes tokens, `lanes` (a power of two)
// threads each, which walk the row kN values a thread.  A row's last piece is
// its last kN values, in part those of the piece in front: written twice, with
// the same bits.
struct RowPlace {
    uint32_t token, column, step;
};
template <uint32_t kN>
__device__ __forceinline__ RowPlace row_place(uint32_t lanes_log2) {
    const uint32_t lanes = 1u << lanes_log2;
    return RowPlace{blockIdx.x * (kRowThreads >> lanes_log2) + (threadIdx.x >> lanes_log2),
                    (threadIdx.x & (lanes - 1u)) * kN, lanes * kN};
}

// rows[inverse[t k + r]] = x[t] for every kept route: a token is read once and written
// top_k times.  32,768 x 10 rows of 2,048 bf16: 257 us, 5.7 TB/s of 1.48 GB, nearly all of
// it writes.
template <typename T, uint32_t kN, bool kStream>
__global__ __launch_bounds__(kRowThreads) void permute_kernel(
    const T* __restrict__ x, const uint32_t* __restrict__ inverse, uint32_t tokens,
    uint32_t top_k, uint32_t width, uint32_t lanes_log2, T* __restrict__ rows) {
    const RowPlace p = row_place<kN>(lanes_log2);
    if (p.token >= tokens) return;
    const uint32_t routes = tokens * top_k;
    const uint32_t* at = inverse + static_cast<size_t>(p.token) * top_k;
    for (uint32_t c0 = p.column; c0 < width; c0 += p.step) {
        const uint32_t c = min(c0, width - kN);
        const auto v = Piece<T, kN>::template get<false>(x + static_cast<size_t>(p.token) * width + c);
        for (uint32_t r = 0; r < top_k; ++r)
            if (in_range(at[r], routes)) v.template put<kStream>(rows + static_cast<size_t>(at[r]) * width + c);
    }
}

// y[t] = sum over t's kept routes, in rank order, of weight * row.  The rows of kRanks
// routes are under way at once; y goes past the caches (21 MB of rows: 4.3 us, cached 5.0).
// 32,768 x 10 rows of 2,048 bf16: 239 us, 6.2 TB/s of 1.48 GB.
template <typename T, uint32_t kN, bool kStream>
__global__ __launch_bounds__(kRowThreads) void unpermute_kernel(
    const T* __restrict__ rows, const uint32_t* __restrict__ inverse,
    const float* __restrict__ weights, uint32_t tokens, uint32_t top_k, uint32_t width,
    uint32_t lanes_log2, T* __restrict__ y) {
    constexpr uint32_t kRanks = 16;
    const RowPlace p = row_place<kN>(lanes_log2);
    if (p.token >= tokens) return;
    const uint32_t routes = tokens * top_k;
    const size_t first = static_cast<size_t>(p.token) * top_k;
    for (uint32_t c0 = p.column; c0 < width; c0 += p.step) {
        const uint32_t c = min(c0, width - kN);
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
            Piece<T, kN> row[kRanks];
#pragma unroll
            for (uint32_t i = 0; i < kRanks; ++i) {
                row[i] = Piece<T, kN>{};
                if (in_range(at[i], routes))
                    row[i] = Piece<T, kN>::template get<kStream>(rows + static_cast<size_t>(at[i]) * width + c);
            }
#pragma unroll
            for (uint32_t i = 0; i < kRanks; ++i) {
                if (at[i] >= routes) w[i] = 0.0f;  // of a row of zeros
                float v[kN];
                row[i].widen(v);
#pragma unroll
                for (uint32_t j = 0; j < kN; ++j) sum[j] = __builtin_fmaf(w[i], v[j], sum[j]);
            }
        }
        Piece<T, kN>::round(sum).template put<true>(y + static_cast<size_t>(p.token) * width + c);
    }
}

// d_rows[at] = w dy[t], d_weights[route] = <dy[t], rows[at]>: up to a wave's lanes (a power of
// two) for each route.  dy[t] is read by each of its routes, from the caches but for the first.
// 16,384 x 10 rows of 2,048
// bf16: 275 us, 5.1 TB/s of 1.41 GB, read and written in nearly equal parts, as in a copy,
// which reaches as much.
template <typename T, uint32_t kN, bool kStream>
__global__ __launch_bounds__(kRowThreads) void unpermute_backward_kernel(
    const T* __restrict__ dy, const T* __restrict__ rows, const uint32_t* __restrict__ inverse,
    const float* __restrict__ weights, uint32_t routes, uint32_t top_k, uint32_t width,
    uint32_t lanes_log2, T* __restrict__ d_rows, float* __restrict__ d_weights) {
    const RowPlace p = row_place<kN>(lanes_log2);
    const uint32_t route = p.token;
    if (route >= routes) return;
    const uint32_t at = inverse[route];
    float dot = 0.0f;
    if (in_range(at, routes)) {
        const float w = weights[route];
        const T* from = dy + static_cast<size_t>(route / top_k) * width;
        const size_t row = static_cast<size_t>(at) * width;
        for (uint32_t c0 = p.column; c0 < width; c0 += p.step) {
            const uint32_t c = min(c0, width - kN);
            float g[kN], v[kN];
            Piece<T, kN>::template get<false>(from + c).widen(g);
            if (d_weights) {
                Piece<T, kN>::template get<kStream>(rows + row + c).widen(v);
#pragma unroll
                for (uint32_t i = 0; i < kN; ++i)  // those of the piece in front are in its sum
                    if (c + i >= c0) dot = __builtin_fmaf(g[i], v[i], dot);
            }
            if (d_rows) {
#pragma unroll
                for (uint32_t i = 0; i < kN; ++i) g[i] *= w;
                Piece<T, kN>::round(g).template put<kStream>(d_rows + row + c);
            }
        }
    }
    if (!d_weights) return;
    for (uint32_t d = 1u << lanes_log2 >> 1; d != 0u; d >>= 1) dot += __shfl_xor(dot, d);
    if (p.column == 0u) d_weights[route] = dot;
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

// Calls f with the values a piece has and whether the rows (`sides` of them: read, written or
// both) go past the caches: where they are more than the 256 MB behind the L2s hold.  10 rows
// of 2,048 bf16 a token, cached / past the caches, us: written 20.8 / 23.7 for 120 MB, 139 /
// 128 for 655, 283 / 257 for 1,342; back 20.5 / 21.4, 88.3 / 87.8 (492 MB), 265 / 239; both
// ways in the gradient 288 / 275 for 1,342.
template <typename T, typename F>
void with_piece(uint32_t sides, uint32_t tokens, uint32_t top_k, uint32_t width, F f) {
    constexpr uint64_t kCachedBytes = 256u << 20;
    constexpr std::integral_constant<uint32_t, 16u / sizeof(T)> kWide{};
    constexpr std::integral_constant<uint32_t, 1u> kNarrow{};
    const bool streamed = static_cast<uint64_t>(tokens) * top_k * width * sizeof(T) * sides > kCachedBytes;
    if (width >= kWide.value) {
        if (streamed) f(kWide, std::true_type{});
        else f(kWide, std::false_type{});
    } else {
        f(kNarrow, std::false_type{});
    }
}

template <typename T>
hipError_t permute(const T* x, const uint32_t* inverse, uint32_t tokens, uint32_t top_k,
                   uint32_t width, T* rows, hipStream_t stream) {
    with_piece<T>(1u, tokens, top_k, width, [&](auto piece, auto streamed) {
        constexpr uint32_t kN = decltype(piece)::value;
        const uint32_t lanes = row_lanes_log2(width, kN);
        permute_kernel<T, kN, decltype(streamed)::value><<<row_grid(tokens, lanes), kRowThreads, 0, stream>>>(
            x, inverse, tokens, top_k, width, lanes, rows);
    });
    return hipGetLastError();
}

template <typename T>
hipError_t unpermute(const T* rows, const uint32_t* inverse, const float* weights,
                     uint32_t tokens, uint32_t top_k, uint32_t width, T* y, hipStream_t stream) {
    with_piece<T>(1u, tokens, top_k, width, [&](auto piece, auto streamed) {
        constexpr uint32_t kN = decltype(piece)::value;
        const uint32_t lanes = row_lanes_log2(width, kN);
        unpermute_kernel<T, kN, decltype(streamed)::value><<<row_grid(tokens, lanes), kRowThreads, 0, stream>>>(
            rows, inverse, weights, tokens, top_k, width, lanes, y);
    });
    return hipGetLastError();
}

template <typename T>
hipError_t unpermute_backward(const T* dy, const T* rows, const uint32_t* inverse,
                              const float* weights, uint32_t tokens, uint32_t top_k,
                              uint32_t width, T* d_rows, float* d_weights, hipStream_t stream) {
    with_piece<T>(2u, tokens, top_k, width, [&](auto piece, auto streamed) {
        constexpr uint32_t kN = decltype(piece)::value;
        const uint32_t routes = tokens * top_k, lanes = std::min(row_lanes_log2(width, kN), 6u);
        unpermute_backward_kernel<T, kN, decltype(streamed)::value>
            <<<row_grid(routes, lanes), kRowThreads, 0, stream>>>(
                dy, rows, inverse, weights, routes, top_k, width, lanes, d_rows, d_weights);
    });
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
