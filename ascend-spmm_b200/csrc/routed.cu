// Rows to their experts and back.
//
//   dispatch   rows[r] = x[source[r] / k]                    (source < 0: zeros)
//   combine    y[t] = sum_j w[t, j] rows[position[t, j]]      (position < 0: nothing; no weights: ones)
//   backward   drows[r] = w[source[r]] dy[source[r] / k],  dw[t, j] = <rows[position[t, j]], dy[t]>
//
// position [tokens, k] and source [tokens * k] are each other's inverse (see
// bucket.cu).  Dispatch and the unweighted combine are each other's gradient.
// All are bound by memory.  A team of lanes owns a token and has up to four
// vectors a lane of each row in flight.  Rows whose width is no multiple of 16
// bytes start anywhere; they are stored in whole vectors between a few loose
// elements and read as pairs of vectors (vec.cuh).
//
// Measured (TB/s of the bytes above; a plain copy reaches 6.5): 32771 rows of
// 1024 bf16, eight choices, dispatch 93 us 6.4, combine 110 us 5.5, backward
// 209 us 5.5; 55507 rows of 477, seven choices, 103 us 4.1, 135 us 3.1, 253 us
// 3.1; nine rows of 1024, four choices, 3 us each, the launch.
#include <algorithm>

#include "../../include/spmm_b200.h"
#include "common.cuh"
#include "engine.h"
#include "layer.cuh"
#include "layer.h"
#include "vec.cuh"

namespace spmmb {

namespace {

constexpr unsigned kFull = 0xffffffffu;

struct RowsArgs {
    const void *x;          // dispatch: [tokens, width]; combine: rows
    const void *grad;       // combine's backward
    void *out;              // may be null in combine's backward
    const int *position, *source;
    const float *weights;   // may be null
    float *dweights;        // may be null
    int64_t tokens, width;
    int k;
    int lanes;              // of a row's team
    DevStatus *status;
};

// A valid position, -1 where there is none.
__device__ __forceinline__ int place_of(const RowsArgs &a, int64_t choice)
{
    const int p = __ldg(a.position + choice);
    if (p < -1 || p >= a.tokens * a.k) {
        raise_status(a.status, SPMM_DEV_BAD_COLUMN, choice);
        return -1;
    }
    return p;
}

// Vectors of a row that a lane has in flight, and blocks of 256 threads on an
// SM.  Rows that are read as pairs of vectors take registers for each, and
// more warps pay more there: combine of 55507 rows of 477 bf16, seven choices,
// with four vectors and two blocks 253 us, two and four 156, one and six 135.
// 32771 aligned rows of 1024, eight choices, with four vectors and two, three,
// four blocks 129, 107, 159 us.
constexpr int at_once(bool aligned) { return aligned ? 4 : 1; }
constexpr int blocks_per_sm(bool aligned) { return aligned ? 3 : 6; }

// A row's team of lanes (a power of two) among those of the grid: as many as
// have the row in flight at once, so that narrow rows share a warp.
struct Team {
    int lanes, lane;
    int64_t index, count;
    __device__ __forceinline__ Team(int lanes)
        : lanes(lanes), lane(threadIdx.x & (lanes - 1)),
          index(((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / lanes), count((int64_t)gridDim.x * blockDim.x / lanes)
    {
    }
};

// Zeros in the rows without a source.
template <bool ALIGNED, typename T> __device__ __forceinline__ void zero_rows(const RowsArgs &a, const Team &team)
{
    const int64_t total = a.tokens * a.k, warps = (int64_t)gridDim.x * (blockDim.x / 32);
    const int lane = threadIdx.x & 31;
    constexpr int kChunk = 8;   // rows that a warp looks at together: those of a plan lie at the end, one after the other
    for (int64_t r = ((int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32) * kChunk; r < total; r += warps * kChunk) {
        unsigned empty = __ballot_sync(kFull, lane < kChunk && r + lane < total && __ldg(a.source + r + lane) < 0);
        while (empty) {   // the warp's teams take the next one each
            unsigned mine = empty;
            for (int i = 0; i < 32 / team.lanes; ++i) {
                if (i < lane / team.lanes) mine &= mine - 1;
                empty &= empty - 1;
            }
            if (!mine) continue;
            T *out = static_cast<T *>(a.out) + (r + __ffs(mine) - 1) * a.width;
            const RowSpan<ALIGNED, T> span(out, a.width);
            for (int64_t c = team.lane; c < span.vectors; c += team.lanes)
                __stcs(reinterpret_cast<uint4 *>(out + span.head) + c, make_uint4(0, 0, 0, 0));
            for (int64_t i = team.lane; i < span.loose(a.width); i += team.lanes) out[span.loose_at(i)] = elem_of<T>(0.f);
        }
    }
}

template <bool ALIGNED, typename T> __global__ void __launch_bounds__(256, blocks_per_sm(ALIGNED)) dispatch_kernel(const RowsArgs a)
{
    constexpr int kAtOnce = at_once(ALIGNED);
    constexpr int kElems = Pack16<T>::kElems;
    const Team team(a.lanes);
    for (int64_t t = team.index; t < a.tokens; t += team.count) {
        const T *x = static_cast<const T *>(a.x) + t * a.width;
        if constexpr (ALIGNED) {
            const int64_t vectors = a.width / kElems;
            for (int64_t c0 = team.lane; c0 < vectors; c0 += team.lanes * kAtOnce) {
                Pack16<T> v[kAtOnce];
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i)
                    if (c0 + i * team.lanes < vectors) v[i].raw = __ldcs(reinterpret_cast<const uint4 *>(x) + c0 + i * team.lanes);
                for (int j = 0; j < a.k; ++j) {
                    const int p = place_of(a, t * a.k + j);
                    if (p < 0) continue;
                    uint4 *out = reinterpret_cast<uint4 *>(static_cast<T *>(a.out) + p * a.width);
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i)
                        if (c0 + i * team.lanes < vectors) __stcs(out + c0 + i * team.lanes, v[i].raw);
                }
            }
        } else {
            // whole vectors start at another place in each result: the row is read again for each choice (from L1)
            for (int j = 0; j < a.k; ++j) {
                const int p = place_of(a, t * a.k + j);
                if (p < 0) continue;
                T *out = static_cast<T *>(a.out) + p * a.width;
                const RowSpan<false, T> span(out, a.width);
                for (int64_t c0 = team.lane; c0 < span.vectors; c0 += team.lanes * kAtOnce) {
                    Pack16<T> v[kAtOnce];
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i)
                        if (c0 + i * team.lanes < span.vectors)
                            v[i] = load16<false>(x + span.head + (c0 + i * team.lanes) * kElems);
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i)
                        if (c0 + i * team.lanes < span.vectors)
                            __stcs(reinterpret_cast<uint4 *>(out + span.head) + c0 + i * team.lanes, v[i].raw);
                }
                for (int64_t i = team.lane; i < span.loose(a.width); i += team.lanes) out[span.loose_at(i)] = x[span.loose_at(i)];
            }
        }
    }
    zero_rows<ALIGNED, T>(a, team);
}

// WHOLE: a team is a warp.
template <bool ALIGNED, bool WHOLE, typename T>
__global__ void __launch_bounds__(256, blocks_per_sm(ALIGNED)) combine_kernel(const RowsArgs a)
{
    constexpr int kAtOnce = at_once(ALIGNED);
    constexpr int kElems = Pack16<T>::kElems;
    const Team team(a.lanes);
    const T *rows = static_cast<const T *>(a.x);
    for (int64_t t = team.index; t < a.tokens; t += team.count) {
        T *y = static_cast<T *>(a.out) + t * a.width;
        const RowSpan<ALIGNED, T> span(y, a.width);
        auto weight_of = [&](int j) { return a.weights ? __ldg(a.weights + t * a.k + j) : 1.f; };
        // kAtOnce vectors a lane of each row: a warp reads 2 KB of it in one go
        for (int64_t c0 = team.lane; c0 - (WHOLE ? team.lane : 0) < span.vectors; c0 += team.lanes * kAtOnce) {
            float sum[kAtOnce][kElems];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
                for (int e = 0; e < kElems; ++e) sum[i][e] = 0.f;
            auto add = [&](int p, float w) {
                if (p < 0) return;
                const T *row = rows + p * a.width + span.head;
                Pack16<T> v[kAtOnce];
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) {   // past the last one (whole warps): read again and not stored
                    const int64_t c = c0 + i * team.lanes;
                    v[i].raw = make_uint4(0, 0, 0, 0);
                    if (WHOLE || c < span.vectors) v[i] = load16<ALIGNED>(row + (WHOLE ? min(c, span.vectors - 1) : c) * kElems);
                }
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) {
                    float f[kElems];
                    v[i].get(f);
#pragma unroll
                    for (int e = 0; e < kElems; ++e) sum[i][e] = fmaf(w, f[e], sum[i][e]);
                }
            };
            if constexpr (WHOLE) {   // a lane reads a choice's position, the others get it from there
                for (int first = 0; first < a.k; first += 32) {
                    const int count = min(32, a.k - first);
                    int place = -1;
                    float weight = 1.f;
                    if (team.lane < count) {
                        place = place_of(a, t * a.k + first + team.lane);
                        weight = weight_of(first + team.lane);
                    }
#pragma unroll 2
                    for (int j = 0; j < count; ++j) add(__shfl_sync(kFull, place, j), __shfl_sync(kFull, weight, j));
                }
            } else {
                constexpr int kAhead = 4;   // choices whose positions are read at once
                for (int j0 = 0; j0 < a.k; j0 += kAhead) {
                    int p[kAhead];
                    float w[kAhead];
#pragma unroll
                    for (int j = 0; j < kAhead; ++j) {
                        p[j] = j0 + j < a.k ? place_of(a, t * a.k + j0 + j) : -1;
                        w[j] = j0 + j < a.k ? weight_of(j0 + j) : 0.f;
                    }
#pragma unroll
                    for (int j = 0; j < kAhead; ++j) add(p[j], w[j]);
                }
            }
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i)
                if (c0 + i * team.lanes < span.vectors) {
                    Pack16<T> v;
                    v.set(sum[i]);
                    __stcs(reinterpret_cast<uint4 *>(y + span.head) + c0 + i * team.lanes, v.raw);
                }
        }
        for (int64_t i = team.lane; i < span.loose(a.width); i += team.lanes) {
            const int64_t c = span.loose_at(i);
            float sum = 0.f;
            for (int j = 0; j < a.k; ++j) {
                const int p = place_of(a, t * a.k + j);
                if (p >= 0) sum = fmaf(weight_of(j), elem_f32<T>(rows[p * a.width + c]), sum);
            }
            y[c] = elem_of<T>(sum);
        }
    }
}

// A team per choice: the token's gradient is in L1 or L2 for the others.
template <bool ALIGNED, typename T>
__global__ void __launch_bounds__(256, 8) combine_backward_kernel(const RowsArgs a)
{
    constexpr int kAtOnce = 1;   // with 32 registers a thread: 211 us for 32771 rows of 1024 bf16, eight choices (four: 225)
    constexpr int kElems = Pack16<T>::kElems;
    const Team team(a.lanes);
    const int64_t choices = a.tokens * a.k;
    for (int64_t i0 = team.index - team.index % (32 / team.lanes); i0 < choices; i0 += team.count) {
        const int64_t i = i0 + team.index % (32 / team.lanes);   // the warp's teams take the same turns
        const int64_t p = i < choices ? place_of(a, i) : -1;
        float dot = 0.f;
        if (p >= 0) {
            const float w = a.weights ? __ldg(a.weights + i) : 1.f;
            const T *dy = static_cast<const T *>(a.grad) + i / a.k * a.width;
            const T *row = static_cast<const T *>(a.x) + p * a.width;
            T *out = static_cast<T *>(a.out) + p * a.width;   // where it is wanted; rows and drows are alike aligned
            const RowSpan<ALIGNED, T> span(row, a.width);
            for (int64_t c0 = team.lane; c0 < span.vectors; c0 += team.lanes * kAtOnce) {
                Pack16<T> gv[kAtOnce], fv[kAtOnce];
#pragma unroll
                for (int n = 0; n < kAtOnce; ++n) {
                    const int64_t c = c0 + n * team.lanes;
                    gv[n].raw = fv[n].raw = make_uint4(0, 0, 0, 0);
                    if (c < span.vectors) {
                        gv[n] = load16<ALIGNED>(dy + span.head + c * kElems);
                        if (a.dweights) fv[n].raw = __ldcs(reinterpret_cast<const uint4 *>(row + span.head) + c);
                    }
                }
#pragma unroll
                for (int n = 0; n < kAtOnce; ++n) {
                    const int64_t c = c0 + n * team.lanes;
                    float g[kElems], f[kElems];
                    gv[n].get(g);
                    fv[n].get(f);
#pragma unroll
                    for (int e = 0; e < kElems; ++e) dot = fmaf(f[e], g[e], dot);
#pragma unroll
                    for (int e = 0; e < kElems; ++e) g[e] *= w;
                    gv[n].set(g);
                    if (a.out && c < span.vectors) __stcs(reinterpret_cast<uint4 *>(out + span.head) + c, gv[n].raw);
                }
            }
            for (int64_t n = team.lane; n < span.loose(a.width); n += team.lanes) {
                const int64_t at = span.loose_at(n);
                const float g = elem_f32<T>(dy[at]);
                if (a.dweights) dot = fmaf(elem_f32<T>(row[at]), g, dot);
                if (a.out) out[at] = elem_of<T>(g * w);
            }
        }
        if (a.dweights) {
            for (int o = team.lanes / 2; o > 0; o >>= 1) dot += __shfl_xor_sync(kFull, dot, o);
            if (team.lane == 0 && i < choices) a.dweights[i] = dot;
        }
    }
    if (a.out) zero_rows<ALIGNED, T>(a, team);
}

// Calls f with whether every row starts on 16 bytes, and the type.
template <typename F> cudaError_t by_rows(int dtype, int64_t width, F f)
{
    auto run = [&](auto type) {
        return width * (int)sizeof(type) % 16 == 0 ? f(std::true_type(), type) : f(std::false_type(), type);
    };
    switch (dtype) {
        case SPMM_F16: return run(__half());
        case SPMM_BF16: return run(__nv_bfloat16());
        default: return run(float());
    }
}

RowsArgs args_of(const RoutedLaunch &r)
{
    RowsArgs a{r.x, r.grad, r.out, r.position, r.source, r.weights, r.dweights, r.tokens, r.width, r.k, 2, r.status};
    const int64_t bytes = r.width * (r.dtype == SPMM_F32 ? 4 : 2);
    while (a.lanes < 32 && a.lanes * at_once(bytes % 16 == 0) < bytes / 16) a.lanes *= 2;
    return a;
}

// Blocks of 256 threads for `items` teams, and for the sources (eight a warp).
unsigned blocks_for(const RowsArgs &a, int64_t items)
{
    const int64_t threads = std::max(items * a.lanes, a.source ? a.tokens * a.k * 4 : 0);
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>((threads + 255) / 256, 32 * (int64_t)device_sm_count()));
}

}  // namespace

cudaError_t launch_dispatch(const RoutedLaunch &r, cudaStream_t stream)
{
    const RowsArgs a = args_of(r);
    return by_rows(r.dtype, r.width, [&](auto aligned, auto type) {
        dispatch_kernel<decltype(aligned)::value, decltype(type)><<<blocks_for(a, r.tokens), 256, 0, stream>>>(a);
        return cudaGetLastError();
    });
}

cudaError_t launch_combine(const RoutedLaunch &r, cudaStream_t stream)
{
    const RowsArgs a = args_of(r);
    return by_rows(r.dtype, r.width, [&](auto aligned, auto type) {
        constexpr bool kAligned = decltype(aligned)::value;
        auto kernel = kAligned && a.lanes == 32 ? combine_kernel<kAligned, kAligned, decltype(type)>
                                                : combine_kernel<kAligned, false, decltype(type)>;
        kernel<<<blocks_for(a, r.tokens), 256, 0, stream>>>(a);
        return cudaGetLastError();
    });
}

cudaError_t launch_combine_backward(const RoutedLaunch &r, cudaStream_t stream)
{
    const RowsArgs a = args_of(r);
    return by_rows(r.dtype, r.width, [&](auto aligned, auto type) {
        combine_backward_kernel<decltype(aligned)::value, decltype(type)><<<blocks_for(a, r.tokens * r.k), 256, 0, stream>>>(a);
        return cudaGetLastError();
    });
}

}  // namespace spmmb
