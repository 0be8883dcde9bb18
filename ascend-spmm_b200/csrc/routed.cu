// Rows to their experts and back.
//
//   dispatch   rows[r] = x[source[r] / k]                    (source < 0: zeros)
//   combine    y[t] = sum_j w[t, j] rows[position[t, j]]      (position < 0: nothing; no weights: ones)
//   backward   drows[r] = w[source[r]] dy[source[r] / k],  dw[t, j] = <rows[position[t, j]], dy[t]>
//
// position [tokens, k] and source [tokens * k] are each other's inverse (see
// bucket.cu).  Dispatch and the unweighted combine are each other's gradient.
// All are bound by memory.  A warp owns a token: it reads the token's row once
// and has the rows of all of its choices in flight.  Rows whose width is no
// multiple of 16 bytes start anywhere; they are stored in whole vectors
// between a few loose elements and read as pairs of vectors (vec.cuh).
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

// Up to 32 of a token's choices, one per lane.
struct Choices {
    int place = -1;
    float weight = 1.f;
    int count;
    __device__ __forceinline__ Choices(const RowsArgs &a, int64_t token, int first)
    {
        const int lane = threadIdx.x & 31;
        count = min(32, a.k - first);
        if (lane < count) {
            place = place_of(a, token * a.k + first + lane);
            if (a.weights) weight = __ldg(a.weights + token * a.k + first + lane);
        }
    }
    __device__ __forceinline__ int place_at(int j) const { return __shfl_sync(kFull, place, j); }
    __device__ __forceinline__ float weight_at(int j) const { return __shfl_sync(kFull, weight, j); }
};

// Zeros in the rows without a source: a warp per 32 rows.
template <bool ALIGNED, typename T> __device__ __forceinline__ void zero_rows(const RowsArgs &a, int64_t warp, int64_t warps)
{
    const int lane = threadIdx.x & 31;
    const int64_t total = a.tokens * a.k;
    for (int64_t r = warp * 32; r < total; r += warps * 32) {
        unsigned empty = __ballot_sync(kFull, r + lane < total && __ldg(a.source + r + lane) < 0);
        while (empty) {
            T *out = static_cast<T *>(a.out) + (r + __ffs(empty) - 1) * a.width;
            empty &= empty - 1;
            const RowSpan<ALIGNED, T> span(out, a.width);
            for (int64_t c = lane; c < span.vectors; c += 32)
                reinterpret_cast<uint4 *>(out + span.head)[c] = make_uint4(0, 0, 0, 0);
            for (int64_t i = lane; i < span.loose(a.width); i += 32) out[span.loose_at(i)] = elem_of<T>(0.f);
        }
    }
}

constexpr int kAtOnce = 4;   // vectors of a row that a lane has in flight

template <bool ALIGNED, typename T> __global__ void __launch_bounds__(256) dispatch_kernel(const RowsArgs a)
{
    constexpr int kElems = Pack16<T>::kElems;
    const int lane = threadIdx.x & 31;
    const int64_t warp = (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
    const int64_t warps = (int64_t)gridDim.x * (blockDim.x / 32);
    for (int64_t t = warp; t < a.tokens; t += warps) {
        const T *x = static_cast<const T *>(a.x) + t * a.width;
        for (int first = 0; first < a.k; first += 32) {
            const Choices choice(a, t, first);
            // the token's row, kAtOnce vectors a lane at a time; whole vectors of a result start at another place in each
            // row where rows are not aligned, so that there a row is read again for each choice (from L1)
            for (int64_t c0 = 0; ALIGNED && c0 < a.width; c0 += 32 * kElems * kAtOnce) {
                Pack16<T> v[kAtOnce];
#pragma unroll
                for (int i = 0; i < kAtOnce; ++i) {
                    const int64_t c = c0 + (32 * i + lane) * kElems;
                    if (c < a.width) v[i].raw = __ldcs(reinterpret_cast<const uint4 *>(x + c));
                }
                for (int j = 0; j < choice.count; ++j) {
                    const int p = choice.place_at(j);
                    if (p < 0) continue;
                    T *out = static_cast<T *>(a.out) + p * a.width;
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i) {
                        const int64_t c = c0 + (32 * i + lane) * kElems;
                        if (c < a.width) __stcs(reinterpret_cast<uint4 *>(out + c), v[i].raw);
                    }
                }
            }
            for (int j = 0; !ALIGNED && j < choice.count; ++j) {
                const int p = choice.place_at(j);
                if (p < 0) continue;
                T *out = static_cast<T *>(a.out) + p * a.width;
                const RowSpan<false, T> span(out, a.width);
                for (int64_t c0 = lane; c0 < span.vectors; c0 += 32 * kAtOnce) {
                    Pack16<T> v[kAtOnce];
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i)   // past the last one: it is read again
                        v[i] = load16<false>(x + span.head + min(c0 + 32 * i, span.vectors - 1) * kElems);
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i)
                        if (c0 + 32 * i < span.vectors) __stcs(reinterpret_cast<uint4 *>(out + span.head) + c0 + 32 * i, v[i].raw);
                }
                if (lane < span.loose(a.width)) out[span.loose_at(lane)] = x[span.loose_at(lane)];
            }
        }
    }
    zero_rows<ALIGNED, T>(a, warp, warps);
}

template <bool ALIGNED, typename T> __global__ void __launch_bounds__(256) combine_kernel(const RowsArgs a)
{
    constexpr int kElems = Pack16<T>::kElems;
    const int lane = threadIdx.x & 31;
    const int64_t warps = (int64_t)gridDim.x * (blockDim.x / 32);
    for (int64_t t = (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32; t < a.tokens; t += warps) {
        T *y = static_cast<T *>(a.out) + t * a.width;
        const T *rows = static_cast<const T *>(a.x);
        const RowSpan<ALIGNED, T> span(y, a.width);
        // kAtOnce vectors a lane of each row: a warp reads 2 KB of it in one go
        for (int64_t c0 = lane; c0 - lane < span.vectors; c0 += 32 * kAtOnce) {
            float sum[kAtOnce][kElems];
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i)
#pragma unroll
                for (int e = 0; e < kElems; ++e) sum[i][e] = 0.f;
            for (int first = 0; first < a.k; first += 32) {
                const Choices choice(a, t, first);
#pragma unroll 2
                for (int j = 0; j < choice.count; ++j) {
                    const int p = choice.place_at(j);
                    const float w = choice.weight_at(j);
                    if (p < 0) continue;
                    const T *row = rows + p * a.width + span.head;
                    Pack16<T> v[kAtOnce];
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i)   // past the last one: read again and not stored
                        v[i] = load16<ALIGNED>(row + min(c0 + 32 * i, span.vectors - 1) * kElems);
#pragma unroll
                    for (int i = 0; i < kAtOnce; ++i) {
                        float f[kElems];
                        v[i].get(f);
#pragma unroll
                        for (int e = 0; e < kElems; ++e) sum[i][e] = fmaf(w, f[e], sum[i][e]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < kAtOnce; ++i)
                if (c0 + 32 * i < span.vectors) {
                    Pack16<T> v;
                    v.set(sum[i]);
                    __stcs(reinterpret_cast<uint4 *>(y + span.head) + c0 + 32 * i, v.raw);
                }
        }
        if constexpr (!ALIGNED) {
            const bool on = lane < span.loose(a.width);
            const int64_t c = on ? span.loose_at(lane) : 0;
            float sum = 0.f;
            for (int first = 0; first < a.k; first += 32) {
                const Choices choice(a, t, first);
                for (int j = 0; j < choice.count; ++j) {
                    const int p = choice.place_at(j);
                    const float w = choice.weight_at(j);
                    if (p >= 0 && on) sum = fmaf(w, elem_f32<T>(rows[p * a.width + c]), sum);
                }
            }
            if (on) y[c] = elem_of<T>(sum);
        }
    }
}

// A warp per choice: the token's gradient is in L1 or L2 for the others.
template <bool ALIGNED, typename T> __global__ void __launch_bounds__(256) combine_backward_kernel(const RowsArgs a)
{
    constexpr int kElems = Pack16<T>::kElems;
    const int lane = threadIdx.x & 31;
    const int64_t warp = (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
    const int64_t warps = (int64_t)gridDim.x * (blockDim.x / 32);
    for (int64_t i = warp; i < a.tokens * a.k; i += warps) {
        const int64_t t = i / a.k, p = place_of(a, i);
        float dot = 0.f;
        if (p >= 0) {
            const float w = a.weights ? __ldg(a.weights + i) : 1.f;
            const T *dy = static_cast<const T *>(a.grad) + t * a.width;
            const T *row = static_cast<const T *>(a.x) + p * a.width;
            T *out = static_cast<T *>(a.out) + p * a.width;   // where it is wanted; rows and drows are alike aligned
            const RowSpan<ALIGNED, T> span(row, a.width);
            for (int64_t c0 = lane; c0 < span.vectors; c0 += 32 * kAtOnce) {
                Pack16<T> gv[kAtOnce], fv[kAtOnce];
#pragma unroll
                for (int j = 0; j < kAtOnce; ++j) {
                    const int64_t c = c0 + 32 * j;
                    gv[j].raw = fv[j].raw = make_uint4(0, 0, 0, 0);
                    if (c < span.vectors) {
                        gv[j] = load16<ALIGNED>(dy + span.head + c * kElems);
                        if (a.dweights) fv[j].raw = __ldcs(reinterpret_cast<const uint4 *>(row + span.head) + c);
                    }
                }
#pragma unroll
                for (int j = 0; j < kAtOnce; ++j) {
                    const int64_t c = c0 + 32 * j;
                    float g[kElems], f[kElems];
                    gv[j].get(g);
                    fv[j].get(f);
#pragma unroll
                    for (int e = 0; e < kElems; ++e) dot = fmaf(f[e], g[e], dot);
#pragma unroll
                    for (int e = 0; e < kElems; ++e) g[e] *= w;
                    gv[j].set(g);
                    if (a.out && c < span.vectors) __stcs(reinterpret_cast<uint4 *>(out + span.head) + c, gv[j].raw);
                }
            }
            if (lane < span.loose(a.width)) {
                const int64_t at = span.loose_at(lane);
                const float g = elem_f32<T>(dy[at]);
                if (a.dweights) dot = fmaf(elem_f32<T>(row[at]), g, dot);
                if (a.out) out[at] = elem_of<T>(g * w);
            }
        }
        if (a.dweights) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(kFull, dot, o);
            if (lane == 0) a.dweights[i] = dot;
        }
    }
    if (a.out) zero_rows<ALIGNED, T>(a, warp, warps);
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

unsigned warp_blocks(int64_t items)
{
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>((items + 7) / 8, 32 * (int64_t)device_sm_count()));
}

RowsArgs args_of(const RoutedLaunch &r)
{
    return RowsArgs{r.x, r.grad, r.out, r.position, r.source, r.weights, r.dweights, r.tokens, r.width, r.k, r.status};
}

}  // namespace

cudaError_t launch_dispatch(const RoutedLaunch &r, cudaStream_t stream)
{
    return by_rows(r.dtype, r.width, [&](auto aligned, auto type) {
        dispatch_kernel<decltype(aligned)::value, decltype(type)><<<warp_blocks(r.tokens), 256, 0, stream>>>(args_of(r));
        return cudaGetLastError();
    });
}

cudaError_t launch_combine(const RoutedLaunch &r, cudaStream_t stream)
{
    return by_rows(r.dtype, r.width, [&](auto aligned, auto type) {
        combine_kernel<decltype(aligned)::value, decltype(type)><<<warp_blocks(r.tokens), 256, 0, stream>>>(args_of(r));
        return cudaGetLastError();
    });
}

cudaError_t launch_combine_backward(const RoutedLaunch &r, cudaStream_t stream)
{
    return by_rows(r.dtype, r.width, [&](auto aligned, auto type) {
        combine_backward_kernel<decltype(aligned)::value, decltype(type)>
            <<<warp_blocks(r.tokens * r.k), 256, 0, stream>>>(args_of(r));
        return cudaGetLastError();
    });
}

}  // namespace spmmb
