// Rows to their experts and back.
//
//   dispatch   rows[r] = x[source[r] / k]                    (source < 0: zeros)
//   combine    y[t] = sum_j w[t, j] rows[position[t, j]]      (position < 0: nothing; no weights: ones)
//   backward   drows[r] = w[source[r]] dy[source[r] / k],  dw[t, j] = <rows[position[t, j]], dy[t]>
//
// position [tokens, k] and source [tokens * k] are each other's inverse (see
// bucket.cu).  Dispatch and the unweighted combine are each other's gradient.
// All are bound by memory.
#include <algorithm>

#include "../../include/spmm_b200.h"
#include "common.cuh"
#include "engine.h"
#include "layer.cuh"
#include "layer.h"

namespace spmmb {

namespace {

constexpr unsigned kFull = 0xffffffffu;

// E consecutive elements as one access.
template <typename T, int E> struct Piece {
    static constexpr int kBytes = E * (int)sizeof(T);
    using V = std::conditional_t<kBytes == 16, uint4, std::conditional_t<kBytes == 8, uint2, std::conditional_t<kBytes == 4, unsigned, unsigned short>>>;
    V raw;
    __device__ __forceinline__ void load(const T *p) { raw = __ldg(reinterpret_cast<const V *>(p)); }
    __device__ __forceinline__ void store(T *p) const { *reinterpret_cast<V *>(p) = raw; }
    __device__ __forceinline__ void zero() { raw = V{}; }
    __device__ __forceinline__ void get(float *f) const
    {
        const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
        for (int i = 0; i < E; ++i) f[i] = elem_f32<T>(e[i]);
    }
    __device__ __forceinline__ void set(const float *f)
    {
        T *e = reinterpret_cast<T *>(&raw);
#pragma unroll
        for (int i = 0; i < E; ++i) e[i] = elem_of<T>(f[i]);
    }
};

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
__device__ __forceinline__ int64_t place_of(const RowsArgs &a, int64_t choice)
{
    const int p = __ldg(a.position + choice);
    if (p < -1 || p >= a.tokens * a.k) {
        raise_status(a.status, SPMM_DEV_BAD_COLUMN, choice);
        return -1;
    }
    return p;
}

// Zeros in the rows without a source: a warp per 32 rows.
template <typename T, int E> __device__ __forceinline__ void zero_rows(const RowsArgs &a, int64_t warp, int64_t warps)
{
    const int lane = threadIdx.x & 31;
    const int64_t total = a.tokens * a.k;
    for (int64_t r = warp * 32; r < total; r += warps * 32) {
        unsigned empty = __ballot_sync(kFull, r + lane < total && __ldg(a.source + r + lane) < 0);
        while (empty) {
            const int64_t row = r + __ffs(empty) - 1;
            empty &= empty - 1;
            Piece<T, E> z;
            z.zero();
            for (int64_t c = lane * E; c < a.width; c += 32 * E) z.store(static_cast<T *>(a.out) + row * a.width + c);
        }
    }
}

template <typename T, int E> __global__ void __launch_bounds__(256) dispatch_kernel(const RowsArgs a)
{
    const int lane = threadIdx.x & 31;
    const int64_t warp = (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
    const int64_t warps = (int64_t)gridDim.x * (blockDim.x / 32);
    for (int64_t t = warp; t < a.tokens; t += warps) {
        const T *x = static_cast<const T *>(a.x) + t * a.width;
        for (int64_t c = lane * E; c < a.width; c += 32 * E) {
            Piece<T, E> v;
            v.load(x + c);
            for (int j = 0; j < a.k; ++j) {
                const int64_t p = place_of(a, t * a.k + j);
                if (p >= 0) v.store(static_cast<T *>(a.out) + p * a.width + c);
            }
        }
    }
    zero_rows<T, E>(a, warp, warps);
}

template <typename T, int E> __global__ void __launch_bounds__(256) combine_kernel(const RowsArgs a)
{
    const int lane = threadIdx.x & 31;
    const int64_t warp = (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32;
    const int64_t warps = (int64_t)gridDim.x * (blockDim.x / 32);
    for (int64_t t = warp; t < a.tokens; t += warps) {
        for (int64_t c = lane * E; c < a.width; c += 32 * E) {
            float sum[E];
#pragma unroll
            for (int i = 0; i < E; ++i) sum[i] = 0.f;
#pragma unroll 4
            for (int j = 0; j < a.k; ++j) {
                const int64_t p = place_of(a, t * a.k + j);
                if (p < 0) continue;
                const float w = a.weights ? __ldg(a.weights + t * a.k + j) : 1.f;
                Piece<T, E> v;
                v.load(static_cast<const T *>(a.x) + p * a.width + c);
                float f[E];
                v.get(f);
#pragma unroll
                for (int i = 0; i < E; ++i) sum[i] = fmaf(w, f[i], sum[i]);
            }
            Piece<T, E> y;
            y.set(sum);
            y.store(static_cast<T *>(a.out) + t * a.width + c);
        }
    }
}

// A warp per choice.
template <typename T, int E> __global__ void __launch_bounds__(256) combine_backward_kernel(const RowsArgs a)
{
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
            T *out = static_cast<T *>(a.out) + p * a.width;
            for (int64_t c = lane * E; c < a.width; c += 32 * E) {
                Piece<T, E> v;
                float g[E];
                v.load(dy + c);
                v.get(g);
                if (a.dweights) {
                    float f[E];
                    v.load(row + c);
                    v.get(f);
#pragma unroll
                    for (int e = 0; e < E; ++e) dot = fmaf(f[e], g[e], dot);
                }
                if (a.out) {
#pragma unroll
                    for (int e = 0; e < E; ++e) g[e] *= w;
                    v.set(g);
                    v.store(out + c);
                }
            }
        }
        if (a.dweights) {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) dot += __shfl_xor_sync(kFull, dot, o);
            if (lane == 0) a.dweights[i] = dot;
        }
    }
    if (a.out) zero_rows<T, E>(a, warp, warps);
}

// Calls f with the type and the elements of the widest access that every row's start allows.
template <typename F> cudaError_t by_rows(int dtype, int64_t width, F f)
{
    auto run = [&](auto type) {
        using T = decltype(type);
        constexpr int kSize = (int)sizeof(T);
        if (width * kSize % 16 == 0) return f(type, std::integral_constant<int, 16 / kSize>());
        if (width * kSize % 8 == 0) return f(type, std::integral_constant<int, 8 / kSize>());
        if (width * kSize % 4 == 0) return f(type, std::integral_constant<int, 4 / kSize>());
        return f(type, std::integral_constant<int, 1>());
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
    return by_rows(r.dtype, r.width, [&](auto type, auto elems) {
        dispatch_kernel<decltype(type), decltype(elems)::value><<<warp_blocks(r.tokens), 256, 0, stream>>>(args_of(r));
        return cudaGetLastError();
    });
}

cudaError_t launch_combine(const RoutedLaunch &r, cudaStream_t stream)
{
    return by_rows(r.dtype, r.width, [&](auto type, auto elems) {
        combine_kernel<decltype(type), decltype(elems)::value><<<warp_blocks(r.tokens), 256, 0, stream>>>(args_of(r));
        return cudaGetLastError();
    });
}

cudaError_t launch_combine_backward(const RoutedLaunch &r, cudaStream_t stream)
{
    return by_rows(r.dtype, r.width, [&](auto type, auto elems) {
        combine_backward_kernel<decltype(type), decltype(elems)::value>
            <<<warp_blocks(r.tokens * r.k), 256, 0, stream>>>(args_of(r));
        return cudaGetLastError();
    });
}

}  // namespace spmmb
