// Rows of a table by id, and the gradient of the table.
//
//   forward    y[i] = scale * table[id[i]]
//   backward   dtable[v] = scale * sum over i with id[i] == v of dy[i]
//
// The backward pass sorts the ids (stable counting sorts of up to 10 bits,
// bucket.cu) and adds each id's rows in their order, so it has no float
// atomics and a result does not depend on timing.  The sorted ids are cut into
// parts of kPart; an id's run that lies in one part is added and stored by
// it, a run over several leaves one fp32 sum per part, which the part that
// the run starts in adds up afterwards (a few ids of a power law hold
// thousands of rows).  Both passes are bound by memory.
//
// An id outside the table gives a row of zeros, no gradient, and the device status.
#include <algorithm>

#include "../../include/spmm_b200.h"
#include "common.cuh"
#include "engine.h"
#include "layer.cuh"
#include "layer.h"

namespace spmmb {

namespace {

constexpr int kPart = 32;      // sorted ids of a part

struct EmbedArgs {
    const void *ids;
    bool wide;
    const void *table;      // backward: dy
    void *out;              // backward: dtable
    const int *order;       // backward: input indexes by id, -1 past the last
    float *partial;         // backward: [2 * parts][width]
    int64_t n, rows, width;
    float scale;
    DevStatus *status;
    __device__ __forceinline__ int64_t id(int64_t i) const
    {
        return wide ? ld_idx(static_cast<const int64_t *>(ids) + i) : ld_idx(static_cast<const int *>(ids) + i);
    }
};

template <typename T, int E> struct Piece {
    static constexpr int kBytes = E * (int)sizeof(T);
    using V = std::conditional_t<kBytes == 16, uint4, std::conditional_t<kBytes == 8, uint2, std::conditional_t<kBytes == 4, unsigned, unsigned short>>>;
    V raw;
    __device__ __forceinline__ void load(const T *p) { raw = __ldg(reinterpret_cast<const V *>(p)); }
    __device__ __forceinline__ void store(T *p) const { *reinterpret_cast<V *>(p) = raw; }
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

// A warp per row.
template <typename T, int E> __global__ void __launch_bounds__(256) embedding_kernel(const EmbedArgs a)
{
    const int lane = threadIdx.x & 31;
    const int64_t warps = (int64_t)gridDim.x * (blockDim.x / 32);
    for (int64_t i = (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32; i < a.n; i += warps) {
        const int64_t id = a.id(i);
        const bool found = id >= 0 && id < a.rows;
        if (!found && lane == 0) raise_status(a.status, SPMM_DEV_BAD_COLUMN, i);
        const T *row = static_cast<const T *>(a.table) + (found ? id : 0) * a.width;
        T *out = static_cast<T *>(a.out) + i * a.width;
#pragma unroll 4
        for (int64_t c = lane * E; c < a.width; c += 32 * E) {
            float f[E];
            Piece<T, E> v;
            if (found) {
                v.load(row + c);
                v.get(f);
            }
#pragma unroll
            for (int e = 0; e < E; ++e) f[e] = found ? f[e] * a.scale : 0.f;
            v.set(f);
            v.store(out + c);
        }
    }
}

// A block per part (and a slice of the columns: blockIdx.y).
template <typename T, int E> __global__ void __launch_bounds__(128) embedding_sum_kernel(const EmbedArgs a)
{
    __shared__ int at[kPart];
    __shared__ int64_t key[kPart + 2];   // of the place before the part, of the part, of the place behind it
    const int64_t first = (int64_t)blockIdx.x * kPart;
    for (int i = threadIdx.x; i < kPart + 2; i += blockDim.x) {
        const int64_t p = first + i - 1;
        const int o = p >= 0 && p < a.n ? a.order[p] : -1;
        key[i] = o >= 0 ? a.id(o) : -1;
        if (i >= 1 && i <= kPart) at[i - 1] = o;
    }
    __syncthreads();
    if (at[0] < 0) return;
    const int64_t c = ((int64_t)blockIdx.y * blockDim.x + threadIdx.x) * E;
    if (c >= a.width) return;
    float sum[E];
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e] = 0.f;
    int run = 0;   // where the run began
#pragma unroll 8
    for (int i = 0; i < kPart; ++i) {
        if (at[i] < 0) break;
        Piece<T, E> v;
        v.load(static_cast<const T *>(a.table) + (int64_t)at[i] * a.width + c);
        float f[E];
        v.get(f);
#pragma unroll
        for (int e = 0; e < E; ++e) sum[e] += f[e];
        const int64_t k = key[i + 1];
        if (i + 1 < kPart && key[i + 2] == k) continue;
        // the run ends here, or with the part
        const bool from_before = run == 0 && key[0] == k, goes_on = i + 1 == kPart && key[kPart + 1] == k;
        if (from_before || goes_on) {
            float *p = a.partial + ((int64_t)blockIdx.x * 2 + (from_before ? 0 : 1)) * a.width + c;
#pragma unroll
            for (int e = 0; e < E; ++e) p[e] = sum[e];
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) sum[e] *= a.scale;
            v.set(sum);
            v.store(static_cast<T *>(a.out) + k * a.width + c);
        }
        run = i + 1;
#pragma unroll
        for (int e = 0; e < E; ++e) sum[e] = 0.f;
    }
}

// Adds the sums of a run that starts in part blockIdx.x and goes on behind it.
template <typename T> __global__ void __launch_bounds__(128) embedding_join_kernel(const EmbedArgs a)
{
    const int64_t part = blockIdx.x, last = (part + 1) * kPart - 1;
    if (last + 1 >= a.n) return;
    const int o = a.order[last], next = a.order[last + 1];
    if (o < 0 || next < 0) return;
    const int64_t k = a.id(o);
    if (a.id(next) != k) return;
    const int64_t first = part * kPart;
    if (first > 0 && a.id(a.order[first]) == k && a.id(a.order[first - 1]) == k) return;   // it starts further up
    // the parts that it goes on in: those whose first id is k
    int64_t end = part + 1;
    for (int more = blockDim.x; more == (int)blockDim.x; end += more) {
        const int64_t p = (end + threadIdx.x) * kPart;
        const int i = p < a.n ? a.order[p] : -1;
        more = __syncthreads_count(i >= 0 && a.id(i) == k);
    }
    const int64_t c = (int64_t)blockIdx.y * blockDim.x + threadIdx.x;
    if (c >= a.width) return;
    float sum = a.partial[(part * 2 + 1) * a.width + c];
#pragma unroll 8
    for (int64_t p = part + 1; p < end; ++p) sum += a.partial[p * 2 * a.width + c];
    static_cast<T *>(a.out)[k * a.width + c] = elem_of<T>(sum * a.scale);
}

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

size_t align256(size_t b) { return (b + 255) & ~size_t(255); }

}  // namespace

cudaError_t launch_embedding(const EmbeddingLaunch &l, cudaStream_t stream)
{
    EmbedArgs a{l.ids, l.itype == SPMM_I64, l.in, l.out, nullptr, nullptr, l.n, l.rows, l.width, l.scale, l.status};
    const unsigned blocks = (unsigned)std::max<int64_t>(1, std::min<int64_t>((l.n + 7) / 8, 32 * (int64_t)device_sm_count()));
    return by_rows(l.dtype, l.width, [&](auto type, auto elems) {
        embedding_kernel<decltype(type), decltype(elems)::value><<<blocks, 256, 0, stream>>>(a);
        return cudaGetLastError();
    });
}

size_t embedding_backward_workspace(int64_t n, int64_t width)
{
    const int64_t parts = (n + kPart - 1) / kPart;
    return 2 * align256((size_t)n * 4) + (size_t)parts * 2 * width * sizeof(float);
}

cudaError_t launch_embedding_backward(const EmbeddingLaunch &l, int64_t skip, void *workspace, cudaStream_t stream)
{
    const size_t size = l.dtype == SPMM_F32 ? 4 : 2;
    cudaError_t e = cudaMemsetAsync(l.out, 0, (size_t)l.rows * l.width * size, stream);
    if (e != cudaSuccess || l.n == 0) return e;
    char *ws = static_cast<char *>(workspace);
    int *orders[2] = {reinterpret_cast<int *>(ws), reinterpret_cast<int *>(ws + align256((size_t)l.n * 4))};
    float *partial = reinterpret_cast<float *>(ws + 2 * align256((size_t)l.n * 4));
    int bits = 1;
    while (bits < 62 && (int64_t(1) << bits) < l.rows) ++bits;
    const int passes = (bits + kBucketBits - 1) / kBucketBits, each = (bits + passes - 1) / passes;
    for (int p = 0; p < passes; ++p) {
        BucketSort s{};
        s.keys = l.ids;
        s.wide = l.itype == SPMM_I64;
        s.order_in = p ? orders[(p - 1) & 1] : nullptr;
        s.n = l.n;
        s.buckets = 1 << each;
        s.shift = p * each;
        s.mask = (1 << each) - 1;
        s.limit = l.rows;
        s.skip = skip;
        s.order = orders[p & 1];
        s.status = l.status;
        if ((e = launch_bucket_sort(s, stream)) != cudaSuccess) return e;
    }
    EmbedArgs a{l.ids, l.itype == SPMM_I64, l.in, l.out, orders[(passes - 1) & 1], partial, l.n, l.rows, l.width, l.scale,
                l.status};
    const unsigned parts = (unsigned)((l.n + kPart - 1) / kPart);
    return by_rows(l.dtype, l.width, [&](auto type, auto elems) {
        using T = decltype(type);
        constexpr int E = decltype(elems)::value;
        const dim3 grid(parts, (unsigned)((l.width + 128 * E - 1) / (128 * E)));
        embedding_sum_kernel<T, E><<<grid, 128, 0, stream>>>(a);
        if (parts > 1) {
            const dim3 join(parts, (unsigned)((l.width + 127) / 128));
            embedding_join_kernel<T><<<join, 128, 0, stream>>>(a);
        }
        return cudaGetLastError();
    });
}

}  // namespace spmmb
