// Rows of a table by id, and the gradient of the table.
//
//   forward    y[i] = scale * table[id[i]]
//   backward   dtable[v] = scale * sum over i with id[i] == v of dy[i]
//
// The backward pass sorts the ids (stable counting sorts of up to 10 bits,
// bucket.cu) and adds each id's rows in their order, so it has no float
// atomics and a result does not depend on timing.  The rows without an id are
// zeroed beside the sort, which takes a few SMs.  The sorted ids are cut into
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
#include "vec.cuh"

namespace spmmb {

namespace {

constexpr int kPart = 32;      // sorted ids of a part
constexpr int kJoin = 8;       // groups of threads that add a run's parts side by side

struct EmbedArgs {
    const void *ids;        // forward
    bool wide;
    const void *in;         // the table; backward: dy
    void *out;              // y; backward: dtable
    const int *order;       // backward: input indexes by id, -1 past the last
    const int *sorted;      // backward: their ids
    float *partial;         // backward: [2 * parts][width]
    int64_t n, rows, width;
    float scale;
    DevStatus *status;
};

// A warp per row.
template <bool ALIGNED, typename T> __global__ void __launch_bounds__(256) embedding_kernel(const EmbedArgs a)
{
    constexpr int kElems = Pack16<T>::kElems;
    const int lane = threadIdx.x & 31;
    const int64_t warps = (int64_t)gridDim.x * (blockDim.x / 32);
    for (int64_t i = (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32; i < a.n; i += warps) {
        const int64_t id = a.wide ? ld_idx(static_cast<const int64_t *>(a.ids) + i) : ld_idx(static_cast<const int *>(a.ids) + i);
        const bool found = id >= 0 && id < a.rows;
        if (!found && lane == 0) raise_status(a.status, SPMM_DEV_BAD_COLUMN, i);
        const T *row = static_cast<const T *>(a.in) + (found ? id : 0) * a.width;
        T *out = static_cast<T *>(a.out) + i * a.width;
        const RowSpan<ALIGNED, T> span(out, a.width);
#pragma unroll 4
        for (int64_t c = lane; c < span.vectors; c += 32) {
            Pack16<T> v;
            v.raw = make_uint4(0, 0, 0, 0);
            if (found) {
                float f[kElems];
                load16<ALIGNED>(row + span.head + c * kElems).get(f);
#pragma unroll
                for (int e = 0; e < kElems; ++e) f[e] *= a.scale;
                v.set(f);
            }
            __stcs(reinterpret_cast<uint4 *>(out + span.head) + c, v.raw);
        }
        if (lane < span.loose(a.width)) {
            const int64_t c = span.loose_at(lane);
            out[c] = elem_of<T>(found ? elem_f32<T>(row[c]) * a.scale : 0.f);
        }
    }
}

// E columns of a row from column c on.
template <bool ALIGNED, typename T, int E> __device__ __forceinline__ void load_columns(const T *p, float (&f)[E])
{
    if constexpr (E == 1) f[0] = elem_f32<T>(*p);
    else load16<ALIGNED>(p).get(f);
}
template <bool ALIGNED, typename T, int E> __device__ __forceinline__ void store_columns(T *p, const float (&f)[E])
{
    if constexpr (ALIGNED) {
        Pack16<T> v;
        v.set(f);
        *reinterpret_cast<uint4 *>(p) = v.raw;
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) p[e] = elem_of<T>(f[e]);
    }
}

// The sorted ids `at` (input indexes) of a part, E columns from c on.
// key: the id before the part, the part's, the id behind it.
template <bool ALIGNED, typename T, int E>
__device__ __forceinline__ void sum_part(const EmbedArgs &a, int64_t part, const int *at, const int *key, int64_t c)
{
    const T *dy = static_cast<const T *>(a.in) + c;
    float sum[E];
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e] = 0.f;
    bool first = true;   // the run is the part's first
    constexpr int kAhead = 8;
#pragma unroll
    for (int i0 = 0; i0 < kPart; i0 += kAhead) {
        if (at[i0] < 0) break;
        float f[kAhead][E];
#pragma unroll
        for (int j = 0; j < kAhead; ++j)   // past the last one: the row is read again and not added
            load_columns<ALIGNED, T, E>(dy + (int64_t)max(at[i0 + j], 0) * a.width, f[j]);
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int i = i0 + j;
            if (at[i] < 0) break;
#pragma unroll
            for (int e = 0; e < E; ++e) sum[e] += f[j][e];
            const int k = key[i + 1];
            if (i + 1 < kPart && key[i + 2] == k) continue;
            // the run ends here, or with the part
            const bool from_before = first && key[0] == k, goes_on = i + 1 == kPart && key[kPart + 1] == k;
            if (from_before || goes_on) {
                float *p = a.partial + (part * 2 + (from_before ? 0 : 1)) * a.width + c;
#pragma unroll
                for (int e = 0; e < E; ++e) p[e] = sum[e];
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) sum[e] *= a.scale;
                store_columns<ALIGNED, T, E>(static_cast<T *>(a.out) + (int64_t)k * a.width + c, sum);
            }
            first = false;
#pragma unroll
            for (int e = 0; e < E; ++e) sum[e] = 0.f;
        }
    }
}

// A block per part (and a slice of the columns: blockIdx.y).
template <bool ALIGNED, typename T> __global__ void __launch_bounds__(128) embedding_sum_kernel(const EmbedArgs a)
{
    constexpr int kElems = Pack16<T>::kElems;
    __shared__ int at[kPart], key[kPart + 2];
    const int64_t part = blockIdx.x, first = part * kPart;
    for (int i = threadIdx.x; i < kPart + 2; i += blockDim.x) {
        const int64_t p = first + i - 1;
        const bool in = p >= 0 && p < a.n;
        key[i] = in ? a.sorted[p] : -1;
        if (i >= 1 && i <= kPart) at[i - 1] = in ? a.order[p] : -1;
    }
    __syncthreads();
    const int64_t vectors = a.width / kElems, t = (int64_t)blockIdx.y * blockDim.x + threadIdx.x;
    if (t < vectors) {
        sum_part<ALIGNED, T, kElems>(a, part, at, key, t * kElems);
    } else if (!ALIGNED && t - vectors < a.width - vectors * kElems) {   // the columns behind the last whole vector
        sum_part<false, T, 1>(a, part, at, key, vectors * kElems + t - vectors);
    }
}

// Adds the sums of a run that starts in part blockIdx.x and goes on behind it:
// 32 columns a block, kJoin warps with every kJoin-th part each, in a fixed order.
template <typename T> __global__ void __launch_bounds__(32 * kJoin) embedding_join_kernel(const EmbedArgs a)
{
    __shared__ float sums[kJoin][32];
    const int64_t part = blockIdx.x, last = (part + 1) * kPart - 1;
    if (last + 1 >= a.n) return;
    const int k = a.sorted[last];
    if (k < 0 || a.sorted[last + 1] != k) return;
    const int64_t first = part * kPart;
    if (first > 0 && a.sorted[first] == k && a.sorted[first - 1] == k) return;   // it starts further up
    // the parts that it goes on in: those whose first id is k
    int64_t end = part + 1;
    for (int more = blockDim.x; more == (int)blockDim.x; end += more) {
        const int64_t p = (end + threadIdx.x) * kPart;
        more = __syncthreads_count(p < a.n && a.sorted[p] == k);
    }
    const int group = threadIdx.x / 32;
    for (int64_t c0 = (int64_t)blockIdx.y * 32; c0 < a.width; c0 += (int64_t)gridDim.y * 32) {
        const int64_t c = c0 + threadIdx.x % 32;
        float sum = 0.f;
        if (c < a.width) {
            if (group == 0) sum = a.partial[(part * 2 + 1) * a.width + c];
#pragma unroll 8
            for (int64_t p = part + 1 + group; p < end; p += kJoin) sum += a.partial[p * 2 * a.width + c];
        }
        sums[group][threadIdx.x % 32] = sum;
        __syncthreads();
        if (group == 0 && c < a.width) {
#pragma unroll
            for (int g = 1; g < kJoin; ++g) sum += sums[g][threadIdx.x];
            static_cast<T *>(a.out)[(int64_t)k * a.width + c] = elem_of<T>(sum * a.scale);
        }
        __syncthreads();
    }
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

size_t align256(size_t b) { return (b + 255) & ~size_t(255); }

}  // namespace

cudaError_t launch_embedding(const EmbeddingLaunch &l, cudaStream_t stream)
{
    EmbedArgs a{};
    a.ids = l.ids; a.wide = l.itype == SPMM_I64; a.in = l.in; a.out = l.out; a.n = l.n; a.rows = l.rows;
    a.width = l.width; a.scale = l.scale; a.status = l.status;
    const unsigned blocks = (unsigned)std::max<int64_t>(1, std::min<int64_t>((l.n + 7) / 8, 32 * (int64_t)device_sm_count()));
    return by_rows(l.dtype, l.width, [&](auto aligned, auto type) {
        embedding_kernel<decltype(aligned)::value, decltype(type)><<<blocks, 256, 0, stream>>>(a);
        return cudaGetLastError();
    });
}

size_t embedding_backward_workspace(int64_t n, int64_t width)
{
    const int64_t parts = (n + kPart - 1) / kPart;
    return 4 * align256((size_t)n * 4) + (size_t)parts * 2 * width * sizeof(float);
}

cudaError_t launch_embedding_backward(const EmbeddingLaunch &l, int64_t skip, void *workspace, cudaStream_t stream)
{
    const size_t bytes = (size_t)l.rows * l.width * (l.dtype == SPMM_F32 ? 4 : 2);
    cudaError_t e;
    if (l.n == 0) return cudaMemsetAsync(l.out, 0, bytes, stream);
    if (bytes % 16)   // the sort writes whole vectors of zeros
        if ((e = cudaMemsetAsync(static_cast<char *>(l.out) + bytes / 16 * 16, 0, bytes % 16, stream)) != cudaSuccess) return e;
    char *ws = static_cast<char *>(workspace);
    int *array[4];   // order and ids of two passes
    for (int i = 0; i < 4; ++i) array[i] = reinterpret_cast<int *>(ws + i * align256((size_t)l.n * 4));
    int bits = 1;
    while (bits < 31 && (int64_t(1) << bits) < l.rows) ++bits;
    const int passes = (bits + kBucketBits - 1) / kBucketBits, each = (bits + passes - 1) / passes;
    const int64_t vectors = (int64_t)(bytes / 16);
    for (int p = 0; p < passes; ++p) {
        BucketSort s{};
        s.keys = p ? static_cast<const void *>(array[2 + (p - 1) % 2]) : l.ids;
        s.wide = p == 0 && l.itype == SPMM_I64;
        s.order_in = p ? array[(p - 1) % 2] : nullptr;
        s.n = l.n;
        s.buckets = 1 << each;
        s.shift = p * each;
        s.mask = (1 << each) - 1;
        s.limit = l.rows;
        s.skip = skip;
        s.order = array[p % 2];
        s.key_out = array[2 + p % 2];
        s.zero = static_cast<uint4 *>(l.out) + vectors * p / passes;   // a share of the zeros beside each pass
        s.zero_vectors = vectors * (p + 1) / passes - vectors * p / passes;
        s.status = l.status;
        if ((e = launch_bucket_sort(s, stream)) != cudaSuccess) return e;
    }
    EmbedArgs a{};
    a.in = l.in; a.out = l.out; a.order = array[(passes - 1) % 2]; a.sorted = array[2 + (passes - 1) % 2];
    a.partial = reinterpret_cast<float *>(ws + 4 * align256((size_t)l.n * 4));
    a.n = l.n; a.rows = l.rows; a.width = l.width; a.scale = l.scale; a.status = l.status;
    const unsigned parts = (unsigned)((l.n + kPart - 1) / kPart);
    return by_rows(l.dtype, l.width, [&](auto aligned, auto type) {
        using T = decltype(type);
        constexpr bool kAligned = decltype(aligned)::value;
        constexpr int kElems = Pack16<T>::kElems;
        const int64_t threads = l.width / kElems + l.width % kElems;
        embedding_sum_kernel<kAligned, T><<<dim3(parts, (unsigned)((threads + 127) / 128)), 128, 0, stream>>>(a);
        if (parts > 1)
            embedding_join_kernel<T><<<dim3(parts, (unsigned)std::min<int64_t>((l.width + 31) / 32, 64)), 32 * kJoin, 0, stream>>>(a);
        return cudaGetLastError();
    });
}

}  // namespace spmmb
