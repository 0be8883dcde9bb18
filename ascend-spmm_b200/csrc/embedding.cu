// Rows of a table by id, and the gradient of the table.
//
//   forward    y[i] = scale * table[id[i]]
//   backward   dtable[v] = scale * sum over i with id[i] == v of dy[i]
//
// The backward pass sorts the ids (stable counting sorts of up to 10 bits,
// bucket.cu) and adds each id's rows in their order, so it has no float
// atomics and a result does not depend on timing.  The rows without an id are
// zeroed beside the sort, which takes a few SMs.  The sorted ids are cut into
// parts of kPart; an id's run of at most that many is added and stored by the
// part that it starts in, a longer one leaves an fp32 sum in each of its parts,
// which are added up afterwards (a few ids of a power law hold thousands of
// rows).  Both passes are bound by memory.
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
constexpr int kFew = 8;        // a run over at most so many parts is added up by a warp, a longer one by a block
constexpr int kJoin = 16;      // of so many warps

struct EmbedArgs {
    const void *ids;        // forward
    bool wide;
    const void *in;         // the table; backward: dy
    void *out;              // y; backward: dtable
    const int2 *sorted;     // backward: input indexes and their ids, by id; -1 past the last
    float *partial;         // backward: [2 * parts][width]
    // backward: the numbers of long runs of few parts and of many, then the parts that they start in (in any order), the
    // former from the front and the latter from the back
    int *runs;
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

// The sorted ids of a part, as a block keeps them in shared memory: those
// around it too, since a run of at most kPart rows over a border is added whole
// by the part that it starts in.
struct Part {
    int key[3 * kPart + 2];   // key[kPart + 1 + i]: the id at place i of the part, -1 outside the ids
    int at[2 * kPart];        // input indexes of the part and of kPart places behind it
    int begin, end;           // the places that this part adds
    bool more;                // the last run is longer and goes on: its sum is a partial one
    bool before;              // the first run comes from before: its sum is a partial one
};

// E columns of the part's sums, from column c on.
template <bool ALIGNED, typename T, int E>
__device__ __forceinline__ void sum_part(const EmbedArgs &a, int64_t part, const Part &s, int64_t c)
{
    const T *dy = static_cast<const T *>(a.in) + c;
    const int *key = s.key + kPart + 1;
    float sum[E];
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e] = 0.f;
    bool before = s.before;
    constexpr int kAhead = 8;
    for (int i0 = s.begin; i0 < s.end; i0 += kAhead) {
        float f[kAhead][E];
#pragma unroll
        for (int j = 0; j < kAhead; ++j)   // past the last one: a row is read again and not added
            load_columns<ALIGNED, T, E>(dy + (int64_t)s.at[min(i0 + j, s.end - 1)] * a.width, f[j]);
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int i = i0 + j;
            if (i >= s.end) break;
#pragma unroll
            for (int e = 0; e < E; ++e) sum[e] += f[j][e];
            const int k = key[i];
            if (i + 1 < s.end && key[i + 1] == k) continue;
            const bool more = i + 1 == s.end && s.more;
            if (before || more) {
                float *p = a.partial + (part * 2 + (before ? 0 : 1)) * a.width + c;
#pragma unroll
                for (int e = 0; e < E; ++e) p[e] = sum[e];
                if (!before && c == 0) {
                    const int64_t far = (part + kFew) * kPart, parts = (a.n + kPart - 1) / kPart;
                    const bool many = far < a.n && a.sorted[far].y == k;
                    const int i = atomicAdd(a.runs + many, 1);
                    a.runs[many ? parts + 1 - i : 2 + i] = (int)part;
                }
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) sum[e] *= a.scale;
                store_columns<ALIGNED, T, E>(static_cast<T *>(a.out) + (int64_t)k * a.width + c, sum);
            }
            before = false;
#pragma unroll
            for (int e = 0; e < E; ++e) sum[e] = 0.f;
        }
    }
}

// A block per part (and a slice of the columns: blockIdx.y).
template <bool ALIGNED, typename T> __global__ void __launch_bounds__(128) embedding_sum_kernel(const EmbedArgs a)
{
    constexpr int kElems = Pack16<T>::kElems;
    __shared__ Part s;
    const int64_t part = blockIdx.x, first = part * kPart;
    for (int i = threadIdx.x; i < 3 * kPart + 2; i += blockDim.x) {
        const int64_t p = first + i - (kPart + 1);
        const int2 v = p >= 0 && p < a.n ? __ldg(a.sorted + p) : make_int2(-1, -1);
        s.key[i] = v.y;
        if (i > kPart && i <= 3 * kPart) s.at[i - (kPart + 1)] = v.x;
    }
    __syncthreads();
    if (threadIdx.x < 32) {
        const int lane = threadIdx.x, *key = s.key + kPart + 1;
        static_assert(kPart == 32, "a lane per place");
        // places of the first run where it comes from before, and places behind the part where the last one goes on
        const unsigned valid = __ballot_sync(0xffffffffu, key[lane] >= 0);
        const unsigned as_before = __ballot_sync(0xffffffffu, key[lane] >= 0 && key[lane] == key[-1]);
        const unsigned as_last = __ballot_sync(0xffffffffu, key[lane] >= 0 && key[lane] == key[kPart - 1]);
        const unsigned beyond = __ballot_sync(0xffffffffu, key[kPart + lane] >= 0 && key[kPart + lane] == key[kPart - 1]);
        if (lane == 0) {
            const int rest = as_before == ~0u ? kPart : __ffs(~as_before) - 1;
            const int start = as_last == ~0u ? 0 : 32 - __clz(~as_last), over = beyond == ~0u ? kPart : __ffs(~beyond) - 1;
            // a run is long if it has the place kPart before its last one, or behind its first one
            const bool long_before = rest == kPart || (rest > 0 && key[rest - 1 - kPart] == key[rest - 1]);
            const bool long_last = over > 0 && (rest == kPart || key[start + kPart] == key[kPart - 1]);
            s.before = long_before;
            s.begin = long_before ? 0 : rest;
            s.more = long_last;
            s.end = __popc(valid) + (long_last ? 0 : over);
        }
    }
    __syncthreads();
    if (s.begin >= s.end) return;
    const int64_t vectors = a.width / kElems, t = (int64_t)blockIdx.y * blockDim.x + threadIdx.x;
    if (t < vectors) {
        sum_part<ALIGNED, T, kElems>(a, part, s, t * kElems);
    } else if (!ALIGNED && t - vectors < a.width - vectors * kElems) {   // the columns behind the last whole vector
        sum_part<false, T, 1>(a, part, s, vectors * kElems + t - vectors);
    }
}

// Adds the sums of each long run, kOwn columns a lane (32 apart): those over
// few parts a warp each, then those over many a block each, whose warps have
// every kJoin-th part; both in a fixed order.
template <typename T> __global__ void __launch_bounds__(32 * kJoin) embedding_join_kernel(const EmbedArgs a)
{
    constexpr int kOwn = 4, kColumns = 32 * kOwn;
    __shared__ float sums[kJoin][kColumns];
    const int lane = threadIdx.x % 32, warp = threadIdx.x / 32;
    const int64_t chunks = (a.width + kColumns - 1) / kColumns, parts = (a.n + kPart - 1) / kPart;
    auto add = [&](float (&sum)[kOwn], int64_t row, int64_t c) {   // row of the partial sums
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
            if (c + 32 * i < a.width) sum[i] += __ldcs(a.partial + row * a.width + c + 32 * i);
    };
    for (int64_t item = (int64_t)blockIdx.x * kJoin + warp; item < a.runs[0] * chunks; item += (int64_t)gridDim.x * kJoin) {
        const int64_t part = a.runs[2 + item / chunks], c = item % chunks * kColumns + lane;
        const int k = a.sorted[(part + 1) * kPart - 1].y;
        // the parts that it goes on in: those whose first id is k
        const int64_t p = (part + 1 + lane) * kPart;
        const unsigned in = __ballot_sync(0xffffffffu, lane < kFew && p < a.n && a.sorted[p].y == k);
        const int more = __ffs(~in) - 1;
        float sum[kOwn] = {};
        add(sum, part * 2 + 1, c);
#pragma unroll
        for (int i = 1; i <= kFew; ++i)
            if (i <= more) add(sum, (part + i) * 2, c);
#pragma unroll
        for (int i = 0; i < kOwn; ++i)
            if (c + 32 * i < a.width) static_cast<T *>(a.out)[(int64_t)k * a.width + c + 32 * i] = elem_of<T>(sum[i] * a.scale);
    }
    for (int64_t item = blockIdx.x; item < a.runs[1] * chunks; item += gridDim.x) {
        const int64_t part = a.runs[parts + 1 - item / chunks], c = item % chunks * kColumns + lane;
        const int k = a.sorted[(part + 1) * kPart - 1].y;
        int64_t end = part + 1;
        for (int more = blockDim.x; more == (int)blockDim.x; end += more) {
            const int64_t p = (end + threadIdx.x) * kPart;
            more = __syncthreads_count(p < a.n && a.sorted[p].y == k);
        }
        float sum[kOwn] = {};
        if (warp == 0) add(sum, part * 2 + 1, c);
#pragma unroll 8
        for (int64_t p = part + 1 + warp; p < end; p += kJoin) add(sum, p * 2, c);
#pragma unroll
        for (int i = 0; i < kOwn; ++i) sums[warp][lane + 32 * i] = sum[i];
        __syncthreads();
        if (threadIdx.x < kColumns) {
            const int64_t at = item % chunks * kColumns + threadIdx.x;
            float all = 0.f;
#pragma unroll
            for (int g = 0; g < kJoin; ++g) all += sums[g][threadIdx.x];
            if (at < a.width) static_cast<T *>(a.out)[(int64_t)k * a.width + at] = elem_of<T>(all * a.scale);
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

// What the backward pass keeps in its workspace.
struct Places {
    size_t sorted[2], runs, counts, partial, bytes;   // sorted: of two sorting passes in turn
};
Places places_of(int64_t n, int64_t width)
{
    const int64_t parts = (n + kPart - 1) / kPart;
    Places p{};
    auto take = [&](size_t bytes) {
        const size_t at = p.bytes;
        p.bytes += (bytes + 255) & ~size_t(255);
        return at;
    };
    for (size_t &at : p.sorted) at = take((size_t)n * sizeof(int2));
    p.runs = take((size_t)(parts + 2) * 4);
    p.counts = take(bucket_workspace(n, kMostBuckets));
    p.partial = take((size_t)parts * 2 * width * sizeof(float));
    return p;
}

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
    return places_of(n, width).bytes;
}

cudaError_t launch_embedding_backward(const EmbeddingLaunch &l, int64_t skip, void *workspace, cudaStream_t stream)
{
    const size_t bytes = (size_t)l.rows * l.width * (l.dtype == SPMM_F32 ? 4 : 2);
    cudaError_t e;
    if (l.n == 0) return cudaMemsetAsync(l.out, 0, bytes, stream);
    if (bytes % 16)   // the sort writes whole vectors of zeros
        if ((e = cudaMemsetAsync(static_cast<char *>(l.out) + bytes / 16 * 16, 0, bytes % 16, stream)) != cudaSuccess) return e;
    char *ws = static_cast<char *>(workspace);
    const Places places = places_of(l.n, l.width);
    int2 *const sorted[2] = {reinterpret_cast<int2 *>(ws + places.sorted[0]), reinterpret_cast<int2 *>(ws + places.sorted[1])};
    int *const runs = reinterpret_cast<int *>(ws + places.runs);
    const unsigned parts = (unsigned)((l.n + kPart - 1) / kPart);
    int bits = 1;
    while (bits < 31 && (int64_t(1) << bits) < l.rows) ++bits;
    const int passes = (bits + kBucketBits - 1) / kBucketBits, each = (bits + passes - 1) / passes;
    const int64_t vectors = (int64_t)(bytes / 16);
    for (int p = 0; p < passes; ++p) {
        BucketSort s{};
        if (p == 0) s.keys = l.ids;
        else s.pairs_in = sorted[(p - 1) % 2];
        s.wide = l.itype == SPMM_I64;
        s.n = l.n;
        s.buckets = 1 << each;
        s.shift = p * each;
        s.mask = (1 << each) - 1;
        s.limit = l.rows;
        s.skip = skip;
        s.pairs = sorted[p % 2];
        s.counts = reinterpret_cast<int *>(ws + places.counts);
        s.clear = runs;
        s.zero = static_cast<uint4 *>(l.out) + vectors * p / passes;   // a share of the zeros beside each pass
        s.zero_vectors = vectors * (p + 1) / passes - vectors * p / passes;
        s.status = l.status;
        if ((e = launch_bucket_sort(s, stream)) != cudaSuccess) return e;
    }
    EmbedArgs a{};
    a.in = l.in; a.out = l.out; a.sorted = sorted[(passes - 1) % 2];
    a.runs = runs;
    a.partial = reinterpret_cast<float *>(ws + places.partial);
    a.n = l.n; a.rows = l.rows; a.width = l.width; a.scale = l.scale; a.status = l.status;
    return by_rows(l.dtype, l.width, [&](auto aligned, auto type) {
        using T = decltype(type);
        constexpr bool kAligned = decltype(aligned)::value;
        constexpr int kElems = Pack16<T>::kElems;
        const int64_t threads = l.width / kElems + l.width % kElems;
        embedding_sum_kernel<kAligned, T><<<dim3(parts, (unsigned)((threads + 127) / 128)), 128, 0, stream>>>(a);
        if (parts > 1)
            embedding_join_kernel<T><<<(unsigned)std::min<int64_t>(parts * ((l.width + 127) / 128), 4 * (int64_t)device_sm_count()),
                                       32 * kJoin, 0, stream>>>(a);
        return cudaGetLastError();
    });
}

}  // namespace spmmb
