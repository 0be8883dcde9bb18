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
// rows).  Both passes are bound by memory: 524287 ids of 131071 rows of 512
// fp32, density 1 / rank, forward 215 us (1.25 GB, 5.8 TB/s), backward 316 us
// (sorting and zeros 90, sums 196, long runs 30); 16411 ids of 50021 rows of 1024
// bf16 10 us and 59 us (sorting and zeros 34, sums 18, long runs 7).
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
constexpr int kJoin = 32;      // of so many warps (16: 39 us for the 30 below, 6 for the 7)

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
    int lanes;              // forward: of a row's team
    float scale;
    DevStatus *status;
};

// A team of a.lanes lanes per row, kAtOnce vectors a lane in flight.
constexpr int kAtOnce = 4;
template <bool ALIGNED, typename T> __global__ void __launch_bounds__(256) embedding_kernel(const EmbedArgs a)
{
    constexpr int kElems = Pack16<T>::kElems;
    const int lane = threadIdx.x & (a.lanes - 1);
    const int64_t teams = (int64_t)gridDim.x * blockDim.x / a.lanes;
    for (int64_t i = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) / a.lanes; i < a.n; i += teams) {
        const int64_t id = a.wide ? ld_idx(static_cast<const int64_t *>(a.ids) + i) : ld_idx(static_cast<const int *>(a.ids) + i);
        const bool found = id >= 0 && id < a.rows;
        if (!found && lane == 0) raise_status(a.status, SPMM_DEV_BAD_COLUMN, i);
        const T *row = static_cast<const T *>(a.in) + (found ? id : 0) * a.width;
        T *out = static_cast<T *>(a.out) + i * a.width;
        const RowSpan<ALIGNED, T> span(out, a.width);
        for (int64_t c0 = lane; c0 < span.vectors; c0 += a.lanes * kAtOnce) {
            Pack16<T> v[kAtOnce];
#pragma unroll
            for (int n = 0; n < kAtOnce; ++n) {
                v[n].raw = make_uint4(0, 0, 0, 0);
                if (found && c0 + n * a.lanes < span.vectors) v[n] = load16<ALIGNED>(row + span.head + (c0 + n * a.lanes) * kElems);
            }
#pragma unroll
            for (int n = 0; n < kAtOnce; ++n) {
                float f[kElems];
                v[n].get(f);
#pragma unroll
                for (int e = 0; e < kElems; ++e) f[e] *= a.scale;
                if (found) v[n].set(f);   // else zeros, whatever the scale's sign
                if (c0 + n * a.lanes < span.vectors) __stcs(reinterpret_cast<uint4 *>(out + span.head) + c0 + n * a.lanes, v[n].raw);
            }
        }
        for (int64_t n = lane; n < span.loose(a.width); n += a.lanes) {
            const int64_t c = span.loose_at(n);
            out[c] = elem_of<T>(found ? elem_f32<T>(row[c]) * a.scale : 0.f);
        }
    }
}

// The sorted ids of a part, as a block keeps them in shared memory: those
// around it too, since a run of at most kPart rows over a border is added whole
// by the part that it starts in.
struct Part {
    int key[3 * kPart + 2];   // key[kPart + 1 + i]: the id at place i of the part, -1 outside the ids
    int at[2 * kPart];        // input indexes of the part and of kPart places behind it
    int head[2 * kPart];      // elements before the first whole vector of their ids' rows of dtable
    int begin, end;           // the places that this part adds
    bool more;                // the last run is longer and goes on: its sum is a partial one
    bool before;              // the first run comes from before: its sum is a partial one
};

// The part's sums, of E columns: the `slot`-th whole vector of an id's row of
// dtable or, with E == 1, its `slot`-th loose element.  Where they lie in the
// row goes by the id, so that a result is stored in whole vectors.
template <bool ALIGNED, typename T, int E>
__device__ __forceinline__ void sum_part(const EmbedArgs &a, int64_t part, const Part &s, int64_t slot)
{
    constexpr int kElems = Pack16<T>::kElems;
    const int *key = s.key + kPart + 1;
    // the column of the slot in the row of the id at place i, -1 where the row has no such one
    const int width = (int)a.width;
    auto column = [&](int i) -> int {
        if constexpr (ALIGNED) return (int)slot * kElems;
        const int head = s.head[i], vectors = (width - head) / kElems;
        if constexpr (E == 1) {
            const int c = slot < head ? (int)slot : (int)slot + vectors * kElems;
            return c < width ? c : -1;
        }
        return slot < vectors ? head + (int)slot * kElems : -1;
    };
    float sum[E];
#pragma unroll
    for (int e = 0; e < E; ++e) sum[e] = 0.f;
    bool before = s.before;
    constexpr int kAhead = 8;
    using Raw = std::conditional_t<E == 1, T, Pack16<T>>;
    for (int i0 = s.begin; i0 < s.end; i0 += kAhead) {
        Raw raw[kAhead];
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {   // past the last one: a row is read again and not added
            const int i = min(i0 + j, s.end - 1), c = max(column(i), 0);
            const T *p = static_cast<const T *>(a.in) + (int64_t)s.at[i] * a.width + c;
            if constexpr (E == 1) raw[j] = *p;
            else raw[j] = load16<ALIGNED>(p);
        }
#pragma unroll
        for (int j = 0; j < kAhead; ++j) {
            const int i = i0 + j;
            if (i >= s.end) break;
            float f[E];
            if constexpr (E == 1) f[0] = elem_f32<T>(raw[j]);
            else raw[j].get(f);
#pragma unroll
            for (int e = 0; e < E; ++e) sum[e] += f[e];
            const int k = key[i];
            if (i + 1 < s.end && key[i + 1] == k) continue;
            const bool more = i + 1 == s.end && s.more;
            const int c = column(i);
            if (before || more) {
                float *p = a.partial + (part * 2 + (before ? 0 : 1)) * a.width + c;
#pragma unroll
                for (int e = 0; e < E; ++e)
                    if (c >= 0) p[e] = sum[e];
            } else if (c >= 0) {
#pragma unroll
                for (int e = 0; e < E; ++e) sum[e] *= a.scale;
                T *p = static_cast<T *>(a.out) + (int64_t)k * a.width + c;
                if constexpr (E == 1) {
                    *p = elem_of<T>(sum[0]);
                } else {
                    Pack16<T> v;
                    v.set(sum);
                    *reinterpret_cast<uint4 *>(p) = v.raw;
                }
            }
            before = false;
#pragma unroll
            for (int e = 0; e < E; ++e) sum[e] = 0.f;
        }
    }
}

// Threads that a part needs: one for each whole vector of a row, and one for
// each element that can lie outside them.
template <typename T> int64_t part_threads(int64_t width)
{
    constexpr int64_t kElems = Pack16<T>::kElems;
    return width % kElems == 0 ? width / kElems : width / kElems + 2 * (kElems - 1);
}

// blockDim.x threads of blockDim.y parts (and of a slice of the columns: blockIdx.y).
constexpr int kSumThreads = 128, kMostParts = 16;
template <bool ALIGNED, typename T> __global__ void __launch_bounds__(kSumThreads, 8) embedding_sum_kernel(const EmbedArgs a)
{
    constexpr int kElems = Pack16<T>::kElems;
    static_assert(kPart == 32, "a lane per place");
    __shared__ Part shared[kMostParts];
    const int warp = (threadIdx.y * blockDim.x + threadIdx.x) / 32, lane = (threadIdx.y * blockDim.x + threadIdx.x) % 32;
    const int64_t parts = (a.n + kPart - 1) / kPart, part0 = (int64_t)blockIdx.x * blockDim.y;
    for (int n = warp; n < (int)blockDim.y; n += kSumThreads / 32) {   // a warp lays out a part
        Part &s = shared[n];
        const int64_t first = (part0 + n) * kPart;
        for (int i = lane; i < 3 * kPart + 2; i += 32) {
            const int64_t p = first + i - (kPart + 1);
            const int2 v = p >= 0 && p < a.n ? __ldg(a.sorted + p) : make_int2(-1, -1);
            s.key[i] = v.y;
            if (i > kPart && i <= 3 * kPart) {
                s.at[i - (kPart + 1)] = v.x;
                if (!ALIGNED)
                    s.head[i - (kPart + 1)] = RowSpan<false, T>(static_cast<T *>(a.out) + (int64_t)max(v.y, 0) * a.width, a.width).head;
            }
        }
        __syncwarp();
        const int *key = s.key + kPart + 1;
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
            // a long run that starts here: for the join, beside those of few parts or of many
            if (blockIdx.y == 0 && long_last && rest < kPart) {
                const int64_t far = first + kFew * kPart;
                const bool many = far < a.n && a.sorted[far].y == key[kPart - 1];
                const int i = atomicAdd(a.runs + many, 1);
                a.runs[many ? parts + 1 - i : 2 + i] = (int)(part0 + n);
            }
        }
    }
    __syncthreads();
    const Part &s = shared[threadIdx.y];
    const int64_t part = part0 + threadIdx.y;
    if (part >= parts || s.begin >= s.end) return;
    const int64_t vectors = a.width / kElems, t = (int64_t)blockIdx.y * blockDim.x + threadIdx.x;
    if (t < vectors) sum_part<ALIGNED, T, kElems>(a, part, s, t);
    else if (!ALIGNED && t - vectors < 2 * (kElems - 1)) sum_part<false, T, 1>(a, part, s, t - vectors);
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
    // N rows of the partial sums, 2 * stride apart, all of their loads in flight; `count` of them are there
    auto add = [&](float (&sum)[kOwn], auto rows, int64_t row, int64_t stride, int count, int64_t c) {
        constexpr int N = decltype(rows)::value;
        float f[N][kOwn];
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int i = 0; i < kOwn; ++i)   // what is not there: the last one again, not added
                f[n][i] = __ldcs(a.partial + (row + 2 * stride * min(n, count - 1)) * a.width + min(c + 32 * i, a.width - 1));
#pragma unroll
        for (int n = 0; n < N; ++n)
#pragma unroll
            for (int i = 0; i < kOwn; ++i)
                if (n < count) sum[i] += f[n][i];
    };
    std::integral_constant<int, 1> one;
    std::integral_constant<int, kFew> several;
    for (int64_t item = (int64_t)blockIdx.x * kJoin + warp; item < a.runs[0] * chunks; item += (int64_t)gridDim.x * kJoin) {
        const int64_t part = a.runs[2 + item / chunks], c = item % chunks * kColumns + lane;
        const int k = a.sorted[(part + 1) * kPart - 1].y;
        // the parts that it goes on in: those whose first id is k
        const int64_t p = (part + 1 + lane) * kPart;
        const unsigned in = __ballot_sync(0xffffffffu, lane < kFew && p < a.n && a.sorted[p].y == k);
        const int more = __ffs(~in) - 1;
        float sum[kOwn] = {};
        add(sum, one, part * 2 + 1, 0, 1, c);
        if (more > 0) add(sum, several, (part + 1) * 2, 1, more, c);
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
        if (warp == 0) add(sum, one, part * 2 + 1, 0, 1, c);
        for (int64_t p = part + 1 + warp; p < end; p += kJoin * kFew)
            add(sum, several, p * 2, kJoin, (int)min((int64_t)kFew, (end - p + kJoin - 1) / kJoin), c);
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
    const int64_t vectors = l.width * (l.dtype == SPMM_F32 ? 4 : 2) / 16;
    for (a.lanes = 2; a.lanes < 32 && a.lanes * kAtOnce < vectors;) a.lanes *= 2;
    const unsigned blocks = (unsigned)std::max<int64_t>(
        1, std::min<int64_t>((l.n * a.lanes + 255) / 256, 32 * (int64_t)device_sm_count()));
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
    BucketPasses sort{};
    static_assert(4 * kBucketBits >= 31, "passes for every id");
    sort.passes = passes;
    for (int p = 0; p < passes; ++p) {
        BucketSort &s = sort.pass[p];
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
    }
    if ((e = launch_bucket_sort(sort, stream)) != cudaSuccess) return e;
    EmbedArgs a{};
    a.in = l.in; a.out = l.out; a.sorted = sorted[(passes - 1) % 2];
    a.runs = runs;
    a.partial = reinterpret_cast<float *>(ws + places.partial);
    a.n = l.n; a.rows = l.rows; a.width = l.width; a.scale = l.scale; a.status = l.status;
    return by_rows(l.dtype, l.width, [&](auto aligned, auto type) {
        using T = decltype(type);
        constexpr bool kAligned = decltype(aligned)::value;
        const int64_t threads = part_threads<T>(l.width);
        int each = kSumThreads;   // threads of a part
        while (each > kSumThreads / kMostParts && each / 2 >= threads) each /= 2;
        const dim3 block(each, kSumThreads / each);
        const dim3 grid((parts + block.y - 1) / block.y, (unsigned)((threads + each - 1) / each));
        embedding_sum_kernel<kAligned, T><<<grid, block, 0, stream>>>(a);
        if (parts > 1)
            embedding_join_kernel<T><<<(unsigned)std::min<int64_t>(parts * ((l.width + 127) / 128), 2 * (int64_t)device_sm_count()),
                                       32 * kJoin, 0, stream>>>(a);
        return cudaGetLastError();
    });
}

}  // namespace spmmb
