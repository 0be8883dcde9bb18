// Stable counting sort of keys: the places that rows of equal keys get when
// the keys are put in order, each key's rows in their own order.
//
// Each warp owns a contiguous slice of the keys and counts them per bucket in
// shared memory; its keys' places are the keys of smaller buckets, those of
// the same one in earlier slices, and their own rank among the slice's.  Places
// come from counts alone (the order of the shared atomics that count does not
// show), so a result never depends on timing.  One block does it all for few
// keys, every pass of a sort by more bits than a pass takes in one launch; for
// many a first launch counts per block and a second one, whose blocks add the
// counts of the others up, places.  Further blocks, where a caller asks for
// them, write zeros beside the first phase: few SMs sort.
//
// What bounds it: the latency of its phases, and with many keys the scattered
// stores.  36 keys 3.6 us; 262144 keys, 64 buckets, 6 and 12 us; 524287, 512
// buckets, 18 us for the second launch; both passes of 6144 ids of 131071 rows in
// one launch 1.8 us less than in two, and 2.5 us less of the host's time.  One
// cluster of 16 blocks with all phases in a launch took 36 and 58 us.
#include <algorithm>

#include "../../include/spmm_b200.h"
#include "common.cuh"
#include "engine.h"
#include "layer.cuh"
#include "layer.h"

namespace spmmb {

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kBatch = 8;             // keys of a lane in flight
constexpr int kMostWarps = 32, kMostBlocks = 128;

// Shared memory: counts [warps][buckets], then the block's totals [buckets]
// and the scan's sums per warp.
size_t bucket_smem(int buckets, int warps) { return (size_t)(warps + 1) * buckets * 4 + warps * 4; }

// The blocks behind the first `blocks`, which sort.
__device__ __forceinline__ void write_zeros(const BucketSort &a, int blocks)
{
    const int64_t threads = (int64_t)(gridDim.x - blocks) * blockDim.x;
    for (int64_t i = (int64_t)((int)blockIdx.x - blocks) * blockDim.x + threadIdx.x; i < a.zero_vectors; i += threads)
        __stcs(static_cast<uint4 *>(a.zero) + i, make_uint4(0, 0, 0, 0));
}

// COUNT: only the counts per block, [blocks][buckets] to a.counts.
template <bool COUNT> __device__ __forceinline__ void sort_pass(const BucketSort &a, const int blocks)
{
    extern __shared__ int smem[];
    const int block = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x / 32, B = a.buckets;
    const int bits = 32 - __clz(B - 1);   // of a bucket (none with a single one)
    int *mine = smem + warp * B, *totals = smem + warps * B, *sums = totals + B;
    for (int i = threadIdx.x; i < warps * B; i += blockDim.x) smem[i] = 0;
    __syncthreads();

    // this warp's keys: [begin, end), multiples of 32 apart
    const int64_t slices = (int64_t)blocks * warps;
    const int64_t each = ((a.n + slices - 1) / slices + 31) / 32 * 32;
    const int64_t begin = min(a.n, ((int64_t)block * warps + warp) * each), end = min(a.n, begin + each);
    // kBatch x 32 keys from i on: each lane's input and key, and its bucket, -1 where it is left out.
    int input[kBatch], bucket[kBatch], key[kBatch];
    auto read = [&](int64_t i, bool raise) {
        int64_t wide[kBatch];
#pragma unroll
        for (int s = 0; s < kBatch; ++s) {
            const int64_t at = i + s * 32 + lane;
            input[s] = -1;
            wide[s] = -1;
            if (at < end && a.pairs_in) {
                const int2 v = __ldcg(a.pairs_in + at);   // this launch may have written them
                input[s] = v.x;
                wide[s] = v.y;
            } else if (at < end) {
                input[s] = (int)at;
                wide[s] = a.wide ? ld_idx(static_cast<const int64_t *>(a.keys) + at) : ld_idx(static_cast<const int *>(a.keys) + at);
            }
        }
#pragma unroll
        for (int s = 0; s < kBatch; ++s) {
            bool in = input[s] >= 0 && wide[s] != a.skip;
            if (in && (wide[s] < 0 || wide[s] >= a.limit)) {
                if (raise) raise_status(a.status, SPMM_DEV_BAD_COLUMN, input[s]);
                in = false;
            }
            key[s] = (int)wide[s];
            bucket[s] = in ? key[s] >> a.shift & a.mask : -1;
        }
    };
    const bool once = end - begin <= 32 * kBatch;   // they stay in registers
    for (int64_t i = begin; i < end; i += 32 * kBatch) {
        read(i, COUNT || blocks == 1);
#pragma unroll
        for (int s = 0; s < kBatch; ++s)
            if (bucket[s] >= 0) atomicAdd(mine + bucket[s], 1);
    }
    __syncthreads();
    // per bucket: this block's keys before each warp's, their number
    for (int b = threadIdx.x; b < B; b += blockDim.x) {
        int sum = 0;
#pragma unroll 8
        for (int w = 0; w < warps; ++w) {
            const int c = smem[w * B + b];
            smem[w * B + b] = sum;
            sum += c;
        }
        totals[b] = sum;
        if (COUNT) a.counts[block * B + b] = sum;
    }
    if constexpr (COUNT) {
        return;
    } else {
        __syncthreads();
        // per bucket: the keys of smaller buckets, and of this one in earlier blocks
        int carry = 0;   // keys of the buckets before the current blockDim.x
        for (int b0 = 0; b0 < B; b0 += blockDim.x) {
            const int b = b0 + threadIdx.x;
            int before = 0, all = 0;
            if (b < B) {
                if (blocks == 1) {
                    all = totals[b];
                } else {
#pragma unroll 16
                    for (int c = 0; c < blocks; ++c) {
                        const int v = __ldg(a.counts + c * B + b);
                        before += c < block ? v : 0;
                        all += v;
                    }
                }
            }
            int scan = all;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(kFull, scan, o);
                if (lane >= o) scan += u;
            }
            if (lane == 31) sums[warp] = scan;
            __syncthreads();
            if (warp == 0) {
                int v = lane < warps ? sums[lane] : 0;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const int u = __shfl_up_sync(kFull, v, o);
                    if (lane >= o) v += u;
                }
                if (lane < warps) sums[lane] = v;
            }
            __syncthreads();
            const int start = carry + scan - all + (warp ? sums[warp - 1] : 0);
            if (b < B) {
                totals[b] = start + before;
                if (a.ptr && block == 0) a.ptr[b] = start;
            }
            carry += sums[warps - 1];
            __syncthreads();
        }
        const int kept = carry;
        if (block == 0 && threadIdx.x == 0) {
            if (a.ptr) a.ptr[B] = kept;
            if (a.clear) a.clear[0] = a.clear[1] = 0;
        }
        for (int i = lane; i < B; i += 32) mine[i] += totals[i];
        __syncwarp();

        for (int64_t i = begin; i < end; i += 32 * kBatch) {
            if (!once) read(i, false);
#pragma unroll
            for (int s = 0; s < kBatch; ++s) {
                if (i + s * 32 >= end) break;
                // the lanes with this one's bucket, bit by bit (match_any takes a turn per distinct value)
                unsigned peers = __ballot_sync(kFull, bucket[s] >= 0);
                for (int bit = 0; bit < bits; ++bit) {
                    const bool set = bucket[s] >> bit & 1;
                    const unsigned ones = __ballot_sync(kFull, set);
                    peers &= set ? ones : ~ones;
                }
                const int rank = __popc(peers & ((1u << lane) - 1));
                int place = -1;
                if (bucket[s] >= 0) place = mine[bucket[s]] + rank;
                __syncwarp();
                if (bucket[s] >= 0 && rank == 0) mine[bucket[s]] += __popc(peers);
                __syncwarp();
                if (place >= 0) {
                    if (a.pairs) a.pairs[place] = make_int2(input[s], key[s]);
                    else a.order[place] = input[s];
                }
                if (a.position && input[s] >= 0) a.position[input[s]] = place;
            }
        }
        for (int64_t i = kept + (int64_t)block * blockDim.x + threadIdx.x; i < a.n; i += (int64_t)blocks * blockDim.x) {
            if (a.pairs) a.pairs[i] = make_int2(-1, -1);
            else a.order[i] = -1;
        }
    }
}

template <bool COUNT> __global__ void __launch_bounds__(kMostWarps * 32) bucket_kernel(const BucketSort a, const int blocks)
{
    if ((int)blockIdx.x >= blocks) write_zeros(a, blocks);
    else sort_pass<COUNT>(a, blocks);
}

// All passes of a sort by one block.
__global__ void __launch_bounds__(kMostWarps * 32) bucket_passes_kernel(const BucketPasses a)
{
    if (blockIdx.x > 0) {
        for (int p = 0; p < a.passes; ++p) write_zeros(a.pass[p], 1);
        return;
    }
    for (int p = 0; p < a.passes; ++p) {
        if (p > 0) __syncthreads();   // the pass before: its pairs, and shared memory
        sort_pass<false>(a.pass[p], 1);
    }
}

// Blocks that sort, and their warps.  One block for as many keys as stay in
// its registers (8192; 7000 ids of 50021 rows, width 64: 36 us, of two blocks
// 40).  Else one for every 2048 keys, of 16 warps (16384 ids 39 us; 4096 keys
// and 32 warps 44), as long as there are few of them, since each adds up the
// counts of all (262144 ids: 56 us; 4096 keys and 32 warps 53).
struct Blocks {
    int count, warps;
};
Blocks blocks_for(int64_t n, int buckets)
{
    if (n <= 2048 && buckets <= 256) return {1, 8};   // few warps, whose barriers are short
    if (n <= kMostWarps * 32 * kBatch) return {1, kMostWarps};
    if (n <= 131072) return {(int)((n + 2047) / 2048), 16};
    return {(int)std::min<int64_t>(kMostBlocks, (n + 4095) / 4096), kMostWarps};
}

}  // namespace

size_t bucket_workspace(int64_t n, int buckets)
{
    const int blocks = blocks_for(n, buckets).count;
    return blocks == 1 ? 0 : (size_t)blocks * buckets * sizeof(int);
}

cudaError_t launch_bucket_sort(const BucketPasses &all, cudaStream_t stream)
{
    const BucketSort &a = all.pass[0];
    static PerDevice<bool> ready;   // the attributes outlast the call
    bool *done = ready.here();
    if (!done || !*done) {
        for (auto kernel : {bucket_kernel<false>, bucket_kernel<true>}) {
            const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                       (int)bucket_smem(kMostBuckets, kMostWarps));
            if (e != cudaSuccess) return e;
        }
        const cudaError_t e = cudaFuncSetAttribute(bucket_passes_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   (int)bucket_smem(kMostBuckets, kMostWarps));
        if (e != cudaSuccess) return e;
        if (done) *done = true;
    }
    const Blocks sorting = blocks_for(a.n, a.buckets);
    const int blocks = sorting.count, warps = sorting.warps;
    const size_t smem = bucket_smem(a.buckets, warps);
    auto zeroing = [&](int64_t vectors) {
        return (unsigned)std::min<int64_t>((vectors + warps * 32 - 1) / (warps * 32),
                                           2 * (int64_t)device_sm_count() * kMostWarps / warps);
    };
    if (blocks == 1) {
        int64_t vectors = 0;
        for (int p = 0; p < all.passes; ++p) vectors += all.pass[p].zero_vectors;
        if (all.passes == 1) bucket_kernel<false><<<1 + zeroing(vectors), warps * 32, smem, stream>>>(a, 1);
        else bucket_passes_kernel<<<1 + zeroing(vectors), warps * 32, smem, stream>>>(all);
        return cudaGetLastError();
    }
    for (int p = 0; p < all.passes; ++p) {
        const BucketSort &s = all.pass[p];
        bucket_kernel<true><<<blocks + zeroing(s.zero_vectors), warps * 32, smem, stream>>>(s, blocks);
        const cudaError_t e = cudaGetLastError();
        if (e != cudaSuccess) return e;
        bucket_kernel<false><<<blocks, warps * 32, smem, stream>>>(s, blocks);
        const cudaError_t e2 = cudaGetLastError();
        if (e2 != cudaSuccess) return e2;
    }
    return cudaSuccess;
}

}  // namespace spmmb
