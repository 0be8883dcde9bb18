// Stable counting sort of keys: the places that rows of equal keys get when
// the keys are put in order, each key's rows in their own order.
//
// One cluster of blocks.  A warp owns a contiguous slice of the keys; its
// counts per bucket are kept in shared memory, and the blocks read each
// other's totals through distributed shared memory, so that a launch counts,
// scans and places.  Places come from counts alone (the order of the shared
// atomics that count does not show), so a result never depends on timing.
//
// What bounds it: the latency of its phases.
#include <cooperative_groups.h>

#include <algorithm>

#include "../../include/spmm_b200.h"
#include "common.cuh"
#include "engine.h"
#include "layer.cuh"
#include "layer.h"

namespace spmmb {

namespace {

namespace cg = cooperative_groups;

constexpr unsigned kFull = 0xffffffffu;
constexpr int kWarps = 32, kCluster = 8;

// Shared memory: counts [kWarps][buckets], then the block's totals [buckets]
// and the scan's sums per warp.
size_t bucket_smem(int buckets) { return (size_t)(kWarps + 1) * buckets * 4 + kWarps * 4; }

__global__ void __launch_bounds__(kWarps * 32) bucket_kernel(const BucketSort a)
{
    extern __shared__ int smem[];
    const cg::cluster_group cluster = cg::this_cluster();
    const int blocks = (int)cluster.num_blocks(), block = (int)cluster.block_rank();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, B = a.buckets;
    int *mine = smem + warp * B, *totals = smem + kWarps * B, *sums = totals + B;
    for (int i = threadIdx.x; i < kWarps * B; i += blockDim.x) smem[i] = 0;
    __syncthreads();

    // this warp's keys: [begin, end), multiples of 32 apart
    const int64_t slices = (int64_t)blocks * kWarps;
    const int64_t each = ((a.n + slices - 1) / slices + 31) / 32 * 32;
    const int64_t begin = min(a.n, ((int64_t)block * kWarps + warp) * each), end = min(a.n, begin + each);
    // The input at place i of this pass and its bucket, -1 where it is left out.
    auto read = [&](int64_t i, int *input, bool raise) {
        *input = -1;
        if (i >= end) return -1;
        const int at = a.order_in ? a.order_in[i] : (int)i;
        if (at < 0) return -1;
        *input = at;
        const int64_t key = a.wide ? static_cast<const int64_t *>(a.keys)[at] : static_cast<const int *>(a.keys)[at];
        if (key == a.skip) return -1;
        if (key < 0 || key >= a.limit) {
            if (raise) raise_status(a.status, SPMM_DEV_BAD_COLUMN, at);
            return -1;
        }
        return (int)(key >> a.shift) & a.mask;
    };
    for (int64_t i = begin; i < end; i += 32) {
        int input;
        const int b = read(i + lane, &input, true);
        if (b >= 0) atomicAdd(mine + b, 1);
    }
    __syncthreads();
    // per bucket: this warp's keys before each warp's, the block's total
    for (int b = threadIdx.x; b < B; b += blockDim.x) {
        int sum = 0;
        for (int w = 0; w < kWarps; ++w) {
            const int c = smem[w * B + b];
            smem[w * B + b] = sum;
            sum += c;
        }
        totals[b] = sum;
    }
    cluster.sync();
    // per bucket: the keys of smaller buckets, and of this one in earlier blocks
    const int b = threadIdx.x;
    int before = 0, all = 0;
    if (b < B)
        for (int c = 0; c < blocks; ++c) {
            const int v = cluster.map_shared_rank(totals, c)[b];
            before += c < block ? v : 0;
            all += v;
        }
    int scan = all;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(kFull, scan, o);
        if (lane >= o) scan += u;
    }
    if (lane == 31) sums[warp] = scan;
    cluster.sync();   // the other blocks have read this one's totals
    if (warp == 0) {
        int v = sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int u = __shfl_up_sync(kFull, v, o);
            if (lane >= o) v += u;
        }
        sums[lane] = v;
    }
    __syncthreads();
    const int start = scan - all + (warp ? sums[warp - 1] : 0), kept = sums[kWarps - 1];
    if (b < B) {
        totals[b] = start + before;
        if (a.ptr && block == 0) a.ptr[b] = start;
    }
    if (a.ptr && block == 0 && threadIdx.x == 0) a.ptr[B] = kept;
    __syncthreads();
    for (int i = threadIdx.x; i < kWarps * B; i += blockDim.x) smem[i] += totals[i % B];
    __syncthreads();

    for (int64_t i = begin; i < end; i += 32) {
        int input;
        const int bucket = read(i + lane, &input, false);
        const unsigned peers = __match_any_sync(kFull, bucket);
        const int rank = __popc(peers & ((1u << lane) - 1));
        int place = -1;
        if (bucket >= 0) place = mine[bucket] + rank;
        __syncwarp();
        if (bucket >= 0 && rank == 0) mine[bucket] += __popc(peers);
        __syncwarp();
        if (place >= 0) a.order[place] = input;
        if (a.position && input >= 0) a.position[input] = place;
    }
    for (int64_t i = kept + (int64_t)block * blockDim.x + threadIdx.x; i < a.n; i += (int64_t)blocks * blockDim.x)
        a.order[i] = -1;
}

}  // namespace

cudaError_t launch_bucket_sort(const BucketSort &a, cudaStream_t stream)
{
    const size_t smem = bucket_smem(a.buckets);
    static PerDevice<bool> ready;   // the attribute outlasts the call
    bool *done = ready.here();
    if (!done || !*done) {
        const cudaError_t e = cudaFuncSetAttribute(bucket_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   (int)bucket_smem(kMostBuckets));
        if (e != cudaSuccess) return e;
        if (done) *done = true;
    }
    const unsigned blocks = a.n <= 4096 ? 1 : kCluster;
    cudaLaunchConfig_t config{};
    config.gridDim = blocks;
    config.blockDim = kWarps * 32;
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.x = blocks;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    config.attrs = &attr;
    config.numAttrs = 1;
    return cudaLaunchKernelEx(&config, bucket_kernel, a);
}

}  // namespace spmmb
