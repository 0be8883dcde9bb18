// Stable counting sort of keys: the places that rows of equal keys get when
// the keys are put in order, each key's rows in their own order.
//
// One cluster of blocks.  A warp owns a contiguous slice of the keys; its
// counts per bucket are kept in shared memory, and the blocks read each
// other's totals through distributed shared memory, so that a launch counts,
// scans and places.  Places come from counts alone (the order of the shared
// atomics that count does not show), so a result never depends on timing.
// Further clusters of the launch, where a caller asks for them, write zeros
// meanwhile: the sort leaves nearly all of the GPU to them.
//
// What bounds it: the latency of its phases, and of a warp's turns (256 keys
// each, whose loads are in flight together).
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
constexpr int kWarps = 32, kBatch = 8;

// Shared memory: counts [kWarps][buckets], then the block's totals [buckets]
// and the scan's sums per warp.
size_t bucket_smem(int buckets) { return (size_t)(kWarps + 1) * buckets * 4 + kWarps * 4; }

__global__ void __launch_bounds__(kWarps * 32) bucket_kernel(const BucketSort a)
{
    extern __shared__ int smem[];
    const cg::cluster_group cluster = cg::this_cluster();
    const int blocks = (int)cluster.num_blocks(), block = (int)cluster.block_rank();
    if ((int)blockIdx.x >= blocks) {   // not the first cluster
        const int64_t threads = (int64_t)(gridDim.x - blocks) * blockDim.x;
        for (int64_t i = (int64_t)(blockIdx.x - blocks) * blockDim.x + threadIdx.x; i < a.zero_vectors; i += threads)
            __stcs(static_cast<uint4 *>(a.zero) + i, make_uint4(0, 0, 0, 0));
        return;
    }
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, B = a.buckets;
    int *mine = smem + warp * B, *totals = smem + kWarps * B, *sums = totals + B;
    for (int i = threadIdx.x; i < kWarps * B; i += blockDim.x) smem[i] = 0;
    __syncthreads();

    // this warp's keys: [begin, end), multiples of 32 apart
    const int64_t slices = (int64_t)blocks * kWarps;
    const int64_t each = ((a.n + slices - 1) / slices + 31) / 32 * 32;
    const int64_t begin = min(a.n, ((int64_t)block * kWarps + warp) * each), end = min(a.n, begin + each);
    // kBatch x 32 keys from i on: each lane's input and key, and its bucket, -1 where it is left out.
    int input[kBatch], bucket[kBatch];
    int64_t key[kBatch];
    auto read = [&](int64_t i, bool raise) {
#pragma unroll
        for (int s = 0; s < kBatch; ++s) {
            const int64_t at = i + s * 32 + lane;
            input[s] = -1;
            key[s] = -1;
            if (at < end) {
                input[s] = a.order_in ? __ldg(a.order_in + at) : (int)at;
                key[s] = a.wide ? ld_idx(static_cast<const int64_t *>(a.keys) + at) : ld_idx(static_cast<const int *>(a.keys) + at);
            }
        }
#pragma unroll
        for (int s = 0; s < kBatch; ++s) {
            bool in = input[s] >= 0 && key[s] != a.skip;
            if (in && (key[s] < 0 || key[s] >= a.limit)) {
                if (raise) raise_status(a.status, SPMM_DEV_BAD_COLUMN, input[s]);
                in = false;
            }
            bucket[s] = in ? (int)(key[s] >> a.shift) & a.mask : -1;
        }
    };
    for (int64_t i = begin; i < end; i += 32 * kBatch) {
        read(i, true);
#pragma unroll
        for (int s = 0; s < kBatch; ++s)
            if (bucket[s] >= 0) atomicAdd(mine + bucket[s], 1);
    }
    __syncthreads();
    // per bucket: this warp's keys before each warp's, the block's total
    for (int b = threadIdx.x; b < B; b += blockDim.x) {
        int sum = 0;
#pragma unroll 8
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
#pragma unroll 8
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
    for (int i = lane; i < B; i += 32) mine[i] += totals[i];
    __syncwarp();

    for (int64_t i = begin; i < end; i += 32 * kBatch) {
        read(i, false);
#pragma unroll
        for (int s = 0; s < kBatch; ++s) {
            const unsigned peers = __match_any_sync(kFull, bucket[s]);
            const int rank = __popc(peers & ((1u << lane) - 1));
            int place = -1;
            if (bucket[s] >= 0) place = mine[bucket[s]] + rank;
            __syncwarp();
            if (bucket[s] >= 0 && rank == 0) mine[bucket[s]] += __popc(peers);
            __syncwarp();
            if (place >= 0) {
                a.order[place] = input[s];
                if (a.key_out) a.key_out[place] = (int)key[s];
            }
            if (a.position && input[s] >= 0) a.position[input[s]] = place;
        }
    }
    for (int64_t i = kept + (int64_t)block * blockDim.x + threadIdx.x; i < a.n; i += (int64_t)blocks * blockDim.x) {
        a.order[i] = -1;
        if (a.key_out) a.key_out[i] = -1;
    }
}

}  // namespace

cudaError_t launch_bucket_sort(const BucketSort &a, cudaStream_t stream)
{
    // Blocks of the cluster: one for few keys, 16 for many where the device can hold such a cluster.
    static PerDevice<int> most;   // outlasts the call
    int *known = most.here(), widest = known ? *known : 0;
    cudaLaunchConfig_t config{};
    config.blockDim = kWarps * 32;
    config.stream = stream;
    cudaLaunchAttribute attr{};
    attr.id = cudaLaunchAttributeClusterDimension;
    attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
    config.attrs = &attr;
    config.numAttrs = 1;
    if (!widest) {
        cudaError_t e = cudaFuncSetAttribute(bucket_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)bucket_smem(kMostBuckets));
        if (e != cudaSuccess) return e;
        int clusters = 0;
        config.gridDim = attr.val.clusterDim.x = 16;
        config.dynamicSmemBytes = bucket_smem(kMostBuckets);
        if (cudaFuncSetAttribute(bucket_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess ||
            cudaOccupancyMaxActiveClusters(&clusters, bucket_kernel, &config) != cudaSuccess)
            clusters = 0;
        (void)cudaGetLastError();
        widest = clusters > 0 ? 16 : 8;
        if (known) *known = widest;
    }
    const unsigned blocks = a.n <= 4096 ? 1 : a.n <= 32768 ? 8 : (unsigned)widest;
    unsigned extra = 0;
    if (a.zero_vectors > 0) {
        const int64_t useful = (a.zero_vectors + kWarps * 32 - 1) / (kWarps * 32);
        extra = (unsigned)std::min<int64_t>(useful, 2 * (int64_t)device_sm_count());
        extra = (extra + blocks - 1) / blocks * blocks;   // whole clusters
    }
    config.gridDim = blocks + extra;
    attr.val.clusterDim.x = blocks;
    config.dynamicSmemBytes = bucket_smem(a.buckets);
    return cudaLaunchKernelEx(&config, bucket_kernel, a);
}

}  // namespace spmmb
