// Products of row ranges with one matrix each, and their gradients.
//
//   rows product      out[r] = x[r] W_g       (or x[r] W_g^T) for the rows r of group g
//   weight gradient   dW_g  = x_g^T dy_g      (a sum over the rows of group g)
//
// The group of a row tile is found on the device from the row ranges, so no
// length crosses to the host and a launch can be captured in a graph.
#include <algorithm>

#include "../../include/spmm_b200.h"
#include "common.cuh"
#include "engine.h"
#include "gemm_tc.cuh"
#include "layer.cuh"
#include "layer.h"

namespace spmmb {

namespace {

constexpr int kTile = 64, kDepth = 16, kThreads = 256;

__host__ __device__ Ranges ranges_of(const GroupedLaunch &a)
{
    return Ranges{a.ptr, a.itype == SPMM_I64, a.groups, a.rows};
}

// acc[4][4] of thread (ty, tx) += A[m, k] B[k, n] over one 64 x 64 tile, operands read by strides.
template <typename T>
__device__ __forceinline__ void simt_tile(const T *A, int64_t ars, int64_t acs, int64_t m, const T *B, int64_t brs,
                                          int64_t bcs, int64_t n, int64_t depth, float (&acc)[4][4])
{
    __shared__ float As[kDepth][kTile + 4], Bs[kDepth][kTile + 4];
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    for (int64_t k0 = 0; k0 < depth; k0 += kDepth) {
        for (int i = threadIdx.x; i < kTile * kDepth; i += kThreads) {
            const int r = i / kDepth, k = i % kDepth;
            As[k][r] = r < m && k0 + k < depth ? elem_f32<T>(A[r * ars + (k0 + k) * acs]) : 0.f;
            const int kk = i / kTile, c = i % kTile;
            Bs[kk][c] = c < n && k0 + kk < depth ? elem_f32<T>(B[(k0 + kk) * brs + c * bcs]) : 0.f;
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kDepth; ++k) {
            float a[4], b[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) { a[i] = As[k][ty * 4 + i]; b[i] = Bs[k][tx * 4 + i]; }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(a[i], b[j], acc[i][j]);
        }
        __syncthreads();
    }
}

template <typename T>
__device__ __forceinline__ void simt_store(T *C, int64_t ldc, int64_t m, int64_t n, const float (&acc)[4][4])
{
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
            if (ty * 4 + i < m && tx * 4 + j < n) C[(ty * 4 + i) * ldc + tx * 4 + j] = elem_of<T>(acc[i][j]);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) grouped_rows_simt_kernel(const GroupedLaunch a)
{
    __shared__ int64_t where[4];
    if (threadIdx.x < 32) {
        TileWalk walk;
        int64_t seg = -1, b = 0, e = 0, inner = 0;
        if (!walk.find(ranges_of(a), kTile, 1, blockIdx.x, a.status, &seg, &b, &e, &inner)) seg = -1;
        if (threadIdx.x == 0) { where[0] = seg; where[1] = b; where[2] = e; where[3] = inner; }
    }
    __syncthreads();
    const int64_t seg = where[0];
    if (seg < 0) return;
    const int64_t depth = a.transposed ? a.N : a.K, width = a.transposed ? a.K : a.N;
    const int64_t r0 = where[1] + where[3] * kTile, m = min((int64_t)kTile, where[2] - r0);
    const int64_t c0 = (int64_t)blockIdx.y * kTile, n = min((int64_t)kTile, width - c0);
    float acc[4][4] = {};
    if (seg >= 1 && seg <= a.groups) {
        const T *w = static_cast<const T *>(a.w) + (seg - 1) * a.K * a.N;
        const int64_t brs = a.transposed ? 1 : a.N, bcs = a.transposed ? a.N : 1;
        simt_tile<T>(static_cast<const T *>(a.x) + r0 * depth, depth, 1, m, w + c0 * bcs, brs, bcs, n, depth, acc);
    }
    simt_store<T>(static_cast<T *>(a.out) + r0 * width + c0, width, m, n, acc);
}

template <typename T>
__global__ void __launch_bounds__(kThreads) grouped_weight_grad_simt_kernel(const GroupedLaunch a)
{
    const int64_t tiles = (a.K + kTile - 1) / kTile;
    const int64_t g = blockIdx.x / tiles, i0 = blockIdx.x % tiles * kTile, c0 = (int64_t)blockIdx.y * kTile;
    int64_t b, e;
    segment_rows(ranges_of(a), g + 1, &b, &e, a.status);
    const int64_t m = min((int64_t)kTile, a.K - i0), n = min((int64_t)kTile, a.N - c0);
    float acc[4][4] = {};
    simt_tile<T>(static_cast<const T *>(a.x) + b * a.K + i0, 1, a.K, m, static_cast<const T *>(a.w) + b * a.N + c0, a.N,
                 1, n, e - b, acc);
    simt_store<T>(static_cast<T *>(a.out) + (g * a.K + i0) * a.N + c0, a.N, m, n, acc);
}

template <typename T> cudaError_t rows_simt(const GroupedLaunch &a, cudaStream_t stream)
{
    const int64_t width = a.transposed ? a.K : a.N;
    const dim3 grid((unsigned)((a.rows + kTile - 1) / kTile + a.groups + 2), (unsigned)((width + kTile - 1) / kTile));
    grouped_rows_simt_kernel<T><<<grid, kThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

template <typename T> cudaError_t weight_grad_simt(const GroupedLaunch &a, cudaStream_t stream)
{
    const dim3 grid((unsigned)((a.K + kTile - 1) / kTile * a.groups), (unsigned)((a.N + kTile - 1) / kTile));
    grouped_weight_grad_simt_kernel<T><<<grid, kThreads, 0, stream>>>(a);
    return cudaGetLastError();
}

// ---- 16-bit types: the tensor-core kernels of gemm_tc.cuh ------------------

// Columns per tile: the widest that the output's width fills and that still
// gives every SM a tile (a narrower tile reads the row operand more often).
int tile_columns(int64_t row_tiles, int64_t width)
{
    const int sms = device_sm_count();
    if (width > 128 && row_tiles * ((width + 255) / 256) >= sms) return 256;
    if (width > 64 && row_tiles * ((width + 127) / 128) >= sms) return 128;
    return 64;
}

template <int BN> cudaError_t rows_tc(const GroupedLaunch &a, tc::GemmArgs &g, int64_t row_tiles, cudaStream_t stream)
{
    CUtensorMap ma, mb;
    const bool bf = g.bf16;
    const int64_t tiles = row_tiles * ((g.n + BN - 1) / BN);
    if (!tc::make_map(&ma, a.x, g.k, a.rows, 1, g.k, 0, tc::kBM, bf)) return cudaErrorInvalidValue;
    const int64_t groups = std::max<int64_t>(a.groups, 1);
    const void *w = a.groups > 0 ? a.w : a.x;   // no group: the map is never read
    if (!tc::make_map(&mb, w, a.N, a.groups > 0 ? a.K : 1, groups, a.N, a.K * a.N, a.transposed ? BN : 64, bf))
        return cudaErrorInvalidValue;
    if (a.transposed) return tc::launch_gemm<tc::kRows, BN, false, false, tc::kStore>(ma, mb, g, tiles, stream);
    return tc::launch_gemm<tc::kRows, BN, false, true, tc::kStore>(ma, mb, g, tiles, stream);
}

cudaError_t launch_rows_tc(const GroupedLaunch &a, cudaStream_t stream)
{
    tc::GemmArgs g{};
    g.ranges = ranges_of(a);
    g.n = a.transposed ? a.K : a.N;
    g.k = a.transposed ? a.N : a.K;
    g.out = a.out;
    g.ldo = g.n;
    g.bf16 = a.dtype == SPMM_BF16;
    g.out_type = g.bf16 ? tc::kOutBf16 : tc::kOutF16;
    g.passes = 1;
    g.status = a.status;
    // every group can end in a partial tile; segments outside the groups too
    const int64_t row_tiles = std::min(a.rows, (a.rows + tc::kBM - 1) / tc::kBM + a.groups + 1);
    switch (tile_columns(row_tiles, g.n)) {
        case 256: return rows_tc<256>(a, g, row_tiles, stream);
        case 128: return rows_tc<128>(a, g, row_tiles, stream);
        default: return rows_tc<64>(a, g, row_tiles, stream);
    }
}

template <int BN> cudaError_t weight_grad_tc(const GroupedLaunch &a, tc::GemmArgs &g, cudaStream_t stream)
{
    CUtensorMap ma, mb;
    const bool bf = g.bf16;
    const int64_t rows = std::max<int64_t>(a.rows, 1);
    const void *x = a.rows > 0 ? a.x : a.out, *dy = a.rows > 0 ? a.w : a.out;   // no rows: the maps are never read
    if (!tc::make_map(&ma, x, a.K, rows, 1, a.K, 0, 64, bf) || !tc::make_map(&mb, dy, a.N, rows, 1, a.N, 0, 64, bf))
        return cudaErrorInvalidValue;
    const int64_t tiles = a.groups * ((a.K + tc::kBM - 1) / tc::kBM) * ((a.N + BN - 1) / BN);
    return tc::launch_gemm<tc::kRagged, BN, true, true, tc::kStore>(ma, mb, g, tiles, stream);
}

cudaError_t launch_weight_grad_tc(const GroupedLaunch &a, cudaStream_t stream)
{
    tc::GemmArgs g{};
    g.ranges = ranges_of(a);
    g.m = a.K;
    g.n = a.N;
    g.out = a.out;
    g.ldo = a.N;
    g.out_batch = a.K * a.N;
    g.bf16 = a.dtype == SPMM_BF16;
    g.out_type = g.bf16 ? tc::kOutBf16 : tc::kOutF16;
    g.passes = 1;
    g.status = a.status;
    switch (tile_columns(a.groups * ((a.K + tc::kBM - 1) / tc::kBM), a.N)) {
        case 256: return weight_grad_tc<256>(a, g, stream);
        case 128: return weight_grad_tc<128>(a, g, stream);
        default: return weight_grad_tc<64>(a, g, stream);
    }
}

}  // namespace

size_t grouped_rows_workspace(int64_t, int64_t, int64_t, int64_t, bool, int) { return 0; }
size_t grouped_weight_grad_workspace(int64_t, int64_t, int64_t, int64_t, int) { return 0; }

cudaError_t launch_grouped_rows(const GroupedLaunch &a, void *, cudaStream_t stream)
{
    return a.dtype == SPMM_F32 ? rows_simt<float>(a, stream) : launch_rows_tc(a, stream);
}

cudaError_t launch_grouped_weight_grad(const GroupedLaunch &a, void *, cudaStream_t stream)
{
    return a.dtype == SPMM_F32 ? weight_grad_simt<float>(a, stream) : launch_weight_grad_tc(a, stream);
}

}  // namespace spmmb
