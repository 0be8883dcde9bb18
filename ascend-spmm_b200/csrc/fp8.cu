// Products of row ranges in 8-bit floating point (e4m3) with a scale for each
// block of 128 elements of the reduction.
//
//   rows       s[r, b] = max |x[r, block b]| / 448,  q = e4m3(x / s)
//   weights    s[g, c, b]: the same over blocks of 128 x 128; q is laid out
//              [groups, N, K], so that both operands have the reduction contiguous
//   product    y[r] = sum over b of sx[r, b] sw[g, n / 128, b] (q_x q_w over block b)
//
// The scales are fp32, of a maximum of at least 2^-100 over the finite values
// (smaller ones would make x / s leave fp32's normal range); infinities and
// NaN become NaN, which e4m3 has.
//
// A slice of the product's ring (gemm_tc.cuh) is 128 bytes deep, one block of
// the scales: each goes into an accumulator of its own, and the epilogue warps
// add it to their registers times its scales while the next one is computed.
#include <cuda_fp8.h>

#include <algorithm>

#include "../../include/spmm_b200.h"
#include "common.cuh"
#include "engine.h"
#include "gemm_tc.cuh"
#include "layer.cuh"
#include "layer.h"

namespace spmmb {

namespace {

constexpr int kBlock = 128;
constexpr float kLargest = 448.f, kTiny = 0x1p-100f;
constexpr unsigned kFull = 0xffffffffu;

__device__ __forceinline__ float finite_abs(float x) { return isfinite(x) ? fabsf(x) : 0.f; }
__device__ __forceinline__ float scale_of(float amax) { return __fdiv_rn(fmaxf(amax, kTiny), kLargest); }
// e4m3 of x / s, to nearest; not finite: NaN.
__device__ __forceinline__ unsigned char quantized(float x, float s)
{
    const float v = isfinite(x) ? __fdiv_rn(x, s) : NAN;
    return (unsigned char)__nv_cvt_float_to_fp8(v, __NV_SATFINITE, __NV_E4M3);
}

// 16 lanes per block of a row, 8 elements a lane; width is a multiple of 16.
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T *x, unsigned char *q, float *scale, int64_t rows,
                                                            int64_t width)
{
    const int64_t blocks = (width + kBlock - 1) / kBlock, items = rows * blocks;
    const int lane = threadIdx.x & 15;
    const int64_t step = (int64_t)gridDim.x * (blockDim.x / 16);
    const int64_t base = (int64_t)blockIdx.x * (blockDim.x / 16);
    for (int64_t b = base; b < items; b += step) {   // the same number of turns for both halves of a warp
        const int64_t i = b + threadIdx.x / 16;
        const int64_t r = i / blocks, c = i % blocks * kBlock + lane * 8;
        const bool on = i < items && c < width;
        float f[8];
        if (on) {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = elem_f32<T>(x[r * width + c + e]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = 0.f;
        }
        float m = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) m = fmaxf(m, finite_abs(f[e]));
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
        const float s = scale_of(m);
        if (i < items && lane == 0) scale[i] = s;
        if (on) {
            uint2 raw;
            unsigned char *o = reinterpret_cast<unsigned char *>(&raw);
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = quantized(f[e], s);
            *reinterpret_cast<uint2 *>(q + r * width + c) = raw;
        }
    }
}

// A block of threads per 128 x 128 block: w [groups, K, N] to q [groups, N, K].
template <typename T>
__global__ void __launch_bounds__(256) quantize_weight_kernel(const T *w, unsigned char *q, float *scale, int64_t groups,
                                                              int64_t K, int64_t N)
{
    __shared__ unsigned char tile[kBlock][kBlock + 4];   // [n][k]
    __shared__ float most[8];
    const int64_t kb = (K + kBlock - 1) / kBlock, nb = (N + kBlock - 1) / kBlock;
    for (int64_t i = blockIdx.x; i < groups * nb * kb; i += gridDim.x) {
        const int64_t g = i / (nb * kb), n0 = i / kb % nb * kBlock, k0 = i % kb * kBlock;
        const int64_t n = n0 + threadIdx.x % kBlock;
        const T *src = w + g * K * N + n;
        float m = 0.f;
        for (int64_t k = k0 + threadIdx.x / kBlock; k < min(k0 + kBlock, K); k += 2)
            if (n < N) m = fmaxf(m, finite_abs(elem_f32<T>(src[k * N])));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
        if (threadIdx.x % 32 == 0) most[threadIdx.x / 32] = m;
        __syncthreads();
        m = 0.f;
#pragma unroll
        for (int v = 0; v < 8; ++v) m = fmaxf(m, most[v]);
        const float s = scale_of(m);
        if (threadIdx.x == 0) scale[i] = s;
        for (int64_t k = k0 + threadIdx.x / kBlock; k < min(k0 + kBlock, K); k += 2)
            if (n < N) tile[threadIdx.x % kBlock][k - k0] = quantized(elem_f32<T>(src[k * N]), s);
        __syncthreads();
        for (int r = threadIdx.x / kBlock; r < kBlock && n0 + r < N; r += 2)
            if (k0 + threadIdx.x % kBlock < K)
                q[(g * N + n0 + r) * K + k0 + threadIdx.x % kBlock] = tile[r][threadIdx.x % kBlock];
        __syncthreads();
    }
}

unsigned blocks_for(int64_t items, int64_t per)
{
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>((items + per - 1) / per, 16 * (int64_t)device_sm_count()));
}

template <typename F> cudaError_t by_type(int dtype, F f)
{
    switch (dtype) {
        case SPMM_F16: return f(__half());
        case SPMM_BF16: return f(__nv_bfloat16());
        default: return f(float());
    }
}

template <int BN, bool PAIR = false>
cudaError_t fp8_tc(const Fp8Launch &a, tc::GemmArgs &g, int64_t row_tiles, cudaStream_t stream)
{
    tc::Maps m;
    const int64_t tiles = row_tiles * ((g.n + g.bn - 1) / g.bn);
    const int cols = PAIR ? BN / 2 : g.bn;   // of the weight that a block brings in
    if (!tc::make_byte_map(&m.a, a.x, a.K, a.rows, 1, tc::kBM) ||
        !tc::make_byte_map(&m.b, a.groups > 0 ? a.w : a.x, a.K, a.groups > 0 ? a.N : 1, std::max<int64_t>(a.groups, 1),
                           cols) ||
        !tc::make_out_map(&m.o, a.out, g.n, a.rows, 1, g.n, 0, g.out_type))
        return cudaErrorInvalidValue;
    m.p = m.o;
    return tc::launch_gemm<tc::kRows, BN, false, false, tc::kStoreScaled, PAIR>(m, g, tiles, stream);
}

}  // namespace

cudaError_t launch_quantize_rows(const void *x, void *q, float *scale, int64_t rows, int64_t width, int dtype,
                                 cudaStream_t stream)
{
    return by_type(dtype, [&](auto type) {
        using T = decltype(type);
        const int64_t items = rows * ((width + kBlock - 1) / kBlock);
        quantize_rows_kernel<T><<<blocks_for(items, 16), 256, 0, stream>>>(
            static_cast<const T *>(x), static_cast<unsigned char *>(q), scale, rows, width);
        return cudaGetLastError();
    });
}

cudaError_t launch_quantize_weight(const void *w, void *q, float *scale, int64_t groups, int64_t K, int64_t N, int dtype,
                                   cudaStream_t stream)
{
    return by_type(dtype, [&](auto type) {
        using T = decltype(type);
        const int64_t items = groups * ((K + kBlock - 1) / kBlock) * ((N + kBlock - 1) / kBlock);
        quantize_weight_kernel<T><<<blocks_for(items, 1), 256, 0, stream>>>(
            static_cast<const T *>(w), static_cast<unsigned char *>(q), scale, groups, K, N);
        return cudaGetLastError();
    });
}

cudaError_t launch_grouped_fp8(const Fp8Launch &a, cudaStream_t stream)
{
    tc::GemmArgs g{};
    g.ranges = Ranges{a.ptr, a.itype == SPMM_I64, a.groups, a.rows};
    g.n = a.N;
    g.k = a.K;
    g.out = a.out;
    g.ldo = a.N;
    g.out_type = a.out_dtype == SPMM_F32 ? tc::kOutF32 : a.out_dtype == SPMM_BF16 ? tc::kOutBf16 : tc::kOutF16;
    g.scale_a = a.x_scale;
    g.scale_b = a.w_scale;
    g.blocks_k = (a.K + kBlock - 1) / kBlock;
    g.blocks_n = (a.N + kBlock - 1) / kBlock;
    g.status = a.status;
    const int64_t row_tiles = std::min(a.rows, (a.rows + tc::kBM - 1) / tc::kBM + a.groups + 1);
    g.bn = tc::tile_columns(row_tiles, g.n, 256);
    if (g.bn <= 64) return fp8_tc<64>(a, g, row_tiles, stream);
    if (g.bn <= 128) return fp8_tc<128>(a, g, row_tiles, stream);
    return fp8_tc<256>(a, g, row_tiles, stream);
}

}  // namespace spmmb
