// Products of row ranges in 8-bit floating point (e4m3) with a scale for each
// block of 128 elements of the reduction.
//
//   rows       s[b, r] = max |x[r, block b]| / 448,  q = e4m3(x / s); a block's scales lie together, as the
//              product's lanes read them
//   weights    s[g, c, b]: the same over blocks of 128 x 128; q is laid out
//              [groups, N, K], so that both operands have the reduction contiguous
//   product    y[r] = sum over b of sx[b, r] sw[g, n / 128, b] (q_x q_w over block b)   (fp8_gemm.cuh)
//
// The scales are fp32, of a maximum of at least 2^-100 over the finite values
// (smaller ones would make x / s leave fp32's normal range); infinities and
// NaN become NaN, which e4m3 has.
//
// Quantising is bound by memory and, near it, by instructions (14 for an
// element): 65537 rows of 1024 bf16 41 us, 203 MB, 0.76 of the copy bandwidth.
// Weights are quantised once, element by element and read twice: 64 x 1024 x 2048
// bf16 307 us, 1.3 TB/s of their 403 MB.
#include <cuda_fp8.h>

#include <algorithm>

#include "../../include/spmm_b200.h"
#include "common.cuh"
#include "engine.h"
#include "fp8_gemm.cuh"
#include "layer.cuh"
#include "layer.h"

namespace spmmb {

namespace {

constexpr int kBlock = 128;
constexpr float kLargest = 448.f, kTiny = 0x1p-100f;
constexpr unsigned kFull = 0xffffffffu;

__device__ __forceinline__ float finite_abs(float x) { return isfinite(x) ? fabsf(x) : 0.f; }
__device__ __forceinline__ float scale_of(float amax) { return __fdiv_rn(fmaxf(amax, kTiny), kLargest); }

// x / s correctly rounded, from the correctly rounded reciprocal of s
// (Markstein 1990: one residual and one correction of x * (1 / s)).  The scale
// keeps all of it in fp32's normal range, but for quotients that round to zero
// in e4m3.  Not finite: NaN (the residual of an infinity is).
__device__ __forceinline__ float quotient(float x, float s, float inverse)
{
    const float q = x * inverse;
    return copysignf(fmaf(fmaf(-q, s, x), inverse, q), x);   // -0 stays so
}
// Two of them in e4m3, to nearest.
__device__ __forceinline__ unsigned short quantized(float x0, float x1, float s, float inverse)
{
    return __nv_cvt_float2_to_fp8x2(make_float2(quotient(x0, s, inverse), quotient(x1, s, inverse)), __NV_SATFINITE,
                                    __NV_E4M3);
}

// 8 lanes per block of a row, 16 elements a lane (which share the scale's
// arithmetic); width is a multiple of 16.
template <typename T>
__global__ void __launch_bounds__(256) quantize_rows_kernel(const T *x, unsigned char *q, float *scale, int64_t rows,
                                                            int64_t width)
{
    tc::let_next_kernel_start();   // it waits for this one before it reads
    const int64_t blocks = (width + kBlock - 1) / kBlock, items = rows * blocks;
    const int lane = threadIdx.x & 7;
    const int64_t step = (int64_t)gridDim.x * (blockDim.x / 8);
    const int64_t step_rows = step / blocks, step_blocks = step % blocks;   // no division per block
    int64_t i = (int64_t)blockIdx.x * (blockDim.x / 8) + threadIdx.x / 8;
    int64_t r = i / blocks, b = i % blocks;
    for (int64_t base = (int64_t)blockIdx.x * (blockDim.x / 8); base < items; base += step) {
        // all lanes of a warp take the same turns
        const int64_t c = b * kBlock + lane * 16;
        const bool on = i < items && c < width;
        __align__(16) T raw[16];
#pragma unroll
        for (int v = 0; v < (int)sizeof(raw) / 16; ++v) {
            uint4 &to = reinterpret_cast<uint4 *>(raw)[v];
            to = make_uint4(0, 0, 0, 0);
            if (on) to = __ldcs(reinterpret_cast<const uint4 *>(x + r * width + c) + v);
        }
        float f[16];
#pragma unroll
        for (int e = 0; e < 16; ++e) f[e] = elem_f32<T>(raw[e]);
        auto largest = [&](auto of) {
            float m = 0.f;
#pragma unroll
            for (int e = 0; e < 16; ++e) m = fmaxf(m, of(f[e]));   // NaN is not the larger one
#pragma unroll
            for (int o = 4; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(kFull, m, o));
            return m;
        };
        float m = largest([](float v) { return fabsf(v); });
        if (__any_sync(kFull, isinf(m))) m = largest(finite_abs);
        const float s = scale_of(m), inverse = __frcp_rn(s);
        if (i < items && lane == 0) scale[b * rows + r] = s;
        if (on) {
            __align__(16) unsigned short o[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) o[e] = quantized(f[2 * e], f[2 * e + 1], s, inverse);
            *reinterpret_cast<uint4 *>(q + r * width + c) = *reinterpret_cast<const uint4 *>(o);
        }
        i += step;
        r += step_rows;
        b += step_blocks;
        if (b >= blocks) {
            b -= blocks;
            ++r;
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
        const float s = scale_of(m), inverse = __frcp_rn(s);
        if (threadIdx.x == 0) scale[i] = s;
        for (int64_t k = k0 + threadIdx.x / kBlock; k < min(k0 + kBlock, K); k += 2)
            if (n < N) tile[threadIdx.x % kBlock][k - k0] = (unsigned char)quantized(elem_f32<T>(src[k * N]), 0.f, s, inverse);
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

// Row tiles, at most: every group can end in a partial one; the rows outside
// the groups too.
int64_t row_tiles_of(const Fp8Launch &l, int height)
{
    return std::min(l.rows, (l.rows + height - 1) / height + l.groups + 1);
}

template <int BN, bool PAIR = false> cudaError_t launch_tiles(const Fp8Launch &l, const tc::Fp8Args &a, cudaStream_t stream)
{
    using S = tc::Fp8Shape<BN, PAIR>;
    auto kernel = tc::fp8_gemm_kernel<BN, PAIR>;
    static PerDevice<bool> ready;   // the attribute outlasts the call
    bool *done = ready.here();
    if (!done || !*done) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes);
        if (e != cudaSuccess) return e;
        if (done) *done = true;
    }
    CUtensorMap x, w, out;
    if (!tc::make_byte_map(&x, l.x, l.K, l.rows, 1, tc::kBM) ||
        !tc::make_byte_map(&w, l.groups > 0 ? l.w : l.x, l.K, l.groups > 0 ? l.N : 1, std::max<int64_t>(l.groups, 1),
                           PAIR ? BN / 2 : BN) ||
        // 16-bit results are stored 64 columns at a time, those of 32-column warps and fp32 ones 32
        !(S::kOwn == 64 && a.out_type != tc::kOutF32
              ? tc::make_map(&out, l.out, l.N, l.rows, 1, l.N, 0, 32, a.out_type == tc::kOutBf16)
              : tc::make_out_map(&out, l.out, l.N, l.rows, 1, l.N, 0, a.out_type)))
        return cudaErrorInvalidValue;
    constexpr int kBlocks = PAIR ? 2 : 1;   // per tile
    const int64_t tiles = row_tiles_of(l, kBlocks * tc::kBM) * ((l.N + BN - 1) / BN);
    const unsigned grid = kBlocks * (unsigned)std::max<int64_t>(1, std::min<int64_t>(tiles, device_sm_count() / kBlocks));
    return tc::launch_overlapped(kernel, grid, kBlocks, S::kThreads, S::kBytes, stream, x, w, out, a);
}

}  // namespace

cudaError_t launch_quantize_rows(const void *x, void *q, float *scale, int64_t rows, int64_t width, int dtype,
                                 cudaStream_t stream)
{
    return by_type(dtype, [&](auto type) {
        using T = decltype(type);
        const int64_t items = rows * ((width + kBlock - 1) / kBlock);
        quantize_rows_kernel<T><<<blocks_for(items, 32), 256, 0, stream>>>(
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
    tc::Fp8Args g{};
    g.ranges = Ranges{a.ptr, a.itype == SPMM_I64, a.groups, a.rows};
    g.n = (int)a.N;
    g.blocks_k = (int)((a.K + kBlock - 1) / kBlock);
    g.blocks_n = (int)((a.N + kBlock - 1) / kBlock);
    g.scale_a = a.x_scale;
    g.scale_b = a.w_scale;
    g.out = a.out;
    g.out_type = a.out_dtype == SPMM_F32 ? tc::kOutF32 : a.out_dtype == SPMM_BF16 ? tc::kOutBf16 : tc::kOutF16;
    g.status = a.status;
    // Pairs of blocks, 256 x 256, where there are tiles for all of them and groups are long enough that their last tile's
    // missing rows do not matter; 128 x 128 and the pairs, K = 1024, N = 2048: 65536 rows of 64 groups 183 and 165 us,
    // of 256 groups 202 and 179; 16384 rows of 8 47 and 45; 4096 rows of 4, N = 512, 7.4 and 10.3.  Tiles of 64 columns
    // where those of 128 would not fill the GPU: 512 rows of 4 groups, K = N = 1024, 6.8 and 6.2 us, 2048 rows of 8
    // groups 7.6 and 9.1.
    if (a.N % 256 == 0 && a.rows >= 256 * std::max<int64_t>(a.groups, 1) &&
        a.rows / 256 * (a.N / 256) >= device_sm_count() / 2)
        return launch_tiles<256, true>(a, g, stream);
    if (row_tiles_of(a, tc::kBM) * ((a.N + 127) / 128) >= device_sm_count()) return launch_tiles<128>(a, g, stream);
    return launch_tiles<64>(a, g, stream);
}

}  // namespace spmmb
