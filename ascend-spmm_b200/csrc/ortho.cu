// Orthogonalised updates: X0 = U / (|U|_F + eps), then `steps` times
//   G = X X^T,  P = b G + c G G,  X <- a X + P X
// on the smaller side s of the matrix (a tall matrix is worked on as its
// transpose).  Each step is two symmetric s x s products and one s x s by
// s x r product.
#include <algorithm>

#include "../../include/spmm_b200.h"
#include "common.cuh"
#include "engine.h"
#include "layer.cuh"
#include "layer.h"

namespace spmmb {

namespace {

constexpr int kTile = 64, kDepth = 16, kThreads = 256;

// 1 / (|U|_F + eps) of each matrix: one block per matrix, squares summed in
// 64 bits (an fp32 update's squares can pass fp32's range).
template <typename T>
__global__ void __launch_bounds__(1024) ortho_norm_kernel(const T *u, int64_t elems, float eps, float *scale)
{
    __shared__ double red[32];
    const T *p = u + (int64_t)blockIdx.x * elems;
    double s = 0.0;
    for (int64_t i = threadIdx.x; i < elems; i += 1024) {
        const double v = (double)elem_f32<T>(p[i]);
        s += v * v;
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0.0;
        for (int w = 0; w < 32; ++w) s += red[w];
        scale[blockIdx.x] = (float)(1.0 / (sqrt(s) + (double)eps));
    }
}

// X [s, r] in fp32 from the update (transposed when it is tall).
template <typename T>
__global__ void ortho_load_kernel(const T *u, const float *scale, float *x, int64_t m, int64_t n, int64_t batch)
{
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= batch * m * n) return;
    const int64_t q = i / (m * n), e = i % (m * n), r = e / n, c = e % n;
    x[q * m * n + (m > n ? c * m + r : e)] = elem_f32<T>(u[i]) * scale[q];
}

__global__ void ortho_store_kernel(const float *x, __nv_bfloat16 *out, int64_t m, int64_t n, int64_t batch)
{
    const int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (i >= batch * m * n) return;
    const int64_t q = i / (m * n), e = i % (m * n), r = e / n, c = e % n;
    out[i] = __float2bfloat16_rn(x[q * m * n + (m > n ? c * m + r : e)]);
}

// C = alpha * A B + beta * D, all [.., ..] fp32 row-major of one batch entry; TB: B transposed.
template <bool TB>
__global__ void __launch_bounds__(kThreads)
ortho_product_kernel(const float *A, const float *B, const float *D, float *C, int64_t m, int64_t n, int64_t depth,
                     float alpha, float beta)
{
    __shared__ float As[kDepth][kTile + 4], Bs[kDepth][kTile + 4];
    const int64_t q = blockIdx.z, i0 = (int64_t)blockIdx.y * kTile, j0 = (int64_t)blockIdx.x * kTile;
    A += q * m * depth;
    B += q * n * depth;
    const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
    float acc[4][4] = {};
    for (int64_t k0 = 0; k0 < depth; k0 += kDepth) {
        for (int i = threadIdx.x; i < kTile * kDepth; i += kThreads) {
            const int r = i / kDepth, k = i % kDepth;
            As[k][r] = i0 + r < m && k0 + k < depth ? A[(i0 + r) * depth + k0 + k] : 0.f;
            if (TB) {
                Bs[k][r] = j0 + r < n && k0 + k < depth ? B[(j0 + r) * depth + k0 + k] : 0.f;
            } else {
                const int kk = i / kTile, c = i % kTile;
                Bs[kk][c] = j0 + c < n && k0 + kk < depth ? B[(k0 + kk) * n + j0 + c] : 0.f;
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < kDepth; ++k)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(As[k][ty * 4 + i], Bs[k][tx * 4 + j], acc[i][j]);
        __syncthreads();
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t r = i0 + ty * 4 + i, c = j0 + tx * 4 + j;
            if (r < m && c < n) {
                const int64_t at = q * m * n + r * n + c;
                C[at] = alpha * acc[i][j] + (D ? beta * D[at] : 0.f);
            }
        }
}

}  // namespace

size_t ortho_workspace(int64_t batch, int64_t m, int64_t n, int)
{
    const int64_t s = std::min(m, n);
    return (size_t)(256 + 4 * batch + 8 * batch * m * n + 8 * batch * s * s);
}

cudaError_t launch_ortho(const OrthoLaunch &o, void *workspace, cudaStream_t stream)
{
    const int64_t s = std::min(o.m, o.n), r = std::max(o.m, o.n), elems = o.m * o.n, all = o.batch * elems;
    float *x = static_cast<float *>(workspace), *x2 = x + all, *g = x2 + all, *p = g + o.batch * s * s;
    float *scale = p + o.batch * s * s;
    const unsigned blocks = (unsigned)((all + 255) / 256);
    switch (o.dtype) {
        case SPMM_F16:
            ortho_norm_kernel<<<(unsigned)o.batch, 1024, 0, stream>>>(static_cast<const __half *>(o.update), elems, o.eps, scale);
            ortho_load_kernel<<<blocks, 256, 0, stream>>>(static_cast<const __half *>(o.update), scale, x, o.m, o.n, o.batch);
            break;
        case SPMM_BF16:
            ortho_norm_kernel<<<(unsigned)o.batch, 1024, 0, stream>>>(static_cast<const __nv_bfloat16 *>(o.update), elems, o.eps, scale);
            ortho_load_kernel<<<blocks, 256, 0, stream>>>(static_cast<const __nv_bfloat16 *>(o.update), scale, x, o.m, o.n, o.batch);
            break;
        default:
            ortho_norm_kernel<<<(unsigned)o.batch, 1024, 0, stream>>>(static_cast<const float *>(o.update), elems, o.eps, scale);
            ortho_load_kernel<<<blocks, 256, 0, stream>>>(static_cast<const float *>(o.update), scale, x, o.m, o.n, o.batch);
    }
    const dim3 square((unsigned)((s + kTile - 1) / kTile), (unsigned)((s + kTile - 1) / kTile), (unsigned)o.batch);
    const dim3 wide((unsigned)((r + kTile - 1) / kTile), (unsigned)((s + kTile - 1) / kTile), (unsigned)o.batch);
    for (int i = 0; i < o.steps; ++i) {
        ortho_product_kernel<true><<<square, kThreads, 0, stream>>>(x, x, nullptr, g, s, s, r, 1.f, 0.f);
        ortho_product_kernel<true><<<square, kThreads, 0, stream>>>(g, g, g, p, s, s, s, o.c, o.b);   // G is symmetric
        ortho_product_kernel<false><<<wide, kThreads, 0, stream>>>(p, x, x, x2, s, r, s, 1.f, o.a);
        std::swap(x, x2);
    }
    ortho_store_kernel<<<blocks, 256, 0, stream>>>(x, static_cast<__nv_bfloat16 *>(o.out), o.m, o.n, o.batch);
    return cudaGetLastError();
}

}  // namespace spmmb
