// Orthogonalised updates of small matrices (shorter side at most 128, longer
// side at most 256): all steps of one matrix in one block, everything on chip.
//
// With a launch per product such a matrix costs fifteen launches and their
// latencies (105 us for 128 x 64, where the products themselves are a few
// microseconds).  Here a matrix stays in one SM: X in fp32 in registers and
// as high and low fp16 operands in shared memory, G and P in shared memory,
// the accumulators in TMEM.  A tall matrix is held as its transpose, so
// always s <= 128 rows of r <= 256.
//
//   G = X X^T       X both operands, K-major (the reduction runs along rows)
//   P = b G + c G G  G is symmetric, K-major on both sides; b G from TMEM
//   X <- a X + P X  P K-major; X as the second operand MN-major: the bytes
//                   of a K-major [rows][64] tile are also those of an
//                   MN-major tile whose reduction runs down the rows
//
// Every operand is a high and a low fp16 part and every product takes
// high x high, high x low and low x high (22 bits): three times the matrix
// instructions, but the error before the result's rounding falls from 2e-3
// (these coefficients multiply an operand's rounding error by up to four a
// step) to 1e-5.
#include <algorithm>

#include "../../include/spmm_b200.h"
#include "common.cuh"
#include "engine.h"
#include "layer.cuh"
#include "layer.h"
#include "ortho.cuh"
#include "tc.cuh"

namespace spmmb {

namespace {

constexpr int kRows = 128;
constexpr int kAtom = kRows * 128;   // bytes of [128 rows][64 columns] fp16

template <int R> struct SmallShape {
    // warps per 32 rows: each has a share of the columns, at most 64 of X in registers
    static constexpr int kShare = R > 128 ? 4 : 2, kWarps = 4 * kShare, kThreads = 32 * kWarps;
    static constexpr int kAtoms = R / 64;
    static constexpr int kHi = 0, kLo = kHi + kAtoms * kAtom;       // X
    static constexpr int kA = kLo + kAtoms * kAtom, kB = kA + 2 * kAtom;   // G, then P: high and low parts
    static constexpr int kBar = kB + 2 * kAtom, kTmem = kBar + 8, kAbort = kTmem + 4, kScale = kAbort + 4;
    static constexpr int kRed = kScale + 8, kBytes = kRed + 8 * kWarps;
    static_assert(kBytes <= 232448, "shared memory of a block");
};

// Byte offset of columns 8 j .. 8 j + 7 of a row in a buffer of swizzled [128][64] atoms.
__device__ __forceinline__ unsigned piece(int row, int j)
{
    return (unsigned)((j >> 3) * kAtom + row * 128 + (((j & 7) ^ (row & 7)) << 4));
}

__device__ __forceinline__ void put8(unsigned at, const float *v)
{
    const uint4 w = tc::pack8(v, false);
    tc::st_shared16(at, w);
}
// High part at `hi`, the rest at `lo`.
__device__ __forceinline__ void put8_split(unsigned hi, unsigned lo, const float *v)
{
    const uint4 w = tc::pack8(v, false);
    float h[8];
    unpack16<__half>(w, h);
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = v[e] - h[e];
    tc::st_shared16(hi, w);
    put8(lo, h);
}

template <typename T, int R>
__global__ void __launch_bounds__(SmallShape<R>::kThreads, 1) ortho_small_kernel(const OrthoLaunch o)
{
    using S = SmallShape<R>;
    constexpr int kOwn = R / S::kShare;       // columns of X of a thread (of its row)
    constexpr int kSq = kRows / S::kShare;    // columns of G and P
    extern __shared__ __align__(1024) unsigned char smem[];
    const unsigned base = (unsigned)__cvta_generic_to_shared(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row = (warp & 3) * 32 + lane, share = warp >> 2;
    const bool tall = o.m > o.n;
    const int s = (int)min(o.m, o.n), r = (int)max(o.m, o.n);
    volatile int *abort = reinterpret_cast<volatile int *>(smem + S::kAbort);
    const unsigned bar = base + S::kBar;

    if (threadIdx.x == 0) {
        tc::bar_init(bar, 1);
        *abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(base + S::kTmem),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }

    // ---- this thread's part of the matrix, its square sum in 64 bits
    const T *u = static_cast<const T *>(o.update) + (int64_t)blockIdx.x * o.m * o.n;
    float x[kOwn];
    double sum = 0.0;
#pragma unroll
    for (int i = 0; i < kOwn; ++i) x[i] = 0.f;
    const int c0 = share * kOwn;
    if (row < s) {
        constexpr int V = 16 / sizeof(T);
        if (!tall && r % V == 0) {
#pragma unroll
            for (int i = 0; i < kOwn; i += V)
                if (c0 + i < r) {
                    const uint4 w = __ldg(reinterpret_cast<const uint4 *>(u + (int64_t)row * r + c0 + i));
#pragma unroll
                    for (int e = 0; e < V; ++e) x[i + e] = elem_f32<T>(reinterpret_cast<const T *>(&w)[e]);
                }
        } else {
            const T *p = u + (tall ? (int64_t)c0 * s + row : (int64_t)row * r + c0);
            const int step = tall ? s : 1;
#pragma unroll
            for (int i = 0; i < kOwn; ++i)
                if (c0 + i < r) x[i] = elem_f32<T>(p[i * step]);
        }
#pragma unroll
        for (int i = 0; i < kOwn; ++i) sum += (double)x[i] * (double)x[i];
    }
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
    if (lane == 0) reinterpret_cast<double *>(smem + S::kRed)[warp] = sum;
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const unsigned tmem = *reinterpret_cast<volatile unsigned *>(smem + S::kTmem);
    const unsigned lanes = tmem + ((unsigned)((warp & 3) * 32) << 16);
    constexpr unsigned kG = 0, kGG = 128, kX = 256;   // TMEM columns of the accumulators
    sum = 0.0;
#pragma unroll
    for (int w = 0; w < S::kWarps; ++w) sum += reinterpret_cast<const double *>(smem + S::kRed)[w];
    const float scale = (float)(1.0 / (sqrt(sum) + (double)o.eps));
#pragma unroll
    for (int i = 0; i < kOwn; ++i) x[i] = x[i] * scale * kScaleX;

    bool ok = (base & 1023u) == 0;   // the swizzle needs 1024-byte alignment
    unsigned parity = 0;
    // Waits for the products committed to `bar`; the same answer in every thread.
    auto finished = [&]() {
        bool mine = tc::bar_wait(bar, parity, abort);
        parity ^= 1u;
        mine = __syncthreads_and(mine);
        tc::fence_after();
        return mine;
    };
    // Shared memory written by every thread, then read by the tensor core.
    auto publish = [&]() {
        tc::fence_async();
        tc::fence_before();
        __syncthreads();
        tc::fence_after();
    };
    const uint64_t hi = tc::desc128(base + S::kHi, 16, 1024), lo = tc::desc128(base + S::kLo, 16, 1024);
    const uint64_t hi_mn = tc::desc128(base + S::kHi, kAtom, 1024), lo_mn = tc::desc128(base + S::kLo, kAtom, 1024);
    const uint64_t pa = tc::desc128(base + S::kA, 16, 1024), pb = tc::desc128(base + S::kB, 16, 1024);
    // K-major: 16 columns further is 32 bytes, the next 64 an atom; MN-major: 16 rows further is 2048 bytes
    auto along = [](int k) { return (uint64_t)((k >> 2) * (kAtom >> 4) + (k & 3) * 2); };
    auto down = [](int k) { return (uint64_t)(k * 128); };
    constexpr unsigned kSquare = tc::idesc16(false, false, false, 128, 128);
    constexpr unsigned kWide = tc::idesc16(false, false, true, 128, R);
    const int kr = (r + 15) / 16, ks = (s + 15) / 16;

    for (int step = 0; step < o.steps && ok; ++step) {
#pragma unroll
        for (int j = 0; j < kOwn / 8; ++j) {
            const unsigned at = piece(row, c0 / 8 + j);
            put8_split(base + S::kHi + at, base + S::kLo + at, x + 8 * j);
        }
        publish();
        if (warp == 0 && tc::elect()) {
            for (int k = 0; k < kr; ++k) {   // the small products first
                tc::mma(tmem + kG, hi + along(k), lo + along(k), kSquare, k > 0);
                tc::mma(tmem + kG, lo + along(k), hi + along(k), kSquare, 1);
            }
            for (int k = 0; k < kr; ++k) tc::mma(tmem + kG, hi + along(k), hi + along(k), kSquare, 1);
            tc::commit(bar);
        }
        if (!(ok = finished())) break;
        {
            constexpr float f = kScaleG / (kScaleX * kScaleX);
#pragma unroll
            for (int c = 0; c < kSq / 32; ++c) {
                float v[32];
                tc::tmem_ld32(lanes + kG + share * kSq + c * 32, v);
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] *= f;
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const unsigned at = piece(row, share * (kSq / 8) + c * 4 + j);
                    put8_split(base + S::kA + at, base + S::kB + at, v + 8 * j);
                }
            }
        }
        publish();
        if (warp == 0 && tc::elect()) {
            for (int k = 0; k < ks; ++k) {
                tc::mma(tmem + kGG, pa + along(k), pb + along(k), kSquare, k > 0);
                tc::mma(tmem + kGG, pb + along(k), pa + along(k), kSquare, 1);
            }
            for (int k = 0; k < ks; ++k) tc::mma(tmem + kGG, pa + along(k), pa + along(k), kSquare, 1);
            tc::commit(bar);
        }
        if (!(ok = finished())) break;
        {
            const float fg = o.b * (kScaleP / (kScaleX * kScaleX)), fgg = o.c * (kScaleP / (kScaleG * kScaleG));
#pragma unroll
            for (int c = 0; c < kSq / 32; ++c) {
                float g[32], v[32];
                tc::tmem_ld32(lanes + kG + share * kSq + c * 32, g);
                tc::tmem_ld32(lanes + kGG + share * kSq + c * 32, v);
#pragma unroll
                for (int i = 0; i < 32; ++i) v[i] = fmaf(fg, g[i], fgg * v[i]);
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const unsigned at = piece(row, share * (kSq / 8) + c * 4 + j);
                    put8_split(base + S::kA + at, base + S::kB + at, v + 8 * j);
                }
            }
        }
        publish();
        if (warp == 0 && tc::elect()) {
            for (int k = 0; k < ks; ++k) {
                tc::mma(tmem + kX, pb + along(k), hi_mn + down(k), kWide, k > 0);
                tc::mma(tmem + kX, pa + along(k), lo_mn + down(k), kWide, 1);
            }
            for (int k = 0; k < ks; ++k) tc::mma(tmem + kX, pa + along(k), hi_mn + down(k), kWide, 1);
            tc::commit(bar);
        }
        if (!(ok = finished())) break;
#pragma unroll
        for (int c = 0; c < kOwn / 32; ++c) {
            float v[32];
            tc::tmem_ld32(lanes + kX + c0 + c * 32, v);
#pragma unroll
            for (int i = 0; i < 32; ++i) x[c * 32 + i] = fmaf(o.a, x[c * 32 + i], v[i] * (1.f / kScaleP));
        }
    }

    if (ok && row < s) {
        __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(o.out) + (int64_t)blockIdx.x * o.m * o.n;
#pragma unroll
        for (int i = 0; i < kOwn; ++i) x[i] *= 1.f / kScaleX;
        if (!tall && r % 8 == 0) {
#pragma unroll
            for (int i = 0; i < kOwn; i += 8)
                if (c0 + i < r) *reinterpret_cast<uint4 *>(out + (int64_t)row * r + c0 + i) = tc::pack8(x + i, true);
        } else {
            __nv_bfloat16 *p = out + (tall ? (int64_t)c0 * s + row : (int64_t)row * r + c0);
            const int step = tall ? s : 1;
#pragma unroll
            for (int i = 0; i < kOwn; ++i)
                if (c0 + i < r) p[i * step] = __float2bfloat16_rn(x[i]);
        }
    }
    if (!ok && threadIdx.x == 0) {
        raise_status(o.status, SPMM_DEV_TIMEOUT, blockIdx.x);
        // the products issued are complete before TMEM is freed (bounded)
        volatile int never = 0;
        tc::bar_wait(bar, parity ^ 1u, &never);
    }
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    if (warp == 0)
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(512) : "memory");
}

template <typename T, int R> cudaError_t run_small(const OrthoLaunch &o, cudaStream_t stream)
{
    auto kernel = ortho_small_kernel<T, R>;
    static PerDevice<bool> ready;
    bool *done = ready.here();
    if (!done || !*done) {
        const cudaError_t e =
            cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SmallShape<R>::kBytes);
        if (e != cudaSuccess) return e;
        if (done) *done = true;
    }
    kernel<<<(unsigned)o.batch, SmallShape<R>::kThreads, SmallShape<R>::kBytes, stream>>>(o);
    return cudaGetLastError();
}

template <typename T> cudaError_t run_type(const OrthoLaunch &o, cudaStream_t stream)
{
    const int64_t r = std::max(o.m, o.n);
    if (r <= 64) return run_small<T, 64>(o, stream);
    if (r <= 128) return run_small<T, 128>(o, stream);
    return run_small<T, 256>(o, stream);
}

}  // namespace

bool ortho_small_eligible(int64_t m, int64_t n) { return std::min(m, n) <= 128 && std::max(m, n) <= 256; }

cudaError_t launch_ortho_small(const OrthoLaunch &o, cudaStream_t stream)
{
    switch (o.dtype) {
        case SPMM_F16: return run_type<__half>(o, stream);
        case SPMM_BF16: return run_type<__nv_bfloat16>(o, stream);
        default: return run_type<float>(o, stream);
    }
}

}  // namespace spmmb
