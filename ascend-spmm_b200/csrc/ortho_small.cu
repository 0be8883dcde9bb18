// Orthogonalised updates of matrices whose shorter side s is at most 128: all
// steps of one matrix in one block, one launch.
//
// Every step multiplies X from the left by the same polynomial of its own
// G = X X^T, so with T = a I + b G + c G G
//     X <- T X,   G <- T G T
// and five steps of X are one product Q X with Q the product of the T's.  So
// X is read to form G, the steps run on s x s matrices alone,
//     GG = G G;  T = a I + b G + c GG;  [H | Q] = T [G | Q];  G = H T
// (all of them polynomials of the first G: symmetric, and so read with the
// reduction contiguous on both sides), and X is read again for the result.
// With a launch per product such a matrix costs fifteen launches and their
// latencies (105 us for 128 x 64); the products on X were most of the rest.
//
// The block holds 128 x 128 matrices in shared memory and their accumulators
// in TMEM; X passes through in chunks of 256 columns.  A tall matrix is held
// as its transpose.  X as the second operand of Q X is MN-major: the bytes of
// a K-major [rows][64] tile are also those of an MN-major tile whose
// reduction runs down the rows.
//
// Precision: every operand is a high and a low fp16 part and every product
// takes high x high, high x low and low x high (22 bits).  The error before
// the result's rounding is 1e-5 for a gradient's spectrum and 4e-4 for a low
// rank with noise, against 2e-3 and more with 11-bit operands (the
// coefficients multiply an operand's rounding error by up to four a step).
// Along a direction without a singular value Q grows to a^steps, which fp16's
// range has to hold: eight steps with the default coefficients.
#include <algorithm>
#include <cmath>

#include "../../include/spmm_b200.h"
#include "common.cuh"
#include "engine.h"
#include "layer.cuh"
#include "layer.h"
#include "ortho.cuh"
#include "tc.cuh"

namespace spmmb {

namespace {

constexpr int kSide = 128, kChunk = 256;
constexpr int kThreads = 512;            // four threads per row
constexpr int kWarps = kThreads / 32;
constexpr int kAtom = kSide * 128;       // bytes of [128 rows][64 columns] fp16

// Shared memory.  G and Q: per part (high, low) and 64 columns an atom of G
// and below it one of Q, so that [G | Q] is one operand of 256 rows.  A chunk
// of X lies where it overlaps neither Q nor itself: high parts over T, low
// parts over G.
constexpr int kG = 0, kQ = kAtom, kPartGQ = 4 * kAtom, kStepGQ = 2 * kAtom;
constexpr int kT = 8 * kAtom, kPartT = 2 * kAtom, kStepT = kAtom;
constexpr int kBar = 12 * kAtom, kTmem = kBar + 8, kAbort = kTmem + 4, kRed = kAbort + 4, kBytes = kRed + 8 * kWarps;
static_assert(kBytes <= 232448, "shared memory of a block");

// Byte offset of columns 8 j .. 8 j + 7 of a row; `step` between atoms.
__device__ __forceinline__ unsigned piece(int row, int j, int step)
{
    return (unsigned)((j >> 3) * step + row * 128 + (((j & 7) ^ (row & 7)) << 4));
}

// High part at `hi`, the rest at `lo`.
__device__ __forceinline__ void put_split(unsigned hi, unsigned lo, const float *v)
{
    const uint4 w = tc::pack8(v, false);
    float h[8];
    unpack16<__half>(w, h);
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = v[e] - h[e];
    tc::st_shared16(hi, w);
    tc::st_shared16(lo, tc::pack8(h, false));
}

// A thread's columns of a chunk: pieces share, share + 4, ... of eight.
template <typename T>
__device__ __forceinline__ void load_chunk(float (&x)[64], const T *u, int s, int64_t r, bool tall, int row, int share,
                                           int64_t c0)
{
    constexpr int V = 16 / sizeof(T);
#pragma unroll
    for (int i = 0; i < 64; ++i) x[i] = 0.f;
    if (row >= s) return;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int64_t c = c0 + (share + 4 * i) * 8;
        if (c >= r) break;
        if (!tall && r % 8 == 0) {
#pragma unroll
            for (int k = 0; k < 8; k += V) {
                const uint4 w = __ldg(reinterpret_cast<const uint4 *>(u + row * r + c + k));
#pragma unroll
                for (int e = 0; e < V; ++e) x[8 * i + k + e] = elem_f32<T>(reinterpret_cast<const T *>(&w)[e]);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (c + e < r) x[8 * i + e] = elem_f32<T>(tall ? u[(c + e) * s + row] : u[row * r + c + e]);
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads, 1) ortho_small_kernel(const OrthoLaunch o, float scale_q)
{
    extern __shared__ __align__(1024) unsigned char smem[];
    const unsigned base = (unsigned)__cvta_generic_to_shared(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int row = (warp & 3) * 32 + lane, share = warp >> 2;
    const bool tall = o.m > o.n;
    const int s = (int)min(o.m, o.n);
    const int64_t r = max(o.m, o.n);
    volatile int *abort = reinterpret_cast<volatile int *>(smem + kAbort);
    const unsigned bar = base + kBar;
    const T *u = static_cast<const T *>(o.update) + (int64_t)blockIdx.x * o.m * o.n;

    if (threadIdx.x == 0) {
        tc::bar_init(bar, 1);
        *abort = 0;
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
    }
    if (warp == 0) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(base + kTmem),
                     "r"(512)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
    }

    // ---- the norm: squares in 64 bits (an fp32 update's can leave fp32's range)
    float x[64];
    double sum = 0.0;
    for (int64_t c = 0; c < r; c += kChunk) {
        load_chunk<T>(x, u, s, r, tall, row, share, c);
#pragma unroll
        for (int i = 0; i < 64; ++i) sum += (double)x[i] * (double)x[i];
    }
#pragma unroll
    for (int k = 16; k > 0; k >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, k);
    if (lane == 0) reinterpret_cast<double *>(smem + kRed)[warp] = sum;
    tc::fence_before();
    __syncthreads();
    tc::fence_after();
    const unsigned tmem = *reinterpret_cast<volatile unsigned *>(smem + kTmem);
    const unsigned lanes = tmem + ((unsigned)((warp & 3) * 32) << 16);
    constexpr unsigned kAccG = 0, kAccGG = 128, kAccW = 256;   // TMEM columns
    sum = 0.0;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) sum += reinterpret_cast<const double *>(smem + kRed)[w];
    const float scale = (float)(1.0 / (sqrt(sum) + (double)o.eps));

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
    // An operand: descriptors of its parts, 16-byte steps per 16 and per 64 of the reduction.
    struct Operand {
        uint64_t hi, lo;
        unsigned near_hi, far_hi, near_lo, far_lo;
    };
    auto k_major = [&](int at, int part, int step) {
        return Operand{tc::desc128(base + at, 16, 1024), tc::desc128(base + at + part, 16, 1024), 2, (unsigned)step >> 4,
                       2, (unsigned)step >> 4};
    };
    const Operand g = k_major(kG, kPartGQ, kStepGQ), q = k_major(kQ, kPartGQ, kStepGQ), t = k_major(kT, kPartT, kStepT);
    const Operand xk{tc::desc128(base + kT, 16, 1024), tc::desc128(base + kG, 16, 1024), 2, kAtom >> 4, 2, kStepGQ >> 4};
    const Operand xn{tc::desc128(base + kT, kAtom, 1024), tc::desc128(base + kG, kStepGQ, 1024), 128, 512, 128, 512};
    // d (+)= A B over n 16-deep steps, the small products first; by one thread.
    auto product = [&](unsigned d, const Operand &a, const Operand &b, int n, unsigned idesc, bool add) {
        for (int k = 0; k < n; ++k) {
            const unsigned i = k & 3, f = k >> 2;
            tc::mma(d, a.hi + i * a.near_hi + f * a.far_hi, b.lo + i * b.near_lo + f * b.far_lo, idesc, add || k > 0);
            tc::mma(d, a.lo + i * a.near_lo + f * a.far_lo, b.hi + i * b.near_hi + f * b.far_hi, idesc, 1);
        }
        for (int k = 0; k < n; ++k) {
            const unsigned i = k & 3, f = k >> 2;
            tc::mma(d, a.hi + i * a.near_hi + f * a.far_hi, b.hi + i * b.near_hi + f * b.far_hi, idesc, 1);
        }
    };
    const int ks = (s + 15) / 16, pieces = 2 * ks;   // of a square matrix's row
    const unsigned square = tc::idesc16(false, false, false, 128, 16 * ks);
    // This thread's pieces (share, share + 4, ...) of a row of a square accumulator, times f, to both parts at `to`.
    auto move = [&](unsigned column, float f, int to, int part, int step) {
        float v[32];
        tc::tmem_ld8x4(lanes + column + share * 8, 32, v);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            if (share + 4 * j >= pieces) break;
#pragma unroll
            for (int e = 0; e < 8; ++e) v[8 * j + e] *= f;
            const unsigned at = base + to + piece(row, share + 4 * j, step);
            put_split(at, at + part, v + 8 * j);
        }
    };
    // The chunk at column c to shared memory (x already holds an only chunk).
    auto stage = [&](int64_t c) {
        if (r > kChunk) load_chunk<T>(x, u, s, r, tall, row, share, c);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float v[8];
            if ((share + 4 * i) * 8 >= ((r - c + 63) & ~int64_t(63))) break;   // past the last atom that is read
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = x[8 * i + e] * scale * kScaleX;
            put_split(base + kT + piece(row, share + 4 * i, kAtom), base + kG + piece(row, share + 4 * i, kStepGQ), v);
        }
        publish();
    };

    if (o.steps > 0) {
        for (int64_t c = 0; c < r && ok; c += kChunk) {
            stage(c);
            if (warp == 0 && tc::elect()) {
                product(tmem + kAccG, xk, xk, (int)(min(r - c, (int64_t)kChunk) + 15) / 16, square, c > 0);
                tc::commit(bar);
            }
            ok = finished();
        }
        if (ok) move(kAccG, kScaleG / (kScaleX * kScaleX), kG, kPartGQ, kStepGQ);
        float unit_g = 1.f / (kScaleX * kScaleX);   // value of kAccG's units
        for (int step = 0; step < o.steps && ok; ++step) {
            const bool first = step == 0, last = step + 1 == o.steps;
            publish();
            if (warp == 0 && tc::elect()) {
                product(tmem + kAccGG, g, g, ks, square, false);
                tc::commit(bar);
            }
            if (!(ok = finished())) break;
            const float fg = o.b * unit_g, fgg = o.c / (kScaleG * kScaleG);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                float v[8], w[8];
                const int col = (share + 4 * j) * 8;
                if (share + 4 * j >= pieces) break;   // the same for the whole warp
                tc::tmem_ld8(lanes + kAccG + col, v);
                tc::tmem_ld8(lanes + kAccGG + col, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[e] = fmaf(fg, v[e], fgg * w[e]);
                    if (row == col + e && row < s) v[e] += o.a;
                    w[e] = v[e] * scale_q;
                    v[e] *= kScaleP;
                }
                const unsigned at = base + kT + piece(row, share + 4 * j, kStepT);
                put_split(at, at + kPartT, v);
                if (first) {   // Q = T
                    const unsigned to = base + kQ + piece(row, share + 4 * j, kStepGQ);
                    put_split(to, to + kPartGQ, w);
                }
            }
            if (first && last) break;
            publish();
            if (warp == 0 && tc::elect()) {
                if (last || (!first && s <= 64)) product(tmem + kAccW + 128, t, q, ks, square, false);
                if (first || s <= 64) {
                    if (!last) product(tmem + kAccW, t, g, ks, square, false);
                } else if (!last) {   // [G | Q] as one operand: T is read once
                    product(tmem + kAccW, t, g, ks, tc::idesc16(false, false, false, 128, 256), false);
                }
                tc::commit(bar);
            }
            if (!(ok = finished())) break;
            if (!first) move(kAccW + 128, 1.f / kScaleP, kQ, kPartGQ, kStepGQ);
            if (last) break;
            move(kAccW, 1.f / kScaleP, kG, kPartGQ, kStepGQ);   // H
            publish();
            if (warp == 0 && tc::elect()) {
                product(tmem + kAccG, g, t, ks, square, false);
                tc::commit(bar);
            }
            if (!(ok = finished())) break;
            unit_g = 1.f / (kScaleG * kScaleP);
            move(kAccG, 1.f / kScaleP, kG, kPartGQ, kStepGQ);
        }
        __syncthreads();   // T of a single step is written before X takes its place
    }

    // ---- the result
    __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(o.out) + (int64_t)blockIdx.x * o.m * o.n;
    for (int64_t c0 = 0; c0 < r && ok; c0 += kChunk) {
        const int cols = (int)min(r - c0, (int64_t)kChunk);
        if (o.steps > 0) {
            stage(c0);
            if (warp == 0 && tc::elect()) {
                product(tmem + kAccW, q, xn, ks, tc::idesc16(false, false, true, 128, (cols + 15) / 16 * 16), false);
                tc::commit(bar);
            }
            if (!(ok = finished())) break;
        } else if (r > kChunk) {
            load_chunk<T>(x, u, s, r, tall, row, share, c0);
        }
        const float f = o.steps > 0 ? 1.f / (scale_q * kScaleX) : scale;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int col = (share + 4 * i) * 8;
            if (col >= cols) break;   // the same for the whole warp
            float v[8];
            if (o.steps > 0) {
                tc::tmem_ld8(lanes + kAccW + col, v);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = x[8 * i + e];
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= f;
            if (row >= s) continue;
            if (!tall && r % 8 == 0) {
                *reinterpret_cast<uint4 *>(out + row * r + c0 + col) = tc::pack8(v, true);
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e)
                    if (col + e < cols)
                        out[tall ? (c0 + col + e) * s + row : row * r + c0 + col + e] = __float2bfloat16_rn(v[e]);
            }
        }
        if (r > kChunk) {   // the accumulator and the chunk are read before the next one
            tc::fence_before();
            __syncthreads();
            tc::fence_after();
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

template <typename T> cudaError_t run_small(const OrthoLaunch &o, float scale_q, cudaStream_t stream)
{
    auto kernel = ortho_small_kernel<T>;
    static PerDevice<bool> ready;
    bool *done = ready.here();
    if (!done || !*done) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
        if (e != cudaSuccess) return e;
        if (done) *done = true;
    }
    kernel<<<(unsigned)o.batch, kThreads, kBytes, stream>>>(o, scale_q);
    return cudaGetLastError();
}

// A power of two that keeps Q, at most max(1, |a|)^steps, in fp16's range; 0 if none does.
float q_scale(int steps, float a)
{
    const double largest = std::pow(std::max(1.0, std::fabs((double)a)), steps);
    if (!(largest <= 32768.0)) return 0.f;
    return (float)std::min(256.0, std::exp2(std::floor(std::log2(32768.0 / largest))));
}

}  // namespace

// The longer side: one block reads the whole matrix three times.
bool ortho_small_eligible(int64_t m, int64_t n, int steps, float a)
{
    return std::min(m, n) <= kSide && std::max(m, n) <= 4096 && q_scale(steps, a) > 0.f;
}

cudaError_t launch_ortho_small(const OrthoLaunch &o, cudaStream_t stream)
{
    const float scale_q = q_scale(o.steps, o.a);
    switch (o.dtype) {
        case SPMM_F16: return run_small<__half>(o, scale_q, stream);
        case SPMM_BF16: return run_small<__nv_bfloat16>(o, scale_q, stream);
        default: return run_small<float>(o, scale_q, stream);
    }
}

}  // namespace spmmb
