// Orthogonalised updates of matrices whose shorter side s is at most 128: the
// steps of one matrix run in one block.
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
// in TMEM; X passes through in chunks of 256 columns.  A short X stays in one
// block and one launch (kAll); of a long one many blocks form G in parts
// (kGram), one runs the steps and leaves Q in memory (kSteps), and many apply
// it (kApply): 30 x 4000 in one block takes 125 us, in parts 54 us.  A tall matrix is held
// as its transpose.  X as the second operand of Q X is MN-major: the bytes of
// a K-major [rows][64] tile are also those of an MN-major tile whose
// reduction runs down the rows.
//
// Precision: every operand is a high and a low fp16 part and every product
// takes high x high, high x low and low x high (22 bits).  The error before
// the result's rounding is 1e-5 for a gradient's spectrum and up to 8e-4 for a
// low rank with noise, against 2e-3 and more with 11-bit operands (the
// coefficients multiply an operand's rounding error by up to four a step).
//
// Where the form ends.  G <- T G T multiplies what was rounded in G along a
// small singular direction by T^2, a^2 = 11.9 a step with the default
// coefficients, and nothing ties it to X any more: an eigenvalue of 1e-8
// that should be zero, of either sign, is of order one eight steps later.  Low
// rank with noise, 128 x 256: 8e-4 after five steps, 9e-3 after six, 1e-1
// after seven, NaN after eight (the form of ortho.cu, which works on X itself:
// 3e-4 to 3e-3).  So the steps' growth of G's error is held to 2^15, five steps
// with the default coefficients; more go to ortho.cu.  Along a direction
// without a singular value Q grows to a^steps, which fp16's range has to hold,
// and G, T and T G with their fixed scales too: coefficients that leave it go
// to ortho.cu, whose scales follow them.
//
// Measured: 128 x 64 25 us, 46 of 256 x 128 49 us.  About a quarter of the
// time is the tensor core's; a step is three dependent products, each with a
// way through shared memory, a wait and a read of TMEM around it.
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
constexpr int kG_ = 0, kQ_ = kAtom, kPartGQ = 4 * kAtom, kStepGQ = 2 * kAtom;
constexpr int kT_ = 8 * kAtom, kPartT = 2 * kAtom, kStepT = kAtom;
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

enum Phase { kAll, kGram, kSteps, kApply };

// What the phases of a long matrix leave for each other.
struct Between {
    const double *squares;   // [batch][square_parts]
    int square_parts;
    float *gram;             // [batch][parts][128][128], in kScaleX^2 units
    int parts;
    int64_t per;             // columns of a part, a multiple of kChunk
    uint4 *q;                // [batch][2][128][16]: Q's parts, 8 columns each
};

template <typename T, int PHASE>
__global__ void __launch_bounds__(kThreads, 1) ortho_small_kernel(const OrthoLaunch o, float scale_q, const Between w)
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
    const int64_t matrix = blockIdx.y;
    const T *u = static_cast<const T *>(o.update) + matrix * o.m * o.n;
    // the columns of this block
    const int64_t c_begin = PHASE == kAll ? 0 : blockIdx.x * w.per;
    const int64_t c_end = PHASE == kAll ? r : min(r, c_begin + w.per);
    const bool reload = PHASE != kAll || r > kChunk;   // x holds one chunk

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
    if constexpr (PHASE == kAll) {
        for (int64_t c = 0; c < r; c += kChunk) {
            load_chunk<T>(x, u, s, r, tall, row, share, c);
#pragma unroll
            for (int i = 0; i < 64; ++i) sum += (double)x[i] * (double)x[i];
        }
    } else if constexpr (PHASE != kSteps) {
        for (int i = threadIdx.x; i < w.square_parts; i += kThreads) sum += w.squares[matrix * w.square_parts + i];
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
    const Operand g = k_major(kG_, kPartGQ, kStepGQ), q = k_major(kQ_, kPartGQ, kStepGQ), t = k_major(kT_, kPartT, kStepT);
    const Operand xk{tc::desc128(base + kT_, 16, 1024), tc::desc128(base + kG_, 16, 1024), 2, kAtom >> 4, 2, kStepGQ >> 4};
    const Operand xn{tc::desc128(base + kT_, kAtom, 1024), tc::desc128(base + kG_, kStepGQ, 1024), 128, 512, 128, 512};
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
        if (reload) load_chunk<T>(x, u, s, r, tall, row, share, c);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float v[8];
            if ((share + 4 * i) * 8 >= ((r - c + 63) & ~int64_t(63))) break;   // past the last atom that is read
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = x[8 * i + e] * scale * kScaleX;
            put_split(base + kT_ + piece(row, share + 4 * i, kAtom), base + kG_ + piece(row, share + 4 * i, kStepGQ), v);
        }
        publish();
    };

    if (PHASE != kApply && o.steps > 0) {
        float unit_g = 1.f / (kScaleX * kScaleX);   // value of kAccG's units
        float given[PHASE == kSteps ? 32 : 1];      // kSteps: this thread's part of the first G, in those units
        if constexpr (PHASE != kSteps) {
            for (int64_t c = c_begin; c < c_end && ok; c += kChunk) {
                stage(c);
                if (warp == 0 && tc::elect()) {
                    product(tmem + kAccG, xk, xk, (int)(min(r - c, (int64_t)kChunk) + 15) / 16, square, c > c_begin);
                    tc::commit(bar);
                }
                ok = finished();
            }
        }
        if constexpr (PHASE == kGram) {
            float v[32];
            tc::tmem_ld8x4(lanes + kAccG + share * 8, 32, v);
            float *to = w.gram + ((matrix * w.parts + blockIdx.x) * kSide + row) * kSide;
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (ok && row < s && share + 4 * j < pieces)
#pragma unroll
                    for (int e = 0; e < 8; e += 4)
                        *reinterpret_cast<float4 *>(to + (share + 4 * j) * 8 + e) =
                            make_float4(v[8 * j + e], v[8 * j + e + 1], v[8 * j + e + 2], v[8 * j + e + 3]);
        } else if constexpr (PHASE == kSteps) {   // the parts, in their order
#pragma unroll
            for (int i = 0; i < 32; ++i) given[i] = 0.f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if (share + 4 * j >= pieces) break;
                // G is symmetric: read down its columns, so that the lanes read one line
                const int col = (share + 4 * j) * 8;
                const float *from = w.gram + (matrix * w.parts * kSide + col) * kSide + row;
                if (row < s)
#pragma unroll 4
                    for (int k = 0; k < w.parts; ++k)
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            if (col + e < s) given[8 * j + e] += __ldg(from + ((int64_t)k * kSide + e) * kSide);
                float v[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) v[e] = given[8 * j + e] * (kScaleG / (kScaleX * kScaleX));
                const unsigned at = base + kG_ + piece(row, share + 4 * j, kStepGQ);
                put_split(at, at + kPartGQ, v);
            }
        } else if (ok) {
            move(kAccG, kScaleG / (kScaleX * kScaleX), kG_, kPartGQ, kStepGQ);
        }
        for (int step = 0; PHASE != kGram && step < o.steps && ok; ++step) {
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
                float v[8], gg[8];
                const int col = (share + 4 * j) * 8;
                if (share + 4 * j >= pieces) break;   // the same for the whole warp
                if (PHASE == kSteps && first) {
#pragma unroll
                    for (int e = 0; e < 8; ++e) v[e] = given[PHASE == kSteps ? 8 * j + e : 0];
                } else {
                    tc::tmem_ld8(lanes + kAccG + col, v);
                }
                tc::tmem_ld8(lanes + kAccGG + col, gg);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    v[e] = fmaf(fg, v[e], fgg * gg[e]);
                    if (row == col + e && row < s) v[e] += o.a;
                    gg[e] = v[e] * scale_q;
                    v[e] *= kScaleP;
                }
                const unsigned at = base + kT_ + piece(row, share + 4 * j, kStepT);
                put_split(at, at + kPartT, v);
                if (first) {   // Q = T
                    const unsigned to = base + kQ_ + piece(row, share + 4 * j, kStepGQ);
                    put_split(to, to + kPartGQ, gg);
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
            if (!first) move(kAccW + 128, 1.f / kScaleP, kQ_, kPartGQ, kStepGQ);
            if (last) break;
            move(kAccW, 1.f / kScaleP, kG_, kPartGQ, kStepGQ);   // H
            publish();
            if (warp == 0 && tc::elect()) {
                product(tmem + kAccG, g, t, ks, square, false);
                tc::commit(bar);
            }
            if (!(ok = finished())) break;
            unit_g = 1.f / (kScaleG * kScaleP);
            move(kAccG, 1.f / kScaleP, kG_, kPartGQ, kStepGQ);
        }
        __syncthreads();   // T of a single step is written before X takes its place
    }

    // ---- Q between the phases: part, row, piece
    if constexpr (PHASE == kSteps || PHASE == kApply) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int part = i & 1, j = share + 4 * (i >> 1);
            uint4 *at = w.q + ((matrix * 2 + part) * kSide + row) * 16 + j;
            uint4 *mine = reinterpret_cast<uint4 *>(smem + kQ_ + part * kPartGQ + piece(row, j, kStepGQ));
            if (j >= pieces) break;
            if (PHASE == kApply) *mine = *at;
            else if (ok) *at = *mine;   // this thread's own
        }
    }

    // ---- the result
    __nv_bfloat16 *out = static_cast<__nv_bfloat16 *>(o.out) + matrix * o.m * o.n;
    for (int64_t c0 = c_begin; (PHASE == kAll || PHASE == kApply) && c0 < c_end && ok; c0 += kChunk) {
        const int cols = (int)min(r - c0, (int64_t)kChunk);
        if (o.steps > 0) {
            stage(c0);
            if (warp == 0 && tc::elect()) {
                product(tmem + kAccW, q, xn, ks, tc::idesc16(false, false, true, 128, (cols + 15) / 16 * 16), false);
                tc::commit(bar);
            }
            if (!(ok = finished())) break;
        } else if (reload) {
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
        if (c0 + kChunk < c_end) {   // the accumulator and the chunk are read before the next one
            tc::fence_before();
            __syncthreads();
            tc::fence_after();
        }
    }

    if (!ok && threadIdx.x == 0) {
        raise_status(o.status, SPMM_DEV_TIMEOUT, matrix);
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

template <typename T, int PHASE>
cudaError_t run_phase(const OrthoLaunch &o, float scale_q, const Between &w, int64_t blocks, cudaStream_t stream)
{
    auto kernel = ortho_small_kernel<T, PHASE>;
    static PerDevice<bool> ready;
    bool *done = ready.here();
    if (!done || !*done) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, kBytes);
        if (e != cudaSuccess) return e;
        if (done) *done = true;
    }
    kernel<<<dim3((unsigned)blocks, (unsigned)o.batch), kThreads, kBytes, stream>>>(o, scale_q, w);
    return cudaGetLastError();
}

// Blocks of a matrix in parts (1: one block does it all).  A block alone takes
// about 22 us more for every chunk (128 x 1024 125 us, 128 x 4096 393), the
// four launches of a matrix in parts 77 and 88 us.  Many matrices fill the GPU
// by themselves; one block each and in parts, us:
//   128 x 4096:  64 matrices 422 and 304, 75 423 and 361, 100 426 and 437, 148 433 and 611
//   128 x 1024:  64 matrices 127 and 110, 75 127 and 137, 100 128 and 143, 148 135 and 187
//   30 x 4000:   64 matrices 189 and 125, 75 189 and 149, 100 189 and 185, 148 190 and 265
// Half of the SMs is between the crossovers; up to 200 and 300 matrices the two
// stay within 8 %.
int64_t parts_of(int64_t batch, int64_t m, int64_t n)
{
    const int64_t r = std::max(m, n), chunks = (r + kChunk - 1) / kChunk;
    return chunks <= 2 || (chunks <= 16 && batch > device_sm_count() / 2) ? 1 : std::min<int64_t>(chunks, 64);
}

Between between(int64_t batch, int64_t m, int64_t n, void *workspace)
{
    Between w{};
    const int64_t parts = parts_of(batch, m, n), chunks = (std::max(m, n) + kChunk - 1) / kChunk;
    if (parts == 1) return w;
    const int64_t each = (chunks + parts - 1) / parts;
    w.per = each * kChunk;
    w.parts = (int)((chunks + each - 1) / each);
    w.square_parts = ortho_square_parts(batch, m, n);
    w.q = static_cast<uint4 *>(workspace);
    w.gram = reinterpret_cast<float *>(w.q + batch * 2 * kSide * 16);
    w.squares = reinterpret_cast<const double *>(w.gram + batch * w.parts * kSide * kSide);
    return w;
}

template <typename T> cudaError_t run_small(const OrthoLaunch &o, float scale_q, void *workspace, cudaStream_t stream)
{
    const Between w = between(o.batch, o.m, o.n, workspace);
    if (w.parts == 0) return run_phase<T, kAll>(o, scale_q, w, 1, stream);
    cudaError_t e = launch_ortho_squares(o, const_cast<double *>(w.squares), stream);
    if (e == cudaSuccess && o.steps > 0) e = run_phase<T, kGram>(o, scale_q, w, w.parts, stream);
    if (e == cudaSuccess && o.steps > 0) e = run_phase<T, kSteps>(o, scale_q, w, 1, stream);
    if (e == cudaSuccess) e = run_phase<T, kApply>(o, scale_q, w, w.parts, stream);
    return e;
}

}  // namespace

// A power of two that keeps Q, a product of the steps' T, in fp16's range; 0
// for a longer side, and where an operand would leave that range or G's
// rounding would grow too far.
float ortho_small_scale(const OrthoLaunch &o)
{
    if (std::min(o.m, o.n) > kSide) return 0.f;
    OrthoReach at(o.a, o.b, o.c);
    double q = 1.0, growth = 1.0;   // growth: of G's error, up to its last use
    for (int i = 0; i < o.steps; ++i) {
        const double t = at.factor(), g = at.reach * at.reach;
        if (!(std::max(t * kScaleP, g * std::max(1.0, t) * kScaleG) <= kMostStored)) return 0.f;
        q *= std::max(1.0, t);
        if (i + 1 < o.steps) growth *= std::max(1.0, at.growth());
        if (!(growth <= 32768.0) || !(q <= kMostStored)) return 0.f;
        at.step();
    }
    return (float)std::min(256.0, std::exp2(std::floor(std::log2(kMostStored / q))));
}

size_t ortho_small_workspace(int64_t batch, int64_t m, int64_t n)
{
    const Between w = between(batch, m, n, nullptr);
    return w.parts == 0 ? 0
                        : (size_t)batch * (2 * kSide * 256 + (size_t)w.parts * kSide * kSide * 4 + 8 * w.square_parts);
}

cudaError_t launch_ortho_small(const OrthoLaunch &o, float scale_q, void *workspace, cudaStream_t stream)
{
    switch (o.dtype) {
        case SPMM_F16: return run_small<__half>(o, scale_q, workspace, stream);
        case SPMM_BF16: return run_small<__nv_bfloat16>(o, scale_q, workspace, stream);
        default: return run_small<float>(o, scale_q, workspace, stream);
    }
}

}  // namespace spmmb
