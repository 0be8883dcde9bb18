// Products of row ranges with 8-bit operands (e4m3) on the fifth-generation
// tensor cores, a scale for each block of 128 elements of the reduction.
//
//   out[r, c] = sum over b of sx[b, r] sw[g, c / 128, b] P_b[r, c],  P_b = sum over block b of x[r, k] w[g, c, k]
//
// A persistent block (with PAIR two, on a tile of 256 rows) walks output
// tiles of 128 x BN.  Warp 0 finds the tiles, hands them to the others through
// a ring and issues the TMA copies of 128-byte deep slices; a thread of warp 1
// issues their products; warp 2 brings the slices' scales into shared memory;
// the others read the accumulators.  A slice is one block b: its products go
// into an accumulator of their own, which the epilogue warps add to their
// registers times the two scales while the next slices run into the others (a
// sum over blocks cannot stay in TMEM, since the tensor core's own block
// scales are powers of two).  So P_b is the tensor core's fp32 sum of 128
// products, and the blocks are added in fp32 rounded to nearest.
//
// What bounds it, 65536 rows of 64 groups, K = 1024, N = 2048, bf16 results:
// 160 to 165 us, 1700 TFLOP/s (the same product in bf16 212 us).  The copies and
// products alone take 105 us, at the pace of shared memory (a pair's slice is
// written and read at 80 KB a block, 640 cycles for the products' 512).  An
// accumulator's way from the products to the readers and back is as long as
// two slices, and TMEM holds two: 25 us.  Reading them takes 14 us; the end of
// a tile, when the readers store and the products can be two slices ahead
// only, 30 us (K = 4096: 2050 TFLOP/s).  Measured and slower: eight readers of
// 128 columns (registers spill, and come back from L2, since shared memory
// leaves no L1: 187 us), 128-column tiles with four accumulators (184 us),
// stores by the readers' lanes (183 us).
//
// Every wait is bounded; a wait that runs out raises SPMM_DEV_TIMEOUT, and
// the block drains its copies and products, frees its TMEM and returns.
#pragma once

#include "../../include/spmm_b200.h"
#include "engine.h"
#include "gemm_tc.cuh"
#include "layer.cuh"
#include "layer.h"
#include "tc.cuh"

namespace spmmb {
namespace tc {

struct Fp8Args {
    Ranges ranges;
    int n, blocks_k, blocks_n;
    const float *scale_a;     // [blocks_k][rows]
    const float *scale_b;     // [groups][blocks_n][blocks_k]
    void *out;
    int out_type;
    DevStatus *status;
};

constexpr int kSlice = 128;           // bytes of a row, the block of a scale
constexpr int kTiles = 4;             // tiles handed out and not yet taken by every warp
constexpr int kGroup = 4, kScales = 2;   // slices whose scales are handed over at once; such groups in shared memory
constexpr int kEnd = -2, kOutside = -1;   // in the place of a group
// -0 in the place of a scale: its group of slices has products of scales that fp32 does not hold in full (they are 0,
// subnormal or infinite) although it may hold a block's sum times both, and a pair of factors for each row instead.
constexpr unsigned kFarScale = 0x80000000u;

template <int BN, bool PAIR> struct Fp8Shape {
    // epilogue warps: each has 32 rows and at most 64 columns in registers
    static constexpr int kReaders = BN == 256 ? 16 : 8, kOwn = BN / (kReaders / 4);
    static constexpr int kFirstReader = 4, kThreads = 32 * (kFirstReader + kReaders);   // warp 3 has no work
    static constexpr int kA = kBM * kSlice, kB = (PAIR ? BN / 2 : BN) * kSlice;
    static constexpr int kStages = BN == 256 ? 4 : BN == 128 ? 5 : 6, kStaging = 4096;             // of an epilogue warp: 32 rows x 128 bytes
    static constexpr int kAccs = BN == 256 ? 2 : 4, kCols = kAccs * BN;
    static constexpr int kHalves = BN == 256 ? 2 : 1, kScaleBytes = kHalves * kBM * 4;   // of a slice, per block of 128 columns
    static constexpr int kStageOff = kStages * (kA + kB), kScaleOff = kStageOff + kReaders * kStaging;
    static constexpr int kFactorOff = kScaleOff + kScales * kGroup * kScaleBytes;   // pairs of factors, laid out as the scales
    static constexpr int kTileOff = kFactorOff + 2 * kScales * kGroup * kScaleBytes;
    static constexpr int kFull = kTileOff + 16 * kTiles, kEmpty = kFull + 8 * kStages;
    static constexpr int kAccFull = kEmpty + 8 * kStages, kAccEmpty = kAccFull + 8 * kAccs;
    static constexpr int kTileFull = kAccEmpty + 8 * kAccs, kTileEmpty = kTileFull + 8 * kTiles;
    static constexpr int kScaleFull = kTileEmpty + 8 * kTiles, kScaleEmpty = kScaleFull + 8 * kScales;
    static constexpr int kDone = kScaleEmpty + 8 * kScales, kTmem = kDone + 8, kAbort = kTmem + 4, kBytes = kAbort + 4;
    static_assert(kBytes <= 232448 && kCols <= 512, "shared memory of a block, TMEM of an SM");
};

// A place in a ring of N (a power of two) and the parity of its rounds, from one counter.
template <int N> struct Turn {
    unsigned count = 0;
    __device__ __forceinline__ unsigned at() const { return count % N; }
    __device__ __forceinline__ unsigned parity() const { return count / N & 1u; }
    __device__ __forceinline__ void next() { ++count; }
};
// The same for any N.
template <int N> struct Ring {
    unsigned place = 0, turn = 0;
    __device__ __forceinline__ unsigned at() const { return place; }
    __device__ __forceinline__ unsigned parity() const { return turn; }
    __device__ __forceinline__ void next()
    {
        if (++place == N) {
            place = 0;
            turn ^= 1u;
        }
    }
};

// A sum is multiplied by the first factor and the result by the second: 1 and the product where fp32 holds that, else the
// smaller and the larger scale.  The first product leaves the range only where the result does, too: sums are 0 or at least
// 2^-18, scales, as quantising gives them, at least 2^-109 (and it is held to 2^-23 of itself).
__device__ __forceinline__ float2 factors(float a, float b)
{
    const float s = a * b;
    if (fabsf(s) >= 0x1p-126f && fabsf(s) < INFINITY) return make_float2(1.f, s);
    return fabsf(a) < fabsf(b) ? make_float2(a, b) : make_float2(b, a);
}

template <int BN, bool PAIR>
__global__ void __launch_bounds__(Fp8Shape<BN, PAIR>::kThreads, 1)
fp8_gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
                const __grid_constant__ CUtensorMap map_o, const __grid_constant__ Fp8Args a)
{
    using S = Fp8Shape<BN, PAIR>;
    constexpr int kHeight = PAIR ? 2 * kBM : kBM, kReaders = S::kReaders, kFirstReader = S::kFirstReader;
    extern __shared__ __align__(1024) unsigned char smem[];
    const unsigned base = (unsigned)__cvta_generic_to_shared(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int *abort = reinterpret_cast<volatile int *>(smem + S::kAbort);
    const unsigned full = base + S::kFull, empty = base + S::kEmpty;
    const unsigned acc_full = base + S::kAccFull, acc_empty = base + S::kAccEmpty;
    const unsigned scale_full = base + S::kScaleFull, scale_empty = base + S::kScaleEmpty;
    const unsigned tile_full = base + S::kTileFull, tile_empty = base + S::kTileEmpty, done = base + S::kDone;
    const unsigned peer = PAIR ? cluster_rank() : 0;   // 0: the pair's first block

    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kStages; ++i) {
            bar_init(full + 8 * i, 1);
            bar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < S::kAccs; ++i) {
            bar_init(acc_full + 8 * i, 1);
            bar_init(acc_empty + 8 * i, PAIR ? 2 * kReaders : kReaders);
        }
        for (int i = 0; i < kTiles; ++i) {
            bar_init(tile_full + 8 * i, 1);
            bar_init(tile_empty + 8 * i, 2 + kReaders);
        }
        for (int i = 0; i < kScales; ++i) {
            bar_init(scale_full + 8 * i, 1);
            bar_init(scale_empty + 8 * i, kReaders);
        }
        bar_init(done, 1);
        // a misaligned stage ring would break the swizzle: give up before any copy
        *abort = (base & 1023u) ? 1 : 0;
        if (base & 1023u) raise_status(a.status, SPMM_DEV_TIMEOUT, -1);
        asm volatile("fence.mbarrier_init.release.cluster;\n" ::: "memory");
        prefetch_map(&map_a);
        prefetch_map(&map_b);
        prefetch_map(&map_o);
    }
    if (PAIR) {   // the barriers of both blocks are set up
        __syncthreads();
        cluster_sync();
    }
    if (warp == 1) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(base + S::kTmem),
                         "r"(S::kCols)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;\n" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;\n" ::"r"(base + S::kTmem),
                         "r"(S::kCols)
                         : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;\n" ::: "memory");
        }
    }
    fence_before();
    __syncthreads();
    fence_after();
    const unsigned tmem = *reinterpret_cast<volatile unsigned *>(smem + S::kTmem);
    let_next_kernel_start();
    wait_for_earlier_kernels();   // nothing above reads or writes global memory

    bool ok = *abort == 0;
    auto give_up = [&](int code) {
        if (*abort == 0) raise_status(a.status, SPMM_DEV_TIMEOUT, code);
        *abort = 1;
        ok = false;
    };
    int4 *const tiles = reinterpret_cast<int4 *>(smem + S::kTileOff);   // first row, rows, first column, group

    if (warp == 0) {
        // ---- finds the tiles and issues their copies
        TileWalk<false> walk;
        Turn<kTiles> hand;
        Ring<S::kStages> stage;
        unsigned issued = 0;   // slices
        const unsigned nt = (unsigned)((a.n + BN - 1) / BN);
        for (int64_t tile = blockIdx.x / (PAIR ? 2 : 1); ok; tile += gridDim.x / (PAIR ? 2 : 1)) {
            int64_t seg, b, e, inner, slots;
            int4 t = make_int4(0, 0, 0, kEnd);
            if (walk.find(a.ranges, kHeight, nt, tile, a.status, &seg, &b, &e, &inner, &slots)) {
                const int64_t row = b + (int64_t)((unsigned)inner / nt) * kHeight + (PAIR ? (int)peer * kBM : 0);
                t = make_int4((int)row, (int)max((int64_t)0, min((int64_t)kBM, e - row)), (int)((unsigned)inner % nt) * BN,
                              seg >= 1 && seg <= a.ranges.groups ? (int)seg - 1 : kOutside);
            }
            if (!bar_wait(tile_empty + 8 * hand.at(), hand.parity() ^ 1u, abort)) { give_up(6); break; }
            if (lane == 0) {
                tiles[hand.at()] = t;
                bar_arrive(tile_full + 8 * hand.at());
            }
            __syncwarp();
            hand.next();
            if (t.w == kEnd) break;
            if (t.w < 0) continue;
            if (elect()) {
                const int col = t.z + (PAIR ? (int)peer * (BN / 2) : 0);
                for (int k = 0; k < a.blocks_k; ++k) {
                    if (!bar_wait(empty + 8 * stage.at(), stage.parity() ^ 1u, abort)) { give_up(1); break; }
                    const unsigned sa = base + stage.at() * (S::kA + S::kB), sb = sa + S::kA;
                    // a pair's slice, both halves, arrives on the first block's barrier
                    if (peer == 0) bar_expect(full + 8 * stage.at(), (PAIR ? 2 : 1) * (S::kA + S::kB));
                    if constexpr (PAIR) {
                        const unsigned bar = in_block(full + 8 * stage.at(), 0);
                        tma_load_pair(sa, &map_a, k * kSlice, t.x, 0, bar);
                        tma_load_pair(sb, &map_b, k * kSlice, col, t.w, bar);
                    } else {
                        tma_load(sa, &map_a, k * kSlice, t.x, 0, full + 8 * stage.at());
                        tma_load(sb, &map_b, k * kSlice, col, t.w, full + 8 * stage.at());
                    }
                    stage.next();
                }
            }
            __syncwarp();
            issued += a.blocks_k;
            ok = *abort == 0;
        }
        if (!ok && peer == 0) {   // copies in flight land before the block leaves (bounded; one never issued runs out)
            for (unsigned s = issued > 2 * S::kStages ? issued - 2 * S::kStages : 0; s < issued; ++s) {
                volatile int never = 0;
                if (!bar_wait(full + 8 * (s % S::kStages), s / S::kStages & 1u, &never)) break;
            }
        }
    } else if (warp == 1) {
        // ---- one thread issues the products (the second block's only takes the tiles)
        if (elect()) {
            const unsigned idesc = idesc8(kHeight, BN);
            const uint64_t da = desc128(base, 16, 1024), db = desc128(base + S::kA, 16, 1024);
            Turn<kTiles> hand;
            Ring<S::kStages> stage;
            Turn<S::kAccs> acc;
            while (ok) {
                if (!bar_wait(tile_full + 8 * hand.at(), hand.parity(), abort)) { give_up(7); break; }
                const int group = tiles[hand.at()].w;
                bar_arrive(tile_empty + 8 * hand.at());
                hand.next();
                if (group == kEnd) break;
                if (group < 0 || peer != 0) continue;
                for (int k = 0; k < a.blocks_k; ++k) {
                    if (!bar_wait<PAIR>(full + 8 * stage.at(), stage.parity(), abort)) { give_up(3); break; }
                    if (!bar_wait<PAIR>(acc_empty + 8 * acc.at(), acc.parity() ^ 1u, abort)) { give_up(2); break; }
                    fence_after();
                    const unsigned d = tmem + acc.at() * BN, off = stage.at() * (S::kA + S::kB) >> 4;
#pragma unroll
                    for (int i = 0; i < kSlice / 32; ++i) {
                        if constexpr (PAIR) mma_pair<true>(d, da + off + 2 * i, db + off + 2 * i, idesc, i > 0);
                        else mma<true>(d, da + off + 2 * i, db + off + 2 * i, idesc, i > 0);
                    }
                    if constexpr (PAIR) {
                        commit_pair(acc_full + 8 * acc.at());
                        commit_pair(empty + 8 * stage.at());
                    } else {
                        commit(acc_full + 8 * acc.at());
                        commit(empty + 8 * stage.at());
                    }
                    stage.next();
                    acc.next();
                }
            }
            if (!ok && peer == 0) {   // every product issued is complete before TMEM is freed (bounded)
                volatile int never = 0;
                if constexpr (PAIR) commit_pair(done);
                else commit(done);
                bar_wait(done, 0, &never);
            }
        }
        __syncwarp();
    } else if (warp == 2) {
        // ---- the scales of each slice: a row's times that of each block of columns
        float *const scales = reinterpret_cast<float *>(smem + S::kScaleOff);
        Turn<kTiles> hand;
        Turn<kScales> slot;
        while (ok) {
            if (!bar_wait(tile_full + 8 * hand.at(), hand.parity(), abort)) { give_up(9); break; }
            const int4 t = tiles[hand.at()];
            __syncwarp();
            if (lane == 0) bar_arrive(tile_empty + 8 * hand.at());
            hand.next();
            if (t.w == kEnd) break;
            if (t.w < 0) continue;
            for (int k0 = 0; k0 < a.blocks_k && ok; k0 += kGroup) {
                float rows[kGroup][4], cols[kGroup][S::kHalves];
#pragma unroll
                for (int j = 0; j < kGroup; ++j) {
                    const int k = min(k0 + j, a.blocks_k - 1);
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int r = lane + 32 * i;
                        rows[j][i] = r < t.y ? __ldg(a.scale_a + (int64_t)k * a.ranges.rows + t.x + r) : 1.f;
                    }
#pragma unroll
                    for (int h = 0; h < S::kHalves; ++h) {
                        const int block = min(t.z / kSlice + h, a.blocks_n - 1);
                        cols[j][h] = __ldg(a.scale_b + ((int64_t)t.w * a.blocks_n + block) * a.blocks_k + k);
                    }
                }
                if (!bar_wait(scale_empty + 8 * slot.at(), slot.parity() ^ 1u, abort)) { give_up(10); break; }
                float *to = scales + slot.at() * (kGroup * S::kScaleBytes / 4);
                // the extremes' products bound all of them (a NaN is no extreme: its products are NaN either way)
                float row_min = INFINITY, row_max = 0.f, col_min = INFINITY, col_max = 0.f;
#pragma unroll
                for (int j = 0; j < kGroup; ++j) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        row_min = fminf(row_min, fabsf(rows[j][i]));
                        row_max = fmaxf(row_max, fabsf(rows[j][i]));
                    }
#pragma unroll
                    for (int h = 0; h < S::kHalves; ++h) {
                        col_min = fminf(col_min, fabsf(cols[j][h]));
                        col_max = fmaxf(col_max, fabsf(cols[j][h]));
                    }
                }
                const bool far = __any_sync(~0u, !(row_min * col_min >= 0x1p-126f && row_max * col_max < INFINITY));
#pragma unroll
                for (int j = 0; j < kGroup; ++j)
#pragma unroll
                    for (int h = 0; h < S::kHalves; ++h)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            to[(j * S::kHalves + h) * kBM + lane + 32 * i] = far ? __uint_as_float(kFarScale) : rows[j][i] * cols[j][h];
                if (far) {
                    float2 *pair = reinterpret_cast<float2 *>(smem + S::kFactorOff) + slot.at() * (kGroup * S::kScaleBytes / 4);
#pragma unroll
                    for (int j = 0; j < kGroup; ++j)
#pragma unroll
                        for (int h = 0; h < S::kHalves; ++h)
#pragma unroll
                            for (int i = 0; i < 4; ++i)
                                pair[(j * S::kHalves + h) * kBM + lane + 32 * i] = factors(rows[j][i], cols[j][h]);
                }
                __syncwarp();
                if (lane == 0) bar_arrive(scale_full + 8 * slot.at());
                slot.next();
            }
        }
    } else if (warp >= kFirstReader) {
        // ---- epilogue warps: TMEM lanes 32 (warp % 4) .. + 31 are rows of the
        // tile; the warps of a lane quarter share the columns out
        constexpr int kOwn = S::kOwn, kRead = kReaders == 16 ? 8 : 32;   // its columns; read at a time
        const int row0 = (warp & 3) * 32, first = (warp - kFirstReader) / 4 * kOwn;
        const unsigned stage = base + S::kStageOff + (warp - kFirstReader) * S::kStaging;
        const unsigned lanes = tmem + ((unsigned)row0 << 16) + first;
        const float *const scales = reinterpret_cast<const float *>(smem + S::kScaleOff);
        const int place = first / kSlice * kBM + row0 + lane;   // of its row's scale
        const unsigned acc_empty_0 = PAIR ? in_block(acc_empty, 0) : 0;   // the first block's
        Turn<kTiles> hand;
        Turn<S::kAccs> acc;
        Turn<kScales> slot;
        while (ok) {
            if (!bar_wait(tile_full + 8 * hand.at(), hand.parity(), abort)) { give_up(8); break; }
            const int4 t = tiles[hand.at()];
            __syncwarp();
            if (lane == 0) bar_arrive(tile_empty + 8 * hand.at());
            hand.next();
            if (t.w == kEnd) break;
            const bool on = row0 + lane < t.y, any = row0 < t.y && t.z + first < a.n;
            float v[kOwn];
#pragma unroll
            for (int i = 0; i < kOwn; ++i) v[i] = 0.f;
            const int n = t.w >= 0 ? a.blocks_k : 0;
            int k = 0;
            // Adds up the slices from k on; without `two` until a group of them that has factors for its rows instead of
            // scales.  That is seen behind the sums of the group's first slice, to which a scale of -0 adds nothing, so that
            // they do not wait for it (a look ahead of them: 177 us for the 168 of 65536 rows, 64 groups, N 1920).
            auto add = [&](auto two) {
                for (; k < n; ++k) {
                    const int in_group = k % kGroup, at = (slot.at() * kGroup + in_group) * (S::kScaleBytes / 4) + place;
                    if (in_group == 0 && !bar_wait(scale_full + 8 * slot.at(), slot.parity(), abort)) { give_up(11); break; }
                    const float scale = scales[at];
                    if (!bar_wait<PAIR>(acc_full + 8 * acc.at(), acc.parity(), abort)) { give_up(4); break; }
                    fence_after();
                    if (any) {
                        const unsigned from = lanes + acc.at() * BN;
                        if constexpr (decltype(two)::value) {
                            const float2 f = __float_as_uint(scale) == kFarScale
                                                 ? reinterpret_cast<const float2 *>(smem + S::kFactorOff)[at]
                                                 : make_float2(1.f, scale);
#pragma unroll
                            for (int c = 0; c < kOwn; c += 2) {   // few at a time: the registers are those of the other form
                                float w[2];
                                tmem_ld(from + c, w);
                                v[c] = fmaf(w[0] * f.x, f.y, v[c]);
                                v[c + 1] = fmaf(w[1] * f.x, f.y, v[c + 1]);
                            }
                        } else {
#pragma unroll
                            for (int c = 0; c < kOwn; c += kRead) {
                                float w[kRead];
                                tmem_ld(from + c, w);
#pragma unroll
                                for (int i = 0; i < kRead; i += 2) fma2(v[c + i], v[c + i + 1], scale, w[i], w[i + 1]);
                            }
                            if (in_group == 0 && __any_sync(~0u, __float_as_uint(scale) == kFarScale)) break;   // it is added again
                        }
                    }
                    fence_before();
                    __syncwarp();
                    if (lane == 0) {
                        // to the first block's product thread: the TMEM reads above are complete.  A release to the cluster
                        // would do as well, but orders memory too: 282 us for the 163 of 65536 rows of 64 groups
                        if (PAIR) bar_arrive_tmem(acc_empty_0 + 8 * acc.at());
                        else bar_arrive(acc_empty + 8 * acc.at());
                    }
                    acc.next();
                    if (in_group == kGroup - 1 || k + 1 == n) {
                        if (lane == 0) bar_arrive(scale_empty + 8 * slot.at());
                        slot.next();
                    }
                }
            };
            add(std::false_type());
            if (ok && k < n) add(std::true_type());
            if (!ok) break;
            if (!any) continue;
            const int out_size = a.out_type == kOutF32 ? 4 : 2;
            // a group's last rows share the block with the next group's: no box for them
            const bool boxed = row0 + 32 <= t.y;
            const unsigned swz2 = (unsigned)(lane >> 1 & 3), swz4 = (unsigned)(lane & 7);
            if (boxed && out_size == 2) {   // all of the warp's columns in one box
                if (elect()) bulk_wait_read<0>();   // the staging's last store has read it
                __syncwarp();
                auto stage_row = [&](auto bf16) {
#pragma unroll
                    for (unsigned i = 0; i < kOwn / 8; ++i)
                        st_shared16(kOwn == 64 ? stage + lane * 128 + ((i ^ swz4) << 4) : stage + lane * 64 + ((i ^ swz2) << 4),
                                    pack8(v + 8 * i, decltype(bf16)::value));
                };
                if (a.out_type == kOutBf16) stage_row(std::true_type());
                else stage_row(std::false_type());
                fence_async();
                __syncwarp();
                if (elect()) {
                    tma_store(&map_o, stage, t.z + first, t.x + row0, 0);
                    bulk_commit();
                }
                continue;
            }
#pragma unroll
            for (int c = 0; c < kOwn; c += 32) {
                const int x = t.z + first + c;
                if (x >= a.n) break;
                if (boxed) {
                    if (elect()) bulk_wait_read<0>();
                    __syncwarp();
#pragma unroll
                    for (unsigned i = 0; i < 8; ++i)
                        st_shared16(stage + lane * 128 + ((i ^ swz4) << 4),
                                    make_uint4(__float_as_uint(v[c + 4 * i]), __float_as_uint(v[c + 4 * i + 1]),
                                               __float_as_uint(v[c + 4 * i + 2]), __float_as_uint(v[c + 4 * i + 3])));
                    fence_async();
                    __syncwarp();
                    if (elect()) {
                        tma_store(&map_o, stage, x, t.x + row0, 0);
                        bulk_commit();
                    }
                } else if (on) {   // each lane its row
                    char *o = static_cast<char *>(a.out) + ((int64_t)(t.x + row0 + lane) * a.n + x) * out_size;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        if (x + 8 * i >= a.n) break;
                        if (out_size == 4) {
                            float4 *q = reinterpret_cast<float4 *>(o) + 2 * i;
                            q[0] = make_float4(v[c + 8 * i], v[c + 8 * i + 1], v[c + 8 * i + 2], v[c + 8 * i + 3]);
                            q[1] = make_float4(v[c + 8 * i + 4], v[c + 8 * i + 5], v[c + 8 * i + 6], v[c + 8 * i + 7]);
                        } else {
                            reinterpret_cast<uint4 *>(o)[i] = pack8(v + c + 8 * i, a.out_type == kOutBf16);
                        }
                    }
                }
            }
        }
        bulk_wait();
    }
    fence_before();
    __syncthreads();
    if (PAIR) cluster_sync();   // neither block's memory or barriers are used any more
    fence_after();
    if (warp == 1) {
        if constexpr (PAIR)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(S::kCols) : "memory");
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;\n" ::"r"(tmem), "r"(S::kCols) : "memory");
    }
}

}  // namespace tc
}  // namespace spmmb
