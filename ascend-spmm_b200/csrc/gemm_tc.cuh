// Dense products on the fifth-generation tensor cores for the layer
// operators: 16-bit operands brought in by TMA, fp32 accumulators in TMEM.
//
// A persistent block per SM walks output tiles of 128 x bn (bn <= BN, so that
// a width just above a multiple of BN is cut into equal tiles).  One warp issues
// the TMA loads of 64-deep slices into a ring of stages, one warp the
// tcgen05.mma of each slice, and eight warps read a finished accumulator out
// of TMEM, round it and store it by TMA (32 rows x 32 columns at a time)
// while the next tile's products run into the other accumulator.  Operands
// may be stored with the reduction contiguous (K-major) or with the rows or
// columns contiguous (MN-major): both layouts are read as they lie, so no
// product needs a transposed copy.
//
// What a tile multiplies depends on the mode:
//   kRows    a row tile of one group times that group's matrix; the group is
//            found from the row ranges on the device, and rows of a tile
//            past its group's end are computed and not stored
//   kRagged  x_g^T dy_g: the reduction runs over a group's rows, in parts of
//            `part_rows` (a longer group's parts are stored in fp32 and added
//            afterwards); of a group's last slice the rows past its end are
//            set to zero in shared memory (in both operands: a neighbour's
//            infinity times zero would be NaN)
//   kDense   a batch of equal products
//
// What bounds it: a slice of 128 x 256 takes about 840 cycles where its
// products take 512, near the 768 in which its 48 KB are written to shared
// memory and read by the tensor core at 128 bytes a cycle; in pairs of blocks (32 KB
// a slice) the tensor pipe is 85 % busy, at the clock that the power limit
// leaves (1.44 GHz of 1.965).  65536 rows of 64 even groups, K = 1024, N =
// 2048, bf16: 212 us, 1300 TFLOP/s (cuBLAS on one large product: 1391
// sustained, 1647 in a burst).
//
// Every wait is bounded; a wait that runs out raises SPMM_DEV_TIMEOUT, and
// the block drains its copies and products, frees its TMEM and returns.
#pragma once

#include <algorithm>

#include "../../include/spmm_b200.h"
#include "engine.h"
#include "layer.cuh"
#include "layer.h"
#include "tc.cuh"

namespace spmmb {
namespace tc {

enum Mode { kRows, kRagged, kDense };
// The tensor core truncates its accumulator towards zero in every step of 16,
// by up to 2^-22 of what it holds: 16384 products of one sign lose 1e-4 of
// their sum, 65536 4e-4, an fp16 result's rounding.  kRagged and kGram end an
// accumulation there; kRows and the other dense products run over a matrix's
// width in one.
// kStoreSum: fp32 operands in three bf16 planes h, m, l each.  A slice brings
// in the planes once, a ring stage each, for its six products h l, l h, m m,
// h m, m h and h h.  The tensor core truncates each step into its accumulator,
// so an accumulator takes one slice, the smallest products first, and the
// epilogue warps add the slices in registers, rounding to nearest (K = 4096:
// error 1.4e-7, with two slices 5e-7 and 6 % less time, with four 1.2e-6).
// The others but kStore are kDense's: see ortho.cu.  kGram, whose products are
// squares on the diagonal and run down a matrix's long side, takes a new
// accumulator every 256 slices: in a single one 2^20 columns lost 6e-3 of G
// and moved a 136-row update by 6e-3, 16384 lose 1e-4.
enum Epi { kStore, kStoreSum, kGram, kPoly, kUpdate };
enum OutType { kOutF16, kOutBf16, kOutF32 };

struct GemmArgs {
    Ranges ranges;            // kRows, kRagged
    int64_t m, n, k;          // kRows: n, k; kRagged: m, n; kDense: all
    int bn;                   // columns of a tile, at most the kernel's BN: a multiple of 32 (16 for a single one)
    int64_t batch;            // kDense
    int64_t part_rows;        // kRagged: a multiple of 64
    int64_t part_slots;       // kRagged: parts in the second output map ([part_slots][m][n])
    void *out;
    int64_t ldo, out_batch;   // elements
    int out_type;
    bool bf16;                // operand type (else fp16)
    int za, zb;               // kStoreSum: plane p of A starts at batch index p * za, of B at p * zb
    // MN-major operands whose map has the blocks of 64 rows or columns as a
    // dimension (make_blocked_map): a slice is one copy instead of one per
    // block, and the issuing lane keeps up with the tensor core
    bool blocked_a, blocked_b;
    // kGram: x = alpha * accumulator; kPoly, kUpdate: x = alpha * accumulator
    // + beta * (in + in_lo), `in` laid out as the output.  kGram and kPoly
    // are symmetric and, with `symmetric`, compute one of two mirrored tiles
    // and write it twice; kUpdate writes x as fp16 and, with `low`, the rest
    // that the rounding left through the second output map (else x alone, in
    // the output's type).
    float alpha, beta;
    bool symmetric;           // kGram, kPoly: only the tiles on and below the diagonal (bn == 128)
    const __half *in, *in_lo;
    bool low;
    int64_t ldi, in_batch;
    DevStatus *status;
};

constexpr int kBM = 128, kBK = 64;
constexpr int kEpiWarps = 8, kGemmThreads = 64 + 32 * kEpiWarps;   // TMA warp, MMA warp, epilogue warps

constexpr int kSorted = 128;   // most groups that a weight gradient sorts
constexpr int kAsked = 4;      // tiles asked for and not yet done by every warp

template <int BN, bool PAIR = false> struct GemmShape {
    static constexpr int kA = kBM * kBK * 2, kB = (PAIR ? BN / 2 : BN) * kBK * 2;
    static constexpr int kStages = PAIR ? 6 : BN == 256 ? 4 : BN == 128 ? 6 : 8;
    static constexpr int kRows = PAIR ? 2 * kBM : kBM;           // of a tile
    static constexpr int kStageOff = kStages * (kA + kB);
    static constexpr int kStaging = 4096;                        // of an epilogue warp
    static constexpr int kBarOff = kStageOff + kEpiWarps * kStaging;
    static constexpr int kFull = kBarOff, kEmpty = kFull + 8 * kStages, kAccFull = kEmpty + 8 * kStages;
    static constexpr int kAccEmpty = kAccFull + 16, kDone = kAccEmpty + 16, kTmem = kDone + 8, kAbort = kTmem + 4;
    // kRagged: the groups in descending order of length (see Order)
    static constexpr int kOrder = kAbort + 4, kFirst = kOrder + 2 * kSorted, kSlot = kFirst + 4 * (kSorted + 1);
    static constexpr int kBegin = kSlot + 4 * kSorted, kLength = kBegin + 4 * kSorted;
    static constexpr int kAnswer = (kLength + 4 * kSorted + 15) / 16 * 16, kAskFull = kAnswer + 16 * kAsked;
    static constexpr int kAskEmpty = kAskFull + 8 * kAsked, kBytes = kAskEmpty + 8 * kAsked;
    static constexpr int kCols = 2 * BN;                         // TMEM columns of the two accumulators
    static_assert(kBytes <= 232448, "shared memory of a block");
};

// The tiles of a block, for one of its warps.  kRows and kDense deal them out
// in turn.  kRagged, whose tiles differ in length, launches a block per tile,
// and a running block takes over those that have not started, one after the
// other: the TMA warp asks, a few tiles ahead of the others (ring of kAsked).
template <int MODE, int BN, bool PAIR> struct Turns {
    using S = GemmShape<BN, PAIR>;
    static constexpr int kBlocks = PAIR ? 2 : 1;   // per tile
    const unsigned base;
    volatile int *const abort;
    const bool asks;       // the TMA warp
    int64_t tile;
    unsigned turn = 0;

    __device__ Turns(unsigned base, volatile int *abort, bool asks)
        : base(base), abort(abort), asks(asks), tile(blockIdx.x / kBlocks)
    {
    }
    // Warp-wide, at the start of the current tile.
    __device__ __forceinline__ bool ask()
    {
        if (MODE != kRagged || !asks) return true;
        const unsigned slot = turn % kAsked;
        if (!bar_wait(base + S::kAskEmpty + 8 * slot, (turn / kAsked & 1u) ^ 1u, abort)) return false;
        if (elect()) {
            fence_async();   // the slot's last answer was read before
            bar_expect(base + S::kAskFull + 8 * slot, 16);
            ask_for_block(base + S::kAnswer + 16 * slot, base + S::kAskFull + 8 * slot);
        }
        __syncwarp();
        return true;
    }
    // Warp-wide: goes to the next tile; tile < 0 past the last.  False if a wait ran out.
    __device__ __forceinline__ bool next()
    {
        if (MODE != kRagged) {
            tile += gridDim.x / kBlocks;
            return true;
        }
        const unsigned slot = turn % kAsked;
        if (!bar_wait(base + S::kAskFull + 8 * slot, turn / kAsked & 1u, abort)) return false;
        tile = block_given(base + S::kAnswer + 16 * slot);
        fence_async();
        __syncwarp();
        if (elect()) bar_arrive(base + S::kAskEmpty + 8 * slot);
        ++turn;
        return true;
    }
};

// One output tile as each role sees it.
struct Tile {
    int64_t batch_a, batch_b, row0, col0;   // operand batch, first row and column
    int64_t k0, k1;                         // range of the reduction (k0 == k1: zeros)
    int64_t out_row, out_z;                 // first row and batch index in the output
    bool part;                              // kRagged: one part of several
    int rows, cols;                         // what is stored
    bool mirror;                            // kGram, kPoly: also the transposed tile
};

// A weight gradient's groups by length, longest first: its tiles take as long
// as their group's rows (of a part), and handed out in this order to the
// blocks as they become free they end within one short tile of each other.
// Up to kSorted groups, which is what shared memory has room for beside the
// ring; with more the tiles are handed out in the groups' order (not measured
// against a sorted one).
struct Order {
    const unsigned short *group;   // [groups], nullptr: not sorted
    const int *first;              // [groups + 1] tiles before the group of this rank
    const int *slot;               // [groups] by group: its first part's slot, -1 with a single part
    const int *begin, *length;     // [groups] by group: its rows
};

// Every thread of the block.
__device__ __forceinline__ void sort_groups(const GemmArgs &a, int tiles, unsigned short *group, int *first, int *slot,
                                            int *begin, int *length)
{
    const int n = (int)a.ranges.groups, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (int g = threadIdx.x; g < n; g += blockDim.x) {
        int64_t b, e;
        segment_rows(a.ranges, g + 1, &b, &e, a.status);
        begin[g] = (int)b;
        length[g] = (int)(e - b);
    }
    __syncthreads();
    for (int g = threadIdx.x; g < n; g += blockDim.x) {
        int rank = 0;
        for (int i = 0; i < n; ++i) rank += length[i] > length[g] || (length[i] == length[g] && i < g);
        group[rank] = (unsigned short)g;
    }
    __syncthreads();
    if (warp < 2) {   // warp 0: tiles by rank; warp 1: slots by group
        int before = 0;
        for (int base = 0; base < n; base += 32) {
            const int i = base + lane;
            int v = 0;
            if (i < n) {
                const int parts = (int)((length[warp ? i : group[i]] + a.part_rows - 1) / a.part_rows);
                v = warp ? (parts > 1 ? parts : 0) : max(parts, 1) * tiles;
            }
            int sum = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int u = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += u;
            }
            if (i < n) (warp ? slot : first)[i] = warp && v == 0 ? -1 : before + sum - v;
            before += __shfl_sync(0xffffffffu, sum, 31);
        }
        if (warp == 0 && lane == 0) first[n] = before;
    }
    __syncthreads();
}

template <int MODE, int EPI, bool PAIR> struct Walk {
    static constexpr int kHeight = PAIR ? 2 * kBM : kBM;   // rows of a tile
    const GemmArgs &a;
    const Order order;
    TileWalk<MODE == kRagged> ranges;
    unsigned mt, nt;   // tiles down and across (an output that fits the GPU has fewer than 2^32 tiles)
    int rank = 0;
    __device__ Walk(const GemmArgs &a, const Order &order)
        : a(a), order(order), mt((unsigned)((a.m + kHeight - 1) / kHeight)), nt((unsigned)((a.n + a.bn - 1) / a.bn))
    {
    }

    // Warp-wide: the tile of index t; false past the last tile.
    __device__ __forceinline__ bool at(int64_t t, Tile *o)
    {
        if constexpr (MODE == kRows) {
            int64_t seg, b, e, inner, slots;
            if (!ranges.find(a.ranges, kHeight, nt, t, a.status, &seg, &b, &e, &inner, &slots)) return false;
            o->row0 = b + (int64_t)((unsigned)inner / nt) * kHeight;
            o->col0 = (int64_t)((unsigned)inner % nt) * a.bn;
            o->batch_a = 0;
            o->batch_b = seg - 1;
            o->k0 = 0;
            o->k1 = seg >= 1 && seg <= a.ranges.groups ? a.k : 0;
            o->rows = (int)min((int64_t)kHeight, e - o->row0);
            o->out_row = o->row0;
            o->out_z = 0;
        } else if constexpr (MODE == kRagged) {
            int64_t seg, b, e, inner, slots;
            if (order.group) {
                const int groups = (int)a.ranges.groups;
                if (rank >= groups || order.first[rank] > t) rank = 0;
                while (rank < groups && order.first[rank + 1] <= t) ++rank;
                if (rank >= groups) return false;
                seg = order.group[rank] + 1;
                inner = t - order.first[rank];
                slots = order.slot[seg - 1];
                b = order.begin[seg - 1];
                e = b + order.length[seg - 1];
            } else if (!ranges.find(a.ranges, a.part_rows, (int64_t)mt * nt, t, a.status, &seg, &b, &e, &inner, &slots)) {
                return false;
            }
            const int64_t p = (unsigned)inner / (mt * nt);
            const unsigned i = (unsigned)inner % (mt * nt);
            o->k0 = b + p * a.part_rows;
            o->k1 = min(e, o->k0 + a.part_rows);
            o->row0 = (int64_t)(i / nt) * kHeight;
            o->col0 = (int64_t)(i % nt) * a.bn;
            o->batch_a = o->batch_b = 0;
            o->rows = (int)min((int64_t)kHeight, a.m - o->row0);
            o->part = slots >= 0;
            if (o->part && slots + p >= a.part_slots) {   // only overlapping (malformed) ranges can need more
                o->k1 = o->k0;
                o->rows = 0;
            }
            o->out_row = o->row0;
            o->out_z = o->part ? slots + p : seg - 1;
        } else {
            const bool half = a.symmetric;   // the tiles on and below the diagonal
            const unsigned per = half ? mt * (mt + 1) / 2 : mt * nt;
            if (t >= a.batch * per) return false;
            const unsigned q = (unsigned)t / per, r = (unsigned)t % per;
            unsigned i, j;
            if (half) {
                i = (unsigned)((sqrtf(8.f * (float)r + 1.f) - 1.f) * 0.5f);
                while (i * (i + 1) / 2 > r) --i;
                while ((i + 1) * (i + 2) / 2 <= r) ++i;
                j = r - i * (i + 1) / 2;
            } else {
                i = r / nt;
                j = r % nt;
            }
            o->batch_a = o->batch_b = q;
            o->row0 = (int64_t)i * kHeight;
            o->col0 = (int64_t)j * a.bn;
            o->k0 = 0;
            o->k1 = a.k;
            o->rows = (int)min((int64_t)kHeight, a.m - o->row0);
            o->out_row = o->row0;
            o->out_z = q;
            o->mirror = half && i != j;
        }
        o->cols = (int)min((int64_t)a.bn, a.n - o->col0);
        if (PAIR) {   // this block's half of the rows
            const int skip = (int)cluster_rank() * kBM;
            o->row0 += skip;
            o->out_row += skip;
            o->rows = max(0, min(kBM, o->rows - skip));
        }
        return true;
    }
};

// PAIR: two blocks share a tile of 256 rows (tcgen05.mma.cta_group::2).  Each
// brings in its 128 rows of A and half of the columns of B, so a slice of
// 256 columns costs a block 32 KB instead of 48 KB; the first block's MMA
// warp issues the products of both, and each block stores its own rows.
template <int MODE, int BN, bool AMN, bool BMN, int EPI, bool PAIR>
__global__ void __launch_bounds__(kGemmThreads, 1)
gemm_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b,
            const __grid_constant__ CUtensorMap map_o, const __grid_constant__ CUtensorMap map_p,
            const __grid_constant__ GemmArgs a)
{
    static_assert(!PAIR || MODE != kRagged, "a group's zeros are written by one block");
    using S = GemmShape<BN, PAIR>;
    constexpr int kParts = EPI == kStoreSum ? 3 : 1;   // ring stages of a slice
    constexpr int kSlices = EPI == kStoreSum ? 1 : EPI == kGram ? 256 : 0;   // of an accumulator, 0: all
    static_assert(S::kStages >= 2 * kParts, "a slice arrives while another is multiplied");
    extern __shared__ __align__(1024) unsigned char smem[];
    const unsigned base = (unsigned)__cvta_generic_to_shared(smem);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    volatile int *abort = reinterpret_cast<volatile int *>(smem + S::kAbort);
    const unsigned full = base + S::kFull, empty = base + S::kEmpty;
    const unsigned acc_full = base + S::kAccFull, acc_empty = base + S::kAccEmpty, done = base + S::kDone;
    const unsigned peer = PAIR ? cluster_rank() : 0;   // 0: the pair's first block

    if (threadIdx.x == 0) {
        for (int i = 0; i < S::kStages; ++i) {
            bar_init(full + 8 * i, 1);
            bar_init(empty + 8 * i, 1);
        }
        for (int i = 0; i < 2; ++i) {
            bar_init(acc_full + 8 * i, 1);
            bar_init(acc_empty + 8 * i, PAIR ? 2 * kEpiWarps : kEpiWarps);
        }
        bar_init(done, 1);
        for (int i = 0; i < kAsked; ++i) {
            bar_init(base + S::kAskFull + 8 * i, 1);
            bar_init(base + S::kAskEmpty + 8 * i, 2 + kEpiWarps);
        }
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

    Order order{};
    if constexpr (MODE == kRagged)
        if (a.ranges.groups <= kSorted) {
            unsigned short *group = reinterpret_cast<unsigned short *>(smem + S::kOrder);
            int *first = reinterpret_cast<int *>(smem + S::kFirst), *slot = reinterpret_cast<int *>(smem + S::kSlot);
            int *begin = reinterpret_cast<int *>(smem + S::kBegin), *length = reinterpret_cast<int *>(smem + S::kLength);
            sort_groups(a, (int)((a.m + S::kRows - 1) / S::kRows * ((a.n + a.bn - 1) / a.bn)), group, first, slot, begin,
                        length);
            order = Order{group, first, slot, begin, length};
        }
    Walk<MODE, EPI, PAIR> walk(a, order);
    // the columns of B that a slice brings in (MN-major: in blocks of 64), and its bytes
    const int b_cols = PAIR ? BN / 2 : a.bn, b_blocks = BMN ? (b_cols + 63) / 64 : 0;
    const unsigned slice_bytes = S::kA + (BMN ? b_blocks * 8192 : b_cols * 128);
    Tile t;
    bool ok = *abort == 0;
    auto give_up = [&](int code) {
        if (*abort == 0) raise_status(a.status, SPMM_DEV_TIMEOUT, code);
        *abort = 1;
        ok = false;
    };

    if (warp == 0) {
        // ---- TMA warp: all lanes find the tile, one issues its copies
        unsigned slice = 0;   // slices issued
        Turns<MODE, BN, PAIR> turns(base, abort, true);
        for (; ok && turns.tile >= 0; turns.next() ? void() : give_up(5)) {
            if (!turns.ask()) { give_up(6); break; }
            if (!walk.at(turns.tile, &t)) {
                if (MODE == kRagged) continue;
                break;
            }
            const int n = (int)((t.k1 - t.k0 + kBK - 1) / kBK);
            if (elect()) {
                const int row0 = (int)t.row0, col0 = (int)t.col0 + (PAIR ? (int)peer * b_cols : 0);
                unsigned at = slice;
                int k = (int)t.k0;
                for (int i = 0; i < n && ok; ++i, k += kBK)
#pragma unroll
                    for (int j = 0; j < kParts; ++j, ++at) {
                        const int plane = kParts == 1 ? 0 : (j + 2) % 3;   // l, h, m: l is done with first
                        const int za = (int)t.batch_a + plane * a.za, zb = (int)t.batch_b + plane * a.zb;
                        const unsigned st = at % S::kStages;
                        if (!bar_wait(empty + 8 * st, (at / S::kStages & 1u) ^ 1u, abort)) { give_up(1); break; }
                        const unsigned sa = base + st * (S::kA + S::kB), sb = sa + S::kA;
                        // a pair's slice, both halves, arrives on the first block's barrier
                        const unsigned bar = PAIR ? in_block(full + 8 * st, 0) : full + 8 * st;
                        if (peer == 0) bar_expect(full + 8 * st, PAIR ? 2 * slice_bytes : slice_bytes);
                        auto load = [&](unsigned dst, const CUtensorMap *map, int x, int y, int z) {
                            if constexpr (PAIR) tma_load_pair(dst, map, x, y, z, bar);
                            else tma_load(dst, map, x, y, z, bar);
                        };
                        auto load_blocks = [&](unsigned dst, const CUtensorMap *map, int x, int z) {
                            if constexpr (PAIR) tma_load4_pair(dst, map, 0, k, x / 64, z, bar);
                            else tma_load4(dst, map, 0, k, x / 64, z, bar);
                        };
                        if (!AMN) {
                            load(sa, &map_a, k, row0, za);
                        } else if (a.blocked_a) {
                            load_blocks(sa, &map_a, row0, za);
                        } else {
#pragma unroll
                            for (int c = 0; c < kBM / 64; ++c) load(sa + c * 8192, &map_a, row0 + 64 * c, k, za);
                        }
                        if (!BMN) {
                            load(sb, &map_b, k, col0, zb);
                        } else if (a.blocked_b) {
                            load_blocks(sb, &map_b, col0, zb);
                        } else {
#pragma unroll
                            for (int c = 0; c < BN / 64; ++c)
                                if (c < b_blocks) load(sb + c * 8192, &map_b, col0 + 64 * c, k, zb);
                        }
                    }
            }
            __syncwarp();
            slice += kParts * n;
            ok = *abort == 0;
        }
        if (!ok) {   // copies and an answer in flight land before the block leaves (bounded; one never issued runs out)
            volatile int no = 0;
            if (MODE == kRagged) bar_wait(base + S::kAskFull + 8 * (turns.turn % kAsked), turns.turn / kAsked & 1u, &no);
            for (unsigned s = slice > 2 * S::kStages ? slice - 2 * S::kStages : 0; s < slice; ++s) {
                volatile int never = 0;
                if (!bar_wait(full + 8 * (s % S::kStages), s / S::kStages & 1u, &never)) break;
            }
        }
    } else if (warp == 1) {
        // ---- MMA warp: one lane issues
        const unsigned idesc = idesc16(a.bf16, AMN, BMN, S::kRows, PAIR ? BN : a.bn);
        // byte strides of the operands' layouts: K-major, 8 rows of 128 bytes per
        // swizzle atom; MN-major, atoms of 64 rows or columns x 8 deep, 8 KB apart
        const uint64_t da = AMN ? desc128(base, 8192, 1024) : desc128(base, 16, 1024);
        const uint64_t db = BMN ? desc128(base + S::kA, 8192, 1024) : desc128(base + S::kA, 16, 1024);
        constexpr unsigned step_a = (AMN ? 2048 : 32) >> 4, step_b = (BMN ? 2048 : 32) >> 4;
        unsigned slice = 0, used = 0;
        auto mul = [&](unsigned d, uint64_t x, uint64_t y, unsigned add) {
            if constexpr (PAIR) mma_pair(d, x, y, idesc, add);
            else mma(d, x, y, idesc, add);
        };
        auto finish = [&](unsigned bar) {
            if constexpr (PAIR) commit_pair(bar);
            else commit(bar);
        };
        auto product = [&](unsigned at_a, unsigned at_b, int depth, unsigned d, bool first) {
            const unsigned off_a = at_a % S::kStages * (S::kA + S::kB) >> 4;
            const unsigned off_b = at_b % S::kStages * (S::kA + S::kB) >> 4;
            if (depth == kBK) {
#pragma unroll
                for (int i = 0; i < kBK / 16; ++i)
                    mul(d, da + off_a + i * step_a, db + off_b + i * step_b, first && i == 0 ? 0u : 1u);
            } else {
                for (int i = 0; i * 16 < depth; ++i)
                    mul(d, da + off_a + i * step_a, db + off_b + i * step_b, first && i == 0 ? 0u : 1u);
            }
        };
        auto landed = [&](unsigned at) {
            return bar_wait<PAIR>(full + 8 * (at % S::kStages), at / S::kStages & 1u, abort);
        };
        auto release = [&](unsigned at) { finish(empty + 8 * (at % S::kStages)); };
        // The products of the slice at ring position `at` (depth elements deep);
        // false if a wait ran out.
        auto multiply = [&](unsigned at, int depth, unsigned d, bool first) {
            if constexpr (kParts == 1) {
                if (!landed(at)) return false;
                product(at, at, depth, d, first);
                release(at);
            } else {   // the smallest first
                const unsigned l = at, h = at + 1, m = at + 2;
                if (!landed(l) || !landed(h)) return false;
                product(h, l, depth, d, first);
                product(l, h, depth, d, false);
                release(l);
                if (!landed(m)) return false;
                product(m, m, depth, d, false);
                product(h, m, depth, d, false);
                product(m, h, depth, d, false);
                product(h, h, depth, d, false);
                release(h);
                release(m);
            }
            return true;
        };
        Turns<MODE, BN, PAIR> turns(base, abort, false);
        for (; ok && turns.tile >= 0; turns.next() ? void() : give_up(5)) {
            if (!walk.at(turns.tile, &t)) {
                if (MODE == kRagged) continue;
                break;
            }
            const int depth = (int)(t.k1 - t.k0), n = (depth + kBK - 1) / kBK;
            if (n <= 0) continue;
            // kRagged: a last slice that ends within 16 rows needs the whole warp
            const bool ragged = MODE == kRagged && (depth & 15);
            const int whole = ragged ? n - 1 : n;
            const int sum = kSlices ? min(kSlices, n) : n;
            for (int s0 = 0; s0 < n && ok; s0 += sum, ++used) {
                const unsigned d = tmem + (used & 1u) * BN;
                if (peer == 0 && !bar_wait<PAIR>(acc_empty + 8 * (used & 1u), (used >> 1 & 1u) ^ 1u, abort)) {
                    give_up(2);
                    break;
                }
                fence_after();
                const int s1 = min(s0 + sum, n);
                if (peer == 0 && elect())
                    for (int i = s0; i < min(s1, whole); ++i)
                        if (!multiply(slice + kParts * (i - s0), min(kBK, depth - i * kBK), d, i == s0)) {
                            give_up(3);
                            break;
                        }
                __syncwarp();
                slice += kParts * (s1 - s0);
                if (ragged && s1 == n && *abort == 0) {
                    const unsigned at = slice - kParts;
                    // the rows past the group's end, up to the next multiple of 16, of both operands: zero
                    const int deep = depth - (n - 1) * kBK;
                    const int quads = (16 - (deep & 15)) * 8;   // 16-byte pieces of a 64-wide column block
                    for (int p = 0; p < kParts; ++p) {
                        if (!landed(at + p)) give_up(3);
                        const unsigned buf = base + (at + p) % S::kStages * (S::kA + S::kB);
                        for (int i = lane; i < quads * (S::kA / 8192 + b_blocks); i += 32)
                            st_shared16(buf + i / quads * 8192 + deep * 128 + i % quads * 16, make_uint4(0, 0, 0, 0));
                    }
                    fence_async();
                    __syncwarp();
                    if (elect() && !multiply(at, deep, d, n - 1 == s0)) give_up(3);
                    __syncwarp();
                }
                ok = *abort == 0;
                if (!ok) break;
                if (peer == 0 && elect()) finish(acc_full + 8 * (used & 1u));
                __syncwarp();
            }
        }
        if (!ok) {   // every product issued is complete before TMEM is freed (bounded)
            volatile int never = 0;
            if (peer == 0) {
                if (elect()) finish(done);
                __syncwarp();
                bar_wait(done, 0, &never);
            }
        }
    } else {
        // ---- epilogue warps: TMEM lanes 32 (warp % 4) .. + 31 are rows of the
        // tile; of the two warps of a lane quarter one takes the even and one
        // the odd blocks of 32 columns
        const int row0 = (warp & 3) * 32, row = row0 + lane, parity = (warp - 2) / 4;
        const unsigned stage = base + S::kStageOff + (warp - 2) * S::kStaging;
        const unsigned lanes = tmem + ((unsigned)row0 << 16);
        const int out_size = a.out_type == kOutF32 ? 4 : 2;
        // an output whose rows do not start on 16 bytes has no tensor map
        const bool mapped = (a.ldo * out_size & 15) == 0;
        // a 16-byte piece in a row of the staged 64-byte (fp32: 128-byte) wide block, swizzled as its map
        const unsigned swz2 = (unsigned)(lane >> 1 & 3), swz4 = (unsigned)(lane & 7);
        unsigned used = 0;
        Turns<MODE, BN, PAIR> turns(base, abort, false);
        for (; ok && turns.tile >= 0; turns.next() ? void() : give_up(5)) {
            if (!walk.at(turns.tile, &t)) {
                if (MODE == kRagged) continue;
                break;
            }
            const int n = (int)max((t.k1 - t.k0 + kBK - 1) / kBK, (int64_t)0);
            const bool on = row < t.rows, part = MODE == kRagged && t.part;
            const bool wide = part || out_size == 4;
            const int y = (int)t.out_row + row0, z = (int)t.out_z;
            // a group's last rows share the block with the next group's: no box for them
            const bool boxed = (part || mapped) && (MODE != kRows || row0 + 32 <= t.rows);
            const bool any = row0 < t.rows;   // the warp has rows of the tile
            // kPoly, kUpdate: what is added to 32 columns from c on
            struct Addend {
                uint4 hi[4], lo[4];
            };
            auto fetch = [&](int c, Addend &p) {
                const int64_t at = t.batch_a * a.in_batch + (t.row0 + row) * a.ldi + t.col0 + c;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    p.hi[i] = p.lo[i] = make_uint4(0, 0, 0, 0);
                    if (!on || t.col0 + c + 8 * i >= a.ldi) continue;
                    p.hi[i] = *reinterpret_cast<const uint4 *>(a.in + at + 8 * i);
                    if (EPI == kUpdate) p.lo[i] = *reinterpret_cast<const uint4 *>(a.in_lo + at + 8 * i);
                }
            };
            // 32 columns from c on: the epilogue's arithmetic and the store
            auto emit = [&](int c, float (&v)[32], const Addend &p) {
                if constexpr (EPI == kGram) {
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[i] *= a.alpha;
                } else if constexpr (EPI == kPoly || EPI == kUpdate) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        float h[8], l[8];
                        unpack16<__half>(p.hi[i], h);
                        unpack16<__half>(p.lo[i], l);
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            v[8 * i + e] = fmaf(a.alpha, v[8 * i + e], a.beta * (h[e] + l[e]));
                    }
                }
                const int x = (int)t.col0 + c;
                if (boxed) {
                    __syncwarp();
                    if (elect()) bulk_wait_read<0>();   // the staging's last store has read it
                    __syncwarp();
                    if (wide) {
#pragma unroll
                        for (unsigned i = 0; i < 8; ++i)
                            st_shared16(stage + lane * 128 + ((i ^ swz4) << 4),
                                        make_uint4(__float_as_uint(v[4 * i]), __float_as_uint(v[4 * i + 1]),
                                                   __float_as_uint(v[4 * i + 2]), __float_as_uint(v[4 * i + 3])));
                    } else {
#pragma unroll
                        for (unsigned i = 0; i < 4; ++i) {
                            const uint4 w = pack8(v + 8 * i, a.out_type == kOutBf16);
                            const unsigned at = stage + lane * 64 + ((i ^ swz2) << 4);
                            st_shared16(at, w);
                            if (EPI == kUpdate && a.low) {   // what the high part's rounding left
                                float h[8];
                                unpack16<__half>(w, h);
#pragma unroll
                                for (int e = 0; e < 8; ++e) h[e] = v[8 * i + e] - h[e];
                                st_shared16(at + 2048, pack8(h, false));
                            }
                        }
                        if ((EPI == kGram || EPI == kPoly) && t.mirror) {
                            // transposed: column c + i of the tile is a row of 32 elements
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                asm volatile("st.shared.u16 [%0], %1;\n" ::"r"(
                                                 stage + 2048 + i * 64 + (((lane >> 3) ^ (i >> 1 & 3)) << 4) +
                                                 (lane & 7) * 2),
                                             "h"(__half_as_ushort(__float2half_rn(v[i])))
                                             : "memory");
                        }
                    }
                    fence_async();
                    __syncwarp();
                    if (elect()) {
                        tma_store(part ? &map_p : &map_o, stage, x, y, z);
                        if (EPI == kUpdate && a.low) tma_store(&map_p, stage + 2048, x, y, z);
                        if ((EPI == kGram || EPI == kPoly) && t.mirror) tma_store(&map_o, stage + 2048, y, x, z);
                        bulk_commit();
                    }
                } else if (MODE == kRows) {   // each lane its row
                    if (on) {
                        char *o = static_cast<char *>(a.out) + ((t.out_row + row) * a.ldo + x) * out_size;
#pragma unroll
                        for (int i = 0; i < 4; ++i) {
                            if (c + 8 * i >= t.cols) break;
                            if (out_size == 4) {
                                float4 *q = reinterpret_cast<float4 *>(o) + 2 * i;
                                q[0] = make_float4(v[8 * i], v[8 * i + 1], v[8 * i + 2], v[8 * i + 3]);
                                q[1] = make_float4(v[8 * i + 4], v[8 * i + 5], v[8 * i + 6], v[8 * i + 7]);
                            } else {
                                reinterpret_cast<uint4 *>(o)[i] = pack8(v + 8 * i, a.out_type == kOutBf16);
                            }
                        }
                    }
                } else {   // kUpdate's result with rows of any alignment: 16-bit, row by row across the lanes
                    __syncwarp();
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint4 w = pack8(v + 8 * i, a.out_type == kOutBf16);
                        const unsigned at = stage + lane * 68 + i * 16;   // an odd number of words apart
                        asm volatile("st.shared.u32 [%0], %1;\n\tst.shared.u32 [%0+4], %2;\n\t"
                                     "st.shared.u32 [%0+8], %3;\n\tst.shared.u32 [%0+12], %4;\n" ::"r"(at),
                                     "r"(w.x), "r"(w.y), "r"(w.z), "r"(w.w)
                                     : "memory");
                    }
                    __syncwarp();
                    const unsigned char *src = smem + S::kStageOff + (warp - 2) * S::kStaging;
                    unsigned short *o = static_cast<unsigned short *>(a.out) + t.out_z * a.out_batch +
                                        (t.out_row + row0) * a.ldo + x;
                    if (c + lane < t.cols)
                        for (int r = 0; r < 32 && row0 + r < t.rows; ++r)
                            o[r * a.ldo + lane] = *reinterpret_cast<const unsigned short *>(src + r * 68 + lane * 2);
                }
            };
            auto take = [&]() {   // the next accumulator
                const unsigned acc = used & 1u;
                if (!bar_wait<PAIR>(acc_full + 8 * acc, used >> 1 & 1u, abort)) { give_up(4); return 0u; }
                fence_after();
                return lanes + acc * BN;
            };
            auto give_back = [&]() {
                fence_before();
                __syncwarp();
                if (lane == 0) {
                    if (PAIR) bar_arrive_cluster(in_block(acc_empty + 8 * (used & 1u), 0));
                    else bar_arrive(acc_empty + 8 * (used & 1u));
                }
                ++used;
            };
            if constexpr (kSlices > 0) {
                float v[BN / 64][32];
#pragma unroll
                for (int b = 0; b < BN / 64; ++b)
#pragma unroll
                    for (int i = 0; i < 32; ++i) v[b][i] = 0.f;
                for (int i = 0; i < n; i += kSlices) {
                    const unsigned from = take();
                    if (!ok) break;
#pragma unroll
                    for (int b = 0; b < BN / 64; ++b) {
                        const int c = parity * 32 + 64 * b;
                        if (any && c < t.cols) {
                            float w[32];
                            tmem_ld32(from + c, w);
#pragma unroll
                            for (int e = 0; e < 32; ++e) v[b][e] += w[e];
                        }
                    }
                    give_back();
                }
                if (!ok) break;
#pragma unroll
                for (int b = 0; b < BN / 64; ++b) {
                    const int c = parity * 32 + 64 * b;
                    if (any && c < t.cols) emit(c, v[b], Addend{});
                }
            } else {
                constexpr bool kAdds = EPI == kPoly || EPI == kUpdate;
                // the first columns' addend is read while the products run, the next ones' a block ahead
                Addend now, next;
                if (kAdds && any) fetch(parity * 32, now);
                unsigned from = 0;
                if (n > 0) from = take();
                if (!ok) break;
                for (int c = parity * 32; c < t.cols && any; c += 64) {
                    if (kAdds && c + 64 < t.cols) fetch(c + 64, next);
                    float v[32];
                    if (n > 0) {
                        tmem_ld32(from + c, v);
                    } else {
#pragma unroll
                        for (int i = 0; i < 32; ++i) v[i] = 0.f;
                    }
                    emit(c, v, now);
                    now = next;
                }
                if (n > 0) give_back();
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

// Tensor map of a 16-bit operand [batch][rows][inner] (strides in elements),
// read in boxes of 64 elements x box_rows, 128-byte swizzled, zero outside.
bool make_map(CUtensorMap *map, const void *p, int64_t inner, int64_t rows, int64_t batch, int64_t ld,
              int64_t batch_stride, int box_rows, bool bf16);
// As make_map for an MN-major operand read in boxes of `blocks` x 64 rows x 64
// elements: [batch][inner / 64][rows][64].  Only for an inner extent of whole
// blocks; others have a box per block.
bool make_blocked_map(CUtensorMap *map, const void *p, int64_t inner, int64_t rows, int64_t batch, int64_t ld,
                      int64_t batch_stride, int blocks, bool bf16);
// An MN-major operand whose tiles are `tile` wide: the blocked map where it
// can be, else the plain one; *blocked says which.
inline bool make_mn_map(CUtensorMap *map, bool *blocked, const void *p, int64_t inner, int64_t rows, int64_t batch,
                        int64_t ld, int64_t batch_stride, int tile, bool bf16)
{
    *blocked = inner % 64 == 0 && (tile % 64 == 0 || tile >= inner);
    return *blocked ? make_blocked_map(map, p, inner, rows, batch, ld, batch_stride, (tile + 63) / 64, bf16)
                    : make_map(map, p, inner, rows, batch, ld, batch_stride, 64, bf16);
}
// Tensor map of an output, written in boxes of 32 x 32 elements.
bool make_out_map(CUtensorMap *map, void *p, int64_t inner, int64_t rows, int64_t batch, int64_t ld,
                  int64_t batch_stride, int out_type);

// Launch that lets the kernel's set-up overlap the kernel before it.
template <typename K, typename... A>
cudaError_t launch_overlapped(K kernel, dim3 grid, unsigned cluster, int threads, int smem, cudaStream_t stream,
                              const A &...args)
{
    cudaLaunchConfig_t config{};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attr[2] = {};
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = cluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    config.attrs = attr;
    config.numAttrs = cluster > 1 ? 2 : 1;
    return cudaLaunchKernelEx(&config, kernel, args...);
}

struct Maps {
    CUtensorMap a, b, o, p;
};

template <int MODE, int BN, bool AMN, bool BMN, int EPI, bool PAIR = false>
cudaError_t launch_gemm(const Maps &m, const GemmArgs &a, int64_t tiles, cudaStream_t s)
{
    using S = GemmShape<BN, PAIR>;
    auto kernel = gemm_kernel<MODE, BN, AMN, BMN, EPI, PAIR>;
    static PerDevice<bool> ready;   // the attribute outlasts the call
    bool *done = ready.here();
    if (!done || !*done) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, S::kBytes);
        if (e != cudaSuccess) return e;
        if (done) *done = true;
    }
    constexpr int kBlocks = PAIR ? 2 : 1;   // per tile
    const int64_t most = MODE == kRagged ? INT32_MAX / 2 : device_sm_count() / kBlocks;
    const unsigned grid = kBlocks * (unsigned)std::max<int64_t>(1, std::min(tiles, most));
    return launch_overlapped(kernel, grid, kBlocks, kGemmThreads, S::kBytes, s, m.a, m.b, m.o, m.p, a);
}

}  // namespace tc
}  // namespace spmmb
