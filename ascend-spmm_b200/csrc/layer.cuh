// Device helpers shared by the layer operators (norm.cu, grouped.cu, ortho.cu).
#pragma once

#include <cuda_bf16.h>

#include "../../include/spmm_b200.h"
#include "common.cuh"

namespace spmmb {

template <typename T> __device__ __forceinline__ float elem_f32(T x);
template <> __device__ __forceinline__ float elem_f32<__half>(__half x) { return __half2float(x); }
template <> __device__ __forceinline__ float elem_f32<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <> __device__ __forceinline__ float elem_f32<float>(float x) { return x; }

template <typename T> __device__ __forceinline__ T elem_of(float x);
template <> __device__ __forceinline__ __half elem_of<__half>(float x) { return __float2half_rn(x); }
template <> __device__ __forceinline__ __nv_bfloat16 elem_of<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <> __device__ __forceinline__ float elem_of<float>(float x) { return x; }

// The rows of a grouped product as segments: segment 0 is the rows before
// the first group, segment g + 1 is group g, segment groups + 1 the rows
// after the last group (0 and groups + 1 get zeros).  A malformed group is
// empty.
struct Ranges {
    const void *ptr;        // [groups + 1], int32 or int64
    bool wide;              // int64
    int64_t groups, rows;
    __device__ __forceinline__ int64_t operator[](int64_t i) const
    {
        return wide ? ld_idx(static_cast<const int64_t *>(ptr) + i) : ld_idx(static_cast<const int *>(ptr) + i);
    }
};

__device__ __forceinline__ void segment_rows(const Ranges &p, int64_t s, int64_t *begin, int64_t *end, DevStatus *status)
{
    int64_t b = 0, e = 0;
    if (s == 0) {
        e = min(max(p[0], (int64_t)0), p.rows);
    } else if (s <= p.groups) {
        b = p[s - 1];
        e = p[s];
        if (b < 0 || e < b || e > p.rows) {
            raise_status(status, SPMM_DEV_BAD_ROWPTR, s - 1);
            b = e = 0;
        }
    } else if (s == p.groups + 1) {
        b = min(max(p[p.groups], (int64_t)0), p.rows);
        e = p.rows;
    }
    *begin = b;
    *end = e;
}

// Walks the tiles of all segments in order, `mult` column tiles per `height`
// rows.  SPLIT (weight gradients): a group's tiles cover its rows in parts of
// `height`, a group without rows has one, the rows outside the groups none.
// Every lane of the warp calls it with the same arguments; it goes on from the
// last tile's place.
template <bool SPLIT> struct TileWalk {
    int64_t base = 0;      // segments before the current 32
    int64_t before = 0;    // tiles of the segments before `base`
    int64_t kept = 0;      // SPLIT: parts of the groups of several parts before `base`
    int64_t count = -1;    // this lane's segment: its tiles, rows, and what is before it
    int64_t begin = 0, end = 0, first = 0, parts = 0, slot = 0;

    // The segment of `tile` (0 .. groups + 1), its rows and the tile's number
    // within it; false past the last tile.  `slots`: parts of the groups of
    // several parts before this group, -1 where it has a single part.
    __device__ __forceinline__ bool find(const Ranges &p, int64_t height, int64_t mult, int64_t tile, DevStatus *status,
                                         int64_t *seg, int64_t *b, int64_t *e, int64_t *inner, int64_t *slots)
    {
        const int lane = threadIdx.x & 31;
        if (tile < before) {
            base = before = kept = 0;
            count = -1;
        }
        for (;;) {
            if (count < 0) {
                segment_rows(p, base + lane, &begin, &end, status);
                int64_t n = (end - begin + height - 1) / height;
                if (SPLIT) n = base + lane >= 1 && base + lane <= p.groups ? max(n, (int64_t)1) : 0;
                count = n * mult;
                parts = SPLIT && n > 1 ? n : 0;
                first = before_lane(count);
                if (SPLIT) slot = before_lane(parts);
            }
            const unsigned hit = __ballot_sync(0xffffffffu, tile - before >= first && tile - before < first + count);
            if (hit) {
                const int l = __ffs(hit) - 1;
                *seg = base + l;
                *b = __shfl_sync(0xffffffffu, begin, l);
                *e = __shfl_sync(0xffffffffu, end, l);
                *inner = tile - before - __shfl_sync(0xffffffffu, first, l);
                if (SPLIT) *slots = __shfl_sync(0xffffffffu, parts ? kept + slot : -1, l);
                return true;
            }
            before += __shfl_sync(0xffffffffu, first + count, 31);
            if (SPLIT) kept += __shfl_sync(0xffffffffu, slot + parts, 31);
            base += 32;
            count = -1;
            if (base >= p.groups + 2) return false;
        }
    }

private:
    __device__ __forceinline__ int64_t before_lane(int64_t v)
    {
        const int lane = threadIdx.x & 31;
        int64_t sum = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int64_t u = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += u;
        }
        return sum - v;
    }
};

}  // namespace spmmb
