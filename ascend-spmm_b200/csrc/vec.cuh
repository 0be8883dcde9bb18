// Rows in 16-byte vectors whatever their alignment.
#pragma once

#include <cuda_bf16.h>

#include "common.cuh"
#include "layer.cuh"

namespace spmmb {

// Elements of T in 16 bytes.
template <typename T> struct Pack16 {
    static constexpr int kElems = 16 / (int)sizeof(T);
    uint4 raw;
    __device__ __forceinline__ void get(float *f) const
    {
        const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
        for (int i = 0; i < kElems; ++i) f[i] = elem_f32<T>(e[i]);
    }
    __device__ __forceinline__ void set(const float *f)
    {
        T *e = reinterpret_cast<T *>(&raw);
#pragma unroll
        for (int i = 0; i < kElems; ++i) e[i] = elem_of<T>(f[i]);
    }
};

// The 16 bytes at p, which is aligned to its elements: the one or two aligned
// vectors that hold them, shifted together.  Each holds one of these bytes at
// least: of an array that starts on 16 bytes, what is read besides it lies
// behind its end and before the next multiple of 16, up to 14 bytes, which are
// not used (and belong to the array's last vector: no other page, no fault).
// Called with one alignment by a whole warp, so that the branches are uniform.
template <bool ALIGNED, typename T> __device__ __forceinline__ Pack16<T> load16(const T *p)
{
    Pack16<T> v;
    if constexpr (ALIGNED) {
        v.raw = __ldg(reinterpret_cast<const uint4 *>(p));
    } else {
        const unsigned shift = (unsigned)reinterpret_cast<uintptr_t>(p) & 15u;
        const uint4 *at = reinterpret_cast<const uint4 *>(reinterpret_cast<uintptr_t>(p) - shift);
        v.raw = __ldg(at);
        if (shift) {
            const uint4 hi = __ldg(at + 1);
            unsigned q[8] = {v.raw.x, v.raw.y, v.raw.z, v.raw.w, hi.x, hi.y, hi.z, hi.w};
            if (shift & 8u) {
#pragma unroll
                for (int i = 0; i < 6; ++i) q[i] = q[i + 2];
            }
            if (shift & 4u) {
#pragma unroll
                for (int i = 0; i < 5; ++i) q[i] = q[i + 1];
            }
            const unsigned bits = (shift & 3u) * 8;
            v.raw.x = __funnelshift_r(q[0], q[1], bits);
            v.raw.y = __funnelshift_r(q[1], q[2], bits);
            v.raw.z = __funnelshift_r(q[2], q[3], bits);
            v.raw.w = __funnelshift_r(q[3], q[4], bits);
        }
    }
    return v;
}

// A row of `width` elements at p for whole-vector stores: elements before its
// first 16-byte boundary, whole vectors from there on, elements behind them.
template <bool ALIGNED, typename T> struct RowSpan {
    int head;
    int64_t vectors, tail;   // tail: where the last elements begin
    __device__ __forceinline__ RowSpan(const T *p, int64_t width)
    {
        constexpr int kElems = Pack16<T>::kElems;
        head = ALIGNED ? 0 : (int)((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / (int)sizeof(T);
        if (head > width) head = (int)width;
        vectors = (width - head) / kElems;
        tail = head + vectors * kElems;
    }
    // Element `i` of those outside the whole vectors (0 .. loose() - 1).
    __device__ __forceinline__ int64_t loose(int64_t width) const { return ALIGNED ? 0 : head + width - tail; }
    __device__ __forceinline__ int64_t loose_at(int64_t i) const { return i < head ? i : tail + i - head; }
};

}  // namespace spmmb
