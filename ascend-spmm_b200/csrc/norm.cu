// Layer normalisation of node rows, forward and backward.
//
//   forward   y = (x - mean) * rstd * w + b,  rstd = 1 / sqrt(var + eps),
//             var = E[(x - mean)^2] over the row
//   backward  with xhat = (x - mean) * rstd and g = dy * w:
//             dx = rstd * (g - E[g] - xhat * E[g * xhat])
//             dw = sum over rows of dy * xhat,  db = sum over rows of dy
//
// Both are bound by memory: forward reads x and writes y, backward reads x
// and dy and writes dx.  A team of lanes owns a row and keeps it in
// registers, so the mean and then the centred squares are summed from
// registers in fp32 (no E[x^2] - E[x]^2, whose cancellation would lose rows
// with a large mean) and each element crosses memory once.  A team is 8
// lanes for rows of up to sixteen 16-byte vectors, a warp up to 128 vectors,
// a block above.
#include <algorithm>

#include "../../include/spmm_b200.h"
#include "common.cuh"
#include "engine.h"
#include "layer.cuh"
#include "layer.h"

namespace spmmb {

namespace {

constexpr unsigned kFull = 0xffffffffu;

// VE consecutive elements as one load or store.
template <int BYTES> struct Raw;
template <> struct Raw<16> { using Type = uint4; };
template <> struct Raw<4> { using Type = unsigned; };
template <> struct Raw<2> { using Type = unsigned short; };

template <typename T, int VE> union Pack {
    typename Raw<sizeof(T) * VE>::Type raw;
    T e[VE];
    __device__ Pack() {}
};

template <typename T, int VE> __device__ __forceinline__ void unpack(const Pack<T, VE> &p, float *f)
{
#pragma unroll
    for (int i = 0; i < VE; ++i) f[i] = elem_f32<T>(p.e[i]);
}

// VE parameters (weight or bias) starting at column c: of the rows' type or fp32.
template <typename T, int VE>
__device__ __forceinline__ void load_params(const void *p, bool f32, int64_t c, float *f)
{
    if (f32) {
        const float *q = static_cast<const float *>(p) + c;
        if constexpr (VE % 4 == 0) {
#pragma unroll
            for (int i = 0; i < VE / 4; ++i) {
                const float4 v = __ldg(reinterpret_cast<const float4 *>(q) + i);
                f[4 * i] = v.x; f[4 * i + 1] = v.y; f[4 * i + 2] = v.z; f[4 * i + 3] = v.w;
            }
        } else {
#pragma unroll
            for (int i = 0; i < VE; ++i) f[i] = __ldg(q + i);
        }
    } else {
        Pack<T, VE> v;
        v.raw = __ldg(reinterpret_cast<const decltype(v.raw) *>(static_cast<const T *>(p) + c));
        unpack<T, VE>(v, f);
    }
}

// Sum over the lanes of a team of at most a warp, or over a block through
// `red` (one float per warp; the caller alternates two buffers so that one
// barrier per sum is enough).
template <int TEAM> __device__ __forceinline__ float team_sum(float v, float *red)
{
#pragma unroll
    for (int o = (TEAM < 32 ? TEAM : 32) / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    if constexpr (TEAM > 32) {
        if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
        __syncthreads();
        v = 0.f;
#pragma unroll
        for (int w = 0; w < TEAM / 32; ++w) v += red[w];
    }
    return v;
}

struct NormArgs {
    const void *x, *w, *b, *dy;
    void *y;                 // y or dx
    float *mean, *rstd;      // written by forward (may be null), read by backward
    float *part;             // backward: [blocks][2][width] partial dw, db (null: not wanted)
    int64_t rows, width;
    float eps;
    bool pf32;               // weight and bias are fp32
};

// Threads per block for a team size.
template <int TEAM> constexpr int kBlock = TEAM > 32 ? TEAM : 128;

template <typename T, int VE, int NV, int TEAM>
__global__ void __launch_bounds__(kBlock<TEAM>) norm_forward_kernel(const NormArgs a)
{
    __shared__ float red[2][32];
    constexpr int kTeams = kBlock<TEAM> / TEAM;
    const int t = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    const float inv = 1.f / (float)a.width;
    const T *x = static_cast<const T *>(a.x);
    T *y = static_cast<T *>(a.y);
    // every lane of a warp (every thread of a block team) takes the same number of turns
    for (int64_t r0 = (int64_t)blockIdx.x * kTeams; r0 < a.rows; r0 += (int64_t)gridDim.x * kTeams) {
        const int64_t r = r0 + team;
        const bool on = r < a.rows;
        const T *xr = x + r * a.width;
        Pack<T, VE> v[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t c = (int64_t)(t + i * TEAM) * VE;
            if (on && c < a.width) v[i].raw = __ldcs(reinterpret_cast<const decltype(v[i].raw) *>(xr + c));
        }
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (on && (int64_t)(t + i * TEAM) * VE < a.width) {
                float f[VE];
                unpack<T, VE>(v[i], f);
#pragma unroll
                for (int e = 0; e < VE; ++e) s += f[e];
            }
        const float mean = team_sum<TEAM>(s, red[0]) * inv;
        s = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (on && (int64_t)(t + i * TEAM) * VE < a.width) {
                float f[VE];
                unpack<T, VE>(v[i], f);
#pragma unroll
                for (int e = 0; e < VE; ++e) s = fmaf(f[e] - mean, f[e] - mean, s);
            }
        const float rstd = 1.f / sqrtf(team_sum<TEAM>(s, red[1]) * inv + a.eps);
        if (!on) continue;
        if (a.mean && t == 0) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t c = (int64_t)(t + i * TEAM) * VE;
            if (c >= a.width) continue;
            float f[VE], p[VE];
            unpack<T, VE>(v[i], f);
#pragma unroll
            for (int e = 0; e < VE; ++e) f[e] = (f[e] - mean) * rstd;
            if (a.w) {
                load_params<T, VE>(a.w, a.pf32, c, p);
#pragma unroll
                for (int e = 0; e < VE; ++e) f[e] *= p[e];
            }
            if (a.b) {
                load_params<T, VE>(a.b, a.pf32, c, p);
#pragma unroll
                for (int e = 0; e < VE; ++e) f[e] += p[e];
            }
            Pack<T, VE> o;
#pragma unroll
            for (int e = 0; e < VE; ++e) o.e[e] = elem_of<T>(f[e]);
            __stcs(reinterpret_cast<decltype(o.raw) *>(y + r * a.width + c), o.raw);
        }
    }
}

// Rows wider than a block's registers: one block per row, three passes.
template <typename T>
__global__ void __launch_bounds__(512) norm_forward_wide_kernel(const NormArgs a)
{
    __shared__ float red[2][32];
    const float inv = 1.f / (float)a.width;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + r * a.width;
        T *y = static_cast<T *>(a.y) + r * a.width;
        float s = 0.f;
        for (int64_t c = threadIdx.x; c < a.width; c += 512) s += elem_f32<T>(x[c]);
        const float mean = team_sum<512>(s, red[0]) * inv;
        s = 0.f;
        for (int64_t c = threadIdx.x; c < a.width; c += 512) {
            const float d = elem_f32<T>(x[c]) - mean;
            s = fmaf(d, d, s);
        }
        const float rstd = 1.f / sqrtf(team_sum<512>(s, red[1]) * inv + a.eps);
        if (a.mean && threadIdx.x == 0) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
        for (int64_t c = threadIdx.x; c < a.width; c += 512) {
            float f = (elem_f32<T>(x[c]) - mean) * rstd, p;
            if (a.w) { load_params<T, 1>(a.w, a.pf32, c, &p); f *= p; }
            if (a.b) { load_params<T, 1>(a.b, a.pf32, c, &p); f += p; }
            y[c] = elem_of<T>(f);
        }
    }
}

// Backward: the lane that holds a column holds it for every row of its team,
// so dw and db accumulate in its registers; the teams of a block are added
// through shared memory and the block writes one partial row.
template <typename T, int VE, int NV, int TEAM>
__global__ void __launch_bounds__(kBlock<TEAM>) norm_backward_kernel(const NormArgs a)
{
    __shared__ float red[2][2][32];
    constexpr int kTeams = kBlock<TEAM> / TEAM;
    const int t = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    const float inv = 1.f / (float)a.width;
    const T *x = static_cast<const T *>(a.x), *dy = static_cast<const T *>(a.dy);
    T *dx = static_cast<T *>(a.y);
    float dw[NV][VE], db[NV][VE];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VE; ++e) dw[i][e] = db[i][e] = 0.f;
    int turn = 0;
    for (int64_t r0 = (int64_t)blockIdx.x * kTeams; r0 < a.rows; r0 += (int64_t)gridDim.x * kTeams, turn ^= 1) {
        const int64_t r = r0 + team;
        const bool on = r < a.rows;
        Pack<T, VE> vx[NV], vg[NV];
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t c = (int64_t)(t + i * TEAM) * VE;
            if (on && c < a.width) {
                vx[i].raw = __ldcs(reinterpret_cast<const decltype(vx[i].raw) *>(x + r * a.width + c));
                vg[i].raw = __ldcs(reinterpret_cast<const decltype(vg[i].raw) *>(dy + r * a.width + c));
            }
        }
        const float mean = on ? a.mean[r] : 0.f, rstd = on ? a.rstd[r] : 0.f;
        float s1 = 0.f, s2 = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t c = (int64_t)(t + i * TEAM) * VE;
            if (on && c < a.width) {
                float f[VE], g[VE], p[VE];
                unpack<T, VE>(vx[i], f);
                unpack<T, VE>(vg[i], g);
                if (a.w) load_params<T, VE>(a.w, a.pf32, c, p);
#pragma unroll
                for (int e = 0; e < VE; ++e) {
                    const float xh = (f[e] - mean) * rstd;
                    dw[i][e] = fmaf(g[e], xh, dw[i][e]);
                    db[i][e] += g[e];
                    const float gw = a.w ? g[e] * p[e] : g[e];
                    s1 += gw;
                    s2 = fmaf(gw, xh, s2);
                }
            }
        }
        if (!a.y) continue;   // the same for every thread: only dw and db wanted
        const float c1 = team_sum<TEAM>(s1, red[turn][0]) * inv, c2 = team_sum<TEAM>(s2, red[turn][1]) * inv;
        if (!on) continue;
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int64_t c = (int64_t)(t + i * TEAM) * VE;
            if (c >= a.width) continue;
            float f[VE], g[VE], p[VE];
            unpack<T, VE>(vx[i], f);
            unpack<T, VE>(vg[i], g);
            if (a.w) load_params<T, VE>(a.w, a.pf32, c, p);
            Pack<T, VE> o;
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const float xh = (f[e] - mean) * rstd, gw = a.w ? g[e] * p[e] : g[e];
                o.e[e] = elem_of<T>(rstd * (gw - c1 - xh * c2));
            }
            __stcs(reinterpret_cast<decltype(o.raw) *>(dx + r * a.width + c), o.raw);
        }
    }
    if (!a.part) return;
    float *pw = a.part + (int64_t)blockIdx.x * 2 * a.width, *pb = pw + a.width;
    if constexpr (kTeams == 1) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VE; ++e) {
                const int64_t c = (int64_t)(t + i * TEAM) * VE + e;
                if (c < a.width) { pw[c] = dw[i][e]; pb[c] = db[i][e]; }
            }
    } else {
        __shared__ float sums[kTeams][TEAM * VE + 1];
        for (int which = 0; which < 2; ++which)
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                __syncthreads();
#pragma unroll
                for (int e = 0; e < VE; ++e) sums[team][t * VE + e] = which ? db[i][e] : dw[i][e];
                __syncthreads();
                for (int j = threadIdx.x; j < TEAM * VE; j += kBlock<TEAM>) {
                    float v = 0.f;
#pragma unroll
                    for (int k = 0; k < kTeams; ++k) v += sums[k][j];
                    const int64_t c = (int64_t)i * TEAM * VE + j;
                    if (c < a.width) (which ? pb : pw)[c] = v;
                }
            }
    }
}

template <typename T>
__global__ void __launch_bounds__(512) norm_backward_wide_kernel(const NormArgs a)
{
    __shared__ float red[2][2][32];
    const float inv = 1.f / (float)a.width;
    float *pw = a.part ? a.part + (int64_t)blockIdx.x * 2 * a.width : nullptr;
    if (pw)
        for (int64_t c = threadIdx.x; c < 2 * a.width; c += 512) pw[c] = 0.f;
    __syncthreads();
    int turn = 0;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x, turn ^= 1) {
        const T *x = static_cast<const T *>(a.x) + r * a.width, *dy = static_cast<const T *>(a.dy) + r * a.width;
        const float mean = a.mean[r], rstd = a.rstd[r];
        float s1 = 0.f, s2 = 0.f;
        for (int64_t c = threadIdx.x; c < a.width; c += 512) {
            const float g = elem_f32<T>(dy[c]), xh = (elem_f32<T>(x[c]) - mean) * rstd;
            float p = 1.f;
            if (a.w) load_params<T, 1>(a.w, a.pf32, c, &p);
            s1 += g * p;
            s2 = fmaf(g * p, xh, s2);
            if (pw) {   // this thread's own columns
                pw[c] = fmaf(g, xh, pw[c]);
                pw[a.width + c] += g;
            }
        }
        if (!a.y) continue;
        const float c1 = team_sum<512>(s1, red[turn][0]) * inv, c2 = team_sum<512>(s2, red[turn][1]) * inv;
        T *dx = static_cast<T *>(a.y) + r * a.width;
        for (int64_t c = threadIdx.x; c < a.width; c += 512) {
            const float xh = (elem_f32<T>(x[c]) - mean) * rstd;
            float p = 1.f;
            if (a.w) load_params<T, 1>(a.w, a.pf32, c, &p);
            dx[c] = elem_of<T>(rstd * (elem_f32<T>(dy[c]) * p - c1 - xh * c2));
        }
    }
}

// Adds the blocks' partial rows: 32 columns per block, 8 partial rows at a
// time, in an order that depends on the number of partials alone.
template <typename P>
__global__ void __launch_bounds__(256) norm_params_kernel(const float *part, int blocks, int64_t width, P *dw, P *db)
{
    __shared__ float sums[8][33];
    const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;   // over dw's columns, then db's
    float s = 0.f;
    if (c < 2 * width)
        for (int k = row; k < blocks; k += 8) s += part[(int64_t)k * 2 * width + c];
    sums[row][lane] = s;
    __syncthreads();
    if (row == 0 && c < 2 * width) {
#pragma unroll
        for (int k = 1; k < 8; ++k) s += sums[k][lane];
        P *out = c < width ? dw : db;
        if (out) out[c < width ? c : c - width] = elem_of<P>(s);
    }
}

// Blocks of `kernel` that fill the GPU once (a persistent grid), no more than the rows need.
template <auto kernel> int64_t grid_of(int threads, int64_t turns)
{
    static PerDevice<int> resident;
    int *have = resident.here(), per_sm = have ? *have : 0;
    if (per_sm < 1) {
        if (cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kernel, threads, 0) != cudaSuccess || per_sm < 1)
            per_sm = 1;
        if (have) *have = per_sm;
    }
    return std::max<int64_t>(1, std::min<int64_t>((int64_t)per_sm * device_sm_count(), turns));
}

template <typename T, int VE, int NV, int TEAM> cudaError_t run_team(const NormArgs &a, bool backward, int64_t max_blocks,
                                                                     int64_t *blocks, cudaStream_t stream)
{
    constexpr int threads = kBlock<TEAM>, teams = threads / TEAM;
    const int64_t turns = (a.rows + teams - 1) / teams;
    if (backward) {
        *blocks = std::min(max_blocks, grid_of<norm_backward_kernel<T, VE, NV, TEAM>>(threads, turns));
        norm_backward_kernel<T, VE, NV, TEAM><<<(unsigned)*blocks, threads, 0, stream>>>(a);
    } else {
        *blocks = grid_of<norm_forward_kernel<T, VE, NV, TEAM>>(threads, turns);
        norm_forward_kernel<T, VE, NV, TEAM><<<(unsigned)*blocks, threads, 0, stream>>>(a);
    }
    return cudaGetLastError();
}

template <typename T> cudaError_t run_norm(const NormArgs &a, bool backward, int64_t max_blocks, int64_t *blocks,
                                           cudaStream_t s)
{
    constexpr int V = 16 / sizeof(T);
    if (a.width % V == 0) {   // rows of whole 16-byte vectors
        const int64_t v = a.width / V;
        if (v <= 8) return run_team<T, V, 1, 8>(a, backward, max_blocks, blocks, s);
        if (v <= 16) return run_team<T, V, 2, 8>(a, backward, max_blocks, blocks, s);
        if (v <= 32) return run_team<T, V, 1, 32>(a, backward, max_blocks, blocks, s);
        if (v <= 64) return run_team<T, V, 2, 32>(a, backward, max_blocks, blocks, s);
        if (v <= 128) return run_team<T, V, 4, 32>(a, backward, max_blocks, blocks, s);
        if (v <= 256) return run_team<T, V, 2, 128>(a, backward, max_blocks, blocks, s);
        if (v <= 512) return run_team<T, V, 2, 256>(a, backward, max_blocks, blocks, s);
        if (v <= 1024) return run_team<T, V, 2, 512>(a, backward, max_blocks, blocks, s);
        if (v <= 2048) return run_team<T, V, 2, 1024>(a, backward, max_blocks, blocks, s);
    } else {                  // rows that start at any element
        if (a.width <= 32) return run_team<T, 1, 4, 8>(a, backward, max_blocks, blocks, s);
        if (a.width <= 128) return run_team<T, 1, 4, 32>(a, backward, max_blocks, blocks, s);
        if (a.width <= 1024) return run_team<T, 1, 8, 128>(a, backward, max_blocks, blocks, s);
        if (a.width <= 4096) return run_team<T, 1, 8, 512>(a, backward, max_blocks, blocks, s);
        if (a.width <= 8192) return run_team<T, 1, 8, 1024>(a, backward, max_blocks, blocks, s);
    }
    *blocks = std::min<int64_t>(a.rows, 2 * device_sm_count());
    if (backward) {
        *blocks = std::min(*blocks, max_blocks);
        norm_backward_wide_kernel<T><<<(unsigned)*blocks, 512, 0, s>>>(a);
    } else {
        norm_forward_wide_kernel<T><<<(unsigned)*blocks, 512, 0, s>>>(a);
    }
    return cudaGetLastError();
}

cudaError_t dispatch(const NormArgs &a, int dtype, bool backward, int64_t max_blocks, int64_t *blocks, cudaStream_t s)
{
    switch (dtype) {
        case SPMM_F16: return run_norm<__half>(a, backward, max_blocks, blocks, s);
        case SPMM_BF16: return run_norm<__nv_bfloat16>(a, backward, max_blocks, blocks, s);
        default: return run_norm<float>(a, backward, max_blocks, blocks, s);
    }
}

}  // namespace

int64_t norm_backward_blocks(int64_t rows)
{
    // at most 16 resident blocks per SM; few rows need no more blocks than rows
    return std::max<int64_t>(1, std::min<int64_t>(rows, 16 * (int64_t)device_sm_count()));
}

cudaError_t launch_norm_forward(const NormLaunch &n, cudaStream_t stream)
{
    NormArgs a{};
    a.x = n.x; a.w = n.weight; a.b = n.bias; a.y = n.out; a.mean = n.mean; a.rstd = n.rstd;
    a.rows = n.rows; a.width = n.width; a.eps = n.eps; a.pf32 = n.param_dtype == SPMM_F32;
    int64_t blocks = 0;
    return dispatch(a, n.dtype, false, 0, &blocks, stream);
}

cudaError_t launch_norm_backward(const NormLaunch &n, const void *grad, void *dweight, void *dbias, float *workspace,
                                 cudaStream_t stream)
{
    NormArgs a{};
    a.x = n.x; a.w = n.weight; a.dy = grad; a.y = n.out; a.mean = n.mean; a.rstd = n.rstd;
    a.rows = n.rows; a.width = n.width; a.pf32 = n.param_dtype == SPMM_F32;
    a.part = dweight || dbias ? workspace : nullptr;
    int64_t blocks = 0;
    cudaError_t e = dispatch(a, n.dtype, true, norm_backward_blocks(n.rows), &blocks, stream);
    if (e != cudaSuccess || !a.part) return e;
    const unsigned grid = (unsigned)((2 * n.width + 31) / 32);
    switch (n.param_dtype) {
        case SPMM_F16:
            norm_params_kernel<__half><<<grid, 256, 0, stream>>>(a.part, (int)blocks, n.width,
                                                                 static_cast<__half *>(dweight),
                                                                 static_cast<__half *>(dbias));
            break;
        case SPMM_BF16:
            norm_params_kernel<__nv_bfloat16><<<grid, 256, 0, stream>>>(a.part, (int)blocks, n.width,
                                                                        static_cast<__nv_bfloat16 *>(dweight),
                                                                        static_cast<__nv_bfloat16 *>(dbias));
            break;
        default:
            norm_params_kernel<float><<<grid, 256, 0, stream>>>(a.part, (int)blocks, n.width,
                                                                static_cast<float *>(dweight),
                                                                static_cast<float *>(dbias));
    }
    return cudaGetLastError();
}

}  // namespace spmmb
