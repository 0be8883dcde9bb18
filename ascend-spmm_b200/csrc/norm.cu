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
// with a large mean) and each element crosses memory once.  The next row is
// loaded while a row is worked on.
//
// Measured (GB/s of the bytes above; a plain copy reaches 6538): fp16, 524287
// rows of 1024, forward 332 us 6470, backward 556 us 5790; fp32, 100003 rows
// of 256, 35 us 5870 and 50 us 6130; bf16, 164110 rows of 1001 (no row starts
// on a vector), 131 us 5030 and 200 us 4920; 9 rows of 256 2.7 us, the launch.
// The widest rows are slower, 1 GB of x each, forward and backward GB/s: fp16
// 8192 2540 and 5510 (the forward form of 512 lanes spills registers), 16384
// 3060 and 2680; fp32 8192 5950 and 4610; and rows that no block holds, a
// thread per element in three passes, fp32 16384 1770 and 1020, fp16 33000
// 1060 and 440.
#include <algorithm>

#include "../../include/spmm_b200.h"
#include "common.cuh"
#include "engine.h"
#include "layer.cuh"
#include "layer.h"

namespace spmmb {

namespace {

constexpr unsigned kFull = 0xffffffffu;

// A 16-byte vector of a row.
template <typename T, int VE> union Pack {
    uint4 raw;
    T e[VE];
    __device__ Pack() {}
};

template <typename T, int VE> __device__ __forceinline__ void unpack(const Pack<T, VE> &p, float *f)
{
#pragma unroll
    for (int i = 0; i < VE; ++i) f[i] = elem_f32<T>(p.e[i]);
}

template <typename T> __device__ __forceinline__ float load_param(const void *p, bool f32, int64_t c)
{
    return f32 ? __ldg(static_cast<const float *>(p) + c) : elem_f32<T>(static_cast<const T *>(p)[c]);
}

// Sums of N values over a team: shuffles within a warp, then, for a team of
// several warps, one exchange through `red` behind a barrier of the team's
// own threads.  The caller alternates two `red` buffers, so that one barrier
// per sum is enough.
template <int TEAM, int BLOCK> __device__ __forceinline__ void team_barrier(int team)
{
    if constexpr (TEAM == BLOCK) __syncthreads();
    else asm volatile("bar.sync %0, %1;\n" ::"r"(team + 1), "n"(TEAM) : "memory");
}
template <int TEAM, int BLOCK, int N> __device__ __forceinline__ void team_sum(float (&v)[N], float (*red)[N], int team)
{
#pragma unroll
    for (int o = (TEAM < 32 ? TEAM : 32) / 2; o > 0; o >>= 1)
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(kFull, v[i], o);
    if constexpr (TEAM > 32) {
        constexpr int kWarps = TEAM / 32;
        float(*mine)[N] = red + team * kWarps;
        if ((threadIdx.x & 31) == 0)
#pragma unroll
            for (int i = 0; i < N; ++i) mine[threadIdx.x % TEAM >> 5][i] = v[i];
        team_barrier<TEAM, BLOCK>(team);
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = 0.f;
#pragma unroll
        for (int w = 0; w < kWarps; ++w)
#pragma unroll
            for (int i = 0; i < N; ++i) v[i] += mine[w][i];
    }
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

// What a lane holds of its team's rows: NV 16-byte vectors, and with ODD
// (rows that start anywhere in a vector) NS single elements.  An odd row is a
// head of single elements up to the first vector boundary, whole vectors, and
// a tail of single elements.  A team only takes rows that start at the same
// place in a vector (its row stride is a multiple of VE), so each lane keeps
// its columns, and their parameters, for all its rows.
template <typename T, int NV_, int TEAM_, bool ODD_> struct Part {
    static constexpr int NV = NV_, TEAM = TEAM_, VE = 16 / sizeof(T);
    static constexpr bool ODD = ODD_;
    static constexpr int NS = !ODD ? 0 : TEAM < 16 ? 2 : 1, KS = NS ? NS : 1;
    int width, vec, vectors;   // vec: first column of vector 0; vectors: this lane's
    int single[KS];            // column of single element k, -1 for none

    __device__ __forceinline__ Part(int64_t row, int64_t w, int t) : width((int)w)
    {
        int head = 0, body = width / VE;
        if constexpr (ODD) {
            head = min((VE - (int)(row * w % VE)) % VE, width);
            body = (width - head) / VE;
            const int tail = width - head - body * VE;
            if constexpr (NS == 2) {
                single[0] = t < head ? t : -1;
                single[1] = t < tail ? width - tail + t : -1;
            } else {
                single[0] = t < 8 ? (t < head ? t : -1) : t - 8 < tail ? width - tail + t - 8 : -1;
            }
        }
        vec = head + t * VE;
        vectors = t < body ? (body - t + TEAM - 1) / TEAM : 0;
    }
    __device__ __forceinline__ int col(int i) const { return vec + i * TEAM * VE; }
    __device__ __forceinline__ int elements() const
    {
        int n = vectors * VE;
        for (int k = 0; k < NS; ++k) n += single[k] >= 0;
        return n;
    }
};

// One row's elements of a lane.
template <typename P, typename T> struct Row {
    Pack<T, P::VE> v[P::NV];
    T s[P::KS];
    __device__ __forceinline__ void load(const T *x, int64_t r, int64_t rows, const P &p)
    {
        if (r >= rows) return;
        const T *q = x + r * p.width;
#pragma unroll
        for (int i = 0; i < P::NV; ++i)
            if (i < p.vectors) v[i].raw = __ldcs(reinterpret_cast<const uint4 *>(q + p.col(i)));
#pragma unroll
        for (int k = 0; k < P::NS; ++k)
            if (p.single[k] >= 0) s[k] = q[p.single[k]];
    }
};

// Parameters of the lane's columns (`none` where there is no such array).
template <typename P, typename T> struct Params {
    float v[P::NV][P::VE], s[P::KS];
    __device__ __forceinline__ Params(const void *p, bool f32, float none, const P &part)
    {
#pragma unroll
        for (int i = 0; i < P::NV; ++i) {
            if (!P::ODD && p && i < part.vectors) {
                if (f32) {
#pragma unroll
                    for (int e = 0; e < P::VE; e += 4) {
                        const float *q = static_cast<const float *>(p) + part.col(i) + e;
                        const float4 u = __ldg(reinterpret_cast<const float4 *>(q));
                        v[i][e] = u.x; v[i][e + 1] = u.y; v[i][e + 2] = u.z; v[i][e + 3] = u.w;
                    }
                } else {
                    Pack<T, P::VE> u;
                    u.raw = __ldg(reinterpret_cast<const uint4 *>(static_cast<const T *>(p) + part.col(i)));
                    unpack<T, P::VE>(u, v[i]);
                }
            } else {
#pragma unroll
                for (int e = 0; e < P::VE; ++e)
                    v[i][e] = p && i < part.vectors ? load_param<T>(p, f32, part.col(i) + e) : none;
            }
        }
#pragma unroll
        for (int k = 0; k < P::NS; ++k) s[k] = p && part.single[k] >= 0 ? load_param<T>(p, f32, part.single[k]) : none;
    }
};

template <typename T, int NV, int TEAM, int BLOCK, bool ODD>
__global__ void __launch_bounds__(BLOCK) norm_forward_kernel(const NormArgs a)
{
    using P = Part<T, NV, TEAM, ODD>;
    constexpr int kTeams = BLOCK / TEAM, VE = P::VE, kLanes = TEAM < 32 ? TEAM : 32;
    __shared__ float red[2][BLOCK / 32][2], count[BLOCK / 32];
    const int t = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    const float inv = 1.f / (float)a.width;
    const T *x = static_cast<const T *>(a.x);
    const int64_t stride = (int64_t)gridDim.x * kTeams;
    int64_t r = (int64_t)blockIdx.x * kTeams + team;
    const P part(r, a.width, t);
    Row<P, T> row, next;
    row.load(x, r, a.rows, part);
    const Params<P, T> w(a.w, a.pf32, 1.f, part), b(a.b, a.pf32, 0.f, part);
    float inv_n = 0.f;   // of the warp's elements of a row
    if constexpr (TEAM > 32) {
        float n = (float)part.elements();
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) n += __shfl_xor_sync(kFull, n, o);
        inv_n = n > 0.f ? 1.f / n : 0.f;
        count[threadIdx.x >> 5] = n;   // read behind the first row's barrier
    }
    int turn = 0;
    // every lane of a warp (every thread of a block) takes the same number of turns
    for (int64_t r0 = (int64_t)blockIdx.x * kTeams; r0 < a.rows; r0 += stride, r += stride, turn ^= 1) {
        next.load(x, r + stride, a.rows, part);   // in flight while this row is worked on
        const bool on = r < a.rows;
        // the team's (a wider team: the warp's) sum, then its squares around its own mean
        float s = 0.f, q = 0.f;
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (on && i < part.vectors) {
                float f[VE];
                unpack<T, VE>(row.v[i], f);
#pragma unroll
                for (int e = 0; e < VE; ++e) s += f[e];
            }
#pragma unroll
        for (int k = 0; k < P::NS; ++k)
            if (on && part.single[k] >= 0) s += elem_f32<T>(row.s[k]);
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) s += __shfl_xor_sync(kFull, s, o);
        float mean = s * (TEAM > 32 ? inv_n : inv);
#pragma unroll
        for (int i = 0; i < NV; ++i)
            if (on && i < part.vectors) {
                float f[VE];
                unpack<T, VE>(row.v[i], f);
#pragma unroll
                for (int e = 0; e < VE; ++e) q = fmaf(f[e] - mean, f[e] - mean, q);
            }
#pragma unroll
        for (int k = 0; k < P::NS; ++k)
            if (on && part.single[k] >= 0) {
                const float d = elem_f32<T>(row.s[k]) - mean;
                q = fmaf(d, d, q);
            }
#pragma unroll
        for (int o = kLanes / 2; o > 0; o >>= 1) q += __shfl_xor_sync(kFull, q, o);
        if constexpr (TEAM > 32) {
            // join the warps behind one barrier: squares moved to the common mean
            // (sum (x - M)^2 = sum (x - m)^2 + n (m - M)^2)
            constexpr int kWarps = TEAM / 32;
            float(*mine)[2] = red[turn] + team * kWarps;
            if ((threadIdx.x & 31) == 0) {
                mine[t >> 5][0] = mean;
                mine[t >> 5][1] = q;
            }
            team_barrier<TEAM, BLOCK>(team);
            s = 0.f;
#pragma unroll
            for (int k = 0; k < kWarps; ++k) s = fmaf(count[team * kWarps + k], mine[k][0], s);
            mean = s * inv;
            q = 0.f;
#pragma unroll
            for (int k = 0; k < kWarps; ++k) {
                const float d = mine[k][0] - mean;
                q += fmaf(count[team * kWarps + k] * d, d, mine[k][1]);
            }
        }
        const float rstd = 1.f / sqrtf(q * inv + a.eps);
        if (on) {
            if (a.mean && t == 0) {
                a.mean[r] = mean;
                a.rstd[r] = rstd;
            }
            T *y = static_cast<T *>(a.y) + r * part.width;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (i >= part.vectors) continue;
                float f[VE];
                unpack<T, VE>(row.v[i], f);
                Pack<T, VE> o;
#pragma unroll
                for (int e = 0; e < VE; ++e) o.e[e] = elem_of<T>(fmaf((f[e] - mean) * rstd, w.v[i][e], b.v[i][e]));
                __stcs(reinterpret_cast<uint4 *>(y + part.col(i)), o.raw);
            }
#pragma unroll
            for (int k = 0; k < P::NS; ++k)
                if (part.single[k] >= 0)
                    y[part.single[k]] = elem_of<T>(fmaf((elem_f32<T>(row.s[k]) - mean) * rstd, w.s[k], b.s[k]));
        }
        row = next;
    }
}

// Rows wider than a block's registers: one block per row, three passes.
template <typename T>
__global__ void __launch_bounds__(512) norm_forward_wide_kernel(const NormArgs a)
{
    __shared__ float red[2][16][1];
    const float inv = 1.f / (float)a.width;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x) {
        const T *x = static_cast<const T *>(a.x) + r * a.width;
        T *y = static_cast<T *>(a.y) + r * a.width;
        float s[1] = {0.f};
        for (int64_t c = threadIdx.x; c < a.width; c += 512) s[0] += elem_f32<T>(x[c]);
        team_sum<512, 512>(s, red[0], 0);
        const float mean = s[0] * inv;
        s[0] = 0.f;
        for (int64_t c = threadIdx.x; c < a.width; c += 512) {
            const float d = elem_f32<T>(x[c]) - mean;
            s[0] = fmaf(d, d, s[0]);
        }
        team_sum<512, 512>(s, red[1], 0);
        const float rstd = 1.f / sqrtf(s[0] * inv + a.eps);
        if (a.mean && threadIdx.x == 0) {
            a.mean[r] = mean;
            a.rstd[r] = rstd;
        }
        for (int64_t c = threadIdx.x; c < a.width; c += 512) {
            float f = (elem_f32<T>(x[c]) - mean) * rstd;
            if (a.w) { f *= load_param<T>(a.w, a.pf32, c); }
            if (a.b) { f += load_param<T>(a.b, a.pf32, c); }
            y[c] = elem_of<T>(f);
        }
    }
}

// Backward: the lane that holds a column holds it for every row of its team,
// so dw and db accumulate in its registers; the teams of a block are added
// through shared memory and the block writes one partial row.
template <typename T, int NV, int TEAM, int BLOCK, bool ODD>
__global__ void __launch_bounds__(BLOCK) norm_backward_kernel(const NormArgs a)
{
    using P = Part<T, NV, TEAM, ODD>;
    constexpr int kTeams = BLOCK / TEAM, VE = P::VE;
    __shared__ float red[2][BLOCK / 32][2];
    const int t = threadIdx.x % TEAM, team = threadIdx.x / TEAM;
    const float inv = 1.f / (float)a.width;
    const T *x = static_cast<const T *>(a.x), *dy = static_cast<const T *>(a.dy);
    const int64_t stride = (int64_t)gridDim.x * kTeams;
    int64_t r = (int64_t)blockIdx.x * kTeams + team;
    const P part(r, a.width, t);
    Row<P, T> vx, vg, nx, ng;
    vx.load(x, r, a.rows, part);
    vg.load(dy, r, a.rows, part);
    float mean = r < a.rows ? a.mean[r] : 0.f, rstd = r < a.rows ? a.rstd[r] : 0.f;
    const Params<P, T> w(a.w, a.pf32, 1.f, part);
    float dw[NV][VE], db[NV][VE], dws[P::KS], dbs[P::KS];
#pragma unroll
    for (int i = 0; i < NV; ++i)
#pragma unroll
        for (int e = 0; e < VE; ++e) dw[i][e] = db[i][e] = 0.f;
#pragma unroll
    for (int k = 0; k < P::KS; ++k) dws[k] = dbs[k] = 0.f;
    int turn = 0;
    for (int64_t r0 = (int64_t)blockIdx.x * kTeams; r0 < a.rows; r0 += stride, r += stride, turn ^= 1) {
        const bool on = r < a.rows, more = r + stride < a.rows;
        nx.load(x, r + stride, a.rows, part);   // in flight while this row is worked on
        ng.load(dy, r + stride, a.rows, part);
        const float next_mean = more ? a.mean[r + stride] : 0.f, next_rstd = more ? a.rstd[r + stride] : 0.f;
        float s[2] = {0.f, 0.f};
        auto add = [&](float f, float g, float wv, float &dwv, float &dbv) {
            const float xh = (f - mean) * rstd, gw = g * wv;
            dwv = fmaf(g, xh, dwv);
            dbv += g;
            s[0] += gw;
            s[1] = fmaf(gw, xh, s[1]);
        };
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            if (!on || i >= part.vectors) continue;
            float f[VE], g[VE];
            unpack<T, VE>(vx.v[i], f);
            unpack<T, VE>(vg.v[i], g);
#pragma unroll
            for (int e = 0; e < VE; ++e) add(f[e], g[e], w.v[i][e], dw[i][e], db[i][e]);
        }
#pragma unroll
        for (int k = 0; k < P::NS; ++k)
            if (on && part.single[k] >= 0) add(elem_f32<T>(vx.s[k]), elem_f32<T>(vg.s[k]), w.s[k], dws[k], dbs[k]);
        if (a.y) {   // the same for every thread
            team_sum<TEAM, BLOCK>(s, red[turn], team);
            const float c1 = s[0] * inv, c2 = s[1] * inv;
            auto grad = [&](float f, float g, float wv) {
                const float xh = (f - mean) * rstd;
                return elem_of<T>(rstd * (g * wv - c1 - xh * c2));
            };
            T *dx = static_cast<T *>(a.y) + r * part.width;
#pragma unroll
            for (int i = 0; i < NV; ++i) {
                if (!on || i >= part.vectors) continue;
                float f[VE], g[VE];
                unpack<T, VE>(vx.v[i], f);
                unpack<T, VE>(vg.v[i], g);
                Pack<T, VE> o;
#pragma unroll
                for (int e = 0; e < VE; ++e) o.e[e] = grad(f[e], g[e], w.v[i][e]);
                __stcs(reinterpret_cast<uint4 *>(dx + part.col(i)), o.raw);
            }
#pragma unroll
            for (int k = 0; k < P::NS; ++k)
                if (on && part.single[k] >= 0)
                    dx[part.single[k]] = grad(elem_f32<T>(vx.s[k]), elem_f32<T>(vg.s[k]), w.s[k]);
        }
        vx = nx;
        vg = ng;
        mean = next_mean;
        rstd = next_rstd;
    }
    if (!a.part) return;
    float *pw = a.part + (int64_t)blockIdx.x * 2 * a.width;
    auto put = [&](float *at, const float (&v)[NV][VE], const float (&single)[P::KS]) {
#pragma unroll
        for (int i = 0; i < NV; ++i)
#pragma unroll
            for (int e = 0; e < VE; ++e)
                if (i < part.vectors) at[part.col(i) + e] = v[i][e];
#pragma unroll
        for (int k = 0; k < P::NS; ++k)
            if (part.single[k] >= 0) at[part.single[k]] = single[k];
    };
    if constexpr (kTeams == 1) {
        put(pw, dw, dws);
        put(pw + a.width, db, dbs);
    } else {
        __shared__ float sums[kTeams][TEAM * NV * VE + 15];   // by column
        for (int which = 0; which < 2; ++which) {
            __syncthreads();
            if (which) put(sums[team], db, dbs);
            else put(sums[team], dw, dws);
            __syncthreads();
            for (int c = threadIdx.x; c < a.width; c += BLOCK) {
                float v = 0.f;
#pragma unroll
                for (int k = 0; k < kTeams; ++k) v += sums[k][c];
                pw[which * a.width + c] = v;
            }
        }
    }
}

template <typename T>
__global__ void __launch_bounds__(512) norm_backward_wide_kernel(const NormArgs a)
{
    __shared__ float red[2][16][2];
    const float inv = 1.f / (float)a.width;
    float *pw = a.part ? a.part + (int64_t)blockIdx.x * 2 * a.width : nullptr;
    if (pw)
        for (int64_t c = threadIdx.x; c < 2 * a.width; c += 512) pw[c] = 0.f;
    __syncthreads();
    int turn = 0;
    for (int64_t r = blockIdx.x; r < a.rows; r += gridDim.x, turn ^= 1) {
        const T *x = static_cast<const T *>(a.x) + r * a.width, *dy = static_cast<const T *>(a.dy) + r * a.width;
        const float mean = a.mean[r], rstd = a.rstd[r];
        float s[2] = {0.f, 0.f};
        for (int64_t c = threadIdx.x; c < a.width; c += 512) {
            const float g = elem_f32<T>(dy[c]), xh = (elem_f32<T>(x[c]) - mean) * rstd;
            const float p = a.w ? load_param<T>(a.w, a.pf32, c) : 1.f;
            s[0] += g * p;
            s[1] = fmaf(g * p, xh, s[1]);
            if (pw) {   // this thread's own columns
                pw[c] = fmaf(g, xh, pw[c]);
                pw[a.width + c] += g;
            }
        }
        if (!a.y) continue;
        team_sum<512, 512>(s, red[turn], 0);
        const float c1 = s[0] * inv, c2 = s[1] * inv;
        T *dx = static_cast<T *>(a.y) + r * a.width;
        for (int64_t c = threadIdx.x; c < a.width; c += 512) {
            const float xh = (elem_f32<T>(x[c]) - mean) * rstd;
            const float p = a.w ? load_param<T>(a.w, a.pf32, c) : 1.f;
            dx[c] = elem_of<T>(rstd * (elem_f32<T>(dy[c]) * p - c1 - xh * c2));
        }
    }
}

// Adds the blocks' partial rows: 32 columns per block, 32 partial rows at a
// time, in an order that depends on the number of partials alone.
template <typename P>
__global__ void __launch_bounds__(1024) norm_params_kernel(const float *part, int blocks, int64_t width, P *dw, P *db)
{
    __shared__ float sums[32][33];
    const int lane = threadIdx.x & 31, row = threadIdx.x >> 5;
    const int64_t c = (int64_t)blockIdx.x * 32 + lane;   // over dw's columns, then db's
    float s = 0.f;
    if (c < 2 * width) {
#pragma unroll 8
        for (int k = row; k < blocks; k += 32) s += part[(int64_t)k * 2 * width + c];
    }
    sums[row][lane] = s;
    __syncthreads();
    s = sums[lane][row];   // column `row` of the block, its 32 sums across the lanes
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(kFull, s, o);
    const int64_t d = (int64_t)blockIdx.x * 32 + row;
    if (lane == 0 && d < 2 * width) {
        P *out = d < width ? dw : db;
        if (out) out[d < width ? d : d - width] = elem_of<P>(s);
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

template <typename T, int NV, int TEAM, bool ODD, bool BACKWARD>
cudaError_t run_team(const NormArgs &a, int64_t max_blocks, int64_t *blocks, cudaStream_t stream)
{
    constexpr int kBlock = TEAM < 256 ? 256 : TEAM, kTeams = kBlock / TEAM, VE = 16 / sizeof(T);
    const int64_t turns = (a.rows + kTeams - 1) / kTeams;
    constexpr auto kernel = [] {
        if constexpr (BACKWARD) return norm_backward_kernel<T, NV, TEAM, kBlock, ODD>;
        else return norm_forward_kernel<T, NV, TEAM, kBlock, ODD>;
    }();
    *blocks = grid_of<kernel>(kBlock, turns);
    if (BACKWARD) *blocks = std::min(max_blocks, *blocks);
    // a team's rows must start at the same place in a vector
    constexpr int kStep = VE / kTeams > 1 ? VE / kTeams : 1;
    if (ODD && *blocks < turns) *blocks = std::max<int64_t>(kStep, *blocks / kStep * kStep);
    kernel<<<(unsigned)*blocks, kBlock, 0, stream>>>(a);
    return cudaGetLastError();
}

// Vectors per lane, measured side by side (fp16, 524287 x 1024; GB/s of 6538,
// calls back to back): forward 4 on a warp 6390, 2 on two warps 5810 (its two
// sums need a barrier); backward, which also holds two accumulators per column,
// 2 on two warps 5770, 4 on a warp 4710.
template <typename T, bool ODD, bool BACKWARD>
cudaError_t run_width(const NormArgs &a, int64_t max_blocks, int64_t *blocks, cudaStream_t s, bool *wide)
{
    constexpr int V = 16 / sizeof(T), NV = BACKWARD ? 2 : 4;
    const int64_t v = a.width / V;   // whole vectors of a row, at most
    if (v <= 8) return run_team<T, 1, 8, ODD, BACKWARD>(a, max_blocks, blocks, s);
    if (v <= 16) return run_team<T, 2, 8, ODD, BACKWARD>(a, max_blocks, blocks, s);
    if (v <= 16 * NV) return run_team<T, NV, 16, ODD, BACKWARD>(a, max_blocks, blocks, s);
    if (v <= 32 * NV) return run_team<T, NV, 32, ODD, BACKWARD>(a, max_blocks, blocks, s);
    if (v <= 64 * NV) return run_team<T, NV, 64, ODD, BACKWARD>(a, max_blocks, blocks, s);
    if (v <= 128 * NV) return run_team<T, NV, 128, ODD, BACKWARD>(a, max_blocks, blocks, s);
    if (v <= 256 * NV) return run_team<T, NV, 256, ODD, BACKWARD>(a, max_blocks, blocks, s);
    if (v <= 512 * NV) return run_team<T, NV, 512, ODD, BACKWARD>(a, max_blocks, blocks, s);
    if (BACKWARD && v <= 2048) return run_team<T, 2, 1024, ODD, true>(a, max_blocks, blocks, s);
    *wide = true;
    return cudaSuccess;
}

template <typename T> cudaError_t run_norm(const NormArgs &a, bool backward, int64_t max_blocks, int64_t *blocks,
                                           cudaStream_t s)
{
    bool wide = false;
    const bool odd = a.width % (16 / sizeof(T)) != 0;
    const cudaError_t e = backward ? odd ? run_width<T, true, true>(a, max_blocks, blocks, s, &wide)
                                           : run_width<T, false, true>(a, max_blocks, blocks, s, &wide)
                          : odd ? run_width<T, true, false>(a, max_blocks, blocks, s, &wide)
                                  : run_width<T, false, false>(a, max_blocks, blocks, s, &wide);
    if (!wide) return e;
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

int64_t norm_backward_blocks(int64_t rows, int64_t width)
{
    // What an SM's 2048 threads hold of a row's lanes (run_width; 16-bit rows
    // have the fewest): 8 blocks of 256, 4 of 512, 2 of 1024 threads.  Rows
    // wider than a block run on 2 of 512.  Few rows need no more blocks than rows.
    const int64_t per_sm = width / 8 <= 512 ? 8 : width / 8 <= 1024 ? 4 : 2;
    return std::max<int64_t>(1, std::min<int64_t>(rows, per_sm * device_sm_count()));
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
    cudaError_t e = dispatch(a, n.dtype, true, norm_backward_blocks(n.rows, n.width), &blocks, stream);
    if (e != cudaSuccess || !a.part) return e;
    const unsigned grid = (unsigned)((2 * n.width + 31) / 32);
    switch (n.param_dtype) {
        case SPMM_F16:
            norm_params_kernel<__half><<<grid, 1024, 0, stream>>>(a.part, (int)blocks, n.width,
                                                                 static_cast<__half *>(dweight),
                                                                 static_cast<__half *>(dbias));
            break;
        case SPMM_BF16:
            norm_params_kernel<__nv_bfloat16><<<grid, 1024, 0, stream>>>(a.part, (int)blocks, n.width,
                                                                        static_cast<__nv_bfloat16 *>(dweight),
                                                                        static_cast<__nv_bfloat16 *>(dbias));
            break;
        default:
            norm_params_kernel<float><<<grid, 1024, 0, stream>>>(a.part, (int)blocks, n.width,
                                                                static_cast<float *>(dweight),
                                                                static_cast<float *>(dbias));
    }
    return cudaGetLastError();
}

}  // namespace spmmb
