// Orthogonalised updates: X0 = U / (|U|_F + eps), then `steps` times
//   G = X X^T,  P = b G + c G G,  X <- a X + P X
// on the smaller side s of the matrix (for a tall one G = X^T X and
// X <- a X + X P, the same polynomial).  Each step is two symmetric s x s
// products, of which (but in small ones) the tiles on and below the diagonal
// are computed and written twice, and one s x s by s x r product; all run on the tensor cores
// (gemm_tc.cuh), which read X, G and P as they lie, so nothing is transposed.
//
// Precision.  The operands are fp16, not bf16: every singular value stays of
// order one (they start in [0, 1], the default coefficients take them to at
// most 1.2024 and map [0, 1.2637] into itself), so the elements need no
// exponent range, and 11 bits instead of 8 take the result's error from 1e-2
// to about 2e-3.  Other coefficients may take singular values anywhere: the
// operands' scales follow what the steps can reach (ortho.cuh).  X is kept as
// a high and a low fp16 part (22 bits): the products take the high part, the
// term a X both.  Otherwise the rounding of X would be multiplied by a in
// every step along the directions whose singular values are still small: 5e-3
// after five steps on a low-rank update with noise, 2e-4 with the low part.
//
// Matrices with a side of at most 128 run in ortho_small.cu, as long as the
// steps are few enough for it.
//
// Measured: one 4096 x 2048 update 357 us, 300 GFLOP with the symmetric halves
// counted once: of a step's 69 us the symmetric products take 20 and 14, the
// update 33, each about 5 us of launch, first copies and last tile beyond its
// products.  Three of 601 x 1023 137 us: fifteen dependent products of 8 to 12
// us, of which the reduction's slices are 2 to 4.
#include <algorithm>
#include <climits>

#include "../../include/spmm_b200.h"
#include "common.cuh"
#include "engine.h"
#include "gemm_tc.cuh"
#include "layer.cuh"
#include "layer.h"
#include "ortho.cuh"

namespace spmmb {

namespace {

constexpr int kParts = 512;   // partial sums of squares per matrix, at most

int64_t pad8(int64_t x) { return (x + 7) & ~int64_t(7); }

// Sums of squares, in 64 bits (an fp32 update's squares can leave fp32's range).
template <typename T>
__global__ void __launch_bounds__(256) ortho_squares_kernel(const T *u, int64_t elems, double *part)
{
    __shared__ double red[8];
    constexpr int V = 16 / sizeof(T);
    const T *p = u + (int64_t)blockIdx.y * elems;
    double s = 0.0;
    const int64_t step = (int64_t)gridDim.x * 256, first = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (elems % V == 0) {
        for (int64_t i = first; i < elems / V; i += step) {
            const uint4 w = __ldg(reinterpret_cast<const uint4 *>(p) + i);
            const T *e = reinterpret_cast<const T *>(&w);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                const double v = (double)elem_f32<T>(e[k]);
                s += v * v;
            }
        }
    } else {
        for (int64_t i = first; i < elems; i += step) {
            const double v = (double)elem_f32<T>(p[i]);
            s += v * v;
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = s;
    __syncthreads();
    if (threadIdx.x == 0) {
        s = 0.0;
        for (int w = 0; w < 8; ++w) s += red[w];
        part[(int64_t)blockIdx.y * gridDim.x + blockIdx.x] = s;
    }
}

// X0 as its high and low parts [m][ld] (a thread: 8 columns), or, with no
// step to follow, the bf16 result.
template <typename T>
__global__ void __launch_bounds__(256)
ortho_split_kernel(const T *u, const double *part, int parts, float eps, int64_t m, int64_t n, int64_t ld, __half *hi,
                   __half *lo, __nv_bfloat16 *out)
{
    __shared__ float scale;
    if (threadIdx.x < 32) {
        double s = 0.0;
        for (int i = threadIdx.x; i < parts; i += 32) s += part[(int64_t)blockIdx.y * parts + i];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (threadIdx.x == 0) scale = (float)(1.0 / (sqrt(s) + (double)eps));
    }
    __syncthreads();
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, per = ld / 8;
    if (i >= m * per) return;
    const int64_t r = i / per, c = i % per * 8;
    const T *p = u + ((int64_t)blockIdx.y * m + r) * n + c;
    float v[8];
    if (n % 8 == 0) {
        constexpr int V = 16 / sizeof(T);
#pragma unroll
        for (int k = 0; k < 8 / V; ++k) {
            const uint4 w = __ldg(reinterpret_cast<const uint4 *>(p) + k);
#pragma unroll
            for (int e = 0; e < V; ++e) v[k * V + e] = elem_f32<T>(reinterpret_cast<const T *>(&w)[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = c + e < n ? elem_f32<T>(p[e]) : 0.f;
    }
    if (out) {
        for (int e = 0; e < 8 && c + e < n; ++e)
            out[((int64_t)blockIdx.y * m + r) * n + c + e] = __float2bfloat16_rn(v[e] * scale);
        return;
    }
    // one rounding of the normalised value, then scaled by a power of two
    float h[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = v[e] * scale * kScaleX;
    const uint4 w = tc::pack8(v, false);
    unpack16<__half>(w, h);
#pragma unroll
    for (int e = 0; e < 8; ++e) h[e] = v[e] - h[e];
    const int64_t at = ((int64_t)blockIdx.y * m + r) * ld + c;
    *reinterpret_cast<uint4 *>(hi + at) = w;
    *reinterpret_cast<uint4 *>(lo + at) = tc::pack8(h, false);
}

struct Space {
    int64_t ldx, lds, x, s;   // leading dimensions; elements of X and of a square matrix, whole batch
    int parts;
    __half *hi[2], *lo, *gram, *poly;
    double *part;
    Space(int64_t batch, int64_t m, int64_t n, void *ws)
    {
        const int64_t side = std::min(m, n);
        ldx = pad8(n);
        lds = pad8(side);
        x = (batch * m * ldx + 127) & ~int64_t(127);
        s = (batch * side * lds + 127) & ~int64_t(127);
        parts = ortho_square_parts(batch, m, n);
        hi[0] = static_cast<__half *>(ws);
        hi[1] = hi[0] + x;
        lo = hi[1] + x;
        gram = lo + x;
        poly = gram + s;
        part = reinterpret_cast<double *>(poly + s);
    }
    size_t bytes(int64_t batch) const { return (size_t)(3 * x + 2 * s) * 2 + (size_t)batch * parts * 8; }
};

template <typename T> void start(const OrthoLaunch &o, const Space &w, cudaStream_t stream)
{
    const T *u = static_cast<const T *>(o.update);
    const int64_t items = o.m * (w.ldx / 8);
    ortho_split_kernel<T><<<dim3((unsigned)((items + 255) / 256), (unsigned)o.batch), 256, 0, stream>>>(
        u, w.part, w.parts, o.eps, o.m, o.n, w.ldx, w.hi[0], w.lo,
        o.steps == 0 ? static_cast<__nv_bfloat16 *>(o.out) : nullptr);
}

// Columns of a tile of a symmetric product.  In tiles of 128 x 128 one of two
// mirrored ones is computed and stored twice; where narrower tiles of the
// whole square fit one turn of the GPU, their shorter products and single
// store win (1024 x 1024: 231 us in halves, 161 with 64 columns; 5 of 512 x
// 512: 125 and, with 96, 121; but 2 of 1024 x 1024, more than one turn, 158
// and 179).
int square_columns(int64_t row_tiles, int64_t side, int sms)
{
    for (int bn : {64, 96})
        if (row_tiles * ((side + bn - 1) / bn) <= sms) return bn;
    return 128;
}

// Columns of an update's tile: the width with the least turns x time, a slice
// of a tile taking about as long as 70 + bn columns.  12 of 700 x 700: 240 us
// with 128 (3 turns), 259 with 256 (2); 30 of 200 x 900: 220 (4) and 210 (2);
// 601 x 1000: 134 and, with 64, 124 (one turn each).
int update_columns(int64_t row_tiles, int64_t width, int sms)
{
    int best = 0;
    int64_t least = INT64_MAX;
    for (int bn : {64, 96, 128, 256}) {
        const int64_t cost = (row_tiles * ((width + bn - 1) / bn) + sms - 1) / sms * (bn + 70);
        if (cost < least) {
            least = cost;
            best = bn;
        }
    }
    return best;
}

// The tensor maps of a call, each encoded once.
struct OrthoMaps {
    CUtensorMap square[2], x[2];            // X as the operands of G and of the update, by buffer
    CUtensorMap square_b[2], gram_b;        // the second operand of G and of G G: tiles of another width
    CUtensorMap gram, poly;                 // G and P as operands
    CUtensorMap gram_out, poly_out, x_out[2], low_out, out;
};

template <int BN>
cudaError_t gram(bool tall, const tc::Maps &m, const tc::GemmArgs &g, int64_t tiles, cudaStream_t stream)
{
    return tall ? tc::launch_gemm<tc::kDense, BN, true, true, tc::kGram>(m, g, tiles, stream)
                : tc::launch_gemm<tc::kDense, BN, false, false, tc::kGram>(m, g, tiles, stream);
}

template <int BN, bool PAIR = false>
cudaError_t update(const OrthoLaunch &o, const tc::Maps &m, const tc::GemmArgs &g, cudaStream_t stream)
{
    const int64_t height = PAIR ? 2 * tc::kBM : tc::kBM;
    const int64_t tiles = o.batch * ((o.m + height - 1) / height) * ((o.n + g.bn - 1) / g.bn);
    if (o.m > o.n) return tc::launch_gemm<tc::kDense, BN, false, false, tc::kUpdate, PAIR>(m, g, tiles, stream);
    return tc::launch_gemm<tc::kDense, BN, false, true, tc::kUpdate, PAIR>(m, g, tiles, stream);
}

}  // namespace

int ortho_square_parts(int64_t batch, int64_t m, int64_t n)
{
    return (int)std::max<int64_t>(1, std::min({(int64_t)kParts, m * n / 8192, 2048 / batch}));
}

cudaError_t launch_ortho_squares(const OrthoLaunch &o, double *squares, cudaStream_t stream)
{
    const dim3 grid(ortho_square_parts(o.batch, o.m, o.n), (unsigned)o.batch);
    const int64_t elems = o.m * o.n;
    switch (o.dtype) {
        case SPMM_F16:
            ortho_squares_kernel<<<grid, 256, 0, stream>>>(static_cast<const __half *>(o.update), elems, squares);
            break;
        case SPMM_BF16:
            ortho_squares_kernel<<<grid, 256, 0, stream>>>(static_cast<const __nv_bfloat16 *>(o.update), elems, squares);
            break;
        default: ortho_squares_kernel<<<grid, 256, 0, stream>>>(static_cast<const float *>(o.update), elems, squares);
    }
    return cudaGetLastError();
}

size_t ortho_workspace(int64_t batch, int64_t m, int64_t n, int)
{
    // which form runs depends on the steps and coefficients too: room for either
    return std::max(Space(batch, m, n, nullptr).bytes(batch),
                    std::min(m, n) <= 128 ? ortho_small_workspace(batch, m, n) : 0);
}

cudaError_t launch_ortho(const OrthoLaunch &o, void *workspace, cudaStream_t stream)
{
    const float scale_q = ortho_small_scale(o);
    if (scale_q > 0.f) return launch_ortho_small(o, scale_q, workspace, stream);
    const Space w(o.batch, o.m, o.n, workspace);
    cudaError_t e = launch_ortho_squares(o, w.part, stream);
    if (e != cudaSuccess) return e;
    switch (o.dtype) {
        case SPMM_F16: start<__half>(o, w, stream); break;
        case SPMM_BF16: start<__nv_bfloat16>(o, w, stream); break;
        default: start<float>(o, w, stream);
    }
    e = cudaGetLastError();
    if (e != cudaSuccess || o.steps == 0) return e;
    const bool tall = o.m > o.n;
    const int64_t side = std::min(o.m, o.n), long_side = std::max(o.m, o.n), sq = side * w.lds, all = o.m * w.ldx;
    const int sms = device_sm_count();
    const int64_t mt = (side + tc::kBM - 1) / tc::kBM;
    const int square_bn = square_columns(o.batch * mt, side, sms);
    const bool whole = square_bn < tc::kBM;
    const int64_t square_tiles = whole ? o.batch * mt * ((side + square_bn - 1) / square_bn) : o.batch * mt * (mt + 1) / 2;
    const int64_t row_tiles = o.batch * ((o.m + tc::kBM - 1) / tc::kBM);
    const int bn = update_columns(row_tiles, o.n, sms);
    // Two SMs share a tile where the products are deep and take several turns
    // (4 of 2048 x 2048: 879 us alone, 780 in pairs; 4096 x 4096: 1572 and
    // 1332; but 3 of 1024 x 4096: 369 and 381, one 2048 x 2048: 245 and 252).
    const bool pair = bn == 256 && side > 1024 && row_tiles * ((o.n + 255) / 256) > sms;
    // a result whose rows do not start on 16 bytes has no map
    const bool mapped = (o.n & 7) == 0;
    OrthoMaps M;
    bool fine = tc::make_map(&M.gram, w.gram, side, side, o.batch, w.lds, sq, tc::kBM, false) &&
                tc::make_map(&M.gram_b, w.gram, side, side, o.batch, w.lds, sq, square_bn, false) &&
                tc::make_map(&M.poly, w.poly, side, side, o.batch, w.lds, sq, tall ? pair ? bn / 2 : bn : tc::kBM, false) &&
                tc::make_out_map(&M.gram_out, w.gram, side, side, o.batch, w.lds, sq, tc::kOutF16) &&
                tc::make_out_map(&M.poly_out, w.poly, side, side, o.batch, w.lds, sq, tc::kOutF16) &&
                tc::make_out_map(&M.low_out, w.lo, o.n, o.m, o.batch, w.ldx, all, tc::kOutF16);
    bool blocked_square = false, blocked_square_b = false, blocked_x = false;
    for (int i = 0; i < 2 && fine; ++i)   // tall: G reads X down its rows, the update along them; wide: the reverse
        fine = (tall ? tc::make_mn_map(&M.square[i], &blocked_square, w.hi[i], o.n, o.m, o.batch, w.ldx, all, tc::kBM,
                                       false) &&
                           tc::make_mn_map(&M.square_b[i], &blocked_square_b, w.hi[i], o.n, o.m, o.batch, w.ldx, all,
                                           square_bn, false)
                     : tc::make_map(&M.square[i], w.hi[i], o.n, o.m, o.batch, w.ldx, all, tc::kBM, false) &&
                           tc::make_map(&M.square_b[i], w.hi[i], o.n, o.m, o.batch, w.ldx, all, square_bn, false)) &&
               (tall ? tc::make_map(&M.x[i], w.hi[i], o.n, o.m, o.batch, w.ldx, all, tc::kBM, false)
                     : tc::make_mn_map(&M.x[i], &blocked_x, w.hi[i], o.n, o.m, o.batch, w.ldx, all, pair ? bn / 2 : bn,
                                       false)) &&
               tc::make_out_map(&M.x_out[i], w.hi[i], o.n, o.m, o.batch, w.ldx, all, tc::kOutF16);
    M.out = M.x_out[0];
    if (fine && mapped) fine = tc::make_out_map(&M.out, o.out, o.n, o.m, o.batch, o.n, o.m * o.n, tc::kOutBf16);
    if (!fine) return cudaErrorInvalidValue;
    OrthoReach at(o.a, o.b, o.c);
    double scale_x = kScaleX;   // of the stored X; it starts with singular values of at most one
    for (int i = 0; i < o.steps && e == cudaSuccess; ++i) {
        const int now = i & 1, next = now ^ 1;
        const double scale_g = scale_for(kScaleG, at.reach * at.reach), scale_p = scale_for(kScaleP, at.poly());
        at.step();
        const double next_x = i + 1 == o.steps ? 1.0 : scale_for(kScaleX, at.reach);   // the result is not scaled
        tc::GemmArgs g{};
        g.batch = o.batch;
        g.status = o.status;
        g.out_type = tc::kOutF16;
        // G = X X^T (X^T X)
        g.m = g.n = side;
        g.k = long_side;
        g.bn = square_bn;
        g.out = w.gram;
        g.ldo = w.lds;
        g.out_batch = sq;
        g.alpha = (float)(scale_g / (scale_x * scale_x));
        g.symmetric = !whole;
        g.blocked_a = blocked_square;
        g.blocked_b = blocked_square_b;
        tc::Maps m{M.square[now], M.square_b[now], M.gram_out, M.gram_out};
        e = square_bn == 64 ? gram<64>(tall, m, g, square_tiles, stream) : gram<128>(tall, m, g, square_tiles, stream);
        if (e != cudaSuccess) break;
        // P = b G + c G G
        g.k = side;
        g.in = w.gram;
        g.ldi = w.lds;
        g.in_batch = sq;
        g.out = w.poly;
        g.alpha = (float)(o.c * (scale_p / (scale_g * scale_g)));
        g.beta = (float)(o.b * (scale_p / scale_g));
        m = tc::Maps{M.gram, M.gram_b, M.poly_out, M.poly_out};
        e = square_bn == 64
                ? tc::launch_gemm<tc::kDense, 64, false, false, tc::kPoly>(m, g, square_tiles, stream)
                : tc::launch_gemm<tc::kDense, 128, false, false, tc::kPoly>(m, g, square_tiles, stream);
        if (e != cudaSuccess) break;
        // X <- a X + P X (X P); the last step writes the result
        const bool last = i + 1 == o.steps;
        g.symmetric = false;
        g.m = o.m;
        g.n = o.n;
        g.bn = bn;
        g.in = w.hi[now];
        g.in_lo = w.lo;
        g.ldi = w.ldx;
        g.in_batch = all;
        g.out = last ? o.out : static_cast<void *>(w.hi[next]);
        g.low = !last;
        g.ldo = last ? o.n : w.ldx;
        g.out_batch = o.m * g.ldo;
        g.out_type = last ? tc::kOutBf16 : tc::kOutF16;
        g.blocked_a = false;
        g.blocked_b = blocked_x;
        g.alpha = (float)(next_x / (scale_p * scale_x));
        g.beta = (float)(o.a * (next_x / scale_x));
        scale_x = next_x;
        m = tc::Maps{tall ? M.x[now] : M.poly, tall ? M.poly : M.x[now], last ? M.out : M.x_out[next], M.low_out};
        if (pair) e = update<256, true>(o, m, g, stream);
        else if (bn > 128) e = update<256>(o, m, g, stream);
        else if (bn > 64) e = update<128>(o, m, g, stream);
        else e = update<64>(o, m, g, stream);
    }
    return e;
}

}  // namespace spmmb
