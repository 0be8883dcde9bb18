// Products of row ranges with one matrix each, and their gradients.
//
//   rows product      out[r] = x[r] W_g       (or x[r] W_g^T) for the rows r of group g
//   weight gradient   dW_g  = x_g^T dy_g      (a sum over the rows of group g)
//
// The group of a row tile is found on the device from the row ranges, so no
// length crosses to the host and a launch can be captured in a graph.
//
// Measured (us; forward, gradient of x, gradient of the weight): bf16, 65537
// uneven rows of 64 groups, K = 1024, N = 2048 217, 221, 300 in the first
// passes and 256, 254, 340 after some hundred (275 GFLOP each: the products, at
// the clock that the power limit leaves); fp16, 100003 rows of 46 groups, K
// = 256, N = 128 16, 18, 27 (77 MB each: memory, and for the weight the parts);
// fp32, 20011 rows of 8 groups, K = 256, N = 264 39, 40, 56 (12 to 20 of each
// is splitting the operands); bf16, 9 rows of 32 groups, K = 1024, N = 512 10,
// half of it the fixed cost of a launch, its first copies and its last store.
#include <algorithm>
#include <climits>

#include "../../include/spmm_b200.h"
#include "common.cuh"
#include "engine.h"
#include "gemm_tc.cuh"
#include "layer.cuh"
#include "layer.h"

namespace spmmb {

namespace {

__host__ __device__ Ranges ranges_of(const GroupedLaunch &a)
{
    return Ranges{a.ptr, a.itype == SPMM_I64, a.groups, a.rows};
}

// ---- fp32 operands ----------------------------------------------------------
//
// The tensor cores take fp32 as tf32 (11 bits).  To keep fp32's 24 bits each
// operand is written as three bf16 planes x = h + m + l (8 bits each, fp32's
// exponents) and the product is run as the six plane products above 2^-24 of
// the result, the smallest first:  h l, l h, m m, h m, m h, h h.  That is six
// bf16 products, about four times the rate of fp32 FMAs.  The six share a
// slice's planes in shared memory: bringing each product's two operands in by
// themselves took half as long again (51, 55 and 69 us for 39, 40 and 56 in
// the case above), bound by those copies.
//
// An infinite x is split as h = +-1, m = 0, l = +-infinity.  l meets the other
// operand's h alone, so the product is an infinity of the right sign, and NaN
// where the other is zero; an infinite h beside the zero m and l planes of
// ordinary numbers would make it NaN.
constexpr int kPlanes = 3;

// An operand to split: src [groups][elems], planes `plane` apart.  `skip`:
// groups without rows are left out.
struct Split {
    const float *src;
    __nv_bfloat16 *dst;
    int64_t elems, plane, groups;
    bool skip;
    __host__ __device__ int64_t chunks() const { return (elems + 2047) / 2048; }   // of a group
};

// Chunks of 2048 elements, of the first operand and then of the second; a
// thread splits 8 elements.
__global__ void __launch_bounds__(256) split_planes_kernel(const Split first, const Split second, Ranges ranges,
                                                           DevStatus *status)
{
    const int64_t firsts = first.groups * first.chunks(), total = firsts + second.groups * second.chunks();
    for (int64_t item = blockIdx.x; item < total; item += gridDim.x) {
        const Split &s = item < firsts ? first : second;
        const int64_t chunk = item < firsts ? item : item - firsts, g = chunk / s.chunks();
        if (s.skip) {
            int64_t b, e;
            segment_rows(ranges, g + 1, &b, &e, status);
            if (b == e) continue;
        }
        const int64_t in_group = chunk % s.chunks() * 2048 + threadIdx.x * 8, i = g * s.elems + in_group;
        if (in_group >= s.elems) continue;
        const float4 u = __ldg(reinterpret_cast<const float4 *>(s.src + i));
        const float4 w = __ldg(reinterpret_cast<const float4 *>(s.src + i) + 1);
        float v[8] = {u.x, u.y, u.z, u.w, w.x, w.y, w.z, w.w}, last[8];   // last: what only plane l holds
#pragma unroll
        for (int k = 0; k < 8; ++k) {
            last[k] = isinf(v[k]) ? v[k] : 0.f;
            if (isinf(v[k])) v[k] = copysignf(1.f, v[k]);
        }
#pragma unroll
        for (int p = 0; p < kPlanes; ++p) {
            __align__(16) __nv_bfloat16 h[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (p == kPlanes - 1) v[k] += last[k];
                h[k] = __float2bfloat16_rn(v[k]);
                // next to fp32's maximum, rounding up would leave the range
                if (isinf(__bfloat162float(h[k])) && !isinf(v[k])) h[k] = __float2bfloat16_rz(v[k]);
                v[k] = isnan(v[k]) ? 0.f : v[k] - __bfloat162float(h[k]);
            }
            *reinterpret_cast<uint4 *>(s.dst + p * s.plane + i) = *reinterpret_cast<const uint4 *>(h);
        }
    }
}

// The rows operand (x) and a second one: rows too, or the weights of `groups` groups.
cudaError_t split_planes(const void *x, void *px, int64_t x_elems, const void *w, void *pw, int64_t w_elems,
                         int64_t groups, bool skip, const Ranges &ranges, DevStatus *status, cudaStream_t stream)
{
    const Split a{static_cast<const float *>(x), static_cast<__nv_bfloat16 *>(px), x_elems, x_elems, 1, false};
    const Split b{static_cast<const float *>(w), static_cast<__nv_bfloat16 *>(pw), w_elems, groups * w_elems, groups, skip};
    const int64_t blocks = std::min(a.chunks() + groups * b.chunks(), 16 * (int64_t)device_sm_count());
    split_planes_kernel<<<(unsigned)std::max<int64_t>(1, blocks), 256, 0, stream>>>(a, b, ranges, status);
    return cudaGetLastError();
}

size_t plane_bytes(int64_t elems) { return ((size_t)elems * kPlanes * 2 + 255) & ~size_t(255); }

// ---- launches --------------------------------------------------------------

// The widest tile: of fp32's planes two slices fit the ring with 128 columns.
constexpr int kWidest = 256, kWidestSum = 128;
int widest(int dtype) { return dtype == SPMM_F32 ? kWidestSum : kWidest; }

// Columns per tile (a multiple of 16 of at most `most`): the cut into equal
// tiles with the least turns x time.  A 64-deep slice of a tile takes about
// as long as 70 + bn columns (0.19 us at 64, 0.46 us at 256): its rows are
// read however narrow it is.
int tile_columns(int64_t row_tiles, int64_t width, int most)
{
    const int64_t sms = device_sm_count();
    int best = 0;
    int64_t least = INT64_MAX;
    for (int64_t n = (width + most - 1) / most; n <= (width + 63) / 64; ++n) {
        const int64_t step = n > 1 ? 32 : 16;   // a tile is stored 32 columns at a time
        const int64_t bn = ((width + n - 1) / n + step - 1) / step * step;
        const int64_t cost = (row_tiles * n + sms - 1) / sms * (bn + 70);
        if (cost < least) {
            least = cost;
            best = (int)bn;
        }
        if (n > 64 && bn <= 128) break;   // very wide outputs: narrower tiles gain nothing more
    }
    return best;
}

void set_types(tc::GemmArgs &g, int dtype)
{
    const bool f32 = dtype == SPMM_F32;
    g.bf16 = f32 || dtype == SPMM_BF16;
    g.out_type = f32 ? tc::kOutF32 : g.bf16 ? tc::kOutBf16 : tc::kOutF16;
}

template <int BN, bool PAIR = false>
cudaError_t rows_tc(const GroupedLaunch &a, const void *x, const void *w, tc::GemmArgs &g, int64_t row_tiles,
                    cudaStream_t stream)
{
    tc::Maps m;
    const int64_t planes = a.dtype == SPMM_F32 ? kPlanes : 1, groups = std::max<int64_t>(a.groups, 1);
    const int64_t tiles = row_tiles * ((g.n + g.bn - 1) / g.bn);
    const int cols = PAIR ? BN / 2 : g.bn;   // of the weight that a block brings in
    if (!tc::make_map(&m.a, x, g.k, a.rows, planes, g.k, a.rows * g.k, tc::kBM, g.bf16) ||
        !(a.transposed ? tc::make_map(&m.b, w, a.N, a.K, planes * groups, a.N, a.K * a.N, cols, g.bf16)
                       : tc::make_mn_map(&m.b, &g.blocked_b, w, a.N, a.K, planes * groups, a.N, a.K * a.N, cols,
                                         g.bf16)) ||
        !tc::make_out_map(&m.o, a.out, g.n, a.rows, 1, g.n, 0, g.out_type))
        return cudaErrorInvalidValue;
    m.p = m.o;
    if constexpr (BN <= kWidestSum)
        if (a.dtype == SPMM_F32)
            return a.transposed ? tc::launch_gemm<tc::kRows, BN, false, false, tc::kStoreSum>(m, g, tiles, stream)
                                : tc::launch_gemm<tc::kRows, BN, false, true, tc::kStoreSum>(m, g, tiles, stream);
    return a.transposed ? tc::launch_gemm<tc::kRows, BN, false, false, tc::kStore, PAIR>(m, g, tiles, stream)
                        : tc::launch_gemm<tc::kRows, BN, false, true, tc::kStore, PAIR>(m, g, tiles, stream);
}

// Row tiles, at most: every group can end in a partial one; the rows outside
// the groups too.
int64_t row_tiles_of(const GroupedLaunch &a, int height)
{
    return std::min(a.rows, (a.rows + height - 1) / height + a.groups + 1);
}

// Whether pairs of blocks take tiles of 256 rows.  They pay where the products
// bound the kernel and groups are long enough that their last tile's missing
// rows do not matter: 65536 rows in 64 groups, K = 1024, N = 2048, bf16, 244 us
// alone and 212 us in pairs with even groups, 253 and 236 us with uneven ones;
// 100003 rows of 46 groups, K = 128, N = 256 (bound by memory) 18 and 22 us.
// A weight gradient gained almost nothing (274 and 272 us) and has no such form.
bool pair_rows(const GroupedLaunch &a, const tc::GemmArgs &g)
{
    return a.dtype != SPMM_F32 && g.k >= 512 && g.n % 256 == 0 && a.rows >= 512 * std::max<int64_t>(a.groups, 1) &&
           a.rows / 256 * (g.n / 256) >= 2 * device_sm_count();
}

// Rows of one part of a weight gradient.  A group's rows are one reduction
// unless it would keep one SM busy for longer than the others together: parts
// of two thirds of an SM's share of the work end within about that much of
// each other.  More and smaller parts cost more than they even out, since
// each stores its tiles in fp32 and they are read again to be added; measured
// with a sixth, two thirds and the whole of the share: 65537 uneven rows of 64
// groups, K = 1024, N = 2048 413, 331 and 326 us; of 64 even groups, K = N =
// 512 122, 64 and 64 us; 65536 rows of 8 groups 78, 61 and 83 us.  The least
// rows that pay: 512, in fp32 (six products of each) 384 (4000 rows of 3
// groups, K = N = 256: 35 us with 1024, 25 us; 20000 rows of 8 groups, K = N =
// 128: 43 and 35 us; 20011 rows of 8 groups, K = 256, N = 264: 55 and 57 us).
//
// At most 16384 rows, whatever the share: the tensor core truncates into its
// accumulator, up to 2^-22 of what it holds in a step of 16 rows and always
// towards zero, so over a part of products of one sign up to 2^-13 of the sum
// is lost (measured 1e-4).  One group of 2^20 rows, K = N = 2048, fp16, was
// 3.4e-3 too small in parts of 604544 rows, seven roundings to fp16.  The
// price, where parts were longer: 65536 rows of that group 0.41 -> 0.55 ms,
// 2^20 rows 6.06 -> 6.21 ms.
constexpr int64_t kLongestPart = 16384;
int64_t weight_grad_part(int64_t rows, int64_t K, int64_t N, int bn, int dtype)
{
    const int64_t tiles = ((K + tc::kBM - 1) / tc::kBM) * ((N + bn - 1) / bn);
    const int64_t part = rows * tiles * 2 / (3 * device_sm_count());
    return (std::min(kLongestPart, std::max<int64_t>(dtype == SPMM_F32 ? 384 : 512, part)) + 63) & ~int64_t(63);
}

// Equal tiles of the greatest width: the reduction is cut where there are
// too few of them, so they need not be narrower.
int weight_grad_columns(int64_t N, int dtype)
{
    const int most = widest(dtype);
    const int64_t n = (N + most - 1) / most;
    const int64_t step = n > 1 ? 32 : 16;   // a tile is stored 32 columns at a time
    return (int)(((N + n - 1) / n + step - 1) / step * step);
}

// Groups of several parts have more than `part` rows each, and no more than
// one part beyond the whole ones in their rows.
int64_t weight_grad_slots(int64_t rows, int64_t groups, int64_t K, int64_t N, int dtype)
{
    const int64_t part = weight_grad_part(rows, K, N, weight_grad_columns(N, dtype), dtype), whole = rows / part;
    return rows <= part ? 0 : whole + std::min(groups, whole);
}

// Adds the parts of each group that has several, in their order.
template <typename T>
__global__ void __launch_bounds__(256) add_parts_kernel(const float *parts, T *out, int64_t elems, int64_t part_rows,
                                                        int64_t slots, Ranges ranges, DevStatus *status)
{
    __shared__ int64_t before;
    tc::wait_for_earlier_kernels();
    for (int64_t g = blockIdx.y; g < ranges.groups; g += gridDim.y) {
        auto parts_of = [&](int64_t group) {
            int64_t b, e;
            segment_rows(ranges, group + 1, &b, &e, status);
            const int64_t n = (e - b + part_rows - 1) / part_rows;
            return n > 1 ? n : 0;
        };
        const int64_t n = parts_of(g);
        if (n == 0) continue;   // the same for the whole block
        if (threadIdx.x < 32) {   // the parts of the groups before g
            int64_t sum = 0;
            for (int64_t i = threadIdx.x; i < g; i += 32) sum += parts_of(i);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (threadIdx.x == 0) before = sum;
        }
        __syncthreads();
        const int64_t first = before;
        __syncthreads();
        if (first + n > slots) continue;
        for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < elems; i += (int64_t)gridDim.x * 1024) {
            float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
            for (int64_t p = 0; p < n; ++p) {
                const float4 v = __ldcs(reinterpret_cast<const float4 *>(parts + (first + p) * elems + i));
                s.x += v.x; s.y += v.y; s.z += v.z; s.w += v.w;
            }
            T *o = out + g * elems + i;
            if constexpr (sizeof(T) == 4) {
                *reinterpret_cast<float4 *>(o) = s;
            } else {
                __align__(8) T h[4] = {elem_of<T>(s.x), elem_of<T>(s.y), elem_of<T>(s.z), elem_of<T>(s.w)};
                *reinterpret_cast<uint2 *>(o) = *reinterpret_cast<const uint2 *>(h);
            }
        }
    }
}

template <typename T> cudaError_t add_parts(const GroupedLaunch &a, const float *parts, const tc::GemmArgs &g, cudaStream_t stream)
{
    const int64_t elems = a.K * a.N;
    const int64_t per = std::max<int64_t>(1, 16 * device_sm_count() / a.groups);
    const unsigned blocks = (unsigned)std::min((elems + 1023) / 1024, per);
    const dim3 grid(blocks, (unsigned)std::min<int64_t>(a.groups, 65535));
    return tc::launch_overlapped(add_parts_kernel<T>, grid, 1, 256, 0, stream, parts, static_cast<T *>(a.out), elems,
                                 g.part_rows, g.part_slots, g.ranges, a.status);
}

template <int BN>
cudaError_t weight_grad_tc(const GroupedLaunch &a, const void *x, const void *dy, float *parts, tc::GemmArgs &g,
                           cudaStream_t stream)
{
    tc::Maps m;
    const int64_t planes = a.dtype == SPMM_F32 ? kPlanes : 1, rows = std::max<int64_t>(a.rows, 1);
    if (!tc::make_mn_map(&m.a, &g.blocked_a, x, a.K, rows, planes, a.K, rows * a.K, tc::kBM, g.bf16) ||
        !tc::make_mn_map(&m.b, &g.blocked_b, dy, a.N, rows, planes, a.N, rows * a.N, g.bn, g.bf16) ||
        !tc::make_out_map(&m.o, a.out, a.N, a.K, a.groups, a.N, a.K * a.N, g.out_type))
        return cudaErrorInvalidValue;
    m.p = m.o;
    if (g.part_slots > 0 && !tc::make_out_map(&m.p, parts, a.N, a.K, g.part_slots, a.N, a.K * a.N, tc::kOutF32))
        return cudaErrorInvalidValue;
    const int64_t tiles = (a.groups + a.rows / g.part_rows) * ((a.K + tc::kBM - 1) / tc::kBM) *
                          ((a.N + g.bn - 1) / g.bn);
    if constexpr (BN <= kWidestSum)
        if (a.dtype == SPMM_F32)
            return tc::launch_gemm<tc::kRagged, BN, true, true, tc::kStoreSum>(m, g, tiles, stream);
    return tc::launch_gemm<tc::kRagged, BN, true, true, tc::kStore>(m, g, tiles, stream);
}

}  // namespace

size_t grouped_rows_workspace(int64_t rows, int64_t groups, int64_t K, int64_t N, bool transposed, int dtype)
{
    if (dtype != SPMM_F32) return 0;
    return plane_bytes(rows * (transposed ? N : K)) + plane_bytes(groups * K * N);
}

cudaError_t launch_grouped_rows(const GroupedLaunch &a, void *workspace, cudaStream_t stream)
{
    tc::GemmArgs g{};
    g.ranges = ranges_of(a);
    g.n = a.transposed ? a.K : a.N;
    g.k = a.transposed ? a.N : a.K;
    g.out = a.out;
    g.ldo = g.n;
    g.status = a.status;
    set_types(g, a.dtype);
    const void *x = a.x, *w = a.groups > 0 ? a.w : a.x;   // no group: the weight is never read
    if (a.dtype == SPMM_F32) {
        char *px = static_cast<char *>(workspace), *pw = px + plane_bytes(a.rows * g.k);
        const cudaError_t e = split_planes(x, px, a.rows * g.k, a.w, pw, a.K * a.N, a.groups, true, g.ranges, a.status,
                                           stream);
        if (e != cudaSuccess) return e;
        x = px;
        w = a.groups > 0 ? pw : px;
        g.za = 1;
        g.zb = (int)a.groups;
    }
    if (pair_rows(a, g)) {
        g.bn = 256;
        return rows_tc<256, true>(a, x, w, g, row_tiles_of(a, 2 * tc::kBM), stream);
    }
    const int64_t row_tiles = row_tiles_of(a, tc::kBM);
    g.bn = tile_columns(row_tiles, g.n, widest(a.dtype));
    if (g.bn <= 64) return rows_tc<64>(a, x, w, g, row_tiles, stream);
    if (g.bn <= 128) return rows_tc<128>(a, x, w, g, row_tiles, stream);
    return rows_tc<256>(a, x, w, g, row_tiles, stream);
}

size_t grouped_weight_grad_workspace(int64_t rows, int64_t groups, int64_t K, int64_t N, int dtype)
{
    const size_t parts = (size_t)weight_grad_slots(rows, groups, K, N, dtype) * K * N * sizeof(float);
    return parts + (dtype == SPMM_F32 ? plane_bytes(rows * K) + plane_bytes(rows * N) : 0);
}

cudaError_t launch_grouped_weight_grad(const GroupedLaunch &a, void *workspace, cudaStream_t stream)
{
    tc::GemmArgs g{};
    g.ranges = ranges_of(a);
    g.m = a.K;
    g.n = a.N;
    g.out = a.out;
    g.ldo = a.N;
    g.out_batch = a.K * a.N;
    g.status = a.status;
    set_types(g, a.dtype);
    g.bn = weight_grad_columns(a.N, a.dtype);
    g.part_rows = weight_grad_part(a.rows, a.K, a.N, g.bn, a.dtype);
    const int64_t slots = weight_grad_slots(a.rows, a.groups, a.K, a.N, a.dtype);
    const void *x = a.rows > 0 ? a.x : a.out, *dy = a.rows > 0 ? a.w : a.out;   // no rows: never read
    char *ws = static_cast<char *>(workspace);
    if (a.dtype == SPMM_F32 && a.rows > 0) {
        char *px = ws, *pdy = px + plane_bytes(a.rows * a.K);
        ws = pdy + plane_bytes(a.rows * a.N);
        const cudaError_t e = split_planes(x, px, a.rows * a.K, dy, pdy, a.rows * a.N, 1, false, g.ranges, a.status,
                                           stream);
        if (e != cudaSuccess) return e;
        x = px;
        dy = pdy;
        g.za = g.zb = 1;
    }
    float *parts = reinterpret_cast<float *>(ws);
    g.part_slots = slots;
    cudaError_t e;
    if (g.bn <= 64) e = weight_grad_tc<64>(a, x, dy, parts, g, stream);
    else if (g.bn <= 128) e = weight_grad_tc<128>(a, x, dy, parts, g, stream);
    else e = weight_grad_tc<256>(a, x, dy, parts, g, stream);
    if (e != cudaSuccess || slots == 0) return e;
    switch (a.dtype) {
        case SPMM_F16: return add_parts<__half>(a, parts, g, stream);
        case SPMM_BF16: return add_parts<__nv_bfloat16>(a, parts, g, stream);
        default: return add_parts<float>(a, parts, g, stream);
    }
}

}  // namespace spmmb
