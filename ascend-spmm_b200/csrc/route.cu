// Routing of rows to experts.
//
//   s = softmax(x) or sigmoid(x) over a row's experts,  c = s + bias
//   groups: those with the largest sums of their `group_best` largest c are
//           kept (`top_groups` of them); only their experts can be chosen
//   experts: the k largest c, in descending order, the lowest index first
//           among equal ones;  weights: w = s[chosen], divided by their sum
//           + 1e-20 with `renormalize`, times `scale`
//   backward, with g = scale * dw and S the sum:
//           d = renormalized ? (g - sum(g s) / S) / S : g        (chosen ones)
//           dx = s (d - sum(d s)) (softmax),  d s (1 - s) (sigmoid)
//
// A warp owns a row, lane l the experts l * VPL .. + VPL - 1 in registers.
//
// The choice is what 64-bit scores give, from 32-bit ones: where two values
// that the choice tells apart (a pick and the next one, the last group kept
// and the best one left out) are closer than their error bounds, the warp
// decides the row again in 64 bits.  Without a bias the scores grow with the
// logits, which are then compared as they are (exactly).
//
// NaN counts as the lowest value in every choice; a row whose logits are all
// -infinity gets zero weights.
#include <algorithm>

#include "../../include/spmm_b200.h"
#include "common.cuh"
#include "engine.h"
#include "layer.cuh"
#include "layer.h"

namespace spmmb {

namespace {

constexpr unsigned kFull = 0xffffffffu;
constexpr int kNone = INT32_MIN;             // taken, or not a candidate
constexpr int kNanKey = INT32_MIN + 64;      // below every number's key, above kNone; the low bits order NaNs by index
constexpr long long kNone64 = INT64_MIN;

__device__ __forceinline__ int warp_max(int v) { return __reduce_max_sync(kFull, v); }
template <typename F> __device__ __forceinline__ F warp_sum(F v)
{
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}

// Integers in the order of the floats (-0 as 0), NaN below all.
__device__ __forceinline__ int order_key(float f)
{
    const int b = __float_as_int(f + 0.f);
    return isnan(f) ? kNanKey : b ^ ((b >> 31) & 0x7fffffff);
}
__device__ __forceinline__ float key_value(int k) { return __int_as_float(k ^ ((k >> 31) & 0x7fffffff)); }
__device__ __forceinline__ long long order_key(double d)
{
    const long long b = __double_as_longlong(d + 0.0);
    return isnan(d) ? kNone64 + 1 : b ^ ((b >> 63) & INT64_MAX);
}

// Largest of the lanes' values; NaN only where all are.
__device__ __forceinline__ float warp_max(float v)
{
    const int k = warp_max(order_key(v));
    return k == kNanKey ? NAN : key_value(k);
}

// Descending order (a merge network of pairs: Batcher 1968).
template <int N> __device__ __forceinline__ void sort_descending(int (&v)[N])
{
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int k = p; k >= 1; k /= 2)
#pragma unroll
            for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; ++i)
                    if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                        const int a = v[i + j], b = v[i + j + k];
                        v[i + j] = max(a, b);
                        v[i + j + k] = min(a, b);
                    }
}

// The largest and the lowest lane that has it.
__device__ __forceinline__ long long warp_best(long long v, int *lane)
{
    long long best = v;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
        const long long u = __shfl_xor_sync(kFull, best, o);
        best = u > best ? u : best;
    }
    *lane = __ffs(__ballot_sync(kFull, v == best)) - 1;
    return best;
}

struct RouteArgs {
    const void *logits;
    const float *bias;      // may be null
    float *weights;         // [tokens, k]
    int *experts;           // [tokens, k]
    int64_t tokens;
    int n, k;               // experts, chosen
    int groups, top_groups, group_best;
    bool sigmoid, renormalize;
    float scale;
};

// VPL values of a lane from `at` on; those past the row's end are `fill`.
template <typename T, int VPL, bool VEC>
__device__ __forceinline__ void load_lane(const T *row, int at, int n, float fill, float (&v)[VPL])
{
    if constexpr (VEC) {
        constexpr int kBytes = VPL * (int)sizeof(T) < 16 ? VPL * (int)sizeof(T) : 16, kElems = kBytes / (int)sizeof(T);
        using V = std::conditional_t<kBytes == 16, uint4, std::conditional_t<kBytes == 8, uint2, std::conditional_t<kBytes == 4, unsigned, unsigned short>>>;
#pragma unroll
        for (int c = 0; c < VPL / kElems; ++c) {
            if (at + c * kElems < n) {   // n is a multiple of kElems
                const V raw = __ldg(reinterpret_cast<const V *>(row + at) + c);
                const T *e = reinterpret_cast<const T *>(&raw);
#pragma unroll
                for (int i = 0; i < kElems; ++i) v[c * kElems + i] = elem_f32<T>(e[i]);
            } else {
#pragma unroll
                for (int i = 0; i < kElems; ++i) v[c * kElems + i] = fill;
            }
        }
    } else {
#pragma unroll
        for (int j = 0; j < VPL; ++j) v[j] = at + j < n ? elem_f32<T>(row[at + j]) : fill;
    }
}

// exp(x - max) of a row; a row of -infinities has zeros.
__device__ __forceinline__ float safe_max(float m) { return m == -INFINITY ? 0.f : m; }

// ---- the row in 64 bits ------------------------------------------------------
// Returns lane p's pick (p < k).
template <typename T, int VPL> __device__ __noinline__ int choose_exactly(const RouteArgs &a, const T *row, float mx)
{
    const int lane = threadIdx.x & 31;
    const bool by_logit = !a.bias && (a.groups == a.top_groups || a.group_best == 1);
    double c[VPL];
    double z = 0;
    for (int j = 0; j < VPL; ++j) {
        const int i = lane * VPL + j;
        const double x = i < a.n ? (double)elem_f32<T>(row[i]) : -INFINITY;
        if (by_logit) c[j] = x;
        else if (a.sigmoid) c[j] = 1 / (1 + exp(-x));
        else z += c[j] = exp(x - (double)mx);
    }
    if (!by_logit && !a.sigmoid) {
        z = warp_sum(z);
        for (int j = 0; j < VPL; ++j) c[j] = z == 0 ? 0 : c[j] / z;
    }
    if (a.bias)
        for (int j = 0; j < VPL; ++j)
            if (lane * VPL + j < a.n) c[j] += (double)a.bias[lane * VPL + j];
    long long key[VPL];
    for (int j = 0; j < VPL; ++j) key[j] = lane * VPL + j < a.n ? order_key(c[j]) : kNone64;
    if (a.top_groups < a.groups) {
        const int per = a.n / a.groups;
        long long mine = kNone64;
        for (int g = 0; g < a.groups; ++g) {
            double sum = 0;
            long long above = INT64_MAX;   // the group's picks so far are those above (above, first)
            int first = -1;
            for (int b = 0; b < a.group_best; ++b) {
                long long best = kNone64;
                int at = -1;
                for (int j = 0; j < VPL; ++j) {
                    const int i = lane * VPL + j;
                    if (i < g * per || i >= (g + 1) * per || key[j] > above || (key[j] == above && i <= first)) continue;
                    if (key[j] > best) {
                        best = key[j];
                        at = j;
                    }
                }
                int winner;
                above = warp_best(best, &winner);
                const double v = __shfl_sync(kFull, at >= 0 ? c[at] : 0.0, winner);
                first = __shfl_sync(kFull, lane * VPL + at, winner);
                sum += v;
            }
            if (lane == g) mine = order_key(sum);
        }
        int rank = 0;
        for (int h = 0; h < a.groups; ++h) {
            const long long other = __shfl_sync(kFull, mine, h);
            rank += other > mine || (other == mine && h < lane);
        }
        const unsigned kept = __ballot_sync(kFull, lane < a.groups && rank < a.top_groups);
        for (int j = 0; j < VPL; ++j)
            if (lane * VPL + j < a.n && !(kept >> ((lane * VPL + j) / per) & 1u)) key[j] = kNone64;
    }
    int pick = 0;
    for (int p = 0; p < a.k; ++p) {
        long long best = kNone64;
        int at = 0;
        for (int j = 0; j < VPL; ++j)
            if (key[j] > best) {
                best = key[j];
                at = j;
            }
        int winner;
        warp_best(best, &winner);
        if (lane == winner) key[at] = kNone64;
        at = __shfl_sync(kFull, at, winner);
        if (lane == p) pick = winner * VPL + at;
    }
    return pick;
}

// Whether two values that the choice tells apart are closer than their
// errors.  A 32-bit score is off by less than 2^-21 of the row's largest, its
// sum with a bias (or of two) by 2^-23 of itself, and its key has lost
// `lost` bits.
__device__ __forceinline__ bool too_close(float hi, float lo, float largest, float rel)
{
    return !(hi - lo > 0x1p-19f * largest + rel * fmaxf(fabsf(hi), fabsf(lo)));   // true for infinities, too
}

// Blocks of an SM: rows are handled in a long chain of dependent steps, so the
// more warps take turns the better.
constexpr int route_blocks(int vpl) { return vpl <= 2 ? 8 : vpl == 4 ? 6 : vpl == 8 ? 5 : vpl == 16 ? 4 : 2; }

template <typename T, int VPL, bool VEC>
__global__ void __launch_bounds__(256, route_blocks(VPL)) route_kernel(const RouteArgs a)
{
    __shared__ int chosen[8][kMostChosen + 1];
    constexpr int kLow = VPL - 1;   // bits of a key that hold the (reversed) place in the lane
    const int lane = threadIdx.x & 31, n = a.n;
    const int first = lane * VPL;
    const bool grouped = a.top_groups < a.groups;
    const bool by_logit = !a.bias && (!grouped || a.group_best == 1);
    // groups that are whole lanes, a power of two of them
    const int per = n / a.groups, lanes = per / VPL;
    const bool by_lanes = per % VPL == 0 && (lanes & (lanes - 1)) == 0 && lanes <= 32;
    int *const picks = chosen[threadIdx.x / 32];
    const int64_t step = (int64_t)gridDim.x * (blockDim.x / 32);
    for (int64_t t = (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32; t < a.tokens; t += step) {
        const T *row = static_cast<const T *>(a.logits) + t * n;
        float x[VPL];
        load_lane<T, VPL, VEC>(row, first, n, -INFINITY, x);
        float mx = 0.f, inv = 1.f;
        float c[VPL];   // the values to choose by
        if (!a.sigmoid) {
            float m = -INFINITY;
#pragma unroll
            for (int j = 0; j < VPL; ++j) m = fmaxf(m, x[j]);
            mx = safe_max(warp_max(m));
            float z = 0.f;
#pragma unroll
            for (int j = 0; j < VPL; ++j) z += c[j] = __expf(x[j] - mx);
            z = warp_sum(z);
            inv = z == 0.f ? 0.f : 1.f / z;
#pragma unroll
            for (int j = 0; j < VPL; ++j) c[j] *= inv;
        } else if (!by_logit) {
#pragma unroll
            for (int j = 0; j < VPL; ++j) c[j] = __fdividef(1.f, 1.f + __expf(-x[j]));
        }
        if (by_logit) {
#pragma unroll
            for (int j = 0; j < VPL; ++j) c[j] = x[j];
        } else if (a.bias) {
#pragma unroll
            for (int j = 0; j < VPL; ++j)
                if (first + j < n) c[j] += __ldg(a.bias + first + j);
        }
        int key[VPL];
#pragma unroll
        for (int j = 0; j < VPL; ++j)
            key[j] = first + j < n ? (order_key(c[j]) & ~kLow) | (kLow - j) : kNone;

        // by logits: 16-bit ones are compared exactly, 32-bit ones where their keys differ above the low bits
        const float largest = by_logit ? 0.f : a.sigmoid ? 1.f : inv;
        const float rel = by_logit ? VPL * 0x1p-23f : 0x1p-21f + VPL * 0x1p-22f;
        const bool exact = by_logit && (sizeof(T) == 2 || VPL == 1);
        bool again = false;
        if (grouped) {
            // lane g: the score of group g
            int mine = kNone;
            auto sum_of = [&](int top, int next) {   // of two keys without their low bits
                return order_key((top == kNanKey ? NAN : key_value(top)) + (next == kNanKey ? NAN : key_value(next)));
            };
            if (by_lanes) {
                int b1 = kNone, b2 = kNone;
#pragma unroll
                for (int j = 0; j < VPL; ++j) {
                    b2 = max(b2, min(b1, key[j]));
                    b1 = max(b1, key[j]);
                }
                b1 &= ~kLow;
                b2 &= ~kLow;
                for (int o = 1; o < lanes; o <<= 1) {
                    const int o1 = __shfl_xor_sync(kFull, b1, o), o2 = __shfl_xor_sync(kFull, b2, o);
                    b2 = max(min(b1, o1), max(b2, o2));
                    b1 = max(b1, o1);
                }
                const int score = a.group_best == 2 ? sum_of(b1, b2) : b1;
                mine = __shfl_sync(kFull, score, min(lane, a.groups - 1) * lanes);
                if (lane >= a.groups) mine = kNone;
            } else {
                for (int g = 0; g < a.groups; ++g) {
                    int b1 = kNone, b2 = kNone;
#pragma unroll
                    for (int j = 0; j < VPL; ++j) {
                        const int i = first + j, v = i >= g * per && i < (g + 1) * per ? key[j] : kNone;
                        b2 = max(b2, min(b1, v));
                        b1 = max(b1, v);
                    }
                    const int top = warp_max(b1);
                    int score = top & ~kLow;
                    if (a.group_best == 2) {
                        const int winner = __ffs(__ballot_sync(kFull, b1 == top)) - 1;
                        score = sum_of(score, warp_max(lane == winner ? b2 : b1) & ~kLow);
                    }
                    if (lane == g) mine = score;
                }
            }
            int rank = 0;
            for (int h = 0; h < a.groups; ++h) {
                const int other = __shfl_sync(kFull, mine, h);
                rank += other > mine || (other == mine && h < lane);
            }
            const bool stays = lane < a.groups && rank < a.top_groups;
            const unsigned kept = __ballot_sync(kFull, stays);
            const int last = __reduce_min_sync(kFull, stays ? mine : INT32_MAX);
            const int out = warp_max(stays ? kNone : mine);
            if (!exact) again = too_close(key_value(last), key_value(out), largest, 2 * rel);
            if (by_lanes) {
                if (first < n && !(kept >> (lane / lanes) & 1u)) {
#pragma unroll
                    for (int j = 0; j < VPL; ++j) key[j] = kNone;
                }
            } else {
#pragma unroll
                for (int j = 0; j < VPL; ++j)
                    if (first + j < n && !(kept >> ((first + j) / per) & 1u)) key[j] = kNone;
            }
        }
        // each lane's keys in descending order: a pick is the largest of the lanes' first ones
        sort_descending(key);
        int before = 0;
        for (int p = 0; p <= a.k && !again; ++p) {
            const int best = warp_max(key[0] & ~kLow);   // the place in the lane only tells a lane's own values apart
            if (p > 0 && !exact && best != kNone)
                again = too_close(key_value(before), key_value(best), largest, rel);
            before = best;
            if (lane == __ffs(__ballot_sync(kFull, (key[0] & ~kLow) == best)) - 1) {
                picks[p] = first + kLow - (key[0] & kLow);
#pragma unroll
                for (int j = 0; j + 1 < VPL; ++j) key[j] = key[j + 1];
                key[VPL - 1] = kNone;
            }
        }
        __syncwarp();
        int pick = lane < a.k ? picks[lane] : 0;
        __syncwarp();
        if (again) pick = choose_exactly<T, VPL>(a, row, mx);

        const bool on = lane < a.k;
        float s = 0.f;
        if (on) {
            const float v = elem_f32<T>(row[pick]);
            s = a.sigmoid ? 1.f / (1.f + expf(-v)) : expf(v - mx) * inv;
        }
        float w = s;
        if (a.renormalize) w = s / (warp_sum(s) + 1e-20f);
        if (on) {
            a.weights[t * a.k + lane] = w * a.scale;
            a.experts[t * a.k + lane] = pick;
        }
    }
}

struct RouteBackwardArgs {
    const void *logits;
    const int *experts;
    const float *grad;      // [tokens, k]
    void *dlogits;
    int64_t tokens;
    int n, k;
    bool sigmoid, renormalize;
    float scale;
    DevStatus *status;
};

// Lane l has the vectors l, l + 32, ... of the row (without vectors: elements).
template <typename T, int VPL, bool VEC> __global__ void __launch_bounds__(256) route_backward_kernel(const RouteBackwardArgs a)
{
    constexpr int kBytes = VEC ? (VPL * (int)sizeof(T) < 16 ? VPL * (int)sizeof(T) : 16) : (int)sizeof(T);
    constexpr int kElems = kBytes / (int)sizeof(T), kVectors = VPL / kElems;
    using V = std::conditional_t<kBytes == 16, uint4, std::conditional_t<kBytes == 8, uint2, std::conditional_t<kBytes == 4, unsigned, unsigned short>>>;
    const int lane = threadIdx.x & 31, n = a.n;
    const int64_t step = (int64_t)gridDim.x * (blockDim.x / 32);
    for (int64_t t = (int64_t)blockIdx.x * (blockDim.x / 32) + threadIdx.x / 32; t < a.tokens; t += step) {
        const T *row = static_cast<const T *>(a.logits) + t * n;
        T *out = static_cast<T *>(a.dlogits) + t * n;
        bool on = lane < a.k;
        int e = 0;
        float d = 0.f, xe = 0.f;
        if (on) {
            e = __ldg(a.experts + t * a.k + lane);
            d = __ldg(a.grad + t * a.k + lane) * a.scale;
            if (e < 0 || e >= n) {
                raise_status(a.status, SPMM_DEV_BAD_COLUMN, t * a.k + lane);
                on = false;
            } else {
                xe = elem_f32<T>(row[e]);
            }
        }
        float v[VPL], mx = 0.f, inv = 1.f;
        if (!a.sigmoid) {
            float m = -INFINITY;
#pragma unroll
            for (int c = 0; c < kVectors; ++c) {
                const int at = (c * 32 + lane) * kElems;   // n is a multiple of kElems
                V raw;
                if (at < n) raw = __ldg(reinterpret_cast<const V *>(row + at));
                const T *w = reinterpret_cast<const T *>(&raw);
#pragma unroll
                for (int i = 0; i < kElems; ++i) {
                    v[c * kElems + i] = at < n ? elem_f32<T>(w[i]) : -INFINITY;
                    m = fmaxf(m, v[c * kElems + i]);
                }
            }
            mx = safe_max(warp_max(m));
            float z = 0.f;
#pragma unroll
            for (int j = 0; j < VPL; ++j) z += v[j] = expf(v[j] - mx);
            z = warp_sum(z);
            inv = z == 0.f ? 0.f : 1.f / z;
        }
        const float s = !on ? 0.f : a.sigmoid ? 1.f / (1.f + expf(-xe)) : expf(xe - mx) * inv;
        if (!on) d = 0.f;
        if (a.renormalize) {
            const float total = warp_sum(s) + 1e-20f;
            d = (d - warp_sum(d * s) / total) / total;
        }
        float along = 0.f;   // softmax: sum of d s
        if (!a.sigmoid) along = warp_sum(on ? d * s : 0.f);
#pragma unroll
        for (int c = 0; c < kVectors; ++c) {
            const int at = (c * 32 + lane) * kElems;
            if (at >= n) break;
            V raw;
            T *w = reinterpret_cast<T *>(&raw);
#pragma unroll
            for (int i = 0; i < kElems; ++i) w[i] = elem_of<T>(a.sigmoid ? 0.f : -v[c * kElems + i] * inv * along);
            *reinterpret_cast<V *>(out + at) = raw;
        }
        __syncwarp();   // the chosen experts' values replace what the row got
        if (on) out[e] = elem_of<T>(a.sigmoid ? d * s * (1.f - s) : s * (d - along));
    }
}

// Calls f with the values per lane (a power of two) and whether rows are read in vectors.
template <typename T, typename F> cudaError_t by_width(int n, F f)
{
    auto run = [&](auto vpl) {
        constexpr int kVpl = decltype(vpl)::value;
        constexpr int kBytes = std::min(16, kVpl * (int)sizeof(T));
        return n * (int)sizeof(T) % kBytes == 0 ? f(vpl, std::true_type()) : f(vpl, std::false_type());
    };
    if (n <= 32) return run(std::integral_constant<int, 1>());
    if (n <= 64) return run(std::integral_constant<int, 2>());
    if (n <= 128) return run(std::integral_constant<int, 4>());
    if (n <= 256) return run(std::integral_constant<int, 8>());
    if (n <= 512) return run(std::integral_constant<int, 16>());
    return run(std::integral_constant<int, 32>());
}

template <typename F> cudaError_t by_type(int dtype, F f)
{
    switch (dtype) {
        case SPMM_F16: return f(__half());
        case SPMM_BF16: return f(__nv_bfloat16());
        default: return f(float());
    }
}

unsigned row_blocks(int64_t tokens)
{
    return (unsigned)std::max<int64_t>(1, std::min<int64_t>((tokens + 7) / 8, 32 * (int64_t)device_sm_count()));
}

}  // namespace

cudaError_t launch_route(const RouteLaunch &r, cudaStream_t stream)
{
    RouteArgs a{r.logits, r.bias, r.weights, r.experts, r.tokens, r.n, r.k, r.groups, r.top_groups, r.group_best,
                r.sigmoid, r.renormalize, r.scale};
    return by_type(r.dtype, [&](auto type) {
        using T = decltype(type);
        return by_width<T>(r.n, [&](auto vpl, auto vec) {
            route_kernel<T, decltype(vpl)::value, decltype(vec)::value><<<row_blocks(r.tokens), 256, 0, stream>>>(a);
            return cudaGetLastError();
        });
    });
}

cudaError_t launch_route_backward(const RouteLaunch &r, const float *grad, void *dlogits, DevStatus *status,
                                  cudaStream_t stream)
{
    RouteBackwardArgs a{r.logits, r.experts, grad, dlogits, r.tokens, r.n, r.k, r.sigmoid, r.renormalize, r.scale,
                        status};
    return by_type(r.dtype, [&](auto type) {
        using T = decltype(type);
        return by_width<T>(r.n, [&](auto vpl, auto vec) {
            route_backward_kernel<T, decltype(vpl)::value, decltype(vec)::value>
                <<<row_blocks(r.tokens), 256, 0, stream>>>(a);
            return cudaGetLastError();
        });
    });
}

}  // namespace spmmb
