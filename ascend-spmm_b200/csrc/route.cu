// Routing of rows to experts.
//
//   s = softmax(x) or sigmoid(x) over a row's experts,  c = s + bias
//   groups: those with the largest sums of their `group_best` largest c are
//           kept (`top_groups` of them); only their experts can be chosen
//   experts: the k largest c, in descending order, the lowest index first
//           among equal ones;  weights: w = s[chosen], divided by their sum
//           + 1e-20 with `renormalize`, times `scale`
//   backward, with g = scale * dw, S the sum and r = s / S:
//           u = renormalized ? r (g - sum(g r)) : g s           (chosen ones)
//           dx = u - s sum(u) (softmax),  u (1 - s) (sigmoid)
//
// A team of LANES lanes owns a row (a warp where it has more than 128
// experts), lane l the experts l * VPL .. + VPL - 1 in registers, each sorted
// by a network; a pick is then the largest of the lanes' first ones.
//
// The choice is what 64-bit scores give, from 32-bit ones: where two values
// that the choice tells apart (a pick and the next one, the last group kept
// and the best one left out) are closer than their error bounds, the warp
// decides the row again in 64 bits.  Where nothing is added to a score (no bias,
// no groups by sums of two) the logits are compared as they are, which is exact:
// the scores grow with them, also where 64 bits round two of them alike.
//
// NaN counts as the lowest value in every choice; a row whose logits are all
// -infinity gets zero weights.
//
// What bounds it: instructions (some 1000 a warp for a row of 256 experts in
// eight groups, eight picks), not the 4 bytes of a logit.  65537 such rows, fp32,
// sigmoid and bias: 82 us forward (11 us of memory; about 25 are scores, groups and
// bias, 20 the picks, 6 the 0.5 % of rows that are decided in 64 bits, the others
// are not told apart), 26 us backward (a sigmoid's reads the sectors of the chosen
// logits only: some 84 MB, 13 us of memory; a chain of loads, expert and then logit,
// and issue slots 62 % busy); 16411 rows of 64 experts, bf16, six picks: 6.5 and
// 6.3 us.  Rows all of whose logits are equal, which 64 bits decide one by one,
// are the worst: 65537 of 256 experts by softmax 144 us, where random ones take 56.
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
// Over the teams of LANES lanes, each by itself.
template <int LANES = 32, typename F> __device__ __forceinline__ F warp_sum(F v)
{
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}
template <int LANES> __device__ __forceinline__ int team_max(int v)
{
    if constexpr (LANES == 32) {
        return warp_max(v);
    } else {
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(kFull, v, o));
        return v;
    }
}
template <int LANES> __device__ __forceinline__ float team_max(float v)
{
#pragma unroll
    for (int o = LANES / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
    return v;
}

// Integers in the order of the floats (-0 as 0), NaN below all.
__device__ __forceinline__ int order_key(float f)
{
    const int b = __float_as_int(f + 0.f);
    return isnan(f) ? kNanKey : b ^ ((b >> 31) & 0x7fffffff);
}
// The same without a look at NaN and -0: positive NaNs above infinity, others below -infinity.
__device__ __forceinline__ int raw_key(float f)
{
    const int b = __float_as_int(f);
    return b ^ ((b >> 31) & 0x7fffffff);
}
constexpr int kInfKey = 0x7f800000, kMinusInfKey = (int)0x807fffff;
__device__ __forceinline__ float key_value(int k) { return __int_as_float(k ^ ((k >> 31) & 0x7fffffff)); }
__device__ __forceinline__ long long order_key(double d)
{
    const long long b = __double_as_longlong(d + 0.0);
    return isnan(d) ? kNone64 + 1 : b ^ ((b >> 63) & INT64_MAX);
}
__device__ __forceinline__ double key_value(long long k) { return __longlong_as_double(k ^ ((k >> 63) & INT64_MAX)); }

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

// The largest of 64-bit keys and the lowest lane that has it.
__device__ __forceinline__ long long warp_best(long long v, int *lane)
{
    const int hi = warp_max((int)(v >> 32));
    const unsigned lo = __reduce_max_sync(kFull, (int)(v >> 32) == hi ? (unsigned)v : 0u);
    const long long best = (long long)hi << 32 | lo;
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
template <typename T, int VPL, bool VEC, bool SHARED = false>
__device__ __forceinline__ void load_lane(const T *row, int at, int n, float fill, float (&v)[VPL])
{
    if constexpr (VEC) {
        constexpr int kBytes = VPL * (int)sizeof(T) < 16 ? VPL * (int)sizeof(T) : 16, kElems = kBytes / (int)sizeof(T);
        using V = std::conditional_t<kBytes == 16, uint4, std::conditional_t<kBytes == 8, uint2, std::conditional_t<kBytes == 4, unsigned, unsigned short>>>;
#pragma unroll
        for (int c = 0; c < VPL / kElems; ++c) {
            if (at + c * kElems < n) {   // n is a multiple of kElems
                const V *from = reinterpret_cast<const V *>(row + at) + c;
                const V raw = SHARED ? *from : __ldg(from);
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
// The whole warp; returns lane p's pick (p < k).  Few rows need it, but a
// kernel ends with its slowest warp: as short a chain as it can be.
template <typename T, int VPL> __device__ __noinline__ int choose_exactly(const RouteArgs &a, const T *row, float mx)
{
    const int lane = threadIdx.x & 31, first = lane * VPL;
    const bool by_logit = !a.bias && (a.groups == a.top_groups || a.group_best == 1);
    double c[VPL], z = 0;
#pragma unroll
    for (int j = 0; j < VPL; ++j) c[j] = first + j < a.n ? (double)elem_f32<T>(row[first + j]) : -INFINITY;
    if (!by_logit && a.sigmoid) {
#pragma unroll
        for (int j = 0; j < VPL; ++j) c[j] = 1 / (1 + exp(-c[j]));
    } else if (!by_logit) {
#pragma unroll
        for (int j = 0; j < VPL; ++j) z += c[j] = exp(c[j] - (double)mx);
        z = warp_sum(z);
#pragma unroll
        for (int j = 0; j < VPL; ++j) c[j] = z == 0 ? 0 : c[j] / z;
    }
    long long key[VPL];
#pragma unroll
    for (int j = 0; j < VPL; ++j) {
        if (a.bias && first + j < a.n) c[j] += (double)__ldg(a.bias + first + j);
        key[j] = first + j < a.n ? order_key(c[j]) : kNone64;
    }
    if (a.top_groups < a.groups) {
        const int per = a.n / a.groups, lanes = per / VPL;
        auto sum_of = [&](long long top, long long next) {
            return a.group_best == 2 ? order_key(key_value(top) + key_value(next)) : top;
        };
        auto join = [](long long &b1, long long &b2, int o) {
            const long long o1 = __shfl_xor_sync(kFull, b1, o), o2 = __shfl_xor_sync(kFull, b2, o);
            b2 = max(min(b1, o1), max(b2, o2));
            b1 = max(b1, o1);
        };
        long long mine = kNone64;   // lane g: the score of group g
        if (per % VPL == 0 && (lanes & (lanes - 1)) == 0) {
            long long b1 = kNone64, b2 = kNone64;
#pragma unroll
            for (int j = 0; j < VPL; ++j) {
                b2 = max(b2, min(b1, key[j]));
                b1 = max(b1, key[j]);
            }
            for (int o = 1; o < lanes; o <<= 1) join(b1, b2, o);
            mine = __shfl_sync(kFull, sum_of(b1, b2), min(lane, a.groups - 1) * lanes);
        } else {
            for (int g = 0; g < a.groups; ++g) {
                long long b1 = kNone64, b2 = kNone64;
#pragma unroll
                for (int j = 0; j < VPL; ++j) {
                    const long long v = first + j >= g * per && first + j < (g + 1) * per ? key[j] : kNone64;
                    b2 = max(b2, min(b1, v));
                    b1 = max(b1, v);
                }
                for (int o = 1; o < 32; o <<= 1) join(b1, b2, o);
                if (lane == g) mine = sum_of(b1, b2);
            }
        }
        int rank = 0;
#pragma unroll 4
        for (int h = 0; h < a.groups; ++h) {
            const long long other = __shfl_sync(kFull, mine, h);
            rank += other > mine || (other == mine && h < lane);
        }
        const unsigned kept = __ballot_sync(kFull, lane < a.groups && rank < a.top_groups);
#pragma unroll
        for (int j = 0; j < VPL; ++j)
            if (first + j < a.n && !(kept >> ((first + j) / per) & 1u)) key[j] = kNone64;
    }
    int pick = 0;
    for (int p = 0; p < a.k; ++p) {
        long long best = key[0];
        int at = 0;
#pragma unroll
        for (int j = 1; j < VPL; ++j)
            if (key[j] > best) {
                best = key[j];
                at = j;
            }
        int winner;
        warp_best(best, &winner);
#pragma unroll
        for (int j = 0; j < VPL; ++j)
            if (lane == winner && j == at) key[j] = kNone64;
        at = __shfl_sync(kFull, first + at, winner);
        if (lane == p) pick = at;
    }
    return pick;
}

// Whether two values that the choice tells apart may be closer than their
// errors.  A 32-bit score is off by at most 2^-21 of the row's largest one (of
// 1 for a sigmoid) for its exponential and the reciprocal, and, with a
// softmax, by its share of the sum's error, (VPL + 5) 2^-24; `score` is more
// than twice that.  A sum with the bias rounds by 2^-24 of itself, and a key has
// lost the bits that hold the place: `rel`.
__device__ __forceinline__ bool too_close(float hi, float lo, float score, float rel)
{
    return !(hi - lo > score + rel * fmaxf(fabsf(hi), fabsf(lo)));   // true for infinities, too
}

__device__ __forceinline__ float reciprocal(float x)   // within 2^-23 of itself
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// exp(x) within 2^-21 of itself (|x| log2(e) rounds by 2^-24 of it; where x is far from 0, exp(x) or, of a sigmoid, 1 is
// all that is left), 0 below 2^-126.
__device__ __forceinline__ float fast_exp(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x * 1.4426950408889634f));
    return y;
}

// Blocks of an SM: a row is a long chain of dependent steps, so the more warps take turns the better.
constexpr int route_blocks(int vpl) { return vpl == 8 ? 4 : vpl == 16 ? 3 : 2; }

// Calls f with this lane's share of the k choices.
template <int LANES, typename F> __device__ __forceinline__ void each_choice(int lane, int k, F f)
{
    if constexpr (LANES >= kMostChosen) {
        if (lane < k) f(lane);
    } else {
        for (int p = lane; p < k; p += LANES) f(p);
    }
}

template <typename T, int LANES, int VPL, bool VEC>
__global__ void __launch_bounds__(256, route_blocks(VPL)) route_kernel(const RouteArgs a)
{
    extern __shared__ __align__(16) unsigned char staged[];   // VEC: two turns' rows of each warp
    constexpr int kLow = VPL - 1;   // bits of a key that hold the (reversed) place in the lane
    constexpr int kTeams = 32 / LANES;
    constexpr unsigned kTeam = LANES == 32 ? kFull : (1u << LANES) - 1;
    __shared__ int s_pick[8][kTeams][kMostChosen + 1], s_key[8][kTeams][kMostChosen + 1], s_score[8][kTeams][kMostGroups];
    __shared__ float s_slack[8][kTeams][kMostGroups];
    const int warp = threadIdx.x / 32, lane = threadIdx.x % LANES, team = threadIdx.x % 32 / LANES, n = a.n;
    const int first = lane * VPL;
    const bool grouped = a.top_groups < a.groups;
    const bool by_logit = !a.bias && (!grouped || a.group_best == 1);
    // groups that are whole lanes, a power of two of them
    const int per = n / a.groups, lanes = per / VPL;
    const bool by_lanes = per % VPL == 0 && (lanes & (lanes - 1)) == 0;
    // by logits: 16-bit ones are compared exactly, 32-bit ones where their keys differ above the low bits
    const float rel = by_logit ? VPL * 0x1p-23f : 0x1p-21f + VPL * 0x1p-22f;
    const bool exact = by_logit && sizeof(T) == 2;
    // a warp's turn is kTeams rows, which lie together: the next turn's are on their way while this one's are worked on
    const int turn_bytes = kTeams * n * (int)sizeof(T);
    unsigned char *const buffers = staged + warp * 2 * turn_bytes;
    auto fetch = [&](int64_t t0, int buffer) {
        if constexpr (VEC) {
            const int64_t at = t0 * n * (int64_t)sizeof(T), end = a.tokens * n * (int64_t)sizeof(T);
            const unsigned to = (unsigned)__cvta_generic_to_shared(buffers + buffer * turn_bytes);
            for (int i = (threadIdx.x & 31) * 16; i < turn_bytes; i += 512)
                if (at + i < end)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;\n" ::"r"(to + i),
                                 "l"(static_cast<const unsigned char *>(a.logits) + at + i)
                                 : "memory");
            asm volatile("cp.async.commit_group;\n" ::: "memory");
        }
    };
    int *const picks = s_pick[warp][team], *const keys = s_key[warp][team], *const scores = s_score[warp][team];
    float *const slacks = s_slack[warp][team];
    const int64_t step = (int64_t)gridDim.x * 8 * kTeams;
    const int64_t start = ((int64_t)blockIdx.x * 8 + warp) * kTeams;
    if (start < a.tokens) fetch(start, 0);
    int buffer = 0;
    for (int64_t t0 = start; t0 < a.tokens; t0 += step, buffer ^= 1) {
        const int64_t t = min(t0 + team, a.tokens - 1);   // a team past the last row does it again and stores nothing
        const T *row = static_cast<const T *>(a.logits) + t * n;
        if constexpr (VEC) {
            fetch(t0 + step, buffer ^ 1);
            asm volatile("cp.async.wait_group 1;\n" ::: "memory");
            __syncwarp();
            row = reinterpret_cast<const T *>(buffers + buffer * turn_bytes) + (int)(t - t0) * n;
        }
        float c[VPL];   // the values to choose by
        load_lane<T, VPL, VEC, VEC>(row, first, n, -INFINITY, c);
        float mx = 0.f, inv = 1.f;
        if (!a.sigmoid) {
            float m = -INFINITY;
#pragma unroll
            for (int j = 0; j < VPL; ++j) m = fmaxf(m, c[j]);
            mx = safe_max(team_max<LANES>(m));
            float e[VPL], z = 0.f;
#pragma unroll
            for (int j = 0; j < VPL; ++j) z += e[j] = fast_exp(c[j] - mx);
            z = warp_sum<LANES>(z);
            inv = z == 0.f ? 0.f : reciprocal(z);
            if (!by_logit) {
#pragma unroll
                for (int j = 0; j < VPL; ++j) c[j] = e[j] * inv;
            }
        } else if (!by_logit) {
#pragma unroll
            for (int j = 0; j < VPL; ++j) c[j] = reciprocal(1.f + fast_exp(-c[j]));
        }
        if (a.bias) {
            float b[VPL];
            load_lane<float, VPL, VEC>(a.bias, first, n, 0.f, b);
#pragma unroll
            for (int j = 0; j < VPL; ++j) c[j] += b[j];
        }
        int key[VPL];
#pragma unroll
        for (int j = 0; j < VPL; ++j) key[j] = (raw_key(c[j] + 0.f) & ~kLow) | (kLow - j);   // the sum makes -0 a 0
        if (first + VPL > n) {
#pragma unroll
            for (int j = 0; j < VPL; ++j)
                if (first + j >= n) key[j] = kNone;
        }

        const float unsure_by = by_logit ? 0.f : (0x1p-19f + VPL * 0x1p-22f) * (a.sigmoid ? 1.f : inv);
        bool again = false;
        if (grouped) {
            // A group's score, and how far it may be off.  That goes by its terms, which can nearly cancel: each is off by at
            // most half of `unsure_by` and half of `rel` of itself, the sum's own rounding by 2^-24 of them.
            auto put = [&](int g, int top, int next) {
                const bool two = a.group_best == 2;
                const float v = key_value(top), w = two ? key_value(next) : 0.f;
                scores[g] = two ? raw_key(v + w) : top;
                slacks[g] = unsure_by + rel * (fabsf(v) + fabsf(w));
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
                if (lane % lanes == 0 && lane / lanes < a.groups) put(lane / lanes, b1, b2);
            } else {
                for (int g = 0; g < a.groups; ++g) {
                    int b1 = kNone, b2 = kNone;
#pragma unroll
                    for (int j = 0; j < VPL; ++j) {
                        const int i = first + j, v = i >= g * per && i < (g + 1) * per ? key[j] & ~kLow : kNone;
                        b2 = max(b2, min(b1, v));
                        b1 = max(b1, v);
                    }
#pragma unroll
                    for (int o = 1; o < LANES; o <<= 1) {
                        const int o1 = __shfl_xor_sync(kFull, b1, o), o2 = __shfl_xor_sync(kFull, b2, o);
                        b2 = max(min(b1, o1), max(b2, o2));
                        b1 = max(b1, o1);
                    }
                    if (lane == 0) put(g, b1, b2);
                }
            }
            __syncwarp();
            unsigned kept = 0;
            float low = INFINITY, high = -INFINITY;   // what the groups kept have at least, those left out at most
            for (int g = lane; g < a.groups; g += LANES) {
                const int mine = scores[g];
                const float score = key_value(mine), slack = slacks[g];
                int rank = 0;
                for (int h = 0; h < a.groups; ++h) {
                    const int other = scores[h];
                    rank += other > mine || (other == mine && h < g);
                }
                if (rank < a.top_groups) {
                    kept |= 1u << g;
                    low = fminf(low, score - slack);
                    again |= !exact && !(slack < INFINITY);   // its terms are not finite: nothing is known of its order
                } else {
                    high = fmaxf(high, score + slack);   // a cut -infinity is a NaN, which is the smaller one
                }
                again |= mine > kInfKey || mine < (kMinusInfKey & ~kLow);   // NaN
            }
            if constexpr (LANES == 32) {
                kept = __reduce_or_sync(kFull, kept);
                low = key_value(__reduce_min_sync(kFull, raw_key(low)));
                high = key_value(warp_max(raw_key(high)));
            } else {
#pragma unroll
                for (int o = LANES / 2; o > 0; o >>= 1) {
                    kept |= __shfl_xor_sync(kFull, kept, o);
                    low = fminf(low, __shfl_xor_sync(kFull, low, o));
                    high = fmaxf(high, __shfl_xor_sync(kFull, high, o));
                }
            }
            again |= !exact && !(low > high);
            if (by_lanes) {
                if (!(kept >> (lane / lanes) & 1u)) {
#pragma unroll
                    for (int j = 0; j < VPL; ++j) key[j] = kNone;
                }
            } else {
#pragma unroll
                for (int j = 0; j < VPL; ++j)
                    if (first + j < n && !(kept >> ((first + j) / per) & 1u)) key[j] = kNone;
            }
        }
        sort_descending(key);
        for (int p = 0; p <= a.k; ++p) {
            const int best = team_max<LANES>(key[0] & ~kLow);   // the place in the lane only tells a lane's own values apart
            const unsigned has = __ballot_sync(kFull, (key[0] & ~kLow) == best) >> (team * LANES) & kTeam;
            const bool winner = lane == __ffs(has) - 1;
            if (winner) {
                picks[p] = first + kLow - (key[0] & kLow);
                keys[p] = best;
            }
#pragma unroll
            for (int j = 0; j + 1 < VPL; ++j) key[j] = winner ? key[j + 1] : key[j];
            key[VPL - 1] = winner ? kNone : key[VPL - 1];
        }
        __syncwarp();
        // the row is decided in 64 bits where a pick and the next one are too close, and where a NaN was met
        each_choice<LANES>(lane, a.k, [&](int p) {
            const int mine = keys[p], next = keys[p + 1];
            again |= mine > kInfKey || mine < (kMinusInfKey & ~kLow);
            if (!exact && next != kNone) again |= too_close(key_value(mine), key_value(next), unsure_by, rel);
        });
        unsigned unsure = __ballot_sync(kFull, again);
        while (unsure) {
            const int who = (__ffs(unsure) - 1) / LANES;
            unsure &= ~(kTeam << (who * LANES));
            const T *its_row = static_cast<const T *>(a.logits) + min(t0 + who, a.tokens - 1) * n;
            const float its_mx = __shfl_sync(kFull, mx, who * LANES);
            const int pick = choose_exactly<T, (LANES * VPL + 31) / 32>(a, its_row, its_mx);
            if ((int)threadIdx.x % 32 < a.k) s_pick[warp][who][threadIdx.x % 32] = pick;
        }
        __syncwarp();
        auto score = [&](int p) {
            const float v = elem_f32<T>(row[picks[p]]);
            return a.sigmoid ? reciprocal(1.f + expf(-v)) : expf(v - mx) * inv;
        };
        const float own = lane < a.k ? score(lane) : 0.f;   // a row of few lanes has more of them: worked out again
        float factor = a.scale;
        if (a.renormalize) {
            float sum = own;
            if constexpr (LANES < kMostChosen)
                for (int p = lane + LANES; p < a.k; p += LANES) sum += score(p);
            factor *= reciprocal(warp_sum<LANES>(sum) + 1e-20f);
        }
        if (t0 + team < a.tokens)
            each_choice<LANES>(lane, a.k, [&](int p) {
                a.weights[t * a.k + p] = (p == lane ? own : score(p)) * factor;
                a.experts[t * a.k + p] = picks[p];
            });
        __syncwarp();   // the picks have been read
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
        // u: the gradient of log s; with renormalize its sum is g w' times what 1e-20 takes of the sum of the weights, which
        // as a difference would be rounding alone
        const float s = !on ? 0.f : a.sigmoid ? 1.f / (1.f + expf(-xe)) : expf(xe - mx) * inv;
        float u = on ? d * s : 0.f, along;
        if (a.renormalize) {
            const float total = warp_sum(s) + 1e-20f, w = s / total, mean = warp_sum(on ? d * w : 0.f);
            u = on ? w * (d - mean) : 0.f;
            along = mean * (1e-20f / total);
        } else {
            along = warp_sum(u);
        }
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
        if (on) out[e] = elem_of<T>(a.sigmoid ? u / (1.f + expf(xe)) : u - s * along);
    }
}

// Calls f with a row's lanes and the values per lane (powers of two), and whether rows are read in vectors.
template <typename T, bool TEAMS, typename F> cudaError_t by_width(int n, F f)
{
    auto run = [&](auto lanes, auto vpl) {
        constexpr int kBytes = std::min(16, decltype(vpl)::value * (int)sizeof(T));
        return n * (int)sizeof(T) % kBytes == 0 ? f(lanes, vpl, std::true_type()) : f(lanes, vpl, std::false_type());
    };
#define SPMM_ROUTE(LANES, VPL) run(std::integral_constant<int, LANES>(), std::integral_constant<int, VPL>())
    if constexpr (TEAMS) {
        if (n <= 32) return SPMM_ROUTE(4, 8);
        if (n <= 64) return SPMM_ROUTE(8, 8);
        if (n <= 128) return SPMM_ROUTE(16, 8);
    } else {
        if (n <= 32) return SPMM_ROUTE(32, 1);
        if (n <= 64) return SPMM_ROUTE(32, 2);
        if (n <= 128) return SPMM_ROUTE(32, 4);
    }
    if (n <= 256) return SPMM_ROUTE(32, 8);
    if (n <= 512) return SPMM_ROUTE(32, 16);
    return SPMM_ROUTE(32, 32);
#undef SPMM_ROUTE
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
        return by_width<T, true>(r.n, [&](auto lanes, auto vpl, auto vec) {
            constexpr int kLanes = decltype(lanes)::value, kVpl = decltype(vpl)::value;
            const int64_t warps = (r.tokens + 32 / kLanes - 1) / (32 / kLanes);
            const unsigned blocks = (unsigned)std::min<int64_t>((warps + 7) / 8, route_blocks(kVpl) * (int64_t)device_sm_count());
            auto kernel = route_kernel<T, kLanes, kVpl, decltype(vec)::value>;
            const int smem = decltype(vec)::value ? 8 * 2 * (32 / kLanes) * r.n * (int)sizeof(T) : 0;
            if (smem >= 16384) {   // with what the kernel has of its own, more than a block gets unasked
                static PerDevice<bool> ready;   // the attribute outlasts the call
                bool *done = ready.here();
                if (!done || !*done) {
                    const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 65536);
                    if (e != cudaSuccess) return e;
                    if (done) *done = true;
                }
            }
            kernel<<<blocks, 256, smem, stream>>>(a);
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
        return by_width<T, false>(r.n, [&](auto, auto vpl, auto vec) {
            route_backward_kernel<T, decltype(vpl)::value, decltype(vec)::value>
                <<<row_blocks(r.tokens), 256, 0, stream>>>(a);
            return cudaGetLastError();
        });
    });
}

}  // namespace spmmb
