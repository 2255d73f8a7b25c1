// maya_route_groups.cuh - routing over groups of experts, by one warp a token.
//
//   s_e = softmax(l)_e or 1 / (1 + exp(-l_e));  c_e = s_e + bias_e          (the bias chooses, it does not weigh)
//   a group's score: its highest c, or the sum of its two highest;  the n_keep best groups are kept (ties: the lower group)
//   the k highest c of the kept groups' experts (ties: the lower expert);  w = s / max(sum of the k s, 2^-14) * w_scale
//
// The choice compares neighbours - of 256 sigmoid scores two lie within 1e-6 of each other all the time - so it is the one that scores, sums and
// comparisons in 64 bits make, and only the weights are rounded, once.  A score that is no number ranks behind every number.
//
// Nearly always 32 bits can tell: scores of a known error decide every comparison that matters (the border of the kept groups, each of the k choices
// against the next) when the values are further apart than that, and only the k weights are computed in 64 bits, a lane each (route_fast).  Where two are
// nearer - one token in some hundreds - or a score is not finite, everything is done over in 64 bits (route_exact).  8192 tokens of 256 experts: 28 us in 64 bits
// alone, 25 so, 23 with the lanes' scores sorted instead of searched in every round.
//
// A lane holds experts lane, lane + 32, ... in registers as whole numbers that order like the scores.  In 64 bits a warp's maximum of them is three
// warp-wide reductions of 32 bits (high words; low words of the lanes that have the highest; the lowest expert of those that have both), where
// a butterfly would exchange three words five times.  Groups cut across lanes: their scores are found in shared memory, a few lanes a group.
#pragma once

#include <math.h>

#include "maya_common.cuh"

namespace maya {

constexpr int kGroupsMost = 32;                        // one lane a group when they are ranked
constexpr int kRouteKMost = 64;
constexpr int kRouteExpertsMost = 2048;

struct RouteGroups {
    const float* logits;         // [tokens][n_expert]
    const float* bias;           // [n_expert] or NULL
    int n_expert, k, n_group, n_keep;
    int sigmoid, top2, norm_w;
    float w_scale;
    unsigned group_mul;          // ceil(2^32 / experts of a group): e / size is its high word of e * group_mul for e < 2^11 (size > 1)
};

// A number that orders like the score; 0: no expert; a score that is no number: 1.
__device__ __forceinline__ unsigned long long order64(double v) {
    const unsigned long long u = (unsigned long long) __double_as_longlong(v + 0.0);        // (-0 is 0)
    return v != v ? 1ull : u ^ ((long long) u < 0 ? ~0ull : 0x8000000000000000ull);
}
__device__ __forceinline__ double value64(unsigned long long o) {
    return __longlong_as_double((long long) (o ^ ((o >> 63) ? 0x8000000000000000ull : ~0ull)));
}
// The warp's highest `o` and the lowest `id` that has it.
__device__ __forceinline__ unsigned long long warp_best(unsigned long long o, int id, int& best_id) {
    const unsigned hi = (unsigned) (o >> 32), lo = (unsigned) o;
    const unsigned mh = __reduce_max_sync(0xffffffffu, hi);
    const unsigned ml = __reduce_max_sync(0xffffffffu, hi == mh ? lo : 0u);
    best_id = (int) __reduce_min_sync(0xffffffffu, hi == mh && lo == ml ? (unsigned) id : 0x7fffffffu);
    return ((unsigned long long) mh << 32) | ml;
}
__device__ __forceinline__ double warp_sum64(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// Lanes that look through one group: the largest power of two that leaves every group lanes of its own in one round.
__host__ __device__ inline int route_lanes(int n_group) {
    int p = 1;
    while (2 * p * n_group <= 32) p *= 2;
    return p;
}
// Words between the groups in shared memory: the lanes that start on different groups find different banks.
__host__ __device__ inline int route_stride(int size, int lanes) { return ((size + lanes - 1) / lanes) * lanes + lanes; }

// One token by the calling warp, in 64 bits.  keys: n_group * route_stride(...) words of shared memory, this warp's own (not needed when every group is
// kept).  Lane i < 32 returns in id[j], w[j] the choice number j * 32 + i and its weight (j < 2).
template<int PER>
__device__ __noinline__ void route_exact(const RouteGroups& A, int64_t token, unsigned long long* keys, int lane, int (&id)[2], float (&w)[2]) {
    const float* l = A.logits + token * A.n_expert;
    float lv[PER];
    float top = -INFINITY;
    bool some = false;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int e = j * 32 + lane;
        lv[j] = e < A.n_expert ? l[e] : -INFINITY;
        top = fmaxf(top, lv[j]);
        some |= lv[j] != -INFINITY;
    }
    double s[PER];
    if (A.sigmoid) {
#pragma unroll
        for (int j = 0; j < PER; ++j) s[j] = 1.0 / (1.0 + exp(-(double) lv[j]));
    } else {
        top = warp_max(top);
        double sum = 0.0;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            s[j] = j * 32 + lane < A.n_expert ? exp((double) lv[j] - (double) top) : 0.0;
            sum += s[j];
        }
        sum = warp_sum64(sum);
        const bool nothing = !__any_sync(0xffffffffu, some);             // but -inf: every score is 0
        const double inv = 1.0 / sum;
#pragma unroll
        for (int j = 0; j < PER; ++j) s[j] = nothing ? 0.0 : s[j] * inv;
    }
    unsigned long long o[PER];
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int e = j * 32 + lane;
        o[j] = 0ull;
        if (e < A.n_expert) o[j] = order64(A.bias != nullptr ? s[j] + (double) A.bias[e] : s[j]);
    }
    if (A.n_keep < A.n_group) {
        const int size = A.n_expert / A.n_group, lanes = route_lanes(A.n_group), stride = route_stride(size, lanes);
        auto group_of = [&](int e) { return size == 1 ? e : (int) __umulhi((unsigned) e, A.group_mul); };
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int e = j * 32 + lane;
            if (e < A.n_expert) {
                const int q = group_of(e);
                keys[q * stride + e - q * size] = o[j];
            }
        }
        __syncwarp();
        const int g = lane / lanes, part = lane % lanes;
        unsigned long long a = 0ull, b = 0ull;                   // the group's highest and second
        if (g < A.n_group)
            for (int i = part; i < size; i += lanes) {
                const unsigned long long v = keys[g * stride + i];
                if (v > a) { b = a; a = v; }
                else if (v > b) b = v;
            }
        for (int d = 1; d < lanes; d *= 2) {
            const unsigned long long oa = __shfl_xor_sync(0xffffffffu, a, d), ob = __shfl_xor_sync(0xffffffffu, b, d);
            const unsigned long long rest = oa > a ? (a > ob ? a : ob) : (oa > b ? oa : b);
            a = oa > a ? oa : a;
            b = rest;
        }
        // a group's score: no number where its two highest are none (1: none; 0: the group has one expert)
        unsigned long long score = a;
        if (A.top2 && a > 1ull && b != 0ull) score = b > 1ull ? order64(value64(a) + value64(b)) : 1ull;
        const unsigned long long mine = part == 0 && g < A.n_group ? score : 0ull;
        int rank = 0;
        for (int q = 0; q < A.n_group; ++q) {
            const unsigned long long other = __shfl_sync(0xffffffffu, mine, q * lanes);
            rank += other > score || (other == score && q < g);
        }
        const unsigned kept = __ballot_sync(0xffffffffu, part == 0 && g < A.n_group && rank < A.n_keep);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int e = j * 32 + lane;
            if (e < A.n_expert && !((kept >> (group_of(e) * lanes)) & 1u)) o[j] = 0ull;
        }
        __syncwarp();                                            // the keys may be another token's next
    }
    // k rounds: the warp's highest, which its lane then gives up
    double sum = 0.0, mine[2] = {0.0, 0.0};
    id[0] = id[1] = 0;
    for (int i = 0; i < A.k; ++i) {
        unsigned long long best = 0ull;
        int at = 0x7fffffff;
        double sv = 0.0;
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (o[j] > best) { best = o[j]; at = j * 32 + lane; sv = s[j]; }
        int e;
        warp_best(best, at, e);
        const double v = __shfl_sync(0xffffffffu, sv, e & 31);
        sum += v;
        if (lane == (i & 31)) { id[i >> 5] = e; mine[i >> 5] = v; }
#pragma unroll
        for (int j = 0; j < PER; ++j)
            if (j * 32 + lane == e) o[j] = 0ull;
    }
    const double div = !A.norm_w ? 1.0 : sum < 6.103515625e-05 ? 6.103515625e-05 : sum;        // 2^-14; a sum that is no number stays one
#pragma unroll
    for (int j = 0; j < 2; ++j) w[j] = (float) (mine[j] / div * (double) A.w_scale);
}

// Batcher's odd-even merge sort, in registers.
template<int N> __device__ __forceinline__ void sort_descending(uint32_t (&v)[N]) {
#pragma unroll
    for (int p = 1; p < N; p *= 2)
#pragma unroll
        for (int k = p; k >= 1; k /= 2)
#pragma unroll
            for (int j = k % p; j + k < N; j += 2 * k)
#pragma unroll
                for (int i = 0; i < k; ++i)
                    if (i + j + k < N && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
                        const uint32_t a = v[i + j], b = v[i + j + k];
                        v[i + j] = max(a, b);
                        v[i + j + k] = min(a, b);
                    }
}

// The same where 32 bits decide; false: they do not, nothing is returned.
// Errors: expf is within 2 ulp, its argument - for a softmax a difference, rounded - within 2^-24 of itself, at most 104 before the result is 0; quotient and sums round.
// So a score without a bias is within 2^-16 of itself (sums of up to 2048 terms among them), a sigmoid with a bias within 2^-21 and the rounding
// of the sum, a softmax with one within 2^-16; what lies below 2^-110 of the highest is not told apart.  kApart times these has to lie between two values.
// An error that grows with the value itself needs to be looked at between neighbours only: a value further off is off by more than its error grows.  That does not
// hold for the sum of a group's two highest, whose error is that of the two - as large as their biases, when the sum of a large and a very negative one is near 0 - so
// every kept group's sum less its error has to lie above every other group's sum and error.
template<int PER>
__device__ __forceinline__ bool route_fast(const RouteGroups& A, int64_t token, float* keys, int lane, int (&id)[2], float (&w)[2]) {
    const float* l = A.logits + token * A.n_expert;
    float s[PER];
    float top = -INFINITY;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int e = j * 32 + lane;
        s[j] = e < A.n_expert ? l[e] : -INFINITY;
        top = fmaxf(top, s[j]);
    }
    float all = 0.0f;
    if (A.sigmoid) {
#pragma unroll
        for (int j = 0; j < PER; ++j) s[j] = __fdividef(1.0f, 1.0f + expf(-s[j]));       // (1 over more than 2^126: 0)
    } else {
        top = warp_max(top);
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            s[j] = expf(s[j] - top);           // (no number beside +inf, or where nothing is above -inf)
            all += s[j];
        }
        all = warp_sum(all);
        if (A.bias != nullptr) {
            const float inv = __fdividef(1.0f, all);
#pragma unroll
            for (int j = 0; j < PER; ++j) s[j] *= inv;
        }
    }
    constexpr float kApart = 8.0f;
    constexpr float kPlaces = (float) PER * 0x1p-23f;         // (what the places in the lowest bits take from a score)
    const float of_itself = kApart * (A.bias == nullptr ? 0x1p-16f : 0x1p-23f) + kPlaces, fixed = A.bias == nullptr ? 0x1p-110f : kApart * (A.sigmoid ? 0x1p-21f : 0x1p-16f);
    auto near = [&](float a, float b) { return !(a - b > fixed + of_itself * fmaxf(fabsf(a), fabsf(b))); };     // a >= b
    auto ordered = [](float c) {
        const uint32_t u = __float_as_uint(c);
        return u ^ ((uint32_t) ((int32_t) u >> 31) | 0x80000000u);
    };
    uint32_t o[PER];
    bool odd = false;
#pragma unroll
    for (int j = 0; j < PER; ++j) {
        const int e = j * 32 + lane;
        o[j] = 0u;
        if (e < A.n_expert) {
            const float c = (A.bias != nullptr ? s[j] + A.bias[e] : s[j]) + 0.0f;
            odd |= !(fabsf(c) < 1e30f);
            o[j] = ordered(c);
        }
    }
    if (__any_sync(0xffffffffu, odd)) return false;
    auto value = [](uint32_t v) { return __uint_as_float(v ^ ((v >> 31) ? 0x80000000u : 0xffffffffu)); };
    if (A.n_keep < A.n_group) {
        const int size = A.n_expert / A.n_group, lanes = route_lanes(A.n_group), stride = route_stride(size, lanes);
        auto group_of = [&](int e) { return size == 1 ? e : (int) __umulhi((unsigned) e, A.group_mul); };
        uint32_t* k32 = (uint32_t*) keys;
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int e = j * 32 + lane;
            if (e < A.n_expert) {
                const int q = group_of(e);
                k32[q * stride + e - q * size] = o[j];
            }
        }
        __syncwarp();
        const int g = lane / lanes, part = lane % lanes;
        uint32_t a = 0u, b = 0u;
        if (g < A.n_group)
#pragma unroll 4
            for (int i = part; i < size; i += lanes) {
                const uint32_t v = k32[g * stride + i];
                b = max(b, min(a, v));
                a = max(a, v);
            }
        for (int d = 1; d < lanes; d *= 2) {
            const uint32_t oa = __shfl_xor_sync(0xffffffffu, a, d), ob = __shfl_xor_sync(0xffffffffu, b, d);
            b = max(max(b, ob), min(a, oa));
            a = max(a, oa);
        }
        const bool mine = part == 0 && g < A.n_group;
        const float score = A.top2 && b != 0u ? value(a) + value(b) : value(a);
        int rank = 0;
        for (int q = 0; q < A.n_group; ++q) {
            const float other = __shfl_sync(0xffffffffu, score, q * lanes);
            rank += other > score || (other == score && q < g);
        }
        const bool keeps = mine && rank < A.n_keep;
        const unsigned kept = __ballot_sync(0xffffffffu, keeps);
        const float err = 0.5f * (fixed + of_itself * (A.top2 && b != 0u ? fabsf(value(a)) + fabsf(value(b)) : fabsf(score)));        // (half of what two have to be apart)
        const unsigned in = __reduce_min_sync(0xffffffffu, keeps ? ordered(score - err) : 0xffffffffu);
        const unsigned out = __reduce_max_sync(0xffffffffu, mine && !keeps ? ordered(score + err) : 0u);
        if (!(in > out)) return false;         // (all lanes alike)
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int e = j * 32 + lane;
            if (e < A.n_expert && !((kept >> (group_of(e) * lanes)) & 1u)) o[j] = 0u;
        }
        __syncwarp();
    }
    // every lane's scores in order, their places in the lowest bits; a round takes the highest of the lanes' first ones
#pragma unroll
    for (int j = 0; j < PER; ++j)
        if (o[j] != 0u) o[j] = (o[j] & ~(uint32_t) (PER - 1)) | (uint32_t) j;
    sort_descending(o);
    id[0] = id[1] = 0;
    uint32_t before = 0u;
    for (int i = 0; i <= A.k; ++i) {           // one more than is taken: the last has to be apart from it
        const uint32_t best = __reduce_max_sync(0xffffffffu, o[0]);
        if (i > 0 && best != 0u && near(value(before), value(best))) return false;
        if (i == A.k) break;
        before = best;
        const unsigned who = __ballot_sync(0xffffffffu, o[0] == best);
        if (__popc(who) != 1) return false;    // equal ones
        const int from = __ffs(who) - 1;
        if (lane == (i & 31)) id[i >> 5] = (int) (best & (uint32_t) (PER - 1)) * 32 + from;
        if (lane == from) {
#pragma unroll
            for (int j = 0; j + 1 < PER; ++j) o[j] = o[j + 1];
            o[PER - 1] = 0u;
        }
    }
    double v[2] = {0.0, 0.0};
#pragma unroll
    for (int j = 0; j < 2; ++j)
        if (j * 32 + lane < A.k) {
            const double x = (double) l[id[j]];
            v[j] = A.sigmoid ? 1.0 / (1.0 + exp(-x)) : exp(x - (double) top);
        }
    const double sum = warp_sum64(v[0] + v[1]);
    // a softmax's scores lack the division by the sum of all, which nothing but the least divisor asks for: far from it, or in 64 bits
    if (!A.sigmoid && !(sum > 2.0 * 6.103515625e-05 * (double) all)) return false;
    const double div = A.sigmoid ? (A.norm_w ? fmax(sum, 6.103515625e-05) : 1.0) : sum;        // (scores are numbers here)
#pragma unroll
    for (int j = 0; j < 2; ++j) w[j] = (float) (v[j] / div * (double) A.w_scale);
    return true;
}

template<int PER>
__device__ __forceinline__ void route_groups_warp(const RouteGroups& A, int64_t token, unsigned long long* keys, int lane, int (&id)[2], float (&w)[2]) {
    const bool can = A.sigmoid || A.norm_w;    // (a softmax's own scores need the sum of all in 64 bits)
    if (can && route_fast<PER>(A, token, (float*) keys, lane, id, w)) return;
    route_exact<PER>(A, token, keys, lane, id, w);
}

}  // namespace maya
