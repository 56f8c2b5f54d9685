// The moments that the log probabilities and the entropy of a row of logits l are made of: M = max l, S = sum e^(l - M) and
// U = sum e^(l - M) (l - M), of parts of the row and joined; log p(t) = (l_t - M) - log S, the entropy is log S - U / S.
//
// Held is S - 1: the largest number's own 1 is left out, so that what little the others add keeps its 24 bits where a row is nearly sure
// of a token (a sum near 1 would be off by 6e-8, and so would a log probability of -1e-4).
#pragma once
#include "common.cuh"

namespace hos {

struct Moments { float m, s, u; };                     // maximum, sum of e^(l - m) but for one maximum, sum of e^(l - m) (l - m)

__device__ __forceinline__ float exp_of(float d) { return ex2_approx(d * 1.44269504f); }
// All of S: nothing where there is no number above -inf (or not-a-number).
__device__ __forceinline__ float whole_sum(const Moments& a) { return a.m == -INFINITY ? a.s : 1.f + a.s; }
__device__ __forceinline__ float log_sum(const Moments& a) { return a.m == -INFINITY ? logf(a.s) : log1pf(a.s); }
__device__ __forceinline__ float entropy_of(const Moments& a) { return log_sum(a) - a.u / whole_sum(a); }

// Both with the larger maximum.
__device__ __forceinline__ Moments joined(const Moments& a, const Moments& b) {
    const bool first = a.m >= b.m;
    const Moments& high = first ? a : b;
    const Moments& low = first ? b : a;
    const float d = high.m == low.m ? 0.f : low.m - high.m, e = exp_of(d), all = whole_sum(low);
    // a part without a number (nothing, m = -inf) adds nothing; a not-a-number stays one
    return Moments{high.m, high.s + all * e, high.u + (all == 0.f ? 0.f : (low.u + all * d) * e)};
}

// N more numbers, `most` the largest of them; -inf adds nothing, not-a-number makes the sums one.
template <int N>
__device__ __forceinline__ void add_to(Moments& to, const float (&x)[N], float most) {
    const bool higher = most > to.m;
    if (higher) {
        const float d = to.m - most, all = whole_sum(to), e = all == 0.f ? 0.f : exp_of(d);
        to.u = all == 0.f ? 0.f : (to.u + all * d) * e;
        to.s = all * e;
        to.m = most;
    }
    const float m = to.m == -INFINITY ? 0.f : to.m;
    float s[2] = {}, u[2] = {};
    int n = higher ? -1 : 0;                                 // maxima, but for the one that is left out
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const float d = x[j] - m, e = exp_of(d);
        if (d != 0.f) s[j & 1] += e; else ++n;
        u[j & 1] = fmaf(e, fmaxf(d, -1000.f), u[j & 1]);     // (0 times -inf would be no number)
    }
    to.s += s[0] + s[1] + (float)n;
    to.u += u[0] + u[1];
}

}  // namespace hos
