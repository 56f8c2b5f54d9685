// The moments that the log probabilities and the entropy of a row of logits l are made of: M = max l, S = sum e^(l - M) and
// U = sum e^(l - M) (l - M), of parts of the row and joined; log p(t) = (l_t - M) - log S, the entropy is log S - U / S.
#pragma once
#include "common.cuh"

namespace hos {

struct Moments { float m, s, u; };                     // maximum, sum of e^(l - m), sum of e^(l - m) (l - m)

__device__ __forceinline__ float exp_of(float d) { return ex2_approx(d * 1.44269504f); }

// Both with the larger maximum.
__device__ __forceinline__ Moments joined(const Moments& a, const Moments& b) {
    Moments r;
    r.m = fmaxf(a.m, b.m);
    const float da = a.m == r.m ? 0.f : a.m - r.m, db = b.m == r.m ? 0.f : b.m - r.m;
    const float ea = exp_of(da), eb = exp_of(db);
    // a part without a number (s = 0, m = -inf) adds nothing; a not-a-number stays one
    r.s = a.s * ea + b.s * eb;
    r.u = (a.s == 0.f ? 0.f : (a.u + a.s * da) * ea) + (b.s == 0.f ? 0.f : (b.u + b.s * db) * eb);
    return r;
}

// N more numbers, `most` the largest of them; -inf adds nothing, not-a-number makes the sums one.
template <int N>
__device__ __forceinline__ void add_to(Moments& to, const float (&x)[N], float most) {
    if (most > to.m) {
        const float d = to.m - most, e = to.s == 0.f ? 0.f : exp_of(d);
        to.u = to.s == 0.f ? 0.f : (to.u + to.s * d) * e;
        to.s *= e;
        to.m = most;
    }
    const float m = to.m == -INFINITY ? 0.f : to.m;
    float s[2] = {}, u[2] = {};
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const float d = x[j] - m, e = exp_of(d);
        s[j & 1] += e;
        u[j & 1] = fmaf(e, fmaxf(d, -1000.f), u[j & 1]);     // (0 times -inf would be no number)
    }
    to.s += s[0] + s[1];
    to.u += u[0] + u[1];
}

}  // namespace hos
